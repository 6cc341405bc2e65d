// Places of the rows of seeded random trees, up to 40 sequences of up to 64 nodes side by side: the first row's position
// and the nodes ahead.  Of the positions only first rows' are set, any value among them; the others hold int32's ends,
// and whole granules of them are poisoned for AddressSanitizer, as is what lies behind a last tree's first row.
#include <sanitizer/asan_interface.h>

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../qraf_amd/csrc/tree_rows.h"

int main(int argc, char** argv) {
    std::mt19937 rng(argc > 1 ? atoi(argv[1]) : 1);
    const int rounds = argc > 2 ? atoi(argv[2]) : 300;
    auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
    long long past = 0, poisoned = 0;
    for (int k = 0; k < rounds; k++) {
        std::vector<int32_t> ids, first, root;
        for (int s = 0, seqs = 1 + below(40); s < seqs; s++) {
            const int nodes = 1 + below(64), at = (int)ids.size();
            const int32_t pos = below(4) ? below(1 << 20) : (int32_t)(below(2) ? INT32_MAX - below(80) : -below(100));
            ids.insert(ids.end(), nodes, s * 7 % 41);
            first.insert(first.end(), nodes, at);
            root.insert(root.end(), nodes, pos);
        }
        // (no entry at all behind the last sequence's first row)
        const int n = (int)ids.size(), held = first[n - 1] + 1;
        int32_t* positions = (int32_t*)malloc((size_t)held * 4);
        for (int i = 0; i < held; i++) positions[i] = first[i] == i ? root[i] : i & 1 ? INT32_MAX : INT32_MIN;
        for (int i = 0; i + 1 < held; i += 2)
            if (first[i] != i && first[i + 1] != i + 1) {
                __asan_poison_memory_region(positions + i, 8);
                poisoned++;
            }
        std::vector<int32_t> places(n);
        qraf_hip::tree_places(n, ids.data(), positions, places.data());
        for (int i = 0; i < n; i++) {
            const int64_t want = (int64_t)root[i] + (i - first[i]);
            past += want > INT32_MAX;
            if (places[i] != std::min<int64_t>(want, INT32_MAX)) {
                printf("row %d of a sequence at %d, first row %d: %d\n", i, root[i], first[i], places[i]);
                return 1;
            }
        }
        __asan_unpoison_memory_region(positions, (size_t)held * 4);
        free(positions);
    }
    printf("%d steps, %lld places past int32, %lld poisoned\n", rounds, past, poisoned);
    return 0;
}
