// Cuts seeded random jobs, up to 4,096 of up to 2^24 tiles (1,024 rows of 2^30 positions), as attention by group does
// on the device: never more pieces than places, whose number and parts the kernel's storage is made for, never fewer
// than one a job, and no shorter piece length would do.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../qraf_amd/csrc/group_pieces.h"

using namespace qraf_hip;

int main(int argc, char** argv) {
    std::mt19937 rng(argc > 1 ? atoi(argv[1]) : 1);
    const int rounds = argc > 2 ? atoi(argv[2]) : 300;
    long long passed_31 = 0;
    auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
    for (int i = 0; i < rounds; i++) {
        const int jobs = i % 10 == 0 ? 4096 : 1 + below(1 << below(13)), shares = 256 / (1 + below(8)), bits = below(25);
        std::vector<int> tiles(jobs);
        for (int& t : tiles) t = below(8) == 0 ? 0 : i % 10 == 0 ? 1 << 24 : below((1 << bits) + 1);
        uint64_t all = 0;
        int full = 0;
        for (int t : tiles) all += (unsigned)t, full += t > 0;
        passed_31 += all >> 31 != 0;
        const int room = piece_room(full, shares);
        const bool longs = *std::max_element(tiles.begin(), tiles.end()) >= LONG_JOB;
        auto pieces = [&](int t, int most) {
            return longs ? pieces_of_long(t, most) : pieces_of(t, most, 1.f / (float)most);
        };
        auto count = [&](int most) {
            long long n = 0;
            for (int t : tiles) n += pieces(t, most);
            return (int)std::min<long long>(n, 1 << 30);
        };
        const int lo = shortest_piece(all, full, room, count), n = count(lo);
        if (n > room || n < full || n > 0xFFFF || lo < 1) {
            printf("%d jobs, %llu tiles, length %d: %d pieces of %d places\n", jobs, (unsigned long long)all, lo, n, room);
            return 1;
        }
        for (int t : tiles) {  // (the quotient: in fp32 the product may fall one short of it, never pass it)
            const int k = pieces(t, lo), up = (int)(((int64_t)t + lo - 1) / lo);
            if (k > up || k < up - 1 || (t && k < 1) || k > t) {
                printf("%d tiles at %d: %d pieces, %d\n", t, lo, k, up);
                return 1;
            }
        }
        if (lo > 1 && (uint64_t)room * (lo - 1) >= all + (uint64_t)full * (lo - 1) && count(lo - 1) <= room) {
            printf("length %d is not the shortest\n", lo);
            return 1;
        }
    }
    printf("%d sets of jobs, %lld past 2^31 tiles\n", rounds, passed_31);
    return 0;
}
