// tree_rows.h -- where the rows of a step of trees of drafted tokens lie (engine.hip; plain C++, so that
// tests/cpp/tree_rows_check runs it under AddressSanitizer and UndefinedBehaviorSanitizer).
#pragma once

#include <climits>
#include <cstdint>

namespace qraf_hip {

// Row i's place in its sequence's cache: the position of the sequence's first row, and the nodes ahead of row i.  Of
// positions only those of first rows are read: a caller need not set the others.  A sum past int32 is its largest, which
// is past every cache.
inline void tree_places(int n, const int32_t* seq_ids, const int32_t* positions, int32_t* places) {
    for (int i = 0, first = 0; i < n; i++) {
        if (i > 0 && seq_ids[i] != seq_ids[i - 1]) first = i;
        const int64_t place = (int64_t)positions[first] + (i - first);
        places[i] = place < INT32_MAX ? (int32_t)place : INT32_MAX;
    }
}

}  // namespace qraf_hip
