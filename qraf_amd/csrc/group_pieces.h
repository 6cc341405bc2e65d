// group_pieces.h -- how attention by group cuts its jobs along the positions
// (attention_group.hip: by a wave of each workgroup; tests: on the host).
#pragma once
#include <cstdint>

#if defined(__HIPCC__)
#define QH_GROUP_FN __host__ __device__ inline
#else
#define QH_GROUP_FN inline
#endif

namespace qraf_hip {

constexpr int LONG_JOB = 1 << 19;  // tiles

// pieces of a job of `tiles` tiles (at most 2^24: 2^30 positions), of at most `most` each
QH_GROUP_FN int pieces_of_long(int tiles, int most) { return tiles ? (tiles - 1) / most + 1 : 0; }
// The same for fewer than LONG_JOB tiles, by a product in fp32, per_most = 1 / most: the quotient or one less (never one
// more, which would have no place for its parts).
QH_GROUP_FN int pieces_of(int tiles, int most, float per_most) {
    if (!tiles) return 0;
    const int k = (int)((float)(tiles + most - 1) * per_most);
    return k > 1 ? k : 1;
}
// the places of `full` jobs with tiles: `shares`, or as many times that as there are jobs
QH_GROUP_FN int piece_room(int full, int shares) {
    const int rounds = (full + shares - 1) / shares;
    return shares * (rounds > 1 ? rounds : 1);
}
// The length of the shortest piece of which there are at most `room`.  all: the jobs' tiles together (1,024 rows of
// 2^30 positions each are 2^34); count(most): the pieces of all jobs.
template <typename F>
QH_GROUP_FN int shortest_piece(uint64_t all, int full, int room, F count) {
    // (pieces of x tiles are at least all / x, and fewer than all / x + full; a job is one piece at 2^25)
    const int spare = room - full;
    int lo, hi;
    if (all < 1u << 30) {  // (divisions in 64 bits take 0.2 us on the device)
        lo = ((int)all + room - 1) / room;
        hi = spare > 0 ? ((int)all + spare - 1) / spare : (int)all;
    } else {
        const uint64_t most = spare > 0 ? (all + spare - 1) / spare : all;
        lo = (int)((all + room - 1) / room);
        hi = most < 1u << 25 ? (int)most : 1 << 25;
    }
    if (lo < 1) lo = 1;
    if (hi < lo) hi = lo;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (count(mid) <= room) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

}  // namespace qraf_hip
