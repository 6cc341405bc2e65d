// tree.hip -- trees of drafted tokens: the accepted path, and its keys and values
// moved to where the sequence goes on.  (Attention of a tree's nodes:
// attention_group.hip.)
//
// A sequence's tree is its rows of a step: row 0 the last token that is certain (the
// root), every other row a drafted token behind its parent.  Node i's keys and values
// lie at position base + i of the cache, whatever its depth.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace qraf_hip {

// ---------------------------------------------------------------------------
// The walk: with t_i the token sampled from the target's distribution behind node
// i, go from node i to the lowest of its children whose draft is t_i; where there
// is none, t_i is the token that follows.  (Drafts that are given and not drawn:
// taking t_i where it is a child is rejection sampling, so the tokens along the way
// are distributed as the target's samples.)  A child lies behind its parent, so one
// pass over a sequence's rows finds the whole path: a wave a sequence, 64 rows at a
// time in its lanes.
// ---------------------------------------------------------------------------
struct AcceptArgs {
    const uint32_t *picks, *drafts;
    const int32_t *parents, *starts;
    int32_t *accepted, *path;
    uint32_t* tokens;
    int rows;
};

__global__ __launch_bounds__(64) void tree_accept_kernel(AcceptArgs a) {
    const int s = blockIdx.x, lane = threadIdx.x;
    const int r0 = max(0, min(a.starts[s], a.rows)), n = max(0, min(a.starts[s + 1], a.rows) - r0);
    int at = 0, len = 0;
    uint32_t token = 0;
    for (int c = 0; c < n; c += 64) {
        const int i = c + lane, r = r0 + min(i, n - 1);
        const int parent = i < n ? a.parents[r] : -1;
        const uint32_t draft = a.drafts[r], pick = a.picks[r];
        if (c == 0) token = __shfl(pick, 0);
        for (;;) {
            const unsigned long long hit = __ballot(i > at && parent == at && draft == token);
            if (!hit) break;
            const int l = __ffsll(hit) - 1;
            if (lane == 0) {
                a.path[r0 + len] = at;
                a.tokens[r0 + len] = token;
            }
            at = c + l;
            token = __shfl(pick, l);
            len++;
        }
    }
    if (n > 0 && lane == 0) {
        a.path[r0 + len] = at;
        a.tokens[r0 + len] = token;
    }
    for (int i = len + 1 + lane; i < n; i += 64) {
        a.path[r0 + i] = -1;
        a.tokens[r0 + i] = 0xFFFFFFFFu;
    }
    if (lane == 0) a.accepted[s] = len;
}

int launch_tree_accept(const uint32_t* picks, const uint32_t* drafts, const int32_t* parents, const int32_t* starts,
                       int seqs, int rows, int32_t* accepted, int32_t* path, uint32_t* tokens, hipStream_t st) {
    QH_REQUIRE(picks && drafts && parents && starts && accepted && path && tokens, QRAF_HIP_ERR_INVALID,
               "tree_accept: null pointer");
    QH_REQUIRE(seqs > 0 && seqs <= 65535 && rows > 0, QRAF_HIP_ERR_INVALID, "tree_accept: %d rows of %d sequences", rows,
               seqs);
    const AcceptArgs a{picks, drafts, parents, starts, accepted, path, tokens, rows};
    hipLaunchKernelGGL(tree_accept_kernel, dim3(seqs), dim3(64), 0, st, a);
    QH_CHECK_HIP(hipGetLastError());
    return QRAF_HIP_OK;
}

// ---------------------------------------------------------------------------
// position base + j <- base + path[j], in every layer.  The path ascends from 0 or
// more, so path[j] >= j, and no position is written that a later step of the path reads:
// a step need not wait for those before it.
//
// A workgroup per (layer, sequence) and in it a wave for each 64 pieces of a position (16
// or 4 bytes of a head's keys; an element of its values, where these lie by dimension;
// scales).  Every wave finds the moves for itself - the path and the pages that the tree
// spans are requested at once, from lengths alone - and has eight moves in flight: three
// reads one after another, then the writes, without a barrier.  Elements that become
// neighbours (values by dimension) are written together.  One sequence: latency, 4.1 to 4.9 us.
// 64 sequences of 6 nodes in 36 layers, fp16, 23.6 MB of keys and values: 19.6 to 19.8 us, in
// which values by dimension bring every line of the pages that the tree spans, 77 MB read
// and written at 3.9 TB/s.  (Keys alone 7.1; one node after another and keys ahead of
// values 22.0; elements written one by one 20.3.)
// ---------------------------------------------------------------------------
struct CompactArgs {
    uint8_t *kc, *vc;
    size_t layer_bytes;
    const int32_t *table, *base, *starts, *path;
    int max_pages, rows, Hkv, hd, page_size;
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// waves of a position's keys (f32: and values) in pieces of `piece` bytes, of values by dimension, of scales
struct CompactWaves {
    int keys, values, scales;
};
static __host__ __device__ CompactWaves compact_waves(uint32_t kv, int Hkv, int hd, int piece) {
    const int item = kv == DT_F32 ? 4 : kv == DT_F16 ? 2 : 1;
    CompactWaves w;
    w.keys = (Hkv * hd * item / piece + 63) / 64;
    w.values = kv == DT_F32 ? w.keys : (Hkv * hd + 63) / 64;
    w.scales = kv == DT_I8 ? (2 * Hkv + 63) / 64 : 0;
    return w;
}

template <int KV, typename Piece>
__global__ __launch_bounds__(512) void kv_compact_kernel(CompactArgs a) {
    constexpr int ITEM = KV == (int)DT_F32 ? 4 : KV == (int)DT_F16 ? 2 : 1;
    const int s = blockIdx.y, lane = threadIdx.x & 63, ps = a.page_size, hd = a.hd, most = a.max_pages - 1;
    // (a base at or past the table's end, which no path begins ahead of, as that end: at most 2^30, so sums below hold)
    const int base = max(0, min(a.base[s], a.max_pages * ps));
    const int r0 = max(0, min(a.starts[s], a.rows)), n = max(0, min(a.starts[s + 1], a.rows) - r0);
    const int32_t* table = a.table + (size_t)s * a.max_pages;
    const int first = base / ps, page_of = table[min(first + lane, most)];  // the tree's pages, a lane to a page
    const size_t block = (size_t)ps * (KV == (int)DT_I8 ? hd + 4 : hd * ITEM);  // bytes of a (page, KV head)
    uint8_t *kc = a.kc + blockIdx.x * a.layer_bytes, *vc = a.vc + blockIdx.x * a.layer_bytes;
    const CompactWaves waves = compact_waves(KV, a.Hkv, hd, sizeof(Piece));
    int last = -1;  // of the path so far
    for (int c = 0; c < n; c += 64) {
        // ---- the moves of 64 entries, a lane to an entry
        const int j = c + lane, node = j < n ? a.path[r0 + j] : -1;
        int before = __shfl_up(node, 1);
        if (lane == 0) before = last;
        // an entry that does not ascend, is no node of the tree or lies past the table ends the path
        const bool good = node > before && node < n && (long long)base + node < (long long)a.max_pages * ps;
        const unsigned long long bad = ~__ballot(good);
        const int count = bad ? __ffsll(bad) - 1 : 64;
        const int from = base + (lane < count ? node : 0), to = base + (lane < count ? j : 0);
        const int pf = from / ps - first, pt = to / ps - first;
        int page_from = __shfl(page_of, min(pf, 63)), page_to = __shfl(page_of, min(pt, 63));
        if (__any(pf > 63)) {  // (trees over more than 64 pages)
            page_from = pf > 63 ? table[min(pf + first, most)] : page_from;
            page_to = pt > 63 ? table[min(pt + first, most)] : page_to;
        }
        const int off_from = from % ps, off_to = to % ps;
        const unsigned long long moves = __ballot(lane < count && node != j);  // (all behind the first)
        const int begin = moves ? __ffsll(moves) - 1 : count;
        last = __shfl(node, 63);
        // ---- piece i of every position: `of` its bytes behind a block's first, for offset 0, `step` apart
        auto move = [&](uint8_t* pool, int head, size_t of, size_t step, auto one) {
            typedef decltype(one) T;
            uint8_t* p = pool + (size_t)head * block + of;
            for (int k0 = begin, run; k0 < count; k0 += run) {
                const int o = __builtin_amdgcn_readlane(off_to, k0);
                run = min(min(8, count - k0), ps - o);  // neighbours in one page
                T v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int m = min(k0 + k, count - 1);
                    v[k] = *(const T*)(p + (size_t)__builtin_amdgcn_readlane(page_from, m) * a.Hkv * block +
                                       __builtin_amdgcn_readlane(off_from, m) * step);
                }
                uint8_t* to = p + (size_t)__builtin_amdgcn_readlane(page_to, k0) * a.Hkv * block + o * step;
                if constexpr (sizeof(T) <= 2) {  // side by side: eight, four, two, one of them in a write
                    auto write = [&](auto many) {
                        constexpr int M = decltype(many)::value;
                        if (M < 8 ? !(run & M) : run < 8) return;
                        struct __attribute__((packed, aligned(sizeof(T)))) Run {
                            T t[M];
                        } r;
#pragma unroll
                        for (int k = 0; k < M; k++) r.t[k] = v[k];
                        *(Run*)to = r;
                        to += M * sizeof(T);
#pragma unroll
                        for (int k = 0; k + M < 8; k++) v[k] = v[k + M];
                    };
                    write(std::integral_constant<int, 8>());
                    if (run < 8) {
                        write(std::integral_constant<int, 4>());
                        write(std::integral_constant<int, 2>());
                        write(std::integral_constant<int, 1>());
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < run) *(T*)(to + k * step) = v[k];
                }
            }
        };
        const int pieces = hd * ITEM / (int)sizeof(Piece);  // of a head's keys
        for (int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); w < waves.keys + waves.values + waves.scales;
             w += (int)blockDim.x >> 6) {
            if (w < waves.keys || (KV == (int)DT_F32 && w < 2 * waves.keys)) {
                const int i = (w < waves.keys ? w : w - waves.keys) * 64 + lane;
                if (i < a.Hkv * pieces)
                    move(w < waves.keys ? kc : vc, i / pieces, sizeof(Piece) * (size_t)(i % pieces), (size_t)hd * ITEM, Piece());
            } else if (w < waves.keys + waves.values) {
                const int i = (w - waves.keys) * 64 + lane;
                if (i < a.Hkv * hd) {
                    if constexpr (KV == (int)DT_F16) move(vc, i / hd, (size_t)(i % hd) * ps * 2, 2, uint16_t());
                    else move(vc, i / hd, (size_t)(i % hd) * ps, 1, uint8_t());
                }
            } else {
                const int i = (w - waves.keys - waves.values) * 64 + lane;
                if (i < 2 * a.Hkv) move(i < a.Hkv ? kc : vc, i % a.Hkv, (size_t)ps * hd, 4, uint32_t());
            }
        }
        if (count < 64) break;
    }
}

int launch_kv_compact(void* kc, void* vc, uint32_t kv_dtype, int layers, size_t layer_bytes, const int32_t* table,
                      int max_pages, const int32_t* base, const int32_t* starts, const int32_t* path, int seqs, int rows,
                      int Hkv, int hd, int page_size, hipStream_t st) {
    QH_REQUIRE(kc && vc && table && base && starts && path, QRAF_HIP_ERR_INVALID, "kv_compact: null pointer");
    QH_REQUIRE((((uintptr_t)kc | (uintptr_t)vc | layer_bytes) & 3) == 0, QRAF_HIP_ERR_INVALID,
               "kv_compact: caches and layers must be 4-byte aligned");
    QH_REQUIRE(seqs > 0 && seqs <= 65535 && rows > 0, QRAF_HIP_ERR_INVALID, "kv_compact: %d rows of %d sequences", rows,
               seqs);
    QH_REQUIRE(layers > 0 && Hkv > 0 && (long long)Hkv * hd <= 1 << 20, QRAF_HIP_ERR_INVALID,
               "kv_compact: %d layers, %d kv heads", layers, Hkv);
    QH_REQUIRE(hd == 16 || hd == 32 || hd == 64 || hd == 128, QRAF_HIP_ERR_INVALID,
               "kv_compact: head_dim %d (16, 32, 64 or 128 supported)", hd);
    QH_REQUIRE(page_size > 0 && max_pages > 0 && (long long)max_pages * page_size <= 1 << 30, QRAF_HIP_ERR_INVALID,
               "kv_compact: bad page geometry");
    QH_REQUIRE(kv_dtype == DT_F32 || kv_dtype == DT_F16 || kv_dtype == DT_I8, QRAF_HIP_ERR_DTYPE, "kv_compact: KV dtype %u",
               kv_dtype);
    const CompactArgs a{(uint8_t*)kc, (uint8_t*)vc, layer_bytes, table, base, starts, path, max_pages, rows, Hkv, hd,
                        page_size};
    // 16 bytes at a time where every position's keys are aligned to them
    const size_t block = (size_t)page_size * (kv_dtype == DT_I8 ? hd + 4 : hd * (kv_dtype == DT_F32 ? 4 : 2));
    const bool wide = (((uintptr_t)kc | (uintptr_t)vc | layer_bytes | block) & 15) == 0;
    const CompactWaves w = compact_waves(kv_dtype, Hkv, hd, wide ? 16 : 4);
    const dim3 grid(layers, seqs), threads(64 * std::min(8, w.keys + w.values + w.scales));
#define QH_COMPACT(KVv)                                                                                          \
    if (kv_dtype == KVv) {                                                                                       \
        if (wide) hipLaunchKernelGGL((kv_compact_kernel<(int)KVv, u32x4>), grid, threads, 0, st, a);             \
        else hipLaunchKernelGGL((kv_compact_kernel<(int)KVv, uint32_t>), grid, threads, 0, st, a);               \
    }
    QH_COMPACT(DT_F32)
    QH_COMPACT(DT_F16)
    QH_COMPACT(DT_I8)
#undef QH_COMPACT
    QH_CHECK_HIP(hipGetLastError());
    return QRAF_HIP_OK;
}

}  // namespace qraf_hip

using namespace qraf_hip;

extern "C" {

int qraf_hip_tree_accept_dev(const uint32_t* picks, const uint32_t* draft_tokens, const int32_t* parents,
                             const int32_t* row_starts, int32_t n_seqs, int32_t n_rows, int32_t* accepted,
                             int32_t* path, uint32_t* tokens, void* stream) {
    clear_error();
    return launch_tree_accept(picks, draft_tokens, parents, row_starts, n_seqs, n_rows, accepted, path, tokens,
                              as_stream(stream));
}

int qraf_hip_kv_compact_dev(void* k_cache, void* v_cache, uint32_t kv_dtype, int32_t n_layers, uint64_t layer_bytes,
                            const int32_t* page_table, int32_t max_pages_per_seq, const int32_t* base_lens,
                            const int32_t* row_starts, const int32_t* path, int32_t n_seqs, int32_t n_rows,
                            int32_t n_kv_heads, int32_t head_dim, int32_t page_size, void* stream) {
    clear_error();
    return launch_kv_compact(k_cache, v_cache, kv_dtype, n_layers, layer_bytes, page_table, max_pages_per_seq, base_lens,
                             row_starts, path, n_seqs, n_rows, n_kv_heads, head_dim, page_size, as_stream(stream));
}

}  // extern "C"
