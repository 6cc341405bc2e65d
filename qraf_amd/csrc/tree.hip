// tree.hip -- trees of drafted tokens: the accepted path, and its keys and values
// moved to where the sequence goes on.  (Attention of a tree's nodes:
// attention_group.hip.)
//
// A sequence's tree is its rows of a step: row 0 the last token that is certain (the
// root), every other row a drafted token behind its parent.  Node i's keys and values
// lie at position base + i of the cache, whatever its depth.
#include <algorithm>

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
// more, so path[j] >= j and a position is written only by a step no later than the
// one that reads it: each thread takes one element of a position's keys or values
// along the path, and no thread another's.
// ---------------------------------------------------------------------------
struct CompactArgs {
    uint8_t *kc, *vc;
    size_t layer_bytes;
    const int32_t *table, *base, *starts, *path;
    int max_pages, rows, Hkv, hd, page_size;
};
constexpr int CTH = 256, CHUNK = 64;  // threads; steps of the path at a time

template <int KV>
__global__ __launch_bounds__(CTH) void kv_compact_kernel(CompactArgs a) {
    constexpr int ITEM = KV == (int)DT_F32 ? 4 : KV == (int)DT_F16 ? 2 : 1;
    __shared__ int s_page[2][CHUNK], s_off[2][CHUNK], s_n;
    const int s = blockIdx.y, tid = threadIdx.x, ps = a.page_size, hd = a.hd;
    const int r0 = max(0, min(a.starts[s], a.rows)), n = max(0, min(a.starts[s + 1], a.rows) - r0);
    const int base = max(0, a.base[s]);
    const size_t block = (size_t)ps * (KV == (int)DT_I8 ? hd + 4 : hd * ITEM);  // bytes of a (page, KV head)
    uint8_t *kc = a.kc + blockIdx.x * a.layer_bytes, *vc = a.vc + blockIdx.x * a.layer_bytes;
    int last = -1;  // of the path so far
    for (int c = 0; c < n; c += CHUNK) {
        __syncthreads();
        if (tid < CHUNK) {
            const int j = c + tid, node = j < n ? a.path[r0 + j] : -1;
            int before = __shfl_up(node, 1);
            if (tid == 0) before = last;
            // an entry that does not ascend, is no node of the tree or lies past the table ends the path
            const bool good = node > before && node < n && (long long)base + node < (long long)a.max_pages * ps;
            const unsigned long long bad = ~__ballot(good);
            const int count = bad ? __ffsll(bad) - 1 : CHUNK;
            if (tid < count) {
                const int from = base + node, to = base + j;
                s_page[0][tid] = a.table[(size_t)s * a.max_pages + from / ps];
                s_page[1][tid] = a.table[(size_t)s * a.max_pages + to / ps];
                s_off[0][tid] = from % ps;
                s_off[1][tid] = to % ps;
            }
            if (tid == 0) s_n = count;
            last = __shfl(node, CHUNK - 1);
        }
        __syncthreads();
        const int count = s_n;
        auto move = [&](uint8_t* pool, int head, size_t first, size_t step, auto one) {
            typedef decltype(one) T;
            auto at = [&](int w, int j) {
                return (T*)(pool + ((size_t)s_page[w][j] * a.Hkv + head) * block + first + s_off[w][j] * step);
            };
            for (int j = 0; j < count; j++) {
                if (s_page[0][j] == s_page[1][j] && s_off[0][j] == s_off[1][j]) continue;
                *at(1, j) = *at(0, j);
            }
        };
        const int words = hd * ITEM / 4;  // of a position of K (and of f32 V)
        for (int e = tid; e < a.Hkv * words; e += CTH) {
            const int h = e / words, w = e % words;
            move(kc, h, 4 * (size_t)w, (size_t)hd * ITEM, uint32_t());
            if (KV == (int)DT_F32) move(vc, h, 4 * (size_t)w, (size_t)hd * ITEM, uint32_t());
        }
        if (KV != (int)DT_F32)
            for (int e = tid; e < a.Hkv * hd; e += CTH) {  // V by dimension
                const int h = e / hd, d = e % hd;
                if (KV == (int)DT_F16) move(vc, h, (size_t)d * ps * 2, 2, uint16_t());
                else move(vc, h, (size_t)d * ps, 1, uint8_t());
            }
        if (KV == (int)DT_I8)
            for (int e = tid; e < 2 * a.Hkv; e += CTH)  // scales
                move(e < a.Hkv ? kc : vc, e % a.Hkv, (size_t)ps * hd, 4, uint32_t());
        if (count < CHUNK) break;
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
#define QH_COMPACT(KVv)                                                                                            \
    if (kv_dtype == KVv) hipLaunchKernelGGL((kv_compact_kernel<(int)KVv>), dim3(layers, seqs), dim3(CTH), 0, st, a)
    QH_COMPACT(DT_F32);
    QH_COMPACT(DT_F16);
    QH_COMPACT(DT_I8);
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
