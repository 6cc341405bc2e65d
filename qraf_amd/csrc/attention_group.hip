// attention_group.hip -- attention of rows that share the first positions of
// their caches (sequences with one prompt, the rows of one sequence).
//
// Row r of group g attends to positions t < ctx[r]; those below prefix[g] hold
// the same K and V for every row of the group.  Pages as in attention.hip.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace qraf_hip {

struct GroupArgs {
    const float* q;             // [n][H][HD]
    const void* kc;             // layer K pages
    const void* vc;             // layer V pages
    const int32_t* page_table;  // [n][max_pages]
    const int32_t* ctx;         // [n] positions attended
    const int32_t* starts;      // [groups + 1]
    const int32_t* prefix;      // [groups]
    float* out;                 // [n][H][HD]
    int n, groups, H, Hkv, G, page_size, max_pages, max_ctx;
    float scale;
};

// entries of the device-resident layout, taken into their ranges
__device__ __forceinline__ int group_start(const GroupArgs& a, int g) { return max(0, min(a.starts[g], a.n)); }
// the group of row r, a row inside some group: the last that starts at or before it and is not empty
__device__ __forceinline__ int group_of(const GroupArgs& a, int r) {
    int lo = 0, hi = a.groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (group_start(a, mid) <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ int row_ctx(const GroupArgs& a, int r) { return max(0, min(a.ctx[r], a.max_ctx)); }

// ---------------------------------------------------------------------------
// Any head layout and page size: a workgroup per (row, query head), its four
// waves taking 64-position tiles in turn, fp32 arithmetic throughout.  Scores
// with a position per lane; P.V with a dimension per lane (64 / HD positions
// side by side for HD < 64); the running maximum and sum of a softmax per wave,
// joined at the end.
// ---------------------------------------------------------------------------
template <int HD, int KV>
__device__ __forceinline__ float any_k(const GroupArgs& a, size_t block, int off, int d) {
    if (KV == DT_F32) return ((const float*)a.kc)[(block * a.page_size + off) * HD + d];
    if (KV == DT_F16) return (float)((const _Float16*)a.kc)[(block * a.page_size + off) * HD + d];
    return (float)((const int8_t*)a.kc)[block * a.page_size * (HD + 4) + (size_t)off * HD + d];
}
template <int HD, int KV>
__device__ __forceinline__ float any_v(const GroupArgs& a, size_t block, int off, int d) {
    if (KV == DT_F32) return ((const float*)a.vc)[(block * a.page_size + off) * HD + d];
    if (KV == DT_F16) return (float)((const _Float16*)a.vc)[(block * HD + d) * a.page_size + off];
    return (float)((const int8_t*)a.vc)[block * a.page_size * (HD + 4) + (size_t)d * a.page_size + off];
}
// int8 pages: the scale behind a block's bytes
template <int HD, int KV>
__device__ __forceinline__ float any_scale(const GroupArgs& a, const void* pool, size_t block, int off) {
    if (KV != DT_I8) return 1.f;
    return *(const float*)((const int8_t*)pool + block * a.page_size * (HD + 4) + (size_t)a.page_size * HD + 4 * off);
}

template <int HD, int KV>
__global__ __launch_bounds__(256) void group_any_kernel(GroupArgs a) {
    constexpr int DPL = HD > 64 ? HD / 64 : 1;  // dimensions per lane of P.V
    constexpr int NP = HD < 64 ? 64 / HD : 1;   // positions side by side
    __shared__ float s_q[HD];
    __shared__ float s_p[4][64];
    __shared__ uint32_t s_block[4][64];
    __shared__ int s_off[4][64];
    __shared__ float s_m[4], s_l[4], s_o[4][HD];
    const int r = blockIdx.x, h = blockIdx.y, kvh = h / a.G;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (r < group_start(a, 0) || r >= group_start(a, a.groups)) return;  // outside every group
    const int ctx = row_ctx(a, r), g = group_of(a, r), prefix = a.prefix[g], r0 = group_start(a, g);
    const size_t base = ((size_t)r * a.H + h) * HD;
    for (int d = tid; d < HD; d += 256) s_q[d] = a.q[base + d];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; j++) o[j] = 0.f;
    const int dl = lane % HD, pl = HD < 64 ? lane / HD : 0;
    const int tiles = (ctx + 255) / 256;
    for (int it = 0; it < tiles; it++) {
        const int t0 = it * 256 + wave * 64, t = t0 + lane;
        float sc = -INFINITY, vs = 0.f;
        size_t block = 0;
        int off = 0;
        if (t < ctx) {
            const int pg = a.page_table[(size_t)(t < prefix ? r0 : r) * a.max_pages + t / a.page_size];
            block = (size_t)pg * a.Hkv + kvh;
            off = t % a.page_size;
            float acc = 0.f;
#pragma unroll 8
            for (int d = 0; d < HD; d++) acc = __builtin_fmaf(any_k<HD, KV>(a, block, off, d), s_q[d], acc);
            sc = (acc * any_scale<HD, KV>(a, a.kc, block, off)) * a.scale;
            vs = any_scale<HD, KV>(a, a.vc, block, off);
        }
        float mt = sc;
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) mt = fmaxf(mt, __shfl_xor(mt, s));
        const float mn = fmaxf(m, mt), mu = mn == -INFINITY ? 0.f : mn;
        const float alpha = expf(m - mu);
        const float p = t < ctx ? expf(sc - mu) : 0.f;
        float lt = p;
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) lt += __shfl_xor(lt, s);
        l = l * alpha + lt;
        m = mn;
        s_p[wave][lane] = p * vs;
        s_block[wave][lane] = (uint32_t)block;
        s_off[wave][lane] = off;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < DPL; j++) o[j] *= alpha;
        const int here = min(64, ctx - t0);
        for (int k = pl; k < here; k += NP) {
            const float pk = s_p[wave][k];
#pragma unroll
            for (int j = 0; j < DPL; j++)
                o[j] = __builtin_fmaf(pk, any_v<HD, KV>(a, s_block[wave][k], s_off[wave][k], dl + 64 * j), o[j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int s = HD; s < 64; s <<= 1) o[0] += __shfl_xor(o[0], s);  // the positions side by side
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
    if (lane < HD)
#pragma unroll
        for (int j = 0; j < DPL; j++) s_o[wave][lane + 64 * j] = o[j];
    __syncthreads();
    const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), mu = M == -INFINITY ? 0.f : M;
    for (int d = tid; d < HD; d += 256) {
        float O = 0.f, L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float e = expf(s_m[w] - mu);
            O = __builtin_fmaf(s_o[w][d], e, O);
            L = __builtin_fmaf(s_l[w], e, L);
        }
        a.out[base + d] = ctx ? O / L : 0.f;
    }
}

size_t group_attention_workspace_bytes(int n, int groups, int H, int Hkv, int hd, int max_ctx) {
    (void)n, (void)groups, (void)H, (void)Hkv, (void)hd, (void)max_ctx;
    return 16;
}

int launch_group_attention(const float* q, const void* kc, const void* vc, uint32_t kv_dtype,
                           const int32_t* page_table, int max_pages, const int32_t* ctx, const int32_t* group_starts,
                           const int32_t* prefix, int n, int groups, int H, int Hkv, int hd, int page_size, float scale,
                           int max_ctx, float* out, void* ws, size_t ws_bytes, hipStream_t st) {
    QH_REQUIRE(q && kc && vc && page_table && ctx && group_starts && prefix && out && ws, QRAF_HIP_ERR_INVALID,
               "group attention: null pointer");
    QH_REQUIRE(n > 0 && n <= 1024, QRAF_HIP_ERR_INVALID, "group attention: %d rows outside 1..1024", n);
    QH_REQUIRE(groups > 0 && groups <= n, QRAF_HIP_ERR_INVALID, "group attention: %d groups of %d rows", groups, n);
    QH_REQUIRE(Hkv > 0 && H > 0 && H % Hkv == 0, QRAF_HIP_ERR_INVALID,
               "group attention: %d heads not a multiple of %d kv heads", H, Hkv);
    QH_REQUIRE(hd == 16 || hd == 32 || hd == 64 || hd == 128, QRAF_HIP_ERR_INVALID,
               "group attention: head_dim %d (16, 32, 64 or 128 supported)", hd);
    QH_REQUIRE(page_size > 0 && max_pages > 0 && max_ctx > 0 && max_ctx <= (long long)max_pages * page_size,
               QRAF_HIP_ERR_INVALID, "group attention: bad page geometry");
    QH_REQUIRE(kv_dtype == DT_F32 || kv_dtype == DT_F16 || kv_dtype == DT_I8, QRAF_HIP_ERR_DTYPE,
               "group attention: KV dtype %u", kv_dtype);
    QH_REQUIRE(ws_bytes >= group_attention_workspace_bytes(n, groups, H, Hkv, hd, max_ctx), QRAF_HIP_ERR_INVALID,
               "group attention: workspace of %zu bytes, %zu needed", ws_bytes,
               group_attention_workspace_bytes(n, groups, H, Hkv, hd, max_ctx));
    GroupArgs a{q, kc, vc, page_table, ctx, group_starts, prefix, out, n, groups, H, Hkv, H / Hkv, page_size, max_pages,
                max_ctx, scale};
    const dim3 grid(n, H);
#define QH_GROUP_ANY(HDv, KVv)                                                                     \
    if (hd == HDv && kv_dtype == KVv) {                                                            \
        hipLaunchKernelGGL((group_any_kernel<HDv, (int)KVv>), grid, dim3(256), 0, st, a);          \
        QH_CHECK_HIP(hipGetLastError());                                                           \
        return QRAF_HIP_OK;                                                                        \
    }
#define QH_GROUP_ANYS(HDv) QH_GROUP_ANY(HDv, DT_F32) QH_GROUP_ANY(HDv, DT_F16) QH_GROUP_ANY(HDv, DT_I8)
    QH_GROUP_ANYS(16) QH_GROUP_ANYS(32) QH_GROUP_ANYS(64) QH_GROUP_ANYS(128)
#undef QH_GROUP_ANYS
#undef QH_GROUP_ANY
    return QRAF_HIP_OK;
}

}  // namespace qraf_hip

using namespace qraf_hip;

extern "C" {

uint64_t qraf_hip_group_attention_workspace_bytes(int32_t n_rows, int32_t n_groups, int32_t n_heads,
                                                  int32_t n_kv_heads, int32_t head_dim, int32_t max_ctx) {
    if (n_rows <= 0 || n_groups <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_ctx <= 0) return 0;
    return group_attention_workspace_bytes(n_rows, n_groups, n_heads, n_kv_heads, head_dim, max_ctx);
}

int qraf_hip_group_attention_dev(const float* q, const void* k_cache, const void* v_cache, uint32_t kv_dtype,
                                 const int32_t* page_table, int32_t max_pages_per_seq, const int32_t* ctx_lens,
                                 const int32_t* group_starts, const int32_t* prefix_lens, int32_t n_rows,
                                 int32_t n_groups, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                 int32_t page_size, float scale, int32_t max_ctx, float* out, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
    clear_error();
    return launch_group_attention(q, k_cache, v_cache, kv_dtype, page_table, max_pages_per_seq, ctx_lens, group_starts,
                                  prefix_lens, n_rows, n_groups, n_heads, n_kv_heads, head_dim, page_size, scale,
                                  max_ctx, out, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
