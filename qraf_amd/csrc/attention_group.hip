// attention_group.hip -- attention of rows that share the first positions of
// their caches (sequences with one prompt, the rows of one sequence).
//
// Row r of group g attends to positions t < ctx[r]; those below prefix[g] hold
// the same K and V for every row of the group.  Pages as in attention.hip.
//
// The work of one KV head is a list of jobs: per group its query vectors (rows x
// the G query heads of the KV head, "columns") in blocks of up to 128 over the
// positions below the prefix that some row of the block attends to, and the rows,
// four to a job, over their own positions behind the prefix.  Long jobs are cut
// along the positions into pieces of equal length, as many as there are
// workgroups at once (group_tile_kernel), all from the device-resident lengths:
// a long prefix of few columns spreads over the chip, ragged lengths balance, and
// a workgroup has one piece, or as few as may be (what a piece costs beside its
// tiles, q to stage and outputs to join, is what 3 to 5 of them take).  A piece that
// holds all there is of a column writes the output; the others write (max, sum,
// unnormalised output) parts, which group_merge_kernel joins in position order.
// Small calls go without: a workgroup per (row, KV head) takes all its positions.
// group_any_kernel takes the shapes that the tiles do not.
//
// Trees of drafted tokens (qraf_hip_tree_attention_dev) are groups all of whose positions
// are shared: a sequence's rows attend to its cache and, behind it, to the positions that
// their 64-bit masks name.  The same jobs, pieces and tiles; tiles that reach behind the
// cache take a bit for each position instead of a length.  Few rows on f32 pages go to
// attn_few_kernel (attention.hip).
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "group_pieces.h"
#include "wave.h"

namespace qraf_hip {

struct GroupArgs {
    const float* q;             // [n][H][HD]
    const void* kc;             // layer K pages
    const void* vc;             // layer V pages
    const int32_t* page_table;  // [n][max_pages]
    const int32_t* ctx;         // [n] positions attended
    const int32_t* starts;      // [groups + 1]
    const int32_t* prefix;      // [groups]
    float* out;                 // [n][H][HD], or (out_hi != null) the planes a GEMM reads (qraf_hip_split_bf16_dev)
    uint16_t *out_hi, *out_lo;
    float* part_o;              // [Hkv][slots][HD] unnormalised outputs of parts
    float2* part_ml;            // [Hkv][slots] their maxima (in powers of two) and sums
    int4* plan;                 // for the merge: [n][2] where each row's parts lie (group_plan)
    int n, groups, H, Hkv, G, page_size, max_pages, max_ctx;
    float scale;
    int ps_log2, job_cap;       // page_size = 1 << ps_log2; prefix jobs at most
    int tail_log2, tails;       // a tail job is 1 << tail_log2 rows; tail jobs
    long long slots;            // part slots of a KV head
    // Trees: groups are sequences, page_table is [groups][max_pages], prefix their caches' lengths, ctx unused.
    const unsigned long long* masks;  // [n] positions prefix + bit that a row attends to beside its cache
};

// output elements i .. i + 3, i
__device__ __forceinline__ void group_store4(const GroupArgs& a, size_t i, float4 v) {
    if (a.out_hi) {
        ushort4 h, l;
        split_bf16(v.x, &h.x, &l.x);
        split_bf16(v.y, &h.y, &l.y);
        split_bf16(v.z, &h.z, &l.z);
        split_bf16(v.w, &h.w, &l.w);
        *(ushort4*)(a.out_hi + i) = h;
        *(ushort4*)(a.out_lo + i) = l;
    } else {
        *(float4*)(a.out + i) = v;
    }
}
__device__ __forceinline__ void group_store(const GroupArgs& a, size_t i, float v) {
    if (a.out_hi) split_bf16(v, &a.out_hi[i], &a.out_lo[i]);
    else a.out[i] = v;
}

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
__device__ __forceinline__ int prefix_len(const GroupArgs& a, int g) { return max(0, min(a.prefix[g], a.max_ctx)); }
// trees: a mask behind a cache of `base` positions, below max_ctx; row r's; the end of what it attends to
__device__ __forceinline__ unsigned long long below_ctx(const GroupArgs& a, unsigned long long mask, int base) {
    const int room = a.max_ctx - base;
    return room >= 64 ? mask : mask & ((1ull << room) - 1);
}
__device__ __forceinline__ unsigned long long row_mask(const GroupArgs& a, int r, int base) {
    return below_ctx(a, a.masks[r], base);
}
__device__ __forceinline__ int mask_end(unsigned long long mask, int base) { return mask ? base + 64 - __clzll(mask) : base; }

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
    return *(const float*)((const int8_t*)pool + block * a.page_size * (HD + 4) + (size_t)a.page_size * HD + 4 * (size_t)off);
}

template <int HD, int KV, bool TREE>
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
    const int g = group_of(a, r), prefix = TREE ? prefix_len(a, g) : a.prefix[g], r0 = TREE ? g : group_start(a, g);
    const unsigned long long mask = TREE ? row_mask(a, r, prefix) : 0;
    const int ctx = TREE ? mask_end(mask, prefix) : row_ctx(a, r);
    auto attends = [&](int t) { return t < ctx && (!TREE || t < prefix || (mask >> (t - prefix) & 1)); };
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
        int off = TREE ? -1 : 0;  // (of a position that the row does not attend to: no value of it is read)
        const bool in = attends(t);
        if (in) {
            const int pg = a.page_table[(size_t)(TREE || t < prefix ? r0 : r) * a.max_pages + t / a.page_size];
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
        const float p = in ? expf(sc - mu) : 0.f;
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
            if (TREE && s_off[wave][k] < 0) continue;
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
        group_store(a, base + d, ctx ? O / L : 0.f);
    }
}

// ---------------------------------------------------------------------------
// The tiles: head_dim 64 or 128, pages of 16, 32, 64, ... positions, up to 128
// query heads per KV head.
//
// One wave holds 32 columns and takes 32 positions at a time, on the 32x32x16
// fp16 matrix products, transposed:
//     S^T[position][column] = K q^T     A = K (lane: position, 8 dims), B = q
//     O^T[dim][column]     += V^T p^T   A = V (lane: dim, 8 positions), B = p
// In the result of the first, lane l holds 16 scores of column l % 32 (its other
// 16 are in lane l ^ 32), so a softmax row's maximum, sum and rescaling factor
// are one register a lane and one exchange between the halves; and with
// position(A row) permuted as in key_of() those 16 are, 8 by 8, the B operand of
// the second: nothing moves between lanes.  32 columns and not 16: half the
// operand reads per product, and the reads are what bounds it.
//
// q, p and f32 K and V enter as fp16 hi + lo pairs (22 bits), fp16 K and V as they
// are, int8 widened; a product of two pairs is three matrix products (lo x lo is
// below 2^-22).  A choice for speed: three of them run at 383 TFLOP/s where fp32
// matrix products run at 154, and outputs come within 2.8e-7 to 3.5e-7 of 64-bit ones
// (fp32 products: 2.2e-7 to 4.7e-7).  int8 scales: K's on the scores, V's on p.  Sums
// in fp32.  So that neither half leaves fp16's range,
//   q     is over a power of two of its column,
//   K, V  (f32) over one of their tile's, in [2^14, 2^15) at its largest, or, where the
//         positions of a tile lie further apart than SPREAD, each over its own: a
//         position that some row does not attend to costs it no bits of the others;
//   p     of f32 and int8 V takes V's powers of two in, over one of the column's own,
//         which follows the largest weighted V of the tiles so far: what is lost of a
//         weighted V is below 2^-34 of that (2^-20 next to f32 V of no weight just
//         within SPREAD), however large a V of no weight is.
//
// Up to 64 columns, tails and int8: K of the next tile is requested behind this
// tile's scores, V behind its outputs, straight into the wave's registers; two waves
// per SIMD cover each other's waits.  More columns: four waves share tiles in LDS.
// Measured (16/2 heads of 128, us): 48 sequences of 5 rows at 128..4,096 fp16 positions
// 41, of which the tiles 34 (117 MB read in the 28 beside 6 of plan and prologue: the
// rate of a plain read); 128 rows behind 2,048 shared and 512 own ones 27, half of it
// plan, prologue and join; 4 chunks of 128 rows at 400..2,000 f32 positions 41 (matrix
// cores 18% busy, VALU 44%, 23% of the waves' time waiting for an instruction's turn);
// 256 rows of 32,768: fp16 154 (446 TFLOP/s of products with q and p in 22 bits: 893
// of the matrix cores'), int8 198, f32 266.  Powers of two by position and column cost
// f32 3 to 4% over one for a tile and a running one, and int8 nothing.
// ---------------------------------------------------------------------------
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int GW = 8, GTH = 64 * GW;  // waves and threads of a workgroup
constexpr int DIRECT_ROWS = 256;      // rows of a call without a plan, at most
constexpr int BLK = 128;              // columns of a block: 4 waves of 32
// p is held times 2^13 of the running maximum it was taken against, which follows the largest score only
// when that has grown by more than 2^2: outputs and sums are rescaled then, a few times a job and not at
// every tile (some of 32 columns finds a larger score nearly always)
// (int8: times 1, and brought into fp16's range with V's scale)
constexpr float P_UNIT = 13.f, GROWTH = 2.f;
// f32 positions whose largest value lies this far below the tile's get powers of two of their own.  Nearer ones lose
// at most 14 of the 38 bits between the tile's largest and fp16's least step.
constexpr float SPREAD = 0x1p-14f;

// max(m, |x|, |y|) and max(|x|, |y|) in one instruction; a NaN among them, of either kind, gives a NaN (fmaxf, v_max3_f32
// drop a quiet one, and what a signalling one was compared with)
__device__ __forceinline__ float amax3(float m, float x, float y) {
    asm("v_maximum3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(x), "v"(y));
    return m;
}
__device__ __forceinline__ float amax2(float x, float y) {
    float m;
    asm("v_maximum3_f32 %0, |%1|, |%2|, |%2|" : "=v"(m) : "v"(x), "v"(y));
    return m;
}
// some lane's condition, seldom true: its code lies behind the kernel, and registers are spilled there
__device__ __forceinline__ bool seldom(bool x) { return __builtin_expect(__any(x), 0); }
// |x|, or 0 of an infinity or NaN
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
__device__ __forceinline__ float fmax2(float x, float y) { return fmaxf(x, y); }
__device__ __forceinline__ int imax2(int x, int y) { return max(x, y); }
__device__ __forceinline__ int imin2(int x, int y) { return min(x, y); }

// the position, of a tile's 32, that row rho of the first product's A holds
__device__ __forceinline__ int key_of(int rho) {
    return 16 * ((rho >> 4) & 1) + 8 * ((rho >> 2) & 1) + 4 * ((rho >> 3) & 1) + (rho & 3);
}
// the row of the first product's A that holds position p of a tile: key_of(row_of(p)) = p
__device__ __forceinline__ int row_of(int p) { return (p & 0x13) | (p >> 1 & 4) | (p << 1 & 8); }
// power of two that brings a largest magnitude into [2^14, 2^15), as its exponent: -113 (fp32's largest) .. 110
__device__ __forceinline__ int unit_exp(float mx) {
    if (!(mx > 0.f)) return 110;
    int e;
    frexpf(mx, &e);
    return min(15 - e, 110);
}
// floor(x), at most 1000 (of a NaN, an infinity)
__device__ __forceinline__ int floor_to(float x) { return (int)floorf(fminf(x, 1000.f)); }
// of magnitudes the largest (a NaN of a NaN) and the least
struct Spread {
    float most = 0.f;
    uint32_t least = 0x7F800000u;
    __device__ __forceinline__ void add(float x, float y) {
        most = amax3(most, x, y);
        least = min(least, min(__float_as_uint(x), __float_as_uint(y)));
    }
    // whether values of the lane may lie too far below `all`, the largest of all lanes, or are no numbers
    __device__ __forceinline__ bool apart(float all) const { return !(most < INFINITY) || __uint_as_float(least) < all * SPREAD; }
};
// and whether they do (y, of a position; 0 has no bits to lose)
__device__ __forceinline__ bool far_below(float y, float all) { return y > 0.f && y < all * SPREAD; }
// two values as fp16 hi + lo, each to the nearest: 23 bits
__device__ __forceinline__ void split2(float x, float y, f16x2& hi, f16x2& lo) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    hi = __builtin_convertvector((f32x2{x, y}), f16x2);
    // (x - hi as a multiply-add: one instruction with the conversion inside)
    lo = __builtin_convertvector(
        (f32x2{__builtin_fmaf((float)hi[0], -1.f, x), __builtin_fmaf((float)hi[1], -1.f, y)}), f16x2);
}
// 8 values, value i times by(i), a power of two (the products inside the multiply-adds: 5 instructions a pair, 6 with
// them ahead)
template <typename F>
__device__ __forceinline__ void split8_by(const float (&x)[8], F by, f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        f16x2 h;
        h[0] = (_Float16)__builtin_fmaf(x[i], by(i), 0.f);
        h[1] = (_Float16)__builtin_fmaf(x[i + 1], by(i + 1), 0.f);
        uint32_t u = __builtin_bit_cast(uint32_t, h);
        asm("" : "+v"(u));  // one register of two halves, as the products take them
        h = __builtin_bit_cast(f16x2, u);
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = (_Float16)__builtin_fmaf(x[i], by(i), -(float)h[0]);
        lo[i + 1] = (_Float16)__builtin_fmaf(x[i + 1], by(i + 1), -(float)h[1]);
    }
}
__device__ __forceinline__ void split8(const float (&x)[8], float by, f16x8& hi, f16x8& lo) {
    split8_by(x, [by](int) { return by; }, hi, lo);
}
__device__ __forceinline__ void split8(const float (&x)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        f16x2 h, l;
        split2(x[i], x[i + 1], h, l);
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = l[0], lo[i + 1] = l[1];
    }
}
// the fp16 halves of a dword that are not numbers, as 0x1 in each (their exponent is all ones)
__device__ __forceinline__ uint32_t odd16(uint32_t u) { return (((u & 0x7C007C00u) + 0x04000400u) >> 15) & 0x00010001u; }
// 4 int8 (one dword) -> 4 fp16, exactly: the biased byte q + 128 under the
// exponent of 1024, less 1152
__device__ __forceinline__ uint2 widen4(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const f16x2 x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    const f16x2 y = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    return make_uint2(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y));
}
__device__ __forceinline__ f16x8 widen8(uint32_t w0, uint32_t w1) {
    const uint2 x = widen4(w0), y = widen4(w1);
    return __builtin_bit_cast(f16x8, make_uint4(x.x, x.y, y.x, y.y));
}

// A barrier for what lies in LDS: loads and stores to memory stay in flight
// (__syncthreads waits for all of them, 3 to 6 us a segment here).
__device__ __forceinline__ void lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---- the plan: jobs and their pieces, from the device-resident lengths, by every workgroup
struct GroupPlan {
    int* tiles;  // [jobs] tiles of each job: prefix blocks, then tails
    int* upto;   // [jobs + 1] pieces ahead of each job, and from bit 16 on jobs with tiles ahead of it
    int* jb;     // [groups + 1] first prefix job of each group
    int* gs;     // [groups + 1] group starts
    int* pre;    // [groups] prefix lengths
    int* ctx;    // [n] context lengths
    int np;      // prefix jobs
};
// the last entry of ascending v[0..n) at or below x (v[0] <= x)
__device__ __forceinline__ int last_at(const int* v, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// the same of two numbers at once
__device__ __forceinline__ void last_at(const int* v, int n, int x0, int x1, int& at0, int& at1) {
    at0 = at1 = 0;
    for (int step = 1 << (31 - __clz(n)); step; step >>= 1) {
        const int m0 = at0 + step, m1 = at1 + step, v0 = v[min(m0, n - 1)], v1 = v[min(m1, n - 1)];
        at0 = m0 < n && v0 <= x0 ? m0 : at0;
        at1 = m1 < n && v1 <= x1 ? m1 : at1;
    }
}
// the same by a whole wave, n <= 4096, of entries' bits in `mask`: two reads instead of one per halving
__device__ __forceinline__ int wave_last_at(const int* v, int n, int x, int mask = -1) {
    const int lane = threadIdx.x & 63, step = (n + 63) >> 6;
    int i = lane * step;
    const int b = (__popcll(__ballot(i < n && (v[min(i, n - 1)] & mask) <= x)) - 1) * step;
    i = b + lane;
    return b + __popcll(__ballot(lane < step && i < n && (v[min(i, n - 1)] & mask) <= x)) - 1;
}
// x summed over the lanes up to each: rows of 16, then rows 1 and 3, then 2 and 3
__device__ __forceinline__ int over_lanes_ahead(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
}
// v[0..n) to its exclusive prefix sums, v[n] the sum, by one wave
__device__ __forceinline__ void wave_prefix_sum(int* v, int n) {
    const int lane = threadIdx.x & 63, per = (n + 63) >> 6, i0 = min(n, lane * per), i1 = min(n, i0 + per);
    int sum = 0;
    for (int i = i0; i < i1; i++) sum += v[i];
    const int inc = over_lanes_ahead(sum);
    int run = inc - sum;
    for (int i = i0; i < i1; i++) {
        const int x = v[i];
        v[i] = run;
        run += x;
    }
    if (lane == 63) v[n] = inc;
}
// waves of a job of `cols` columns side by side along them (the others along the positions)
__device__ __forceinline__ int waves_over(int cols) { return cols > 64 ? 4 : cols > 32 ? 2 : 1; }
__device__ __forceinline__ int tiles_of(int positions, int cols) {
    const int s = cols > 64 ? 6 : cols > 32 ? 7 : 8;  // 32 positions times GW / waves_over(cols)
    return (positions + (1 << s) - 1) >> s;
}
// a tail begins with the 16 positions that hold the prefix's end, one page's
__device__ __forceinline__ int tail_base(int prefix) { return prefix & ~15; }

// a wave's sum of f(i) over i < n
template <typename F>
__device__ __forceinline__ int wave_sum(int n, F f) {
    int x = 0;
    for (int i = threadIdx.x & 63; i < n; i += 64) x += f(i);
    return over_wave(x, [](int u, int v) { return u + v; });
}
template <bool TREE>
__device__ void group_plan(const GroupArgs& a, GroupPlan& p, int shares) {
    const int tid = threadIdx.x;
    static_assert(2 * GTH >= 1024, "rows by thread");
    unsigned long long masks[2];  // (trees) of rows tid and tid + GTH
    if (TREE) masks[0] = a.masks[min(tid, a.n - 1)], masks[1] = a.masks[min(tid + GTH, a.n - 1)];
    for (int i = tid; i < max(a.n, a.groups + 1); i += GTH) {  // (all requested at once)
        const int c = TREE ? 0 : row_ctx(a, min(i, a.n - 1)), s = group_start(a, min(i, a.groups)),
                  t = group_start(a, min(i + 1, a.groups)), e = prefix_len(a, min(i, a.groups - 1));
        if (i < a.n) p.ctx[i] = c;
        if (i <= a.groups) p.gs[i] = s;
        if (i < a.groups) {
            p.pre[i] = e;
            p.jb[i] = (max(0, t - s) * a.G + BLK - 1) / BLK;
        }
    }
    for (int j = tid; j < a.job_cap + a.tails; j += GTH) p.tiles[j] = 0;
    lds_sync();
    if (tid < 64) wave_prefix_sum(p.jb, a.groups);
    lds_sync();
    p.np = min(p.jb[a.groups], a.job_cap);
    const int jobs = p.np + a.tails;
    const int r_first = p.gs[0], r_end = p.gs[a.groups];
    int group[2];  // of rows tid and tid + GTH
    last_at(p.gs, a.groups, max(tid, r_first), max(tid + GTH, r_first), group[0], group[1]);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int r = tid + k * GTH, g = group[k];
        if (r >= a.n || r < r_first || r >= r_end) continue;
        const int all = (p.gs[g + 1] - p.gs[g]) * a.G;
        int ctx = p.ctx[r], pre = p.pre[g];
        if (TREE) {
            ctx = p.ctx[r] = mask_end(below_ctx(a, masks[k], pre), pre);
            pre = ctx;
        }
        const int c0 = (r - p.gs[g]) * a.G, b1 = (c0 + a.G - 1) / BLK;
        for (int b = c0 / BLK; b <= b1 && p.jb[g] + b < p.np; b++)
            atomicMax(&p.tiles[p.jb[g] + b], tiles_of(min(ctx, pre), min(BLK, all - BLK * b)));
        if (ctx > pre) atomicMax(&p.tiles[p.np + (r >> a.tail_log2)], tiles_of(ctx - tail_base(pre), BLK));
    }
    lds_sync();
    if (tid < 64) {
        // the shortest piece of which there are at most `shares`, or as many times that as there are jobs
        // (from bit 16 on those of LONG_JOB tiles: where there is none, all of the at most 4,096 fit 32 bits)
        const int jobs_full = wave_sum(jobs, [&](int j) { return p.tiles[j] > 0 ? 1 + (p.tiles[j] >= LONG_JOB ? 1 << 16 : 0) : 0; });
        const int full = jobs_full & 0xFFFF, room = piece_room(full, shares);
        const bool longs = __builtin_amdgcn_readfirstlane(jobs_full >> 16) != 0;
        uint64_t all = (unsigned)wave_sum(jobs, [&](int j) { return p.tiles[j]; });
        if (longs) {
            all = (unsigned)wave_sum(jobs, [&](int j) { return p.tiles[j] & 0xFFFF; });
            all += (uint64_t)wave_sum(jobs, [&](int j) { return p.tiles[j] >> 16; }) << 16;
        }
        int few[4];  // up to 256 jobs: a lane's, in registers through the search
#pragma unroll
        for (int k = 0; k < 4; k++) few[k] = p.tiles[max(min(tid + 64 * k, jobs - 1), 0)];
        const int lo = shortest_piece(all, full, room, [&](int most) {
            const float per = 1.f / (float)most;
            if (jobs <= 256 && !longs) {
                int x = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) x += tid + 64 * k < jobs ? pieces_of(few[k], most, per) : 0;
                return __builtin_amdgcn_readfirstlane(over_wave(x, [](int u, int v) { return u + v; }));
            }
            if (longs) return wave_sum(jobs, [&](int j) { return pieces_of_long(p.tiles[j], most); });
            return wave_sum(jobs, [&](int j) { return pieces_of(p.tiles[j], most, per); });
        });
        const float per = 1.f / (float)lo;
        for (int j = tid; j < jobs; j += 64) {
            const int x = longs ? pieces_of_long(p.tiles[j], lo) : pieces_of(p.tiles[j], lo, per);
            p.upto[j] = x | (x ? 1 << 16 : 0);
        }
        wave_prefix_sum(p.upto, jobs);
    }
    lds_sync();
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        // {first column among the prefix jobs' (-1: outside every group), pieces ahead of its block, of the next, of
        // the one behind}, {which parts, pieces ahead of its tail, behind it}; a row's columns are in two blocks at most
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int r = tid + k * GTH;
            if (r >= a.n) continue;
            const bool in = r >= r_first && r < r_end;
            const int g = in ? group[k] : 0;
            const int pos = p.jb[g] * BLK + (r - p.gs[g]) * a.G, b = in ? pos / BLK : 0, t = p.np + (r >> a.tail_log2);
            a.plan[2 * r] = make_int4(in ? pos : -1, p.upto[min(b, jobs)], p.upto[min(b + 1, jobs)], p.upto[min(b + 2, jobs)]);
            if (TREE) a.plan[2 * r + 1] = make_int4(p.ctx[r] > 0 ? 1 : 0, 0, 0, 0);
            else a.plan[2 * r + 1] = make_int4((min(p.ctx[r], p.pre[g]) > 0 ? 1 : 0) | (p.ctx[r] > p.pre[g] ? 2 : 0), p.upto[t],
                                               p.upto[t + 1], 0);
        }
    }
}

// ---- the plan of trees of up to 64 sequences: a lane to a sequence, by each wave for itself, in registers.  A sequence's
// blocks but the last are alike; its positions are taken to end where a mask's highest bit may lie (tiles that no row
// attends to are skipped), so the masks are not waited for.  No barrier, a read, 3,300 cycles to the piece where the plan
// in LDS takes 9,000 to 12,000 (1 to 48 sequences).
struct LanePlan {
    int first, end, base;  // rows, cache
    int blocks, tiles, last;    // blocks of columns; tiles of each, of the last
    int pieces, last_pieces;    // of those
    int upto;                   // pieces ahead of the sequence's, and from bit 16 on its blocks ahead
    int all;                    // pieces of all sequences
};
__device__ __forceinline__ LanePlan lane_plan(const GroupArgs& a, int shares) {
    const int s = threadIdx.x & 63;
    LanePlan p;
    // (ascending, whatever is given: no two sequences share a row, and past the last there are none)
    int first = group_start(a, min(s, a.groups));
    first = max(first, __builtin_amdgcn_update_dpp(0, first, 0x111, 0xF, 0xF, false));
    first = max(first, __builtin_amdgcn_update_dpp(0, first, 0x112, 0xF, 0xF, false));
    first = max(first, __builtin_amdgcn_update_dpp(0, first, 0x114, 0xF, 0xF, false));
    first = max(first, __builtin_amdgcn_update_dpp(0, first, 0x118, 0xF, 0xF, false));
    first = max(first, __builtin_amdgcn_update_dpp(0, first, 0x142, 0xA, 0xF, false));
    p.first = max(first, __builtin_amdgcn_update_dpp(0, first, 0x143, 0xC, 0xF, false));
    p.end = __shfl_down(p.first, 1);
    if (s == 63) p.end = max(p.first, group_start(a, a.groups));
    p.base = prefix_len(a, min(s, a.groups - 1));
    const int cols = (p.end - p.first) * a.G, to = min(p.base + 64, a.max_ctx);
    p.blocks = (cols + BLK - 1) / BLK;
    p.tiles = p.blocks > 1 ? tiles_of(to, BLK) : 0;
    p.last = p.blocks > 0 ? tiles_of(to, cols - BLK * (p.blocks - 1)) : 0;
    auto sum = [](int x) { return __builtin_amdgcn_readfirstlane(over_wave(x, [](int u, int v) { return u + v; })); };
    const bool longs = __any(max(p.tiles, p.last) >= LONG_JOB);
    // (at most 1,088 blocks, of fewer than LONG_JOB tiles or of 2^24)
    const uint64_t mine = (uint64_t)max(p.blocks - 1, 0) * p.tiles + p.last;
    const uint64_t all = longs ? (unsigned)sum((int)(mine & 0xFFFF)) + ((uint64_t)(unsigned)sum((int)(mine >> 16)) << 16)
                               : (unsigned)sum((int)mine);
    const int full = sum(p.blocks), room = piece_room(full, shares);
    auto cut = [&](int most, int& pieces, int& last) {
        const float per = 1.f / (float)most;
        pieces = longs ? pieces_of_long(p.tiles, most) : pieces_of(p.tiles, most, per);
        last = longs ? pieces_of_long(p.last, most) : pieces_of(p.last, most, per);
        return max(p.blocks - 1, 0) * pieces + last;
    };
    int x, y;
    const int most = shortest_piece(all, full, room, [&](int m) { return sum(cut(m, x, y)); });
    const int own = cut(most, p.pieces, p.last_pieces) | p.blocks << 16, inc = over_lanes_ahead(own);
    p.upto = inc - own;
    p.all = __builtin_amdgcn_readlane(inc, 63) & 0xFFFF;
    return p;
}

// ---- a wave's K and V of one tile
template <int HD, int KV>
struct GroupTile;
template <int HD>
struct GroupTile<HD, (int)DT_F16> {
    f16x8 k[HD / 16];
    uint4 v[HD / 32][2];
};
template <int HD>
struct GroupTile<HD, (int)DT_I8> {
    uint4 k[HD / 32];
    uint2 v[HD / 32][2];
    float4 ks[4], vs[4];
};
template <int HD>
struct GroupTile<HD, (int)DT_F32> {
    typedef float vrow __attribute__((ext_vector_type(HD / 32)));
    float4 k[HD / 8];
    vrow v[16];
};

// DIRECT: no plan; workgroup (r, KV head) takes row r alone, its prefix and its tail one behind the other.
// LDS floats for the tiles: the waves' outputs, [GW][32][hd]; before them q, and two f32 tiles that waves share
constexpr int tile_floats(int hd) { return GW * 32 * hd; }

// TREE: rows attend to their sequence's cache and to the positions behind it that their masks name, all of them shared
// (the prefix ends where their attention does): tiles that reach behind the cache go by bits.
// LANES: the plan is lane_plan's.
// Trees, measured (16/2 heads of 128, us a call): 64 nodes at 8,000 positions, fp16, 25.4, of which the join's launch 4.7
// and in the tiles' 40,000 cycles the plan 4,500, the piece and q 10,000, four tiles 18,000 and the outputs 8,000; 48
// trees of up to 16 at 128..4,096, fp16, 52 to 64: 114 MB at a plain read's rate in 30 behind 20 that are fixed; 24 of up
// to 26 at 3,000..8,000, int8, 89 to 95: widening and softmax (VALU) beside the products; 8 of 64 at 777..2,000, f32, 44 to 48.
template <int HD, int KV, bool DIRECT, bool TREE, bool LANES>
__global__ __launch_bounds__(GTH, 2) void group_tile_kernel(GroupArgs a) {
    constexpr int KS = HD / 16, DT = HD / 32;  // products per score tile, 32-dim output tiles
    constexpr bool F32 = KV == (int)DT_F32, F16 = KV == (int)DT_F16, I8 = KV == (int)DT_I8;
    extern __shared__ __align__(16) float s_dyn[];
    __shared__ float s_m[GW][32], s_l[GW][32], s_qs[BLK];
    // f32 tiles that four waves share: the exponents of K's and V's powers of two, of 8 positions each, or (OWN) of each,
    // where the waves' maxima and sums lie behind the tiles
    int(*const s_kx)[32] = (int(*)[32])s_m;
    int(*const s_vx)[32] = (int(*)[32])s_l;
    constexpr int OWN = -(1 << 20);  // (scores over it are infinite)
    __shared__ int s_ku[2][4], s_vu[2][4];
    __shared__ unsigned long long s_mask[TREE ? BLK : 1];
    __shared__ long long s_to[BLK];  // where a column's output goes: an element of out, or ~ a slot of part_o
    constexpr long long NOWHERE = 1ll << 62;
    // [GW][32][HD] the waves' outputs, behind a segment's tiles; 16-byte piece c of a column's row lies at
    // c ^ (column % 16), which spreads a wave's writes over the banks
    float* s_o = s_dyn;
    // q's operands, during them: [lo, hi][4 tiles of 32 columns][KS][2 halves][33] 16-byte pieces of 8 dims, the 33rd
    // unused (a column's pieces, which neighbouring lanes write, are in banks of their own)
    constexpr int QB = 33, QT = 2 * KS * QB, QHI = 4 * QT;
    uint4 *s_qlo = (uint4*)s_dyn, *s_qhi = s_qlo + QHI;
    GroupPlan plan;
    unsigned long long* const masks = (unsigned long long*)(s_dyn + tile_floats(HD));  // LANES: all rows'
    LanePlan lp;
    plan.tiles = (int*)(s_dyn + tile_floats(HD));
    plan.upto = plan.tiles + a.job_cap + a.tails;
    plan.jb = plan.upto + a.job_cap + a.tails + 1;
    plan.gs = plan.jb + a.groups + 1;
    plan.pre = plan.gs + a.groups + 1;
    plan.ctx = plan.pre + a.groups;
    // opaque to the compiler before each use of many (here and below): else addresses made of it are formed once,
    // ahead of the loops, and spilled across them
    int tid = threadIdx.x;
    int lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto lanes_again = [&] {
        asm volatile("" : "+v"(tid));
        lane = tid & 63;
        col = lane & 31;
        half = lane >> 5;
    };
    const int kvh = blockIdx.y, w = blockIdx.x, G = a.G, psl = a.ps_log2, psm = (1 << psl) - 1;
    const float inv_g = 1.f / (float)G;

    int jobs = 0, pieces = w + 1;
    int d_ctx = 0, d_pre = 0, d_first = 0, d_tiles = 0;  // DIRECT: the row's context, prefix, group's first row; prefix tiles
    if constexpr (DIRECT) {
        static_assert(DIRECT_ROWS % 64 == 0, "rows by lane");
        int s[DIRECT_ROWS / 64], e[DIRECT_ROWS / 64];
#pragma unroll
        for (int k = 0; k < DIRECT_ROWS / 64; k++) {  // (groups <= rows <= DIRECT_ROWS)
            s[k] = group_start(a, min(lane + 64 * k, a.groups));
            e[k] = prefix_len(a, min(lane + 64 * k, a.groups - 1));
        }
        if (!TREE) d_ctx = row_ctx(a, w);
        if (w < group_start(a, 0) || w >= group_start(a, a.groups)) return;  // outside every group
        int g = -1;
#pragma unroll
        for (int k = 0; k < DIRECT_ROWS / 64; k++) g += __popcll(__ballot(lane + 64 * k < a.groups && s[k] <= w));
#pragma unroll
        for (int k = 0; k < DIRECT_ROWS / 64; k++)
            if (g >> 6 == k) {
                d_first = __builtin_amdgcn_readlane(s[k], g & 63);
                d_pre = __builtin_amdgcn_readlane(e[k], g & 63);
            }
        if (TREE) {
            d_ctx = mask_end(row_mask(a, w, d_pre), d_pre);
            d_first = g;  // (whose row of the page table is read)
        }
        d_tiles = (TREE ? d_ctx + 31 : min(d_ctx, d_pre) + 31) >> 5;
    } else if constexpr (LANES) {
        const unsigned long long m0 = a.masks[min(tid, a.n - 1)], m1 = a.masks[min(tid + GTH, a.n - 1)];
        lp = lane_plan(a, gridDim.x);
        if (tid < a.n) masks[tid] = m0;
        if (tid + GTH < a.n) masks[tid + GTH] = m1;
        pieces = lp.all;
        lds_sync();
    } else {
        group_plan<TREE>(a, plan, gridDim.x);
        jobs = plan.np + a.tails;
        pieces = plan.upto[jobs] & 0xFFFF;
    }
    // (trees) behind the last position that row r of a sequence with `cache` positions attends to
    auto row_end = [&](int r, int cache) { return LANES ? mask_end(below_ctx(a, masks[r], cache), cache) : plan.ctx[r]; };

    for (int piece = w; piece < pieces; piece += gridDim.x) {
        lanes_again();
        int j = 0, here = 0, i_of = 0, ja = 0, jend = 0;
        bool whole = true;  // tiles [ja, jend) of the job
        int l_seq = 0, l_first = 0, l_end = 0, l_block = 0;  // LANES: the piece's sequence, its rows, the block
        if constexpr (!DIRECT) {
            int tiles, n_of;
            if constexpr (LANES) {
                const int at = lp.upto & 0xFFFF, of = max(lp.blocks - 1, 0) * lp.pieces + lp.last_pieces;
                l_seq = __ffsll((unsigned long long)__ballot(piece >= at && piece < at + of)) - 1;
                auto its = [&](int x) { return __builtin_amdgcn_readlane(x, l_seq); };
                const int upto = its(lp.upto), k = its(lp.pieces), last = its(lp.blocks) - 1, local = piece - (upto & 0xFFFF);
                l_block = last > 0 ? min((int)(((float)local + 0.5f) / (float)k), last) : 0;
                here = upto + l_block * (k | 1 << 16);
                n_of = l_block < last ? k : its(lp.last_pieces);
                tiles = l_block < last ? its(lp.tiles) : its(lp.last);
                l_first = its(lp.first);
                l_end = its(lp.end);
            } else {
                j = __builtin_amdgcn_readfirstlane(wave_last_at(plan.upto, jobs, piece, 0xFFFF));
                here = __builtin_amdgcn_readfirstlane(plan.upto[j]);
                const int next = __builtin_amdgcn_readfirstlane(plan.upto[j + 1]);
                tiles = __builtin_amdgcn_readfirstlane(plan.tiles[j]);
                n_of = (next & 0xFFFF) - (here & 0xFFFF);
            }
            i_of = piece - (here & 0xFFFF);
            const int each = (int)((unsigned)tiles / (unsigned)n_of), odd = tiles - each * n_of;  // `odd` pieces of one more
            ja = i_of * each + min(i_of, odd);
            jend = ja + each + (i_of < odd ? 1 : 0);
            whole = n_of == 1;
        }

        // ---- the wave's place: qt of wq waves side by side along the job's columns, kw of wk along the positions
        bool tail = !DIRECT && !LANES && j >= plan.np;
        int g, trow, first, cols, wq;  // group; the row whose table is read; first column (among all rows'), columns
        int bfirst = 0, bcols = 0;     // those of the workgroup (of a prefix)
        if constexpr (DIRECT) {
            wq = 1;
            first = bfirst = w * G;
            cols = bcols = G;
            // tiles: the prefix's, then the tail's
            jend = d_tiles + (!TREE && d_ctx > d_pre ? (d_ctx - tail_base(d_pre) + 31) >> 5 : 0);
            tail = !TREE && wave >= d_tiles;
            trow = tail ? w : d_first;
            g = 0;
        } else if (!TREE && tail) {    // a row's columns are 1, 2 or 4 waves'
            wq = 4;
            const int side = 4 >> a.tail_log2, c0 = 32 * (wave & (side - 1));
            const int row = ((j - plan.np) << a.tail_log2) + ((wave & 3) >> (2 - a.tail_log2));
            const bool in = row < a.n && row >= plan.gs[0] && row < plan.gs[a.groups];
            trow = min(row, a.n - 1);
            g = in ? wave_last_at(plan.gs, a.groups, trow) : 0;
            first = trow * G + c0;
            cols = in && plan.ctx[trow] > plan.pre[g] ? min(32, G - c0) : 0;
        } else {
            g = LANES ? l_seq : wave_last_at(plan.jb, a.groups, j);
            const int b = LANES ? l_block : j - plan.jb[g];
            trow = LANES ? l_first : plan.gs[g];
            cols = bcols = min(BLK, ((LANES ? l_end : plan.gs[g + 1]) - trow) * G - BLK * b);
            wq = waves_over(cols);
            const int c0 = 32 * (wave & (wq - 1));
            bfirst = trow * G + BLK * b;
            first = bfirst + c0;
            cols = min(32, cols - c0);
        }
        wq = __builtin_amdgcn_readfirstlane(wq);
        cols = __builtin_amdgcn_readfirstlane(max(cols, 0));
        const int wk = GW / wq, qt = wave & (wq - 1), kw = wave / wq;
        const int cache = __builtin_amdgcn_readfirstlane(DIRECT ? d_pre : LANES ? __builtin_amdgcn_readlane(lp.base, l_seq) : plan.pre[g]);  // (trees: ahead of the masks)
        const int pre = TREE ? INT_MAX : cache, base = tail ? tail_base(pre) : 0;
        int lo = tail ? pre : 0;
        // the page table through scalar loads: an id does not wait for vector loads ahead of it
        typedef const __attribute__((address_space(4))) int32_t ConstInt;
        auto table_of = [&](int row) {
            return (ConstInt*)(uintptr_t)(a.page_table + (size_t)__builtin_amdgcn_readfirstlane(row) * a.max_pages);
        };
        ConstInt* ptab = table_of(TREE && !DIRECT ? g : trow);

        // ---- the lane's column (past the last: that again, not written), row and limit
        const int ab = min(first + min(col, max(cols - 1, 0)), a.n * G - 1);
        const int r = DIRECT ? w : (int)(((float)ab + 0.5f) * inv_g);  // (ab < 2^17: exact)
        const size_t orow = ((size_t)r * a.H + kvh * G + (ab - r * G)) * HD;
        const int ctx = DIRECT ? d_ctx : row_end(r, cache);
        int lim = cols == 0 ? 0 : tail ? ctx : min(ctx, pre);
        // behind the last position that some of the wave's columns attends to
        int kend = __builtin_amdgcn_readfirstlane(DIRECT ? lim : over_wave(lim, imax2)), klast = max(kend - 1, 0);
        int least = TREE ? cache : __builtin_amdgcn_readfirstlane(DIRECT ? lim : over_wave(lim, imin2));
        // (trees) the positions of the tile at t that the lane's column attends to, as bits; those of its half from bit 0
        auto attended = [&](int t) {
            const unsigned long long mask = s_mask[qt * 32 + col];
            const int d = t - cache, in = min(max(d, 0), 63), ahead = min(max(-d, 0), 32);  // (ahead: positions of the cache)
            const uint32_t b = d >= 64 ? 0u : (uint32_t)((mask >> in) << ahead | ((1ull << ahead) - 1));
            return b >> (8 * half);
        };
        auto bit_of = [](uint32_t b, int x) { return (b >> (16 * (x >> 3) + (x & 7)) & 1) != 0; };  // of register x

        // ---- loads of the tile at position t
        GroupTile<HD, KV> tl;
        int pg0 = 0, pg1 = 0;
        auto ids = [&](int t) {
            pg0 = ptab[min(t, klast) >> psl];
            pg1 = ptab[min(t + 16, klast) >> psl];
        };
        const size_t blk = (size_t)a.page_size * (I8 ? HD + 4 : F16 ? 2 * HD : 4 * HD);  // bytes of a (page, KV head)
        auto block = [&](const void* pool, int pg) { return (const char*)pool + ((size_t)pg * a.Hkv + kvh) * blk; };
        // (real false: one address for all lanes, a load that nothing uses)
        auto load_k = [&](int t, bool real = true) {
            const int pc = min(t + key_of(col), klast);  // (past the end: the last position's, masked below)
            const char* kp = pc >= t + 16 && real ? block(a.kc, pg1) : block(a.kc, pg0);
            const uint32_t on = real ? 0xFFFFFFFFu : 0u;
            if constexpr (F16) {
                const uint32_t o = ((uint32_t)((pc & psm) * HD + 8 * half) * 2u) & on;
#pragma unroll
                for (int kk = 0; kk < KS; kk++) tl.k[kk] = *(const f16x8*)(kp + (o + 32u * kk));
            } else if constexpr (I8) {
                const uint32_t o = (uint32_t)((pc & psm) * HD + 16 * half) & on;
#pragma unroll
                for (int kk = 0; kk < KS / 2; kk++) tl.k[kk] = *(const uint4*)(kp + (o + 32u * kk));
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const char* sp = block(a.kc, b ? pg1 : pg0) + (size_t)a.page_size * HD + 4 * (((t + 16 * b) & psm) + 8 * half);
                    tl.ks[2 * b] = *(const float4*)sp;
                    tl.ks[2 * b + 1] = *(const float4*)(sp + 16);
                }
            } else {
                const uint32_t o = ((uint32_t)((pc & psm) * HD + 8 * half) * 4u) & on;
#pragma unroll
                for (int kk = 0; kk < KS; kk++) {
                    tl.k[2 * kk] = *(const float4*)(kp + (o + 64u * kk));
                    tl.k[2 * kk + 1] = *(const float4*)(kp + (o + 64u * kk + 16u));
                }
            }
        };
        auto load_v = [&](int t, bool real = true) {
            const uint32_t on = real ? 0xFFFFFFFFu : 0u;
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const char* vp = block(a.vc, b ? pg1 : pg0);
                const int off = ((t + 16 * b) & psm) + 8 * half;
                if constexpr (F16) {
#pragma unroll
                    for (int d = 0; d < DT; d++)
                        tl.v[d][b] = *(const uint4*)(vp + (((uint32_t)((32 * d + col) * a.page_size + off) * 2u) & on));
                } else if constexpr (I8) {
#pragma unroll
                    for (int d = 0; d < DT; d++)
                        tl.v[d][b] = *(const uint2*)(vp + ((uint32_t)((32 * d + col) * a.page_size + off) & on));
                    const char* sp = vp + (size_t)a.page_size * HD + 4 * off;
                    tl.vs[2 * b] = *(const float4*)sp;
                    tl.vs[2 * b + 1] = *(const float4*)(sp + 16);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int pc = min(t + 16 * b + 8 * half + i, klast);
                        const char* xp = pc >= t + 16 ? block(a.vc, pg1) : block(a.vc, pg0);
                        tl.v[8 * b + i] = *(const typename GroupTile<HD, (int)DT_F32>::vrow*)(
                            xp + (((uint32_t)((pc & psm) * HD + DT * col) * 4u) & on));
                    }
                }
            }
        };

        // f32 rows of 128 fill the registers: V is requested behind the scores, the next K behind the outputs
        constexpr bool TURNS = F32 && HD == 128;
        // the wave's tiles: every wk-th 32 positions
        int i = DIRECT ? wave : ja;
        int t = __builtin_amdgcn_readfirstlane(DIRECT ? base + 32 * (i - (tail ? d_tiles : 0)) : base + (i * wk + kw) * 32);
        const int dt = 32 * wk;
        const bool shared = !DIRECT && !I8 && !tail && wq == 4;
        bool more = i < jend && (DIRECT || t < kend);
        ids(more ? t : 0);
        // No load of K and V depends on a branch, here and below (but whether waves share tiles): where paths with more and
        // with fewer loads behind one meet, a wait for it is a wait for all.  A wave without tiles reads its pool's first page.
        pg0 = more ? pg0 : 0;
        pg1 = more ? pg1 : 0;

        // Tiles that four waves share (below): a wave's 8 positions of a tile; fp16's first is requested ahead of q's end.
        constexpr bool SHARES = !DIRECT && !I8;
        constexpr int NP = HD / 64, PCS = HD / 8, RP = 64 / PCS;  // K: passes, pieces of a row, rows of a pass
        typedef float vpart __attribute__((ext_vector_type(NP)));
        std::conditional_t<SHARES && F32, float[NP][8], int> kx;
        std::conditional_t<SHARES && F32, vpart[8], int> vx;
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        std::conditional_t<SHARES && F16, u32x4[NP], int> kr, vr;  // 8 dims of K, 8 positions of V
        int kl = 0, id = 0;  // the last position that some column of the block attends to; the next request's page
        bool some = true;    // (there is one; else no page is named, and the first is read)
        auto id_of = [&](int at) { return some ? ptab[min(at + 8 * qt, kl) >> psl] : 0; };
        auto request = [&](int at, int page) {
            if constexpr (SHARES) {
                const char *kp = block(a.kc, page), *vp = block(a.vc, page);
                lanes_again();
#pragma unroll
                for (int u = 0; u < NP; u++) {
                    const uint32_t off = (uint32_t)((min(at + 8 * qt + u * RP + lane / PCS, kl) & psm) * HD + 8 * (lane % PCS));
                    if constexpr (F32) {
                        const float4 x = *(const float4*)(kp + 4u * off), y = *(const float4*)(kp + (4u * off + 16u));
                        kx[u][0] = x.x, kx[u][1] = x.y, kx[u][2] = x.z, kx[u][3] = x.w;
                        kx[u][4] = y.x, kx[u][5] = y.y, kx[u][6] = y.z, kx[u][7] = y.w;
                    } else {
                        kr[u] = *(const u32x4*)(kp + 2u * off);
                        vr[u] = *(const u32x4*)(vp + 2u * (uint32_t)((64 * u + lane) * a.page_size + ((at + 8 * qt) & psm)));
                    }
                }
                if constexpr (F32) {
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        vx[k] = *(const vpart*)(vp + (uint32_t)(((min(at + 8 * qt + k, kl) & psm) * HD + NP * lane) * 4));
                }
            }
        };
        int id0 = 0;
        if (SHARES && shared) {
#pragma unroll
            for (int c = 0; c < BLK; c += 64)
                kl = max(kl, row_end((int)(((float)(bfirst + min(lane + c, bcols - 1)) + 0.5f) * inv_g), cache));
            kl = min(__builtin_amdgcn_readfirstlane(over_wave(kl, imax2)), pre);
            some = kl > 0;
            kl = max(kl, 1) - 1;
            id0 = id_of(t);
            id = id_of(t + dt);
        }

        // ---- q as fp16 hi + lo, scaled per column: 32 (HD 128) or 16 neighbouring lanes to a column, 16 bytes each,
        // all waves (a lane to a column, as the products take it, is a line of memory per lane and load: 2 us more)
        auto stage_q = [&](auto tiles_c) {
            constexpr int NQ = decltype(tiles_c)::value * 32 * HD / (4 * GTH), CPL = 256 / HD;
            const int d0 = 4 * (lane % (HD / 4)), c0 = wave * NQ * CPL + lane / (HD / 4);
            float4 x[NQ];
#pragma unroll
            for (int u = 0; u < NQ; u++) {
                const int c = c0 + u * CPL;
                int row, h;
                if (!DIRECT && tail) {
                    const int per = 7 - a.tail_log2;  // BLK columns over the rows
                    row = min(((j - plan.np) << a.tail_log2) + (c >> per), a.n - 1);
                    h = min(c & ((1 << per) - 1), G - 1);
                } else {
                    const int at = bfirst + min(c, bcols - 1);
                    row = DIRECT ? w : (int)(((float)at + 0.5f) * inv_g);
                    h = at - row * G;
                }
                x[u] = *(const float4*)(a.q + (uint32_t)((row * a.H + kvh * G + h) * HD + d0));
            }
            // (behind q, which is waited for alone)
            if constexpr (SHARES && decltype(tiles_c)::value == 4) {
                if (!shared) load_k(more ? t : 0);
                else if (F16) request(t, id0);  // (f32: registers)
            } else {
                load_k(more ? t : 0);
            }
            const int kk = I8 ? 2 * (d0 >> 5) + ((d0 >> 3) & 1) : d0 >> 4, hf = I8 ? (d0 >> 4) & 1 : (d0 >> 3) & 1;
#pragma unroll
            for (int u = 0; u < NQ; u++) {
                const int c = c0 + u * CPL;
                float mx = fmaxf(fmaxf(fabsf(x[u].x), fabsf(x[u].y)), fmaxf(fabsf(x[u].z), fabsf(x[u].w)));
                mx = over_row(mx, fmax2);
                if (HD == 128) mx = over_rows(mx, fmax2);
                const int e = mx < INFINITY ? unit_exp(mx) : 0;
                const float sg = copysignf(ldexpf(1.f, e), a.scale);  // (scores take the scale's magnitude)
                f16x2 h0, l0, h1, l1;
                split2(x[u].x * sg, x[u].y * sg, h0, l0);
                split2(x[u].z * sg, x[u].w * sg, h1, l1);
                uint2* to = (uint2*)(s_qlo + (c >> 5) * QT + (2 * kk + hf) * QB + (c & 31)) + ((d0 >> 2) & 1);
                to[0] = make_uint2(__builtin_bit_cast(uint32_t, l0), __builtin_bit_cast(uint32_t, l1));
                to[2 * QHI] = make_uint2(__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1));
                if (d0 == 0) s_qs[c] = ldexpf(fabsf(a.scale) * 1.44269504088896340736f, -e);
            }
        };
        const unsigned long long mask_of =
            LANES ? below_ctx(a, masks[(int)(((float)(bfirst + min(tid % BLK, bcols - 1)) + 0.5f) * inv_g)], cache)
            : TREE ? row_mask(a, DIRECT ? w : (int)(((float)(bfirst + min(tid % BLK, bcols - 1)) + 0.5f) * inv_g), cache) : 0;
        if (DIRECT || wq == 1) stage_q(std::integral_constant<int, 1>());
        else if (wq == 2) stage_q(std::integral_constant<int, 2>());
        else stage_q(std::integral_constant<int, 4>());
        if (!TURNS && !(SHARES && shared)) load_v(more ? t : 0);  // (behind q: their registers)
        if (TREE) s_mask[tid % BLK] = mask_of;
        lds_sync();
        const float qs = s_qs[qt * 32 + col];  // scores in powers of two

        float m = -INFINITY, l = 0.f;  // running maximum; sum of the lane's own positions, times 2^13
        int vexp = 110;                // f32, int8: the column's outputs are held times 2^vexp
        f32x16 o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int x = 0; x < 16; x++) o[d][x] = 0.f;

        // the running maximum to that of a tile, mt, if it has grown (f32, int8: a whole number, so that outputs keep
        // their bits: they and the column's power of two go along)
        auto follow = [&](float mt) {
            if (!__any(mt > m + GROWTH)) return;
            const float mn = fmaxf(m, F16 ? mt : ceilf(mt));
            float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
            if constexpr (!F16) {
                const int up = min(floor_to(mn - m), 110 - vexp);
                vexp += up;
                alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn + (float)up);
            }
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[d][x] *= alpha;
            m = mn;
        };
        // the column's power of two to `lim`, the one that a tile's weighted V need, if it is more than GROWTH above
        auto hold = [&](int lim) {
            if (!__any(vexp > lim + (int)GROWTH)) return;
            const int down = vexp > lim + (int)GROWTH ? lim - vexp : 0;
            const float f = ldexpf(1.f, down);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[d][x] *= f;
            vexp += down;
        };

        if constexpr (SHARES) {
            // Tiles of more than 64 columns: the four waves side by side load a quarter of a tile each, 8 positions, and
            // write it as operands for all of them, f32 split (alone each would load and split it all, and a lane to a
            // position reads a line of memory per lane).  The tiles lie where q's hi halves were, which stay in
            // registers.  f32: K's and V's powers of two are those of the 8 positions, or each position's.  256 rows of
            // 32,768 positions, 16/2 heads of 128: f32 in 0.63 and fp16 in 0.89 of the time of waves alone; int8 gained
            // nothing and goes on alone.
            if (shared) {
                constexpr int HL = F32 ? 2 : 1, KP = HL * QT, VP = 2 * 64 * DT, TP = KP + HL * VP;  // 16-byte pieces: hi, lo
                static_assert((QHI + 2 * TP) * 16 <= 4 * tile_floats(HD), "q's lo halves and a tile of each kw");
                uint4* tile = s_qhi + kw * TP;
                f16x8 qh[KS];
#pragma unroll
                for (int kk = 0; kk < KS; kk++) qh[kk] = __builtin_bit_cast(f16x8, s_qhi[qt * QT + half * QB + col + 2 * QB * kk]);
                if (F32) request(t, id0);
                for (; i < jend; i++, t += dt) {
                    lds_sync();  // what lay there is read
                    // ---- this wave's quarter
                    if constexpr (F32) {
                        Spread sp;
                        float y[NP];  // (a row's 8 values of this lane for the row)
#pragma unroll
                        for (int u = 0; u < NP; u++) {
                            y[u] = amax2(kx[u][0], kx[u][1]);
#pragma unroll
                            for (int k = 2; k < 8; k += 2) y[u] = amax3(y[u], kx[u][k], kx[u][k + 1]);
                        }
                        sp.add(y[0], y[NP - 1]);
                        float most = over_wave(sp.most, fmax2);
                        bool k_own = false, v_own = false;
                        if (seldom(sp.apart(most))) {
                            most = 0.f;
#pragma unroll
                            for (int u = 0; u < NP; u++) {
                                y[u] = 0.f;
#pragma unroll
                                for (int k = 0; k < 8; k++) y[u] = fmaxf(y[u], finite_abs(kx[u][k]));
                                y[u] = PCS == 16 ? over_row(y[u], fmax2) : over_8(y[u], fmax2);
                                most = fmaxf(most, y[u]);
                            }
                            most = over_wave(most, fmax2);
#pragma unroll
                            for (int u = 0; u < NP; u++) k_own = k_own || __any(far_below(y[u], most));
                        }
                        const int e = __builtin_amdgcn_readfirstlane(unit_exp(most));
                        lanes_again();
#pragma unroll
                        for (int u = 0; u < NP; u++) {
                            const int p = 8 * qt + u * RP + lane / PCS;
                            int eu = e;
                            if (__builtin_expect(k_own, 0)) {
                                eu = unit_exp(y[u]);
                                s_kx[kw][p] = eu;
                            }
                            f16x8 h, lw;
                            split8(kx[u], ldexpf(1.f, eu), h, lw);
                            uint4* to = tile + (lane % PCS) * QB + row_of(p);
                            to[0] = __builtin_bit_cast(uint4, h);
                            to[QT] = __builtin_bit_cast(uint4, lw);
                        }
                        sp = Spread();
                        float z[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            if constexpr (NP == 1) z[k] = fabsf(vx[k][0]);
                            else z[k] = amax2(vx[k][0], vx[k][1]);
                            if (NP == 1) z[k] = over_pair(z[k], amax2);  // (of 2 dims: one alone is often small)
                            if (k & 1) sp.add(z[k - 1], z[k]);
                        }
                        most = over_wave(sp.most, fmax2);
                        if (seldom(sp.apart(most))) {
                            most = 0.f;
#pragma unroll
                            for (int k = 0; k < 8; k++) {
                                z[k] = 0.f;
#pragma unroll
                                for (int c = 0; c < NP; c++) z[k] = fmaxf(z[k], finite_abs(vx[k][c]));
                                z[k] = over_wave(z[k], fmax2);
                                most = fmaxf(most, z[k]);
                            }
#pragma unroll
                            for (int k = 0; k < 8; k++) v_own = v_own || __any(far_below(z[k], most));
                        }
                        const int ev = __builtin_amdgcn_readfirstlane(unit_exp(most));
                        float vg = ldexpf(1.f, ev);
                        lanes_again();
                        if (__builtin_expect(v_own, 0)) {
#pragma unroll
                            for (int k = 0; k < 8; k++) {
                                const int ek = __builtin_amdgcn_readfirstlane(unit_exp(z[k]));
#pragma unroll
                                for (int c = 0; c < NP; c++) vx[k][c] = ldexpf(vx[k][c], ek);
                                if (lane == 0) s_vx[kw][8 * qt + k] = ek;
                            }
                            vg = 1.f;
                        }
#pragma unroll
                        for (int c = 0; c < NP; c++) {
                            float x[8];
#pragma unroll
                            for (int k = 0; k < 8; k++) x[k] = vx[k][c];
                            f16x8 h, lw;
                            split8(x, vg, h, lw);
                            const int dim = NP * lane + c;
                            uint4* to = tile + KP + (dim % DT * 2 + (qt >> 1)) * 64 + (qt & 1) * 32 + dim / DT;
                            to[0] = __builtin_bit_cast(uint4, h);
                            to[VP] = __builtin_bit_cast(uint4, lw);
                        }
                        if (lane == 0) {
                            s_ku[kw][qt] = k_own ? OWN : e;
                            s_vu[kw][qt] = v_own ? OWN : ev;
                        }
                    } else {
                        lanes_again();
                        const int valid = kl + 1 - (t + 8 * qt);  // positions of the 8 that are any (V behind: zeros)
#pragma unroll
                        for (int u = 0; u < NP; u++) {
                            const int p = 8 * qt + u * RP + lane / PCS, dim = 64 * u + lane;
                            auto keep = [&](uint32_t x, int k) {
                                return x & (valid >= 2 * k + 2 ? 0xFFFFFFFFu : valid == 2 * k + 1 ? 0xFFFFu : 0u);
                            };
                            const uint4 vv = make_uint4(keep(vr[u][0], 0), keep(vr[u][1], 1), keep(vr[u][2], 2), keep(vr[u][3], 3));
                            tile[lane % PCS * QB + row_of(p)] = __builtin_bit_cast(uint4, kr[u]);
                            tile[KP + ((dim >> 5) * 2 + (qt >> 1)) * 64 + (qt & 1) * 32 + (dim & 31)] = vv;
                        }
                    }
                    lds_sync();
                    request(t + dt, id);
                    id = id_of(t + 2 * dt);
                    if (t >= kend) continue;
                    const bool edge = t + 32 > least;
                    // ---- scores
                    lanes_again();
                    f32x16 s;
#pragma unroll
                    for (int x = 0; x < 16; x++) s[x] = 0.f;
                    const uint4 *kt = tile + half * QB + col, *qtile = s_qlo + qt * QT + half * QB + col;
                    uint4 kf[2][3];  // a product ahead, and no more of them: registers
                    kf[0][0] = kt[0], kf[0][2] = qtile[0];
                    if (F32) kf[0][1] = kt[QT];
#pragma unroll
                    for (int kk = 0; kk < KS; kk++) {
                        if (kk + 1 < KS) {
                            kf[(kk + 1) & 1][0] = kt[2 * QB * (kk + 1)];
                            if (F32) kf[(kk + 1) & 1][1] = kt[QT + 2 * QB * (kk + 1)];
                            kf[(kk + 1) & 1][2] = qtile[2 * QB * (kk + 1)];
                        }
                        const f16x8 kh = __builtin_bit_cast(f16x8, kf[kk & 1][0]);
                        if constexpr (F32)
                            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, kf[kk & 1][1]), qh[kk], s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, __builtin_bit_cast(f16x8, kf[kk & 1][2]), s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[kk], s, 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    // f32: scores and outputs over the positions' powers of two (half's 8 of a quarter of the tile)
                    float fs[2] = {qs, qs};
                    int ve[2] = {0, 0};
                    bool v_own = false;
                    if constexpr (F32) {
                        const int k0 = s_ku[kw][half], k1 = s_ku[kw][2 + half];
                        fs[0] = ldexpf(qs, -k0);
                        fs[1] = ldexpf(qs, -k1);
                        if (seldom(!(fmaxf(fs[0], fs[1]) < INFINITY))) {
                            int qe;
                            const float qm = frexpf(qs, &qe);
#pragma unroll
                            for (int x = 0; x < 16; x++) {
                                const int k = x < 8 ? k0 : k1, e = k == OWN ? s_kx[kw][16 * (x >> 3) + 8 * half + (x & 7)] : k;
                                s[x] = ldexpf(s[x] * qm, qe - e);
                            }
                            fs[0] = fs[1] = 1.f;
                        }
                        ve[0] = t + 8 * half < kend ? s_vu[kw][half] : 110;  // (the wave's columns end ahead of them: no part)
                        ve[1] = t + 16 + 8 * half < kend ? s_vu[kw][2 + half] : 110;
                        v_own = seldom(min(ve[0], ve[1]) == OWN);
                    }
                    // ---- softmax
                    uint32_t seen = 0;
                    if (edge) {
                        if (TREE) seen = attended(t);
#pragma unroll
                        for (int x = 0; x < 16; x++)
                            s[x] = (TREE ? bit_of(seen, x) : t + 16 * (x >> 3) + 8 * half + (x & 7) < lim) ? s[x] : -INFINITY;
                    }
                    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        m0 = fmaxf(m0, s[x]);
                        m1 = fmaxf(m1, s[x + 8]);
                    }
                    m0 = m0 == -INFINITY ? m0 : m0 * fs[0];
                    m1 = m1 == -INFINITY ? m1 : m1 * fs[1];
                    follow(over_halves(fmaxf(m0, m1), fmax2));
                    const float sub = P_UNIT - (m == -INFINITY ? 0.f : m);
                    float vf[2] = {1.f, 1.f};  // V's powers of two over the column's
                    if constexpr (F32) {
                        int lim = 1000;
                        if (__builtin_expect(v_own, 0)) {
#pragma unroll
                            for (int x = 0; x < 16; x++) {
                                const int k = ve[x >> 3], e = k == OWN ? s_vx[kw][16 * (x >> 3) + 8 * half + (x & 7)] : k;
                                lim = min(lim, e + floor_to(m - s[x] * fs[x >> 3]));
                            }
                        } else {
                            lim = min(ve[0] + floor_to(m - m0), ve[1] + floor_to(m - m1));
                        }
                        hold(over_halves(lim, imin2));
                        if (__builtin_expect(!v_own, 1)) {
                            vf[0] = ldexpf(1.f, min(vexp - ve[0], 100));
                            vf[1] = ldexpf(1.f, min(vexp - ve[1], 100));
                        }
                    }
                    f16x8 ph[2], pl[2];
#pragma unroll
                    for (int b2 = 0; b2 < 2; b2++) {
                        float p[8];
#pragma unroll
                        for (int x = 0; x < 8; x++) {
                            p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * b2 + x], fs[b2], sub));
                            if (edge) p[x] = s[8 * b2 + x] == -INFINITY ? 0.f : p[x];
                            l += p[x];
                        }
                        if (__builtin_expect(F32 && v_own, 0)) {
#pragma unroll
                            for (int x = 0; x < 8; x++)
                                p[x] = ldexpf(p[x], min(vexp - (ve[b2] == OWN ? s_vx[kw][16 * b2 + 8 * half + x] : ve[b2]), 100));
                        }
                        if (F32) split8(p, vf[b2], ph[b2], pl[b2]);
                        else split8(p, ph[b2], pl[b2]);
                    }
                    // ---- outputs
                    const uint4* vt = tile + KP + half * 32 + col;
                    bool bad = false;
                    if (edge) {  // (an infinity or NaN where some columns do not attend, as below)
                        uint32_t odd = 0;
#pragma unroll
                        for (int d = 0; d < 2 * DT; d++) {
                            const uint4 u = vt[64 * d];
                            odd |= odd16(u.x) | odd16(u.y) | odd16(u.z) | odd16(u.w);
                        }
                        bad = __any(odd != 0);
                    }
                    if (bad) {
                        f16x8 att[2];
#pragma unroll
                        for (int x = 0; x < 16; x++)
                            att[x >> 3][x & 7] = (TREE ? bit_of(seen, x) : t + 16 * (x >> 3) + 8 * half + (x & 7) < lim)
                                                     ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
                        for (int d = 0; d < DT; d++) {
                            f32x16 c;
#pragma unroll
                            for (int x = 0; x < 16; x++) c[x] = 0.f;
#pragma unroll
                            for (int b2 = 0; b2 < 2; b2++) {
                                uint4 f = vt[64 * (2 * d + b2)];
                                f = make_uint4(odd16(f.x) * 0x3C00u, odd16(f.y) * 0x3C00u, odd16(f.z) * 0x3C00u, odd16(f.w) * 0x3C00u);
                                c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, f), att[b2], c, 0, 0, 0);
                            }
#pragma unroll
                            for (int x = 0; x < 16; x++) o[d][x] = c[x] > 0.f ? NAN : o[d][x];
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        uint4 uh[2], ul[2];  // (fp16: no lo)
#pragma unroll
                        for (int b2 = 0; b2 < 2; b2++) {
                            uh[b2] = vt[64 * (2 * d + b2)];
                            if (F32) ul[b2] = vt[VP + 64 * (2 * d + b2)];
                        }
                        if (bad) {
#pragma unroll
                            for (int b2 = 0; b2 < 2; b2++) {
                                auto good = [](uint32_t u) { return ~(odd16(u) * 0xFFFFu); };
                                const uint4 k = make_uint4(good(uh[b2].x), good(uh[b2].y), good(uh[b2].z), good(uh[b2].w));
                                uh[b2] = make_uint4(uh[b2].x & k.x, uh[b2].y & k.y, uh[b2].z & k.z, uh[b2].w & k.w);
                                if (F32) ul[b2] = make_uint4(ul[b2].x & k.x, ul[b2].y & k.y, ul[b2].z & k.z, ul[b2].w & k.w);
                            }
                        }
#pragma unroll
                        for (int b2 = 0; b2 < 2; b2++) {
                            const f16x8 vh = __builtin_bit_cast(f16x8, uh[b2]);
                            if constexpr (F32)
                                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, ul[b2]), ph[b2], o[d], 0, 0, 0);
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[b2], o[d], 0, 0, 0);
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[b2], o[d], 0, 0, 0);
                        }
                        if (d & 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
                tl = {};  // (nothing of it is held across the loop)
            }
        }
        if (!shared) while (more) {
            lanes_again();
            const uint4* qtile = s_qlo + qt * QT + half * QB + col;
            const bool edge = t < lo || t + 32 > least;  // some column does not attend to all 32
            // ---- scores
            f32x16 s;
#pragma unroll
            for (int x = 0; x < 16; x++) s[x] = 0.f;
            float fs = qs;
            if constexpr (F32) {
                float mx = 0.f;  // of the lane's position
#pragma unroll
                for (int k = 0; k < 2 * KS; k++) mx = amax3(amax3(mx, tl.k[k].x, tl.k[k].y), tl.k[k].z, tl.k[k].w);
                const bool odd = !(mx < INFINITY);
                mx = over_halves(mx, fmax2);
                float most = over_rows(over_row(mx, fmax2), fmax2);
                int e = unit_exp(most);
                fs = ldexpf(qs, -e);
                bool own = false;
                if (seldom(odd || mx < most * SPREAD || !(fs < INFINITY))) {
                    mx = 0.f;  // without infinities and NaN
#pragma unroll
                    for (int k = 0; k < 2 * KS; k++) {
                        const float v[4] = {tl.k[k].x, tl.k[k].y, tl.k[k].z, tl.k[k].w};
#pragma unroll
                        for (int c = 0; c < 4; c++) mx = fmaxf(mx, finite_abs(v[c]));
                    }
                    mx = over_halves(mx, fmax2);
                    most = over_rows(over_row(mx, fmax2), fmax2);
                    e = unit_exp(most);
                    fs = ldexpf(qs, -e);
                    own = __any(far_below(mx, most) || !(fs < INFINITY));
                    if (own) e = unit_exp(mx);
                }
                const float sg = ldexpf(1.f, e);
#pragma unroll
                for (int kk = 0; kk < KS; kk++) {
                    const float4 x = tl.k[2 * kk], y = tl.k[2 * kk + 1];
                    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                    f16x8 kh, kl;
                    split8(v, sg, kh, kl);
                    const f16x8 qh = __builtin_bit_cast(f16x8, qtile[QHI + 2 * QB * kk]);
                    const f16x8 ql = __builtin_bit_cast(f16x8, qtile[2 * QB * kk]);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh, s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql, s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh, s, 0, 0, 0);
                }
                if (__builtin_expect(own, 0)) {
                    int qe;
                    const float qm = frexpf(qs, &qe);
#pragma unroll
                    for (int x = 0; x < 16; x++)
                        s[x] = ldexpf(s[x] * qm, qe - __shfl(e, row_of(16 * (x >> 3) + 8 * half + (x & 7))));
                    fs = 1.f;
                }
            } else {
                // (int8: the wave at its products goes ahead of the one beside it, which widens and weighs meanwhile: 24 trees of
                // 26 nodes at 8,000 positions 100.8 -> 97.2 us; the others gained nothing)
                if (I8) __builtin_amdgcn_s_setprio(2);
#pragma unroll
                for (int kk = 0; kk < KS; kk++) {
                    f16x8 kf;
                    if constexpr (I8) {
                        const uint4 x = tl.k[kk >> 1];
                        kf = (kk & 1) ? widen8(x.z, x.w) : widen8(x.x, x.y);
                    } else {
                        kf = tl.k[kk];
                    }
                    const f16x8 qh = __builtin_bit_cast(f16x8, qtile[QHI + 2 * QB * kk]);
                    const f16x8 ql = __builtin_bit_cast(f16x8, qtile[2 * QB * kk]);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql, s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh, s, 0, 0, 0);
                }
            }
            if (I8) __builtin_amdgcn_s_setprio(0);
            float vsc[16];
            if constexpr (I8) {
#pragma unroll
                for (int x = 0; x < 16; x++) s[x] *= ((const float*)&tl.ks[x >> 2])[x & 3];
#pragma unroll
                for (int x = 0; x < 16; x++) vsc[x] = ((const float*)&tl.vs[x >> 2])[x & 3];
            }
            // the next tile's ids and K
            const bool go = DIRECT ? i + GW < jend : i + 1 < jend && t + dt < kend;
            int tn = go ? t + dt : t;
            const bool turn = DIRECT && go && !tail && i + GW >= d_tiles;  // from the prefix to the tail
            if (TURNS) load_v(t);
            if (turn) {
                tn = tail_base(pre) + 32 * (i + GW - d_tiles);
                ptab = table_of(w);
                klast = ctx - 1;
            }
            ids(tn);
            if (!TURNS) load_k(tn, go);

            // ---- softmax: register x is position t + 16 (x / 8) + 8 half + x % 8
            float mt = -INFINITY;
            uint32_t seen = 0;
            if (edge) {
                if (TREE) seen = attended(t);
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const int pos = t + 16 * (x >> 3) + 8 * half + (x & 7);
                    s[x] = (TREE ? bit_of(seen, x) : pos >= lo && pos < lim) ? s[x] : -INFINITY;
                    if constexpr (I8) vsc[x] = pos < kend ? vsc[x] : 0.f;
                }
            }
#pragma unroll
            for (int x = 0; x < 16; x++) mt = fmaxf(mt, s[x]);
            mt = over_halves(mt, fmax2);
            mt = mt == -INFINITY ? mt : mt * fs;
            follow(mt);
            const float sub = (I8 ? 0.f : P_UNIT) - (m == -INFINITY ? 0.f : m);
            float p[16];
#pragma unroll
            for (int x = 0; x < 16; x++) {
                p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], fs, sub));
                if (edge) p[x] = s[x] == -INFINITY ? 0.f : p[x];  // (a factor of 0 times it)
                l += p[x];
            }
            float vf = 1.f, vg = 1.f;  // V's powers of two over the column's, and those (f32)
            bool v_own = false;
            if constexpr (I8) {
                float mx = 0.f;
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    p[x] = !edge || s[x] > -INFINITY ? p[x] * vsc[x] : 0.f;
                    mx = fmaxf(mx, fabsf(p[x]));
                }
                hold(unit_exp(over_halves(mx, fmax2)) - (int)GROWTH);
                vf = ldexpf(1.f, vexp);
            }
            if constexpr (F32) {
                Spread sp;  // of positions, DT dims of each
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    float x = amax2(tl.v[k][0], tl.v[k][1]), y = amax2(tl.v[k + 1][0], tl.v[k + 1][1]);
#pragma unroll
                    for (int c = 2; c < DT; c += 2) {
                        x = amax3(x, tl.v[k][c], tl.v[k][c + 1]);
                        y = amax3(y, tl.v[k + 1][c], tl.v[k + 1][c + 1]);
                    }
                    sp.add(x, y);
                }
                float most = over_wave(sp.most, fmax2);
                if (seldom(sp.apart(most))) {
                    most = 0.f;
                    float least = INFINITY;
#pragma unroll
                    for (int k = 0; k < 16; k++) {  // (the lanes of a half hold its position)
                        float y = 0.f;
#pragma unroll
                        for (int c = 0; c < DT; c++) y = fmaxf(y, finite_abs(tl.v[k][c]));
                        y = over_rows(over_row(y, fmax2), fmax2);
                        most = fmaxf(most, y);
                        least = y > 0.f ? fminf(least, y) : least;
                        s_m[wave][16 * half + k] = y;
                        __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
                    }
                    most = over_halves(most, fmax2);
                    v_own = __any(far_below(least, most));
                }
                int e = unit_exp(most), lim = e + floor_to(m - mt);
                if (__builtin_expect(v_own, 0)) {
                    int top = -1000;  // log2 of the largest weighted magnitude, at most
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        e = unit_exp(s_m[wave][16 * half + k]);
                        top = max(top, p[k] > 0.f ? __builtin_amdgcn_frexp_expf(p[k]) - e : -1000);
                        s_m[wave][16 * half + k] = ldexpf(1.f, e);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    lim = (int)P_UNIT - over_halves(top, imax2);
                }
                hold(lim);
                if (__builtin_expect(v_own, 0)) {
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        p[k] = ldexpf(p[k], min(vexp + 1 - __builtin_amdgcn_frexp_expf(s_m[wave][16 * half + k]), 100));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
                    s_m[wave][col] = ldexpf(1.f, e);
                    vf = ldexpf(1.f, min(vexp - e, 100));
                }
            }
            f16x8 ph[2], pl[2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const float v[8] = {p[8 * b], p[8 * b + 1], p[8 * b + 2], p[8 * b + 3],
                                    p[8 * b + 4], p[8 * b + 5], p[8 * b + 6], p[8 * b + 7]};
                if constexpr (F16) split8(v, ph[b], pl[b]);
                else split8(v, vf, ph[b], pl[b]);
            }

            // ---- outputs
            if constexpr (!I8) {
                if (edge) {
                    // V past the end: zeros, whatever the page holds there (f32: the last position's)
                    if constexpr (F16) {
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const int valid = kend - (t + 16 * b + 8 * half);
#pragma unroll
                            for (int d = 0; d < DT; d++) {
                                uint32_t* u = (uint32_t*)&tl.v[d][b];
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    u[k] &= valid >= 2 * k + 2 ? 0xFFFFFFFFu : valid == 2 * k + 1 ? 0xFFFFu : 0u;
                            }
                        }
                    }
                    // An infinity or NaN in V times a weight of 0 is NaN, in columns that do not attend to it.
                    // Tiles that hold one: NaN to the outputs of the columns that do (a product of indicators
                    // counts them), then zeros in its place.
                    bool bad = false;
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        if constexpr (F32) {
#pragma unroll
                            for (int k = 0; k < 16; k++) bad |= !(fabsf(tl.v[k][d]) < INFINITY);
                        } else {
                            uint32_t any = 0;
#pragma unroll
                            for (int k = 0; k < 8; k++) any |= odd16(((const uint32_t*)&tl.v[d][k >> 2])[k & 3]);
                            bad |= any != 0;
                        }
                    }
                    if (__any(bad)) {
                        f16x8 att[2];
#pragma unroll
                        for (int x = 0; x < 16; x++) {
                            const int pos = t + 16 * (x >> 3) + 8 * half + (x & 7);
                            att[x >> 3][x & 7] = (TREE ? bit_of(seen, x) : pos >= lo && pos < lim) ? (_Float16)1.f : (_Float16)0.f;
                        }
#pragma unroll
                        for (int d = 0; d < DT; d++) {
                            f32x16 c;
#pragma unroll
                            for (int x = 0; x < 16; x++) c[x] = 0.f;
#pragma unroll
                            for (int b = 0; b < 2; b++) {
                                uint4 f;  // fp16 ones where V is no number
                                uint32_t* fu = (uint32_t*)&f;
                                if constexpr (F32) {
#pragma unroll
                                    for (int k = 0; k < 8; k++) {
                                        const float v = tl.v[8 * b + k][d];
                                        const bool good = fabsf(v) < INFINITY;
                                        const uint32_t one = good ? 0u : k & 1 ? 0x3C000000u : 0x3C00u;
                                        fu[k >> 1] = k & 1 ? fu[k >> 1] | one : one;
                                        tl.v[8 * b + k][d] = good ? v : 0.f;
                                    }
                                } else {
                                    uint32_t* u = (uint32_t*)&tl.v[d][b];
#pragma unroll
                                    for (int k = 0; k < 4; k++) {
                                        const uint32_t w = odd16(u[k]);
                                        fu[k] = w * 0x3C00u;
                                        u[k] &= ~(w * 0xFFFFu);
                                    }
                                }
                                c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, f), att[b], c, 0, 0, 0);
                            }
#pragma unroll
                            for (int x = 0; x < 16; x++) o[d][x] = c[x] > 0.f ? NAN : o[d][x];
                        }
                    }
                }
            }
            // dims DT * row + d of tile d (f32), 32 d + row
            auto product = [&](int d, int b, auto by) {
                if constexpr (F32) {
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = tl.v[8 * b + k][d];
                    f16x8 vh, vl;
                    split8_by(x, by, vh, vl);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[b], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[b], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[b], o[d], 0, 0, 0);
                } else {
                    f16x8 vf;
                    if constexpr (I8) vf = widen8(tl.v[d][b].x, tl.v[d][b].y);
                    else vf = __builtin_bit_cast(f16x8, tl.v[d][b]);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl[b], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph[b], o[d], 0, 0, 0);
                }
            };
            if (I8) __builtin_amdgcn_s_setprio(2);
#pragma unroll
            for (int b = 0; b < 2; b++) {
                float by[8];  // (f32: a half's 8 positions; 8 at a time: registers)
#pragma unroll
                for (int k = 0; k < 8; k++) by[k] = F32 ? s_m[wave][16 * half + 8 * b + k] : 1.f;
#pragma unroll
                for (int d = 0; d < DT; d++) product(d, b, [&](int k) { return by[k]; });
                if (F32) __builtin_amdgcn_sched_barrier(0);
            }
            if (I8) __builtin_amdgcn_s_setprio(0);
            if (TURNS) load_k(tn, go);
            else load_v(tn, go);
            more = go;
            i += DIRECT ? GW : 1;
            t = tn;
            if (turn) {
                tail = true;
                lo = pre;
                lim = kend = least = ctx;
            }
        }

        // ---- join the waves of a column
        lanes_again();
        lds_sync();  // q's operands lie where the outputs go
        l = over_halves(l, [](float x, float y) { return x + y; });
        if (F32) l = ldexpf(l, -(int)P_UNIT);  // weights of 1 again: V next to fp32's largest stay in it
        if (half == 0) {
            s_m[wave][col] = m;
            s_l[wave][col] = l;
        }
        // where a column's joined output goes (pieces ahead, less one for each of their jobs: a job's columns are at most
        // 128, so slots stay apart)
        if (kw == 0 && half == 0) {
            const bool any_pre = min(ctx, pre) > 0, any_tail = ctx > pre;
            const bool alone = DIRECT || (whole && (tail ? !any_pre : any_pre && !any_tail));
            const size_t slot = (size_t)kvh * a.slots + (tail ? (size_t)a.n * G : 0) + ab +
                                (size_t)BLK * ((here & 0xFFFF) - (here >> 16) + i_of);
            const bool mine = col < cols, part = mine && !alone && (tail || any_pre);
            s_to[qt * 32 + col] = mine && alone ? (long long)orow : part ? ~(long long)slot : NOWHERE;
        }
        const float unit = F16 ? 1.f : ldexpf(1.f, -vexp - (F32 ? (int)P_UNIT : 0));
        if (col < cols) {
            float4* row = (float4*)(s_o + (wave * 32 + col) * HD);
            const int x = col & 15;
#pragma unroll
            for (int b = 0; b < 4; b++) {
                if constexpr (F32) {  // register 4 b + c of tile d: dim DT * (8 b + 4 half + c) + d
#pragma unroll
                    for (int c = 0; c < 4; c += 4 / DT) {
                        float v[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) v[k] = o[k % DT][4 * b + c + k / DT] * unit;
                        row[(DT * (8 * b + 4 * half + c) >> 2) ^ x] = make_float4(v[0], v[1], v[2], v[3]);
                    }
                } else {  // dim 32 d + 8 b + 4 half + c
#pragma unroll
                    for (int d = 0; d < DT; d++)
                        row[(8 * d + 2 * b + half) ^ x] = make_float4(o[d][4 * b] * unit, o[d][4 * b + 1] * unit,
                                                                      o[d][4 * b + 2] * unit, o[d][4 * b + 3] * unit);
                }
            }
        }
        lds_sync();
        lanes_again();
        lds_sync();
        auto join = [&](auto wk_c) {
            constexpr int WK = decltype(wk_c)::value, WQ = GW / WK;
            // U pieces of 16 bytes at a time, all read ahead of the first branch (one by one a piece was 600 cycles)
            constexpr int U = 8 / WK < WQ * 32 * (HD / 4) / GTH ? 8 / WK : WQ * 32 * (HD / 4) / GTH;
            for (int e0 = tid; e0 < WQ * 32 * (HD / 4); e0 += U * GTH) {
                long long to[U];
                float4 x[U][WK];
                float f[U][WK], lw[U][WK];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int e = e0 + u * GTH, c = e / (HD / 4), d = e % (HD / 4) * 4, cq = c >> 5, ci = c & 31;
                    to[u] = s_to[c];
#pragma unroll
                    for (int k = 0; k < WK; k++) {
                        x[u][k] = *(const float4*)(s_o + ((cq + WQ * k) * 32 + ci) * HD + (d ^ 4 * (ci & 15)));
                        f[u][k] = s_m[cq + WQ * k][ci];
                        lw[u][k] = s_l[cq + WQ * k][ci];
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int d = (e0 + u * GTH) % (HD / 4) * 4;
                    float M = -INFINITY, L = 0.f;
#pragma unroll
                    for (int k = 0; k < WK; k++) M = fmaxf(M, f[u][k]);
                    const float mu = M == -INFINITY ? 0.f : M;
                    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < WK; k++) {  // (a wave without positions holds zeros)
                        const float by = __builtin_amdgcn_exp2f(f[u][k] - mu);
                        L = __builtin_fmaf(lw[u][k], by, L);
                        O.x = __builtin_fmaf(x[u][k].x, by, O.x);
                        O.y = __builtin_fmaf(x[u][k].y, by, O.y);
                        O.z = __builtin_fmaf(x[u][k].z, by, O.z);
                        O.w = __builtin_fmaf(x[u][k].w, by, O.w);
                    }
                    if (to[u] == NOWHERE) continue;
                    if (to[u] < 0) {
                        *(float4*)(a.part_o + (size_t)~to[u] * HD + d) = O;
                        if (d == 0) a.part_ml[~to[u]] = make_float2(M, L);
                    } else {
                        const float by = DIRECT && d_ctx == 0 ? 0.f : 1.f / L;
                        group_store4(a, to[u] + d, make_float4(O.x * by, O.y * by, O.z * by, O.w * by));
                    }
                }
            }
        };
        if (wk == 2) join(std::integral_constant<int, 2>());
        else if (wk == 4) join(std::integral_constant<int, 4>());
        else join(std::integral_constant<int, 8>());
        lds_sync();  // s_o, s_m, s_l are written again
    }
    // where each row's parts lie, for the join: as group_plan writes it, by the workgroup that has least to do
    if (LANES && blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) {
        int* seq = (int*)s_dyn;  // [7][64]
        if (tid < 64) {
            const int of[7] = {lp.first, lp.end, lp.base, lp.blocks, lp.pieces, lp.last_pieces, lp.upto};
#pragma unroll
            for (int k = 0; k < 7; k++) seq[64 * k + tid] = of[k];
        }
        lds_sync();
        for (int r = tid; r < a.n; r += GTH) {
            const int* q = seq + last_at(seq, a.groups, r);
            const bool in = r >= q[0] && r < q[64];
            const int pos = (r - q[0]) * G, b = pos / BLK, block = q[256] | 1 << 16;
            auto upto = [&](int k) {
                return q[384] + (k < q[192] ? k * block : (q[192] - 1) * block + (q[320] | 1 << 16));
            };
            a.plan[2 * r] = make_int4(in ? pos : -1, upto(b), upto(b + 1), upto(b + 2));
            a.plan[2 * r + 1] = make_int4(in && row_end(r, q[128]) > 0 ? 1 : 0, 0, 0, 0);
        }
    }
}

// The parts of a column, joined in order: one wave per (row, query head).  A row
// whose one part was the output itself is left; one without any is zero.
template <int HD>
__global__ __launch_bounds__(256) void group_merge_kernel(GroupArgs a) {
    constexpr int DPL = HD / 64, FLIGHT = 8;  // dimensions a lane; parts in flight
    const int r = blockIdx.x, h = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (h >= a.H) return;
    const int lane = threadIdx.x & 63, kvh = h / a.G, hh = h - kvh * a.G;
    const int4 at0 = a.plan[2 * r], at1 = a.plan[2 * r + 1];
    if (at0.x < 0) return;  // outside every group
    // (first slot, parts) of the prefix and of the tail
    int first[2] = {0, 0}, count[2] = {0, 0};
    const bool second = (at0.x + hh) / BLK != at0.x / BLK;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int x = k ? at1.y : second ? at0.z : at0.y, y = k ? at1.z : second ? at0.w : at0.z;
        first[k] = (x & 0xFFFF) - (x >> 16);
        count[k] = at1.x >> k & 1 ? (y & 0xFFFF) - (x & 0xFFFF) : 0;
    }
    const int all = count[0] + count[1];
    const size_t out = ((size_t)r * a.H + h) * HD;
    if (all == 0) {
#pragma unroll
        for (int k = 0; k < DPL; k++) group_store(a, out + lane + 64 * k, 0.f);
        return;
    }
    if (all == 1) return;
    const size_t column = (size_t)kvh * a.slots + (size_t)r * a.G + hh;
    auto slot = [&](int i) {
        return i < count[0] ? column + (size_t)BLK * (first[0] + i)
                            : column + (size_t)a.n * a.G + (size_t)BLK * (first[1] + i - count[0]);
    };
    float m = -INFINITY, l = 0.f, O[DPL];  // running, as in the tiles
#pragma unroll
    for (int k = 0; k < DPL; k++) O[k] = 0.f;
    for (int i0 = 0; i0 < all; i0 += FLIGHT) {
        float v[FLIGHT][DPL];
        float2 ml[FLIGHT];
#pragma unroll
        for (int u = 0; u < FLIGHT; u++) {
            const size_t at = slot(min(i0 + u, all - 1));
            ml[u] = a.part_ml[at];
#pragma unroll
            for (int k = 0; k < DPL; k++) v[u][k] = a.part_o[at * HD + lane + 64 * k];
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < FLIGHT; u++) mn = i0 + u < all ? fmaxf(mn, ml[u].x) : mn;
        const float mu = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - mu);
        l *= alpha;
#pragma unroll
        for (int k = 0; k < DPL; k++) O[k] *= alpha;
#pragma unroll
        for (int u = 0; u < FLIGHT; u++) {
            const float f = i0 + u < all ? __builtin_amdgcn_exp2f(ml[u].x - mu) : 0.f;
            l = __builtin_fmaf(ml[u].y, f, l);
#pragma unroll
            for (int k = 0; k < DPL; k++) O[k] = i0 + u < all ? __builtin_fmaf(v[u][k], f, O[k]) : O[k];
        }
        m = mn;
    }
#pragma unroll
    for (int k = 0; k < DPL; k++) group_store(a, out + lane + 64 * k, O[k] / l);
}

// The same of trees, whose columns have parts of one kind: HD / 4 lanes hold a part, so 2 or 4 parts lie side by side in
// a wave's registers, 4 or 8 times; their maxima, sums and outputs meet at the end.  (64 nodes at 8,000 positions, 32
// parts a column: 4.7 us, of which two reads one after another and the launch; eight parts of two dimensions a lane at
// a time 6.1.)
template <int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(GroupArgs a) {
    constexpr int W = HD / 4, NP = 64 / W;
    const int r = blockIdx.x, h = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (h >= a.H) return;
    const int lane = threadIdx.x & 63, kvh = h / a.G, hh = h - kvh * a.G, d = 4 * (lane % W), side = lane / W;
    const int4 at = a.plan[2 * r];
    const bool some = a.plan[2 * r + 1].x != 0;
    if (at.x < 0) return;  // of no sequence
    const bool second = (at.x + hh) / BLK != at.x / BLK;
    const int x = second ? at.z : at.y, y = second ? at.w : at.z;
    const int all = some ? (y & 0xFFFF) - (x & 0xFFFF) : 0;
    const size_t out = ((size_t)r * a.H + h) * HD + d;
    if (all == 0 && side == 0) group_store4(a, out, make_float4(0.f, 0.f, 0.f, 0.f));
    if (all <= 1) return;
    const size_t column = (size_t)kvh * a.slots + (size_t)r * a.G + hh + (size_t)BLK * ((x & 0xFFFF) - (x >> 16));
    float m = -INFINITY, l = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    auto take = [&](int i0, auto many) {
        constexpr int U = decltype(many)::value;
        float4 v[U];
        float2 ml[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t slot = column + (size_t)BLK * min(i0 + u * NP + side, all - 1);
            ml[u] = a.part_ml[slot];
            v[u] = *(const float4*)(a.part_o + slot * HD + d);
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; u++) mn = i0 + u * NP + side < all ? fmaxf(mn, ml[u].x) : mn;
        const float mu = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - mu);
        l *= alpha;
        O = make_float4(O.x * alpha, O.y * alpha, O.z * alpha, O.w * alpha);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool in = i0 + u * NP + side < all;
            const float f = in ? __builtin_amdgcn_exp2f(ml[u].x - mu) : 0.f;
            l = in ? __builtin_fmaf(ml[u].y, f, l) : l;
            O.x = in ? __builtin_fmaf(v[u].x, f, O.x) : O.x;
            O.y = in ? __builtin_fmaf(v[u].y, f, O.y) : O.y;
            O.z = in ? __builtin_fmaf(v[u].z, f, O.z) : O.z;
            O.w = in ? __builtin_fmaf(v[u].w, f, O.w) : O.w;
        }
        m = mn;
    };
    if (all <= 4 * NP) take(0, std::integral_constant<int, 4>());
    else
        for (int i0 = 0; i0 < all; i0 += 8 * NP) take(i0, std::integral_constant<int, 8>());
    auto sides = [](float v, auto op) { return NP == 4 ? over_halves(over_rows(v, op), op) : over_halves(v, op); };
    const float M = sides(m, fmax2), by = __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
    auto sum = [&](float v) { return sides(v * by, [](float p, float q) { return p + q; }); };
    l = sum(l);
    O = make_float4(sum(O.x), sum(O.y), sum(O.z), sum(O.w));
    if (side == 0) group_store4(a, out, make_float4(O.x / l, O.y / l, O.z / l, O.w / l));
}

// workgroups per KV head: as many as are resident at once, one per CU, whose
// registers its 8 waves fill
static int group_grid(int Hkv) { return std::max(1, 256 / Hkv); }

struct GroupSizes {
    int job_cap, tail_log2, tails;
    long long slots;
    size_t plan_bytes, ml_bytes, o_bytes;
};
static GroupSizes group_sizes(int n, int groups, int H, int Hkv, int hd, bool tree = false) {
    const int G = H / Hkv;
    GroupSizes z;
    z.job_cap = (int)((long long)n * G / BLK) + groups;
    z.tail_log2 = G <= 32 ? 2 : G <= 64 ? 1 : 0;
    z.tails = tree ? 0 : (n + (1 << z.tail_log2) - 1) >> z.tail_log2;
    z.slots = 2ll * n * G + (long long)BLK * group_grid(Hkv);
    z.plan_bytes = ((size_t)n * 32 + 255) / 256 * 256;
    z.ml_bytes = ((size_t)Hkv * z.slots * sizeof(float2) + 255) / 256 * 256;
    z.o_bytes = (size_t)Hkv * z.slots * hd * 4;
    return z;
}
static size_t group_lds(int hd, int n, int groups, const GroupSizes& z) {
    return (size_t)tile_floats(hd) * 4 + (size_t)(2 * (z.job_cap + z.tails) + 1 + 3 * groups + 2 + n) * 4;
}
// shapes of the tiles (their LDS bounds what few very wide layouts would need; offsets inside a page, and of q, are
// held in 32 bits)
bool group_attention_tiles(int n, int groups, int H, int Hkv, int hd, int page_size, bool tree) {
    const int G = H / Hkv;
    return (hd == 64 || hd == 128) && G <= BLK && page_size >= 16 && (page_size & (page_size - 1)) == 0 && (long long)page_size * hd <= 1 << 29 &&
           (long long)n * H * hd <= 1 << 30 &&
           group_lds(hd, n, groups, group_sizes(n, groups, H, Hkv, hd, tree)) + (tree ? 6144 : 5120) <= 160 * 1024;
}

// Small calls: one launch without a plan, a workgroup per (row, KV head), which saves the plan (3 us) and the launch
// that joins parts (4) and costs 1 (fp16) to 5 us (f32, head_dim 128) per 256 positions, shared or not.  Planned against
// direct, us: 5 rows of 40 / 300 / 600 / 1,000 positions, fp16, 16/2 heads of 128: 13.9 / 15.0 / 15.2 / 15.6 against
// 8.1 / 9.8 / 11.9 / 15.8; int8 14.2 / 16.0 / 16.1 / 16.3 against 8.7 / 11.0 / 13.3 / 18.2; f32 16.8 / 19.3 / 19.6 /
// 19.8 against 11.1 / 15.2 / 20.6 / 32.0.  250 workgroups of 300 / 600 positions, fp16: 18.5 / 19.5 against 13.3 / 17.7.
static bool group_direct(int n, int H, int Hkv, uint32_t kv_dtype, int max_ctx) {
    const int most = 256 * (kv_dtype == DT_F32 ? 2 : kv_dtype == DT_I8 ? 3 : 4);
    return H / Hkv <= 32 && n <= DIRECT_ROWS && (long long)n * Hkv <= 256 && max_ctx <= (n * Hkv > 128 ? most / 2 : most);
}

int group_attention_init() {
#define QH_GROUP_LDS1(HDv, KVv, DIRECTv, TREEv, LANESv)                                                   \
    QH_CHECK_HIP(hipFuncSetAttribute((const void*)group_tile_kernel<HDv, (int)KVv, DIRECTv, TREEv, LANESv>, \
                                     hipFuncAttributeMaxDynamicSharedMemorySize, (TREEv ? 154 : 155) * 1024));
#define QH_GROUP_LDS(HDv, KVv)                                                                             \
    QH_GROUP_LDS1(HDv, KVv, false, false, false) QH_GROUP_LDS1(HDv, KVv, true, false, false)              \
    QH_GROUP_LDS1(HDv, KVv, false, true, false) QH_GROUP_LDS1(HDv, KVv, true, true, false)                \
    QH_GROUP_LDS1(HDv, KVv, false, true, true)
    QH_GROUP_LDS(64, DT_F32) QH_GROUP_LDS(64, DT_F16) QH_GROUP_LDS(64, DT_I8)
    QH_GROUP_LDS(128, DT_F32) QH_GROUP_LDS(128, DT_F16) QH_GROUP_LDS(128, DT_I8)
#undef QH_GROUP_LDS
#undef QH_GROUP_LDS1
    return QRAF_HIP_OK;
}

// (of any page size: one that the tiles do not take needs less)
size_t group_attention_workspace_bytes(int n, int groups, int H, int Hkv, int hd, int max_ctx) {
    (void)max_ctx;
    if (H % Hkv || !group_attention_tiles(n, groups, H, Hkv, hd, 16)) return 16;
    const GroupSizes z = group_sizes(n, groups, H, Hkv, hd);
    return z.plan_bytes + z.ml_bytes + z.o_bytes;
}

// the tiles, and the join of their parts
template <bool TREE>
static int group_tiles(GroupArgs& a, uint32_t kv_dtype, int hd, void* ws, bool direct, hipStream_t st) {
    const GroupSizes z = group_sizes(a.n, a.groups, a.H, a.Hkv, hd, TREE);
    a.job_cap = z.job_cap;
    a.tail_log2 = z.tail_log2;
    a.tails = z.tails;
    a.slots = z.slots;
    while ((1 << a.ps_log2) < a.page_size) a.ps_log2++;
    a.plan = (int4*)ws;
    a.part_ml = (float2*)((uint8_t*)ws + z.plan_bytes);
    a.part_o = (float*)((uint8_t*)ws + z.plan_bytes + z.ml_bytes);
    const int gx = group_grid(a.Hkv);
    // (A lane to a sequence; more take the plan in LDS.  64 / 65 trees of 8, 16/2 heads of 128, us: at 128..4,096 positions f32
    // 95 / 95, fp16 45.9 / 46.8, int8 44.5 / 45.5, at 300 29.4 / 31.4, 21.0 / 21.3, 21.8 / 21.2.)
    const bool lanes = TREE && a.groups <= 64;
    const size_t lds = lanes ? (size_t)tile_floats(hd) * 4 + (size_t)a.n * 8 : group_lds(hd, a.n, a.groups, z);
#define QH_GROUP_TILE(HDv, KVv)                                                                                            \
    if (hd == HDv && kv_dtype == KVv) {                                                                                    \
        if (direct)                                                                                                        \
            hipLaunchKernelGGL((group_tile_kernel<HDv, (int)KVv, true, TREE, false>), dim3(a.n, a.Hkv), dim3(GTH),        \
                               tile_floats(HDv) * 4, st, a);                                                               \
        else if (lanes)                                                                                                    \
            hipLaunchKernelGGL((group_tile_kernel<HDv, (int)KVv, false, TREE, TREE>), dim3(gx, a.Hkv), dim3(GTH), lds, st, a); \
        else                                                                                                               \
            hipLaunchKernelGGL((group_tile_kernel<HDv, (int)KVv, false, TREE, false>), dim3(gx, a.Hkv), dim3(GTH), lds, st, a); \
    }
    QH_GROUP_TILE(64, DT_F32) QH_GROUP_TILE(64, DT_F16) QH_GROUP_TILE(64, DT_I8)
    QH_GROUP_TILE(128, DT_F32) QH_GROUP_TILE(128, DT_F16) QH_GROUP_TILE(128, DT_I8)
#undef QH_GROUP_TILE
    QH_CHECK_HIP(hipGetLastError());
    if (direct) return QRAF_HIP_OK;
    const dim3 grid(a.n, (a.H + 3) / 4);
    if (hd == 128) hipLaunchKernelGGL((TREE ? tree_merge_kernel<128> : group_merge_kernel<128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((TREE ? tree_merge_kernel<64> : group_merge_kernel<64>), grid, dim3(256), 0, st, a);
    QH_CHECK_HIP(hipGetLastError());
    return QRAF_HIP_OK;
}

// the plain form, of every shape
template <bool TREE>
static int group_any(const GroupArgs& a, uint32_t kv_dtype, int hd, hipStream_t st) {
    const dim3 grid(a.n, a.H);
#define QH_GROUP_ANY(HDv, KVv)                                                                     \
    if (hd == HDv && kv_dtype == KVv) {                                                            \
        hipLaunchKernelGGL((group_any_kernel<HDv, (int)KVv, TREE>), grid, dim3(256), 0, st, a);    \
        QH_CHECK_HIP(hipGetLastError());                                                           \
        return QRAF_HIP_OK;                                                                        \
    }
#define QH_GROUP_ANYS(HDv) QH_GROUP_ANY(HDv, DT_F32) QH_GROUP_ANY(HDv, DT_F16) QH_GROUP_ANY(HDv, DT_I8)
    QH_GROUP_ANYS(16) QH_GROUP_ANYS(32) QH_GROUP_ANYS(64) QH_GROUP_ANYS(128)
#undef QH_GROUP_ANYS
#undef QH_GROUP_ANY
    return QRAF_HIP_OK;
}

int launch_group_attention(const float* q, const void* kc, const void* vc, uint32_t kv_dtype,
                           const int32_t* page_table, int max_pages, const int32_t* ctx, const int32_t* group_starts,
                           const int32_t* prefix, int n, int groups, int H, int Hkv, int hd, int page_size, float scale,
                           int max_ctx, float* out, void* ws, size_t ws_bytes, hipStream_t st, uint16_t* out_hi,
                           uint16_t* out_lo) {
    QH_REQUIRE(q && kc && vc && page_table && ctx && group_starts && prefix && (out || (out_hi && out_lo)) && ws,
               QRAF_HIP_ERR_INVALID, "group attention: null pointer");
    QH_REQUIRE((((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)out | (uintptr_t)ws) & 15) == 0,
               QRAF_HIP_ERR_INVALID, "group attention: q, caches, out and workspace must be 16-byte aligned");
    QH_REQUIRE(n > 0 && n <= 1024, QRAF_HIP_ERR_INVALID, "group attention: %d rows outside 1..1024", n);
    QH_REQUIRE(groups > 0 && groups <= n, QRAF_HIP_ERR_INVALID, "group attention: %d groups of %d rows", groups, n);
    QH_REQUIRE(Hkv > 0 && H > 0 && H % Hkv == 0, QRAF_HIP_ERR_INVALID,
               "group attention: %d heads not a multiple of %d kv heads", H, Hkv);
    QH_REQUIRE(hd == 16 || hd == 32 || hd == 64 || hd == 128, QRAF_HIP_ERR_INVALID,
               "group attention: head_dim %d (16, 32, 64 or 128 supported)", hd);
    QH_REQUIRE(page_size > 0 && max_pages > 0 && max_ctx > 0 && max_ctx <= (long long)max_pages * page_size,
               QRAF_HIP_ERR_INVALID, "group attention: bad page geometry");
    QH_REQUIRE(max_ctx <= 1 << 30, QRAF_HIP_ERR_INVALID, "group attention: max_ctx %d over 2^30", max_ctx);
    QH_REQUIRE(kv_dtype == DT_F32 || kv_dtype == DT_F16 || kv_dtype == DT_I8, QRAF_HIP_ERR_DTYPE,
               "group attention: KV dtype %u", kv_dtype);
    QH_REQUIRE(ws_bytes >= group_attention_workspace_bytes(n, groups, H, Hkv, hd, max_ctx), QRAF_HIP_ERR_INVALID,
               "group attention: workspace of %zu bytes, %zu needed", ws_bytes,
               group_attention_workspace_bytes(n, groups, H, Hkv, hd, max_ctx));
    GroupArgs a{};
    a.q = q;
    a.kc = kc;
    a.vc = vc;
    a.page_table = page_table;
    a.ctx = ctx;
    a.starts = group_starts;
    a.prefix = prefix;
    a.out = out;
    a.out_hi = out_hi;
    a.out_lo = out_lo;
    a.n = n;
    a.groups = groups;
    a.H = H;
    a.Hkv = Hkv;
    a.G = H / Hkv;
    a.page_size = page_size;
    a.max_pages = max_pages;
    a.max_ctx = max_ctx;
    a.scale = scale;
    if (group_attention_tiles(n, groups, H, Hkv, hd, page_size)) {
        return group_tiles<false>(a, kv_dtype, hd, ws, group_direct(n, H, Hkv, kv_dtype, max_ctx), st);
    }
    return group_any<false>(a, kv_dtype, hd, st);
}

size_t tree_attention_workspace_bytes(int n, int seqs, int H, int Hkv, int hd, int max_ctx) {
    (void)max_ctx;
    if (H % Hkv || !group_attention_tiles(n, seqs, H, Hkv, hd, 16, true)) return 16;
    const GroupSizes z = group_sizes(n, seqs, H, Hkv, hd, true);
    return z.plan_bytes + z.ml_bytes + z.o_bytes;
}

int launch_tree_attention(const float* q, const void* kc, const void* vc, uint32_t kv_dtype, const int32_t* page_table,
                          int max_pages, const int32_t* base, const int32_t* row_starts, const uint64_t* masks, int n,
                          int seqs, int H, int Hkv, int hd, int page_size, float scale, int max_ctx, float* out,
                          void* ws, size_t ws_bytes, hipStream_t st, uint16_t* out_hi, uint16_t* out_lo) {
    QH_REQUIRE(q && kc && vc && page_table && base && row_starts && masks && (out || (out_hi && out_lo)) && ws,
               QRAF_HIP_ERR_INVALID, "tree attention: null pointer");
    QH_REQUIRE((((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)out | (uintptr_t)ws) & 15) == 0 &&
                   ((uintptr_t)masks & 7) == 0,
               QRAF_HIP_ERR_INVALID,
               "tree attention: q, caches, out and workspace must be 16-byte, masks 8-byte aligned");
    QH_REQUIRE(n > 0 && n <= 1024, QRAF_HIP_ERR_INVALID, "tree attention: %d rows outside 1..1024", n);
    QH_REQUIRE(seqs > 0 && seqs <= n, QRAF_HIP_ERR_INVALID, "tree attention: %d sequences of %d rows", seqs, n);
    QH_REQUIRE(Hkv > 0 && H > 0 && H % Hkv == 0, QRAF_HIP_ERR_INVALID,
               "tree attention: %d heads not a multiple of %d kv heads", H, Hkv);
    QH_REQUIRE(H <= 65535, QRAF_HIP_ERR_INVALID, "tree attention: %d heads over 65535", H);
    QH_REQUIRE(hd == 16 || hd == 32 || hd == 64 || hd == 128, QRAF_HIP_ERR_INVALID,
               "tree attention: head_dim %d (16, 32, 64 or 128 supported)", hd);
    QH_REQUIRE(page_size > 0 && max_pages > 0 && max_ctx > 0 && max_ctx <= (long long)max_pages * page_size,
               QRAF_HIP_ERR_INVALID, "tree attention: bad page geometry");
    QH_REQUIRE(max_ctx <= 1 << 30, QRAF_HIP_ERR_INVALID, "tree attention: max_ctx %d over 2^30", max_ctx);
    QH_REQUIRE(kv_dtype == DT_F32 || kv_dtype == DT_F16 || kv_dtype == DT_I8, QRAF_HIP_ERR_DTYPE,
               "tree attention: KV dtype %u", kv_dtype);
    const size_t need = tree_attention_workspace_bytes(n, seqs, H, Hkv, hd, max_ctx);
    QH_REQUIRE(ws_bytes >= need, QRAF_HIP_ERR_INVALID, "tree attention: workspace of %zu bytes, %zu needed", ws_bytes,
               need);
    if (const int few = kv_dtype == DT_F32 ? tree_few_heads(n, seqs, H, Hkv, hd, page_size, max_ctx) : 0)
        return launch_tree_few(q, kc, vc, page_table, max_pages, base, row_starts, masks, n, seqs, H, Hkv, hd, page_size, scale,
                               max_ctx, few, out, st, out_hi, out_lo);
    GroupArgs a{};
    a.q = q;
    a.kc = kc;
    a.vc = vc;
    a.page_table = page_table;
    a.starts = row_starts;
    a.prefix = base;
    a.masks = (const unsigned long long*)masks;
    a.out = out;
    a.out_hi = out_hi;
    a.out_lo = out_lo;
    a.n = n;
    a.groups = seqs;
    a.H = H;
    a.Hkv = Hkv;
    a.G = H / Hkv;
    a.page_size = page_size;
    a.max_pages = max_pages;
    a.max_ctx = max_ctx;
    a.scale = scale;
    if (group_attention_tiles(n, seqs, H, Hkv, hd, page_size, true))
        return group_tiles<true>(a, kv_dtype, hd, ws, group_direct(n, H, Hkv, kv_dtype, max_ctx), st);
    return group_any<true>(a, kv_dtype, hd, st);
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

uint64_t qraf_hip_tree_attention_workspace_bytes(int32_t n_rows, int32_t n_seqs, int32_t n_heads, int32_t n_kv_heads,
                                                 int32_t head_dim, int32_t max_ctx) {
    if (n_rows <= 0 || n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_ctx <= 0) return 0;
    return tree_attention_workspace_bytes(n_rows, n_seqs, n_heads, n_kv_heads, head_dim, max_ctx);
}

int qraf_hip_tree_attention_dev(const float* q, const void* k_cache, const void* v_cache, uint32_t kv_dtype,
                                const int32_t* page_table, int32_t max_pages_per_seq, const int32_t* base_lens,
                                const int32_t* row_starts, const uint64_t* masks, int32_t n_rows, int32_t n_seqs,
                                int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t page_size, float scale,
                                int32_t max_ctx, float* out, void* workspace, uint64_t workspace_bytes, void* stream) {
    clear_error();
    return launch_tree_attention(q, k_cache, v_cache, kv_dtype, page_table, max_pages_per_seq, base_lens, row_starts,
                                 masks, n_rows, n_seqs, n_heads, n_kv_heads, head_dim, page_size, scale, max_ctx, out,
                                 workspace, workspace_bytes, as_stream(stream), nullptr, nullptr);
}

}  // extern "C"
