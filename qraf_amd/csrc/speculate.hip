// speculate.hip -- a Sampler's distribution as probabilities, and drafted
// tokens verified against such probabilities (speculative decoding).
//
// qraf_hip_sample_probs_dev: the distribution that Sampler::sample draws from
// (reference src/sampling/sampler.cpp:57-128), written out.  With m the row's
// largest logit and w_i = exp((l_i - m) / T):
//   C     the top_k largest logits (all when top_k is off), equal ones in
//         index order;
//   N     with 0 < top_p < 1 the shortest prefix of C in that order whose
//         weight reaches top_p times the weight of C, else C;
//   p_i = w_i / sum_{j in N} w_j for i in N, 0 elsewhere.
// The kept set is one threshold: the order-preserving key of its smallest
// logit and the number of equal logits it takes, lowest indices first.  It is
// found from a short list of candidates in order, or by a radix select over all
// keys.  Weights are summed as integers there (w times a power of two that keeps
// the row's sum below 2^62, from a 64-bit exponential): integer sums do not depend
// on the order of the atomics, so results repeat bit for bit, and the border of a
// nucleus whose tokens weigh 1e-6 of the row each is the one of the sums in 64-bit
// floating point.  (Steps of 2^-62 times the next power of two above the
// vocabulary: 2^-44 of the largest weight for 151,936 tokens.)  The probabilities
// themselves are 32-bit products, w by a two-part exponent, sums of whole rows in
// 32 bits within a split and in 64 over the splits: within 8 * 2^-24 of a value, which
// a 32-bit result has room for and the draw (64-bit sums of them) takes as it is.
//
// A row of 152K logits is read by many workgroups (one alone reads 600 KB in
// 10 us), in launches that follow one another:
//   stats   per split the largest and smallest logit and, where nothing is cut
//           off, the weight; for a short top_k also the largest of every thread's
//           E logits (a sub-range)
//   select  short top_k: one workgroup per row.  The top_k-th largest of the
//           sub-ranges' maxima bounds the top_k-th largest logit from below;
//           only sub-ranges whose maximum reaches it are read again
//           (probs_topk_kernel)
//           nucleus of the whole row: weights by bins of the logits' distance from
//           the largest (probs_bins_kernel), the logits of the bin in which top_p
//           is reached (probs_gather_kernel), those in order (probs_border_kernel)
//           else (top_k over 512, or of more sub-ranges than the workgroup holds:
//           from 163,841 logits by 8, 655,361 by 32), and where such a list
//           overflows (flat rows): radix select over the keys by one workgroup
//   write   w_i / sum in 32 bits
//
// qraf_hip_verify_draft_dev: row j of a sequence is the target's distribution
// behind its first j drafted tokens.  Draft x_j, drawn from q_j, is accepted
// while u_j q_j(x_j) < p_j(x_j) (probability min(1, p/q)); at the first row that
// rejects, the next token is drawn from max(p_j - q_j, 0), which makes the
// emitted tokens' distribution the target's own; behind the last accepted draft
// it is drawn from the last row's p.  Draws are inverse sums in index order:
// the first token whose running sum passes v times the total.  Products and
// sums in 64 bits.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "logits.h"

namespace qraf_hip {

constexpr int PNT = 1024;  // threads per row

// weight64 in 32 bits, off by at most 3 units of the last place: the exponent's
// rounding errors (of l - m, of its product with log2(e) / T) as a factor behind it.
// l and m by halves: their difference may leave fp32's range where T brings it back
struct Weight32 {
    float m, mh, c, c_lo;
    __device__ __forceinline__ Weight32(float m_, double T) : m(m_), mh(0.5f * m_) {
        const double k = 2 * 1.4426950408889634074 / T;
        c = (float)k;
        c_lo = (float)(k - (double)c);
    }
    __device__ __forceinline__ float operator()(float l) const {
        const float d = __builtin_fmaf(l, 0.5f, -mh), bb = d + mh;  // (l - m) / 2 = d + err (Knuth's two-sum)
        const float err = __builtin_fmaf(l, 0.5f, -bb) + (mh - (bb - d));
        const float h = d * c;
        const float e = __builtin_fmaf(d, c, -h) + __builtin_fmaf(d, c_lo, err * c);
        const float w = __builtin_amdgcn_exp2f(h);
        return l == m ? 1.f : h > -160.f ? __builtin_fmaf(w, e * 0.693147180559945f, w) : 0.f;  // (-inf, NaN: 0)
    }
};

constexpr int STH = 256;       // threads of a split
constexpr int TOPK_MAX = 512;  // largest top_k by sub-range maxima
constexpr int SUB_REGS = 20;   // sub-range maxima a thread of the selection holds
constexpr int LIST = 4096;     // candidates in order at most
constexpr int BINS = 2048;

struct Border {  // the bin of a row in which its nucleus ends (-1: no bins), the weight ahead of it, the weight needed
    int bin;
    float m, scale;
    unsigned long long above, need;
};
struct SplitStats {
    float m, s, least;  // the largest logit, the split's weight against it, the smallest above -inf
    int mi;             // the first index of m
};
struct RowSel {  // what is kept: keys above `key`, and of those equal to it the logits before index `cut`
    double inv;  // 1 / their weight
    float m;
    uint32_t key;
    int cut;
};
constexpr RowSel EMPTY_ROW{0.0, -INFINITY, 0u, 0};  // a row without a token
struct ProbsArgs {
    const float* logits;
    float* probs;
    SplitStats* stats;         // [rows][S]
    float* sub;                // [rows][S * STH] sub-range maxima
    unsigned long long* bins;  // [rows][BINS]
    unsigned long long* list;  // [rows][LIST] (key, ~index)
    int* count;                // [rows]
    Border* border;            // [rows]
    RowSel* sel;               // [rows]
    int V, S, cutoff;
    float T, top_p;
};

// logits of a split: thread's element u of E, its index; VEC: in float4s, of rows aligned to them
template <int E, bool VEC>
__device__ __forceinline__ int split_index(int split, int u) {
    const int b = split * STH * E;
    return VEC ? b + 4 * (threadIdx.x + STH * (u >> 2)) + (u & 3) : b + (int)threadIdx.x + STH * u;
}
// element u of sub-range (split, thread)
template <int E, bool VEC>
__device__ __forceinline__ int sub_index(int sub, int u) {
    const int b = sub / STH * STH * E, t = sub % STH;
    return VEC ? b + 4 * (t + STH * (u >> 2)) + (u & 3) : b + t + STH * u;
}
template <int E, bool VEC>
__device__ __forceinline__ void load_split(const float* l, int V, int split, float (&v)[E]) {
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < E / 4; j++) {
            const int i = split_index<E, VEC>(split, 4 * j);
            const float4 x = *(const float4*)(l + min(i, V - 4));
            const bool in = i < V;
            v[4 * j] = in ? x.x : -INFINITY, v[4 * j + 1] = in ? x.y : -INFINITY;
            v[4 * j + 2] = in ? x.z : -INFINITY, v[4 * j + 3] = in ? x.w : -INFINITY;
        }
    } else {
#pragma unroll
        for (int u = 0; u < E; u++) {
            const int i = split_index<E, VEC>(split, u);
            const float x = l[min(i, V - 1)];
            v[u] = i < V ? x : -INFINITY;
        }
    }
}

// the first of the largest over a workgroup's waves, in every thread (s_f, s_i: an entry for each wave)
__device__ __forceinline__ void block_first_max(float& m, int& mi, float* s_f, int* s_i, int waves) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float om = __shfl_xor(m, o);
        const int oi = __shfl_xor(mi, o);
        if (om > m || (om == m && oi < mi)) {
            m = om;
            mi = oi;
        }
    }
    if ((threadIdx.x & 63) == 0) {
        s_f[threadIdx.x >> 6] = m;
        s_i[threadIdx.x >> 6] = mi;
    }
    __syncthreads();
    for (int w = 0; w < waves; w++)
        if (s_f[w] > m || (s_f[w] == m && s_i[w] < mi)) {
            m = s_f[w];
            mi = s_i[w];
        }
}

// what follows: the write of whole rows, top_k (clear: and the probabilities are zeroed for it), the nucleus' bins, or
// what needs the largest logit alone
enum : int { STATS_SUM = 0, STATS_SUB = 1, STATS_BINS = 2, STATS_MAX = 3 };

template <int E, bool VEC>
__device__ __forceinline__ void store_split(float* p, int V, int split, const float (&v)[E]) {
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < E / 4; j++) {
            const int i = split_index<E, VEC>(split, 4 * j);
            if (i < V) *(float4*)(p + i) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
    } else {
#pragma unroll
        for (int u = 0; u < E; u++) {
            const int i = split_index<E, VEC>(split, u);
            if (i < V) p[i] = v[u];
        }
    }
}

template <int E, bool VEC>
__global__ __launch_bounds__(STH) void probs_stats_kernel(ProbsArgs a, int what, int clear) {
    __shared__ float s_f[4], s_least[4], s_sum[4];
    __shared__ int s_i[4];
    const int split = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float v[E];
    load_split<E, VEC>(a.logits + (size_t)row * a.V, a.V, split, v);
    float m = -INFINITY, least = INFINITY;
    int mi = a.V;
#pragma unroll
    for (int u = 0; u < E; u++) {
        v[u] = clean_logit(v[u]);
        if (v[u] > m) {  // (increasing index)
            m = v[u];
            mi = split_index<E, VEC>(split, u);
        }
        least = v[u] > -INFINITY ? fminf(least, v[u]) : least;
    }
    if (what == STATS_SUB) a.sub[((size_t)row * a.S + split) * STH + tid] = m;
    if (clear) {
        float z[E];
#pragma unroll
        for (int u = 0; u < E; u++) z[u] = 0.f;
        store_split<E, VEC>(a.probs + (size_t)row * a.V, a.V, split, z);
    }
    block_first_max(m, mi, s_f, s_i, 4);
    float sum = 0.f;
    if (what == STATS_SUM && m > -INFINITY) {
        const Weight32 weight(m, a.T);
#pragma unroll
        for (int u = 0; u < E; u++) sum += weight(v[u]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        least = fminf(least, __shfl_xor(least, o));
        sum += __shfl_xor(sum, o);
    }
    if (lane == 0) {
        s_least[wave] = least;
        s_sum[wave] = sum;
    }
    __syncthreads();
    if (tid == 0)
        a.stats[(size_t)row * a.S + split] =
            SplitStats{m, (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]),
                       fminf(fminf(s_least[0], s_least[1]), fminf(s_least[2], s_least[3])), mi};
    if (what == STATS_BINS) {  // cleared for what follows
        for (int i = split * STH + tid; i < BINS; i += a.S * STH) a.bins[(size_t)row * BINS + i] = 0;
        if (split == 0 && tid == 0) a.count[row] = 0;
    }
}

// the row's largest logit, its first index and its smallest above -inf, from its splits, by each wave
struct RowStats {
    float m, least;
    int mi;
};
__device__ __forceinline__ RowStats row_stats(const ProbsArgs& a, int row) {
    const SplitStats* st = a.stats + (size_t)row * a.S;
    RowStats r{-INFINITY, INFINITY, a.V};
    for (int i = threadIdx.x & 63; i < a.S; i += 64) {
        const SplitStats x = st[i];
        if (x.m > r.m) {
            r.m = x.m;
            r.mi = x.mi;
        }
        r.least = fminf(r.least, x.least);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float om = __shfl_xor(r.m, o);
        const int oi = __shfl_xor(r.mi, o);
        if (om > r.m || (om == r.m && oi < r.mi)) {
            r.m = om;
            r.mi = oi;
        }
        r.least = fminf(r.least, __shfl_xor(r.least, o));
    }
    return r;
}
// its weight
__device__ __forceinline__ double row_weight(const ProbsArgs& a, int row, float m) {
    const SplitStats* st = a.stats + (size_t)row * a.S;
    double s = 0.0;
    for (int i = threadIdx.x & 63; i < a.S; i += 64) s += (double)st[i].s * weight64(st[i].m, m, a.T);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    return s;
}

// integer weights: the power of two that keeps a row's sum below 2^62
__device__ __forceinline__ double weight_unit(int V) { return ldexp(1.0, 62 - (32 - __clz(V))); }
__device__ __forceinline__ unsigned long long weigh(float l, float m, double T, double unit) {
    return (unsigned long long)(weight64(l, m, T) * unit + 0.5);
}
// weight that the nucleus has to reach
__device__ __forceinline__ unsigned long long nucleus_need(unsigned long long z, float top_p) {
    return max(1ull, (unsigned long long)ceil((double)z * (double)top_p));
}

// ---- radix select, one workgroup: any row and parameters
struct RadixShared {
    unsigned long long hist[256], sum, need;
    uint32_t key;
    int cut, cnt[PNT];
};
__device__ void radix_select(const ProbsArgs& a, const float* l, float m, RadixShared& sh, RowSel* out) {
    const int tid = threadIdx.x, V = a.V;
    const double t64 = a.T, unit = weight_unit(V);
    uint32_t key = 0;  // the kept set so far
    int cut = V;
    // the kept set's largest logits that reach `need` (a count, or a weight)
    auto select = [&](bool by_weight, unsigned long long need) {
        uint32_t prefix = 0, mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += PNT) {
                const float v = clean_logit(l[i]);
                const uint32_t k = logit_key(v);
                if ((k & mask) != prefix || k < key || (k == key && i >= cut)) continue;
                atomicAdd(&sh.hist[(k >> shift) & 255u], by_weight ? weigh(v, m, t64, unit) : 1ull);
            }
            __syncthreads();
            if (tid == 0) {
                unsigned long long acc = 0;
                int d = 255;
                for (; d > 0; d--) {
                    if (acc + sh.hist[d] >= need) break;
                    acc += sh.hist[d];
                }
                sh.key = prefix | ((uint32_t)d << shift);
                sh.need = need - acc;
            }
            __syncthreads();
            prefix = sh.key;
            need = sh.need;
            mask |= 255u << shift;
            __syncthreads();
        }
        // `need` more at key `prefix`: so many of the equal logits
        unsigned long long ties = need;
        if (by_weight) {
            const uint32_t b = (prefix & 0x80000000u) ? (prefix & 0x7FFFFFFFu) : ~prefix;
            const unsigned long long w = weigh(__uint_as_float(b), m, t64, unit);
            ties = w ? (need + w - 1) / w : (unsigned long long)V;
        }
        // the index behind the ties-th of them
        const int ch = (V + PNT - 1) / PNT, i0 = min(V, tid * ch), i1 = min(V, i0 + ch);
        int c = 0;
        for (int i = i0; i < i1; i++) c += logit_key(clean_logit(l[i])) == prefix;
        sh.cnt[tid] = c;
        if (tid == 0) sh.cut = V;
        __syncthreads();
        unsigned long long before = 0;
        for (int t = 0; t < tid; t++) before += sh.cnt[t];
        if (before < ties && before + c >= ties) {
            int i = i0;
            for (; before < ties; i++) before += logit_key(clean_logit(l[i])) == prefix;
            sh.cut = i;
        }
        __syncthreads();
        cut = prefix == key ? min(cut, sh.cut) : sh.cut;
        key = prefix;
        __syncthreads();
    };
    auto total = [&]() {  // the kept set's weight
        if (tid == 0) sh.sum = 0;
        __syncthreads();
        unsigned long long z = 0;
        for (int i = tid; i < V; i += PNT) {
            const float v = clean_logit(l[i]);
            const uint32_t k = logit_key(v);
            if (k > key || (k == key && i < cut)) z += weigh(v, m, t64, unit);
        }
        atomicAdd(&sh.sum, z);
        __syncthreads();
        z = sh.sum;
        __syncthreads();
        return z;
    };
    if (a.cutoff < V) select(false, (unsigned long long)a.cutoff);
    unsigned long long z = total();
    if (a.top_p > 0.f && a.top_p < 1.f) {
        select(true, nucleus_need(z, a.top_p));
        z = total();
    }
    if (tid == 0) *out = RowSel{unit / (double)z, m, key, cut};
}

__global__ __launch_bounds__(PNT) void probs_radix_kernel(ProbsArgs a) {
    __shared__ RadixShared sh;
    const int row = blockIdx.x;
    const RowStats r = row_stats(a, row);
    if (r.m == -INFINITY) {
        if (threadIdx.x == 0) a.sel[row] = EMPTY_ROW;
        return;
    }
    radix_select(a, a.logits + (size_t)row * a.V, r.m, sh, &a.sel[row]);
}

// ---- candidates in order: n <= LIST entries (key, ~index) of `in`, the largest first, to `sorted`
__device__ __forceinline__ void rank_sort(const unsigned long long* in, unsigned long long* sorted, int n) {
    for (int i = threadIdx.x; i < n; i += PNT) {
        const unsigned long long x = in[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += in[j] > x;
        sorted[rank] = x;
    }
    __syncthreads();
}
// The first nc of `sorted`, or (nucleus) as many of them as bring the weight `above` them to need(all); in every
// thread.  (s_w: a word for each entry)
template <typename F>
__device__ RowSel keep_prefix(const ProbsArgs& a, const unsigned long long* sorted, int nc, float m, bool nucleus,
                              unsigned long long above, F need_of, unsigned long long* s_w, RowSel* s_sel) {
    const int tid = threadIdx.x;
    const double unit = weight_unit(a.V);
    for (int i = tid; i < nc; i += PNT) s_w[i] = weigh(key_logit((uint32_t)(sorted[i] >> 32)), m, a.T, unit);
    __syncthreads();
    if (tid < 64) {  // one wave: lane's entries per * lane ..
        const int per = (nc + 63) >> 6, i0 = min(nc, tid * per), i1 = min(nc, i0 + per);
        unsigned long long w = 0;
        for (int i = i0; i < i1; i++) w += s_w[i];
        unsigned long long inc = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long x = __shfl_up(inc, o);
            inc += tid >= o ? x : 0;
        }
        const unsigned long long all = above + __shfl(inc, 63), need = need_of(all);
        auto keep = [&](int i, unsigned long long sum) {
            const unsigned long long last = sorted[i];
            *s_sel = RowSel{unit / (double)sum, m, (uint32_t)(last >> 32), (int)(0xFFFFFFFFu - (uint32_t)last) + 1};
        };
        unsigned long long sum = above + inc - w;
        if (!nucleus) {
            if (tid == 0) keep(nc - 1, all);
        } else if (sum < need && sum + w >= need) {
            int i = i0;
            for (;; i++) {
                sum += s_w[i];
                if (sum >= need || i + 1 >= i1) break;
            }
            keep(i, sum);
        }
    }
    __syncthreads();
    return *s_sel;
}

// ---- short top_k.  scatter: the probabilities are zero, and the few that are kept are written here
template <int E, bool VEC>
__global__ __launch_bounds__(PNT) void probs_topk_kernel(ProbsArgs a, int scatter) {
    __shared__ RadixShared sh;
    __shared__ unsigned long long s_list[LIST], s_sorted[LIST], s_w[LIST];
    __shared__ uint32_t s_lo[PNT / 64];
    __shared__ int s_subs[PNT], s_cnt[3][8], s_n, s_ns;
    __shared__ RowSel s_sel;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, V = a.V, n_sub = a.S * STH, k = a.cutoff;
    const float* l = a.logits + (size_t)row * V;
    const float* sub = a.sub + (size_t)row * n_sub;
    uint32_t mine[SUB_REGS], lo = 0xFFFFFFFFu;
#pragma unroll
    for (int u = 0; u < SUB_REGS; u++) {
        mine[u] = 0u;
        if (PNT * u < n_sub) {  // (for the whole workgroup)
            const int i = tid + PNT * u;
            const uint32_t x = logit_key(sub[min(i, n_sub - 1)]);
            mine[u] = i < n_sub ? x : 0u;
            lo = min(lo, x);
        }
    }
    const RowStats r = row_stats(a, row);
    if (r.m == -INFINITY) {
        if (tid == 0) a.sel[row] = EMPTY_ROW;
        return;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) lo = min(lo, (uint32_t)__shfl_xor((int)lo, o));
    if (lane == 0) s_lo[tid >> 6] = lo;
    if (tid < 24) s_cnt[tid >> 3][tid & 7] = 0;
    if (tid == 0) s_n = s_ns = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PNT / 64; w++) lo = min(lo, s_lo[w]);
    // a bound that at least k, and not many more, maxima reach: 8 thresholds at a time between the smallest of them
    // and the largest.  (All rows of one value, or masked ones, end with a list that overflows.)
    uint32_t hi = logit_key(r.m);
    const int enough = k + (k >> 2) + 8;
    int reach = n_sub;
    for (int pass = 0; pass < 12 && reach > enough && lo < hi; pass++) {
        uint32_t th[8];
        int c = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            th[j] = lo + (uint32_t)(((unsigned long long)(hi - lo) * (j + 1)) >> 3);
            int x = 0;
#pragma unroll
            for (int u = 0; u < SUB_REGS; u++)
                if (PNT * u < n_sub) x += __popcll(__ballot(mine[u] >= th[j]));
            c = lane == j ? x : c;
        }
        if (lane < 8 && c) atomicAdd(&s_cnt[pass % 3][lane], c);
        __syncthreads();
        uint32_t nlo = lo, nhi = hi;
        int nr = reach;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int x = s_cnt[pass % 3][j];
            if (x >= k) {
                nlo = th[j];
                nr = x;
            } else if (th[j] < nhi) {
                nhi = th[j];
            }
        }
        if (tid < 8) s_cnt[(pass + 2) % 3][tid] = 0;  // last read before this pass's barrier
        if (nlo == lo && nhi == hi) break;
        lo = nlo, hi = nhi, reach = nr;
    }
    // sub-ranges that reach it, then their logits that do
#pragma unroll
    for (int u = 0; u < SUB_REGS; u++)
        if (PNT * u < n_sub && mine[u] >= lo && tid + PNT * u < n_sub) {
            const int x = atomicAdd(&s_ns, 1);
            if (x < PNT) s_subs[x] = tid + PNT * u;
        }
    __syncthreads();
    const int ns = s_ns;
    if (ns <= PNT) {
        for (int i = tid; i < ns * E; i += PNT) {
            const int at = sub_index<E, VEC>(s_subs[i / E], i % E);
            if (at >= V) continue;
            const uint32_t key = logit_key(clean_logit(l[at]));
            if (key >= lo) {
                const int x = atomicAdd(&s_n, 1);
                if (x < LIST) s_list[x] = (unsigned long long)key << 32 | (0xFFFFFFFFu - (uint32_t)at);
            }
        }
    }
    __syncthreads();
    const int n = s_n;
    RowSel sel;
    const bool listed = ns <= PNT && n <= LIST && n >= k;
    if (listed) {
        rank_sort(s_list, s_sorted, n);
        sel = keep_prefix(a, s_sorted, min(n, k), r.m, a.top_p > 0.f && a.top_p < 1.f, 0,
                          [&](unsigned long long z) { return nucleus_need(z, a.top_p); }, s_w, &s_sel);
    } else {
        radix_select(a, l, r.m, sh, &s_sel);
        __syncthreads();
        sel = s_sel;
    }
    if (!scatter) {
        if (tid == 0) a.sel[row] = sel;
        return;
    }
    const Weight32 weight(r.m, a.T);
    float* p = a.probs + (size_t)row * V;
    auto write = [&](float x, int i) {
        const uint32_t key = logit_key(x);
        if (key > sel.key || (key == sel.key && i < sel.cut)) p[i] = weight(x) * (float)sel.inv;
    };
    if (listed) {
        for (int i = tid; i < n; i += PNT)
            write(key_logit((uint32_t)(s_sorted[i] >> 32)), (int)(0xFFFFFFFFu - (uint32_t)s_sorted[i]));
    } else {
        for (int i = tid; i < V; i += PNT) write(clean_logit(l[i]), i);
    }
}

// ---- nucleus of the whole row: bin of a logit by its distance from the largest, up to 32 T or the smallest
__device__ __forceinline__ float bin_scale(const RowStats& r, float T) {
    const float d = fminf((r.m - r.least) / T, 32.f);
    return (float)(BINS - 1) / (fmaxf(d, 1e-30f) * T);
}
__device__ __forceinline__ int bin_of(float l, float m, float scale) {  // monotone in l
    return l == m ? 0 : (int)fminf((m - l) * scale, (float)(BINS - 1));
}
// whether rows of infinities, or of T that leaves the range, have bins at all
__device__ __forceinline__ bool has_bins(const RowStats& r, float scale) {
    return r.m < INFINITY && scale > 0.f && scale < INFINITY;
}

template <int E, bool VEC>
__global__ __launch_bounds__(STH) void probs_bins_kernel(ProbsArgs a, int per_wg) {
    __shared__ unsigned long long s_bin[BINS];
    const int row = blockIdx.y, tid = threadIdx.x;
    const RowStats r = row_stats(a, row);
    const float scale = bin_scale(r, a.T);
    if (r.m == -INFINITY || !has_bins(r, scale)) return;
    for (int i = tid; i < BINS; i += STH) s_bin[i] = 0;
    __syncthreads();
    const double unit = weight_unit(a.V);
    const int s1 = min(a.S, ((int)blockIdx.x + 1) * per_wg);
    for (int split = blockIdx.x * per_wg; split < s1; split++) {
        float v[E];
        load_split<E, VEC>(a.logits + (size_t)row * a.V, a.V, split, v);
#pragma unroll 4
        for (int u = 0; u < E; u++) {
            const float x = clean_logit(v[u]);
            if (x > -INFINITY) atomicAdd(&s_bin[bin_of(x, r.m, scale)], weigh(x, r.m, a.T, unit));
        }
    }
    __syncthreads();
    for (int i = tid; i < BINS; i += STH)
        if (s_bin[i]) atomicAdd(&a.bins[(size_t)row * BINS + i], s_bin[i]);
}

// the border bin of each row, one wave for each: lanes sum their 32 bins, then the one that holds the border looks
__global__ __launch_bounds__(64) void probs_cut_kernel(ProbsArgs a) {
    constexpr int PER = BINS / 64;
    const int row = blockIdx.x, lane = threadIdx.x;
    const ulonglong2* bins = (const ulonglong2*)(a.bins + (size_t)row * BINS + lane * PER);
    unsigned long long x[PER], w = 0;
#pragma unroll
    for (int i = 0; i < PER / 2; i++) {
        const ulonglong2 y = bins[i];
        x[2 * i] = y.x;
        x[2 * i + 1] = y.y;
    }
    const RowStats r = row_stats(a, row);
    const float scale = bin_scale(r, a.T);
    if (r.m == -INFINITY || !has_bins(r, scale)) {
        if (lane == 0) a.border[row] = Border{-1, r.m, 0.f, 0, 0};
        return;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) w += x[i];
    unsigned long long inc = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long y = __shfl_up(inc, o);
        inc += lane >= o ? y : 0;
    }
    const unsigned long long need = nucleus_need(__shfl(inc, 63), a.top_p);
    unsigned long long sum = inc - w;
    if (sum < need && sum + w >= need) {
        int at = 0;
        bool found = false;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            found = found || sum + x[i] >= need;
            if (!found) {
                sum += x[i];
                at = i + 1;
            }
        }
        a.border[row] = Border{lane * PER + at, r.m, scale, sum, need};
    }
}

// (a place in the row's list for all that a workgroup found: an atomic for each of them takes 60 us of 64 rows)
template <int E, bool VEC>
__global__ __launch_bounds__(STH) void probs_gather_kernel(ProbsArgs a) {
    __shared__ unsigned long long s_found[LIST];
    __shared__ int s_n, s_at;
    const int split = blockIdx.x, row = blockIdx.y;
    float v[E];
    load_split<E, VEC>(a.logits + (size_t)row * a.V, a.V, split, v);
    const Border b = a.border[row];
    if (b.bin < 0) return;
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < E; u++) {
        const float x = clean_logit(v[u]);
        if (x > -INFINITY && bin_of(x, b.m, b.scale) == b.bin) {
            const int at = atomicAdd(&s_n, 1);
            if (at < LIST)
                s_found[at] = (unsigned long long)logit_key(x) << 32 | (0xFFFFFFFFu - (uint32_t)split_index<E, VEC>(split, u));
        }
    }
    __syncthreads();
    const int n = s_n;
    if (n == 0) return;
    if (threadIdx.x == 0) s_at = atomicAdd(&a.count[row], n);
    __syncthreads();
    for (int i = threadIdx.x; i < n && s_at + i < LIST; i += STH) a.list[(size_t)row * LIST + s_at + i] = s_found[i];
}

__global__ __launch_bounds__(PNT) void probs_border_kernel(ProbsArgs a) {
    __shared__ RadixShared sh;
    __shared__ unsigned long long s_list[LIST], s_sorted[LIST], s_w[LIST];
    __shared__ RowSel s_sel;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Border b = a.border[row];
    const int n = a.count[row];
    if (b.m == -INFINITY) {
        if (tid == 0) a.sel[row] = EMPTY_ROW;
        return;
    }
    if (b.bin < 0 || n > LIST) {
        radix_select(a, a.logits + (size_t)row * a.V, b.m, sh, &a.sel[row]);
        return;
    }
    for (int i = tid; i < n; i += PNT) s_list[i] = a.list[(size_t)row * LIST + i];
    __syncthreads();
    rank_sort(s_list, s_sorted, n);
    const RowSel sel = keep_prefix(a, s_sorted, n, b.m, true, b.above, [&](unsigned long long) { return b.need; }, s_w, &s_sel);
    if (tid == 0) a.sel[row] = sel;
}

// ---- the probabilities
enum : int { WRITE_ALL = 0, WRITE_SEL = 1, WRITE_FIRST = 2 };  // no cut, the selection's, temperature 0

template <int E, bool VEC>
__global__ __launch_bounds__(STH) void probs_write_kernel(ProbsArgs a, int what) {
    const int split = blockIdx.x, row = blockIdx.y;
    float v[E];
    float* p = a.probs + (size_t)row * a.V;
    if (what == WRITE_FIRST) {
        const RowStats r = row_stats(a, row);
#pragma unroll
        for (int u = 0; u < E; u++) v[u] = split_index<E, VEC>(split, u) == r.mi ? 1.f : 0.f;
        store_split<E, VEC>(p, a.V, split, v);
        return;
    }
    load_split<E, VEC>(a.logits + (size_t)row * a.V, a.V, split, v);
    RowSel sel{0.0, 0.f, 0u, a.V};
    if (what == WRITE_SEL) {
        sel = a.sel[row];
    } else {
        sel.m = row_stats(a, row).m;
        sel.inv = 1.0 / row_weight(a, row, sel.m);
    }
    const float inv = (float)sel.inv;
    const Weight32 weight(sel.m, a.T);
#pragma unroll
    for (int u = 0; u < E; u++) {
        const float x = clean_logit(v[u]);
        const uint32_t k = logit_key(x);
        const bool in = sel.m > -INFINITY && (k > sel.key || (k == sel.key && split_index<E, VEC>(split, u) < sel.cut));
        v[u] = in ? weight(x) * inv : 0.f;
    }
    store_split<E, VEC>(p, a.V, split, v);
}

// Logits of a thread's sub-range: 32 where that still gives every CU a workgroup, else 8 (4 rows x 49152:
// 24 workgroups of 32, 96 of 8).
static int probs_e(int rows, int V) { return V >= 65536 && (long long)rows * V >= 256ll * STH * 32 ? 32 : 8; }
static int probs_splits(int rows, int V) {
    const int e = STH * probs_e(rows, V);
    return (V + e - 1) / e;
}
struct ProbsSizes {
    size_t stats, sub, bins, list, count, border, sel;
};
static ProbsSizes probs_sizes(int rows, int V) {
    const size_t S = probs_splits(rows, V), n = rows;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    return ProbsSizes{up(n * S * sizeof(SplitStats)), up(n * S * STH * 4), up(n * BINS * 8), up(n * LIST * 8),
                      up(n * 4), up(n * sizeof(Border)), up(n * sizeof(RowSel))};
}
size_t sample_probs_workspace_bytes(int rows, int V) {
    const ProbsSizes z = probs_sizes(rows, V);
    return z.stats + z.sub + z.bins + z.list + z.count + z.border + z.sel;
}

int launch_sample_probs(float* logits, int rows, int V, const qraf_sampling_params& sp, const uint32_t* recent,
                        const int32_t* counts, int stride, float* probs, void* ws, size_t ws_bytes, hipStream_t s) {
    QH_REQUIRE(logits && probs && ws && rows > 0 && V > 0, QRAF_HIP_ERR_INVALID, "sample_probs: bad arguments");
    QH_REQUIRE(V <= 1 << 30, QRAF_HIP_ERR_INVALID, "sample_probs: vocabulary %d over 2^30", V);
    QH_REQUIRE(rows <= 65535, QRAF_HIP_ERR_INVALID, "sample_probs: %d rows over 65535", rows);
    QH_REQUIRE(((uintptr_t)ws & 15) == 0, QRAF_HIP_ERR_INVALID, "sample_probs: workspace not 16-byte aligned");
    QH_REQUIRE(ws_bytes >= sample_probs_workspace_bytes(rows, V), QRAF_HIP_ERR_INVALID,
               "sample_probs: workspace of %zu bytes, %zu needed", ws_bytes, sample_probs_workspace_bytes(rows, V));
    QH_TRY(launch_penalty(logits, rows, V, sp.repetition_penalty, recent, counts, stride, s));
    const ProbsSizes z = probs_sizes(rows, V);
    ProbsArgs a{};
    a.logits = logits;
    a.probs = probs;
    uint8_t* w = (uint8_t*)ws;
    a.stats = (SplitStats*)w;
    a.sub = (float*)(w += z.stats);
    a.bins = (unsigned long long*)(w += z.sub);
    a.list = (unsigned long long*)(w += z.bins);
    a.count = (int*)(w += z.list);
    a.border = (Border*)(w += z.count);
    a.sel = (RowSel*)(w += z.border);
    a.V = V;
    a.S = probs_splits(rows, V);
    a.cutoff = (sp.top_k > 0 && sp.top_k < V) ? sp.top_k : V;
    a.T = sp.temperature;
    a.top_p = sp.top_p;
    const bool greedy = !(sp.temperature > 0.f), cut_p = sp.top_p > 0.f && sp.top_p < 1.f;
    const bool cuts = !greedy && (a.cutoff < V || cut_p);
    const bool topk = cuts && a.cutoff < V && a.cutoff <= TOPK_MAX && a.S * STH <= SUB_REGS * PNT;
    const bool bins = cuts && a.cutoff == V;
    const bool vec = V % 4 == 0 && ((uintptr_t)logits & 15) == 0 && ((uintptr_t)probs & 15) == 0;
    const int e = probs_e(rows, V);
    const dim3 grid(a.S, rows);
    // top_k keeps few: the first pass writes zeros as it reads, and the selection what it keeps (160 x 151,936: 33 us
    // for a pass that writes, 15 for the zeros), unless the probabilities take the logits' place
    const bool scatter = topk && (const float*)probs != logits;
    const int per = std::max(1, a.S * rows / 1024);  // splits of a workgroup with bins of its own
#define QH_PROBS(Ev, Vv)                                                                                            \
    if (e == Ev && vec == Vv) {                                                                                     \
        hipLaunchKernelGGL((probs_stats_kernel<Ev, Vv>), grid, dim3(STH), 0, s, a,                                  \
                           topk ? STATS_SUB : bins ? STATS_BINS : cuts || greedy ? STATS_MAX : STATS_SUM, (int)scatter);                         \
        if (topk) {                                                                                                 \
            hipLaunchKernelGGL((probs_topk_kernel<Ev, Vv>), dim3(rows), dim3(PNT), 0, s, a, (int)scatter);          \
        } else if (bins) {                                                                                          \
            hipLaunchKernelGGL((probs_bins_kernel<Ev, Vv>), dim3((a.S + per - 1) / per, rows), dim3(STH), 0, s, a, per); \
            hipLaunchKernelGGL(probs_cut_kernel, dim3(rows), dim3(64), 0, s, a);                                    \
            hipLaunchKernelGGL((probs_gather_kernel<Ev, Vv>), grid, dim3(STH), 0, s, a);                            \
            hipLaunchKernelGGL(probs_border_kernel, dim3(rows), dim3(PNT), 0, s, a);                                \
        } else if (cuts) {                                                                                          \
            hipLaunchKernelGGL(probs_radix_kernel, dim3(rows), dim3(PNT), 0, s, a);                                 \
        }                                                                                                           \
        if (!scatter)                                                                                               \
            hipLaunchKernelGGL((probs_write_kernel<Ev, Vv>), grid, dim3(STH), 0, s, a,                              \
                               greedy ? WRITE_FIRST : cuts ? WRITE_SEL : WRITE_ALL);                                \
    }
    QH_PROBS(8, true) QH_PROBS(8, false) QH_PROBS(32, true) QH_PROBS(32, false)
#undef QH_PROBS
    QH_CHECK_HIP(hipGetLastError());
    return QRAF_HIP_OK;
}

// ---------------------------------------------------------------- verification

struct VerifyArgs {
    const float* p;             // [n_rows][V] the target's probabilities
    const float* q;             // [n_rows][V] the drafts' probabilities, or null (a draft was certain)
    const uint32_t* draft;      // [n_rows] the token drafted behind row j's, unused in a sequence's last row
    const int32_t* row_starts;  // [n + 1]
    const float* u;             // [n_rows] acceptance
    const float* v;             // [n] the next token's draw
    int32_t* accepted;          // [n]
    uint32_t* tokens;           // [n_rows]
    int n, n_rows, V;
};

// The first row of a sequence that does not accept its draft, or its last: all drafts looked at at once, by each wave.
// (a sequence's rows [r0, r1), r0 < r1)
__device__ __forceinline__ int rejecting_row(const VerifyArgs& a, int r0, int r1) {
    for (int base = r0; base < r1 - 1; base += 64) {
        const int r = min(base + (int)(threadIdx.x & 63), r1 - 1);
        const uint32_t x = a.draft[r], xc = min(x, (uint32_t)a.V - 1);
        const double q = a.q ? (double)a.q[(size_t)r * a.V + xc] : 1.0;
        const bool good = x < (uint32_t)a.V && (double)a.u[r] * q < (double)a.p[(size_t)r * a.V + xc];
        const unsigned long long bad = __ballot(r < r1 - 1 && !good);
        if (bad) return base + __builtin_ctzll(bad);
    }
    return r1 - 1;
}
__device__ __forceinline__ void rows_of(const VerifyArgs& a, int s, int& r0, int& r1) {
    r0 = max(0, min(a.row_starts[s], a.n_rows));
    r1 = max(r0, min(a.row_starts[s + 1], a.n_rows));
}

// E consecutive tokens of a row from i on: the weights of the draw, what is left of p behind a rejected draft (less:
// max(p - q, 0), or p without the draft), and p (VEC: rows aligned to float4s)
template <int E, bool VEC>
__device__ __forceinline__ void draw_weights(const VerifyArgs& a, size_t r, bool missed, uint32_t x, int i, float (&p)[E],
                                             double (&less)[E]) {
    const float *pr = a.p + r * a.V, *qr = a.q + r * a.V;
    const bool sub = missed && a.q;
    float q[E];
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < E / 4; j++) {
            const int at = min(i + 4 * j, a.V - 4);
            *(float4*)&p[4 * j] = *(const float4*)(pr + at);
            if (sub) *(float4*)&q[4 * j] = *(const float4*)(qr + at);
        }
    } else {
#pragma unroll
        for (int u = 0; u < E; u++) {
            const int at = min(i + u, a.V - 1);
            p[u] = pr[at];
            if (sub) q[u] = qr[at];
        }
    }
#pragma unroll
    for (int u = 0; u < E; u++) {
        p[u] = i + u < a.V ? p[u] : 0.f;
        less[u] = sub ? fmax((double)p[u] - (double)q[u], 0.0) : missed && (uint32_t)(i + u) == x ? 0.0 : (double)p[u];
        less[u] = i + u < a.V ? less[u] : 0.0;
    }
}

// sums of a split of STH x E tokens of each sequence's deciding row
template <int E, bool VEC>
__global__ __launch_bounds__(STH) void verify_sums_kernel(VerifyArgs a, double2* part, int* decides) {
    __shared__ double s_less[4], s_p[4];
    const int split = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    int r0, r1;
    rows_of(a, s, r0, r1);
    if (r0 == r1) return;
    const int r = rejecting_row(a, r0, r1);
    const bool missed = r < r1 - 1;
    const uint32_t x = a.draft[r];
    double sl = 0.0, sp = 0.0;
#pragma unroll
    for (int j = 0; j < E / 4; j++) {  // (any order within the split: neighbouring threads, neighbouring float4s)
        float p[4];
        double less[4];
        draw_weights<4, VEC>(a, r, missed, x, split * STH * E + 4 * (tid + STH * j), p, less);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            sl += less[u];
            sp += (double)p[u];
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        sl += __shfl_xor(sl, o);
        sp += __shfl_xor(sp, o);
    }
    if ((tid & 63) == 0) {
        s_less[tid >> 6] = sl;
        s_p[tid >> 6] = sp;
    }
    __syncthreads();
    if (tid == 0 && split == 0) decides[s] = r;
    if (tid == 0)
        part[(size_t)s * gridDim.x + split] =
            make_double2((s_less[0] + s_less[1]) + (s_less[2] + s_less[3]), (s_p[0] + s_p[1]) + (s_p[2] + s_p[3]));
}

// inclusive sum over a workgroup's threads in order (s_w: a word for each wave), and the sum of all
__device__ __forceinline__ double block_scan(double w, double* s_w, double& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(w, o);
        w += lane >= o ? x : 0.0;
    }
    if (lane == 63) s_w[wave] = w;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
#pragma unroll
    for (int v = 0; v < STH / 64; v++) {
        before += v < wave ? s_w[v] : 0.0;
        all += s_w[v];
    }
    return before + w;
}

// The first of a workgroup's threads whose inclusive sum passes the target, else the last that adds anything (a sum
// rounds otherwise here than where the target was formed): -1 where none does.  (s_t: two words for each wave)
__device__ __forceinline__ int passing_thread(double inc, double w, double target, int (*s_t)[2]) {
    const int wave = threadIdx.x >> 6;
    const unsigned long long pass = __ballot(w > 0.0 && inc > target), any = __ballot(w > 0.0);
    if ((threadIdx.x & 63) == 0) {
        s_t[wave][0] = pass ? 64 * wave + __builtin_ctzll(pass) : -1;
        s_t[wave][1] = any ? 64 * wave + 63 - __builtin_clzll(any) : -1;
    }
    __syncthreads();
    int first = -1, last = -1;
#pragma unroll
    for (int v = STH / 64 - 1; v >= 0; v--) {
        first = s_t[v][0] >= 0 ? s_t[v][0] : first;
        last = max(last, s_t[v][1]);
    }
    return first >= 0 ? first : last;
}

// The draw: the split in which the running sum passes it, then the token; a workgroup for each sequence
template <int E, bool VEC>
__global__ __launch_bounds__(STH) void verify_pick_kernel(VerifyArgs a, const double2* part, const int* decides, int S) {
    __shared__ double s_w[2][STH / 64], s_ahead;
    __shared__ int s_t[2][STH / 64][2], s_split, s_token;
    const int s = blockIdx.x, tid = threadIdx.x;
    int r0, r1;
    rows_of(a, s, r0, r1);
    if (r0 == r1) {  // a sequence without rows
        if (tid == 0) a.accepted[s] = 0;
        return;
    }
    const int r = decides[s];
    const uint32_t draft = a.draft[r];
    const double2* mine = part + (size_t)s * S;
    const int per = (S + STH - 1) / STH, i0 = min(S, tid * per), i1 = min(S, i0 + per);
    double w = 0.0, w_p = 0.0, all;
    for (int i = i0; i < i1; i++) {
        w += mine[i].x;
        w_p += mine[i].y;
    }
    double inc = block_scan(w, s_w[0], all);
    const bool left = all > 0.0;  // else nothing is left of p: the target's own distribution
    if (!left) {
        w = w_p;
        inc = block_scan(w, s_w[1], all);
    }
    // a draw outside [0, 1) (or NaN) takes the nearest inside
    const double target = (double)fminf(fmaxf(a.v[s], 0.f), 0x1.fffffep-1f) * all;
    if (tid == max(0, passing_thread(inc, w, target, s_t[0]))) {  // among the thread's splits, as among the threads
        double c = inc - w;
        s_split = i0;
        s_ahead = c;
        for (int i = i0; per > 1 && i < i1; i++) {
            const double x = left ? mine[i].x : mine[i].y;
            if (x > 0.0) {
                s_split = i;
                s_ahead = c;
                if (c + x > target) break;
            }
            c += x;
        }
    }
    __syncthreads();
    const int split = min(s_split, S - 1);
    float p[E];
    double less[E], sum;
    draw_weights<E, VEC>(a, r, left && r < r1 - 1, draft, split * STH * E + tid * E, p, less);
    w = 0.0;
#pragma unroll
    for (int u = 0; u < E; u++) w += less[u];
    double c = s_ahead + (block_scan(w, s_w[1], sum) - w);
    if (tid == max(0, passing_thread(c + w, w, target, s_t[1]))) {
        int first = -1, last = 0;
#pragma unroll
        for (int u = 0; u < E; u++) {
            c += less[u];
            last = less[u] > 0.0 ? u : last;
            first = first < 0 && less[u] > 0.0 && c > target ? u : first;
        }
        s_token = split * STH * E + tid * E + (first >= 0 ? first : last);
    }
    __syncthreads();
    if (tid == 0) {
        a.accepted[s] = r - r0;
        for (int i = r0; i < r; i++) a.tokens[i] = a.draft[i];
        a.tokens[r] = s_token < a.V && all > 0.0 ? (uint32_t)s_token : 0u;
        for (int i = r + 1; i < r1; i++) a.tokens[i] = 0xFFFFFFFFu;
    }
}

// Tokens of a thread in a split: 32 where that still gives every CU a workgroup, else 8
static int verify_e(int n, int V) { return (long long)n * V >= 256ll * STH * 32 ? 32 : 8; }
static int verify_splits(int n, int V) {
    const int e = STH * verify_e(n, V);
    return (V + e - 1) / e;
}

size_t verify_draft_workspace_bytes(int n, int V) {
    return (size_t)n * verify_splits(n, V) * sizeof(double2) + (size_t)n * sizeof(int);
}

int launch_verify_draft(const float* probs, const float* draft_probs, const uint32_t* draft_tokens,
                        const int32_t* row_starts, int n, int n_rows, int V, const float* accept_uniforms,
                        const float* pick_uniforms, int32_t* accepted, uint32_t* tokens, void* ws, size_t ws_bytes,
                        hipStream_t s) {
    QH_REQUIRE(probs && draft_tokens && row_starts && accept_uniforms && pick_uniforms && accepted && tokens && ws,
               QRAF_HIP_ERR_INVALID, "verify_draft: null pointer");
    QH_REQUIRE(n > 0 && n_rows > 0 && V > 0, QRAF_HIP_ERR_INVALID, "verify_draft: %d sequences, %d rows, vocabulary %d",
               n, n_rows, V);
    QH_REQUIRE(((uintptr_t)ws & 15) == 0, QRAF_HIP_ERR_INVALID, "verify_draft: workspace not 16-byte aligned");
    QH_REQUIRE(ws_bytes >= verify_draft_workspace_bytes(n, V), QRAF_HIP_ERR_INVALID,
               "verify_draft: workspace of %zu bytes, %zu needed", ws_bytes, verify_draft_workspace_bytes(n, V));
    QH_REQUIRE(V <= 1 << 30 && n <= 65535, QRAF_HIP_ERR_INVALID,
               "verify_draft: vocabulary %d over 2^30, or %d sequences over 65535", V, n);
    const VerifyArgs a{probs, draft_probs, draft_tokens, row_starts, accept_uniforms, pick_uniforms,
                       accepted, tokens, n, n_rows, V};
    const bool vec = V % 4 == 0 && ((uintptr_t)probs & 15) == 0 && ((uintptr_t)draft_probs & 15) == 0;
    const int e = verify_e(n, V), S = verify_splits(n, V);
    double2* part = (double2*)ws;
    int* decides = (int*)(part + (size_t)n * S);
#define QH_VERIFY(Ev, Vv)                                                                                               \
    if (e == Ev && vec == Vv) {                                                                                         \
        hipLaunchKernelGGL((verify_sums_kernel<Ev, Vv>), dim3(S, n), dim3(STH), 0, s, a, part, decides);                \
        hipLaunchKernelGGL((verify_pick_kernel<Ev, Vv>), dim3(n), dim3(STH), 0, s, a, part, decides, S);                \
    }
    QH_VERIFY(8, true) QH_VERIFY(8, false) QH_VERIFY(32, true) QH_VERIFY(32, false)
#undef QH_VERIFY
    QH_CHECK_HIP(hipGetLastError());
    return QRAF_HIP_OK;
}

}  // namespace qraf_hip

using namespace qraf_hip;

extern "C" {

uint64_t qraf_hip_sample_probs_workspace_bytes(int32_t rows, int32_t vocab) {
    return rows > 0 && vocab > 0 ? sample_probs_workspace_bytes(rows, vocab) : 0;
}

int qraf_hip_sample_probs_dev(float* logits, int32_t rows, int32_t vocab, const qraf_sampling_params* params,
                              const uint32_t* recent, const int32_t* recent_count, int32_t recent_stride, float* probs,
                              void* workspace, uint64_t workspace_bytes, void* stream) {
    clear_error();
    QH_REQUIRE(params, QRAF_HIP_ERR_INVALID, "sample_probs: null parameters");
    return launch_sample_probs(logits, rows, vocab, *params, recent, recent_count, recent_stride, probs, workspace,
                               workspace_bytes, as_stream(stream));
}

uint64_t qraf_hip_verify_draft_workspace_bytes(int32_t n_seqs, int32_t vocab) {
    return n_seqs > 0 && vocab > 0 ? verify_draft_workspace_bytes(n_seqs, vocab) : 0;
}

int qraf_hip_verify_draft_dev(const float* probs, const float* draft_probs, const uint32_t* draft_tokens,
                              const int32_t* row_starts, int32_t n_seqs, int32_t n_rows, int32_t vocab,
                              const float* accept_uniforms, const float* pick_uniforms, int32_t* accepted,
                              uint32_t* tokens, void* workspace, uint64_t workspace_bytes, void* stream) {
    clear_error();
    return launch_verify_draft(probs, draft_probs, draft_tokens, row_starts, n_seqs, n_rows, vocab, accept_uniforms,
                               pick_uniforms, accepted, tokens, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
