// logprobs.hip -- what a server says about a token beside it: the log probability
// and rank of given tokens, the entropy of their distributions, the top alternatives.
//
// Of a row l of V logits, with m the largest, d_i = l_i - m and S = sum exp(d_i):
//   log probability   d_t - ln S of the row's given token t
//   rank              how many tokens are ahead of t: larger logits, and equal ones of
//                     lower index
//   entropy           ln S - (1 / S) sum exp(d_i) d_i
//   alternatives      the n tokens ahead of all others, and d_i - ln S of each
// NaN counts as -inf, -0 as +0.  Of infinite logits each has the same share; a row
// without a logit above -inf has log probabilities of -inf and entropy 0.
//
// The logits are read once, by many workgroups a row; nothing else is large.  A wave
// holds E logits a lane and writes its maximum, its sums against that, and how many of
// its tokens are ahead; for alternatives every lane also writes the largest of its own
// (a sub-range).  A second launch, a workgroup a row (a wave without alternatives), joins
// the sums in 64 bits and finds the alternatives: the n-th largest of 512 maxima bounds
// the n-th logit from below, only sub-ranges that reach the bound are read again, and the
// few logits that do are ordered by counting.  Rows of up to 8,192 logits take one
// workgroup and one launch.  Rows with more equal logits at the border than the lists
// hold take a search over the whole row (flat_tops).
// Measured: 512 rows of 151,936 (311 MB) 55.6 us, 5.6 TB/s; 160 rows with 20 alternatives (97 MB) 24.1, of which the
// pass 17 and the join 6.3; 8 rows of 49,152 with 4 7.6.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "logits.h"
#include "wave.h"

namespace qraf_hip {

constexpr int TOP_MAX = 64;
constexpr int STH = 256;        // threads of a split
constexpr int JTH = 512;        // threads that join a row
constexpr int SPLITS = 64;      // splits of a row at most: longer rows give them several chunks
constexpr int SUBS = 128;       // sub-ranges that a wave reads again, at most
constexpr int LIST = 2816;      // candidates: what the lanes that reach a bound of 64 hold, of 32 logits each
constexpr uint32_t KEY_NONE = 0x007FFFFFu;  // logit_key of -inf

struct WaveStats {
    float m, s, e;  // the largest logit, sum exp(l - m), sum exp(l - m) (l - m)
    int ahead;      // tokens ahead of the row's given one
};
struct LogprobArgs {
    const float* logits;
    const uint32_t* tokens;
    float *logprobs, *entropies, *top_logprobs;
    int32_t* ranks;
    uint32_t* top_tokens;
    WaveStats* stats;  // [rows][S * 4]
    float* sub;        // [rows][S * STH] largest logits of sub-ranges
    int V, S, top, rows;
};

// tokens in their order: a is ahead of b  <=>  key(a) > key(b)
__device__ __forceinline__ unsigned long long token_key(uint32_t key, int i) {
    return (unsigned long long)key << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float add2(float x, float y) { return x + y; }
__device__ __forceinline__ int iadd2(int x, int y) { return x + y; }
__device__ __forceinline__ float max2(float x, float y) { return fmaxf(x, y); }
__device__ __forceinline__ uint32_t umax2(uint32_t x, uint32_t y) { return max(x, y); }
__device__ __forceinline__ uint32_t umin2(uint32_t x, uint32_t y) { return min(x, y); }

// 16 bytes of a row, whose alignment is that of a float
struct __attribute__((packed, aligned(4))) Four {
    float v[4];
};
// Chunk c of a row, E logits of TH threads each: element u is index chunk_index(c, u); past the row -inf.
template <int E, int TH = STH>
__device__ __forceinline__ int chunk_index(int c, int t, int u) {
    return c * (TH * E) + 4 * (t + TH * (u >> 2)) + (u & 3);
}
template <int E, int TH = STH>
__device__ __forceinline__ void load_chunk(const float* l, int V, int c, float (&v)[E]) {
    const int t = threadIdx.x;
    if ((c + 1) * (TH * E) <= V) {
#pragma unroll
        for (int j = 0; j < E; j += 4) {
            const Four x = *(const Four*)(l + chunk_index<E, TH>(c, t, j));
#pragma unroll
            for (int k = 0; k < 4; k++) v[j + k] = x.v[k];
        }
    } else if (V >= 4) {
        // (A row's last chunk one logit at a time took four times its loads: 512 rows of 128,256 logits 57 us, so 50.)
        const int end = V & ~3, rest = V & 3;
        float last[3];
#pragma unroll
        for (int k = 0; k < 3; k++) last[k] = l[min(end + k, V - 1)];
#pragma unroll
        for (int j = 0; j < E; j += 4) {
            const int i = chunk_index<E, TH>(c, t, j);
            const Four x = *(const Four*)(l + min(i, V - 4));
#pragma unroll
            for (int k = 0; k < 4; k++) v[j + k] = i < end ? x.v[k] : k < rest && i == end ? last[k % 3] : -INFINITY;
        }
    } else {
#pragma unroll
        for (int u = 0; u < E; u++) {
            const int i = chunk_index<E, TH>(c, t, u);
            const float x = l[min(i, V - 1)];
            v[u] = i < V ? x : -INFINITY;
        }
    }
}

// sums of exp(v - m) and of that times (v - m), by halves: a chain of log2(E) additions.  Below m - 200, and of -inf and
// NaN, nothing is left of either.
template <int E>
__device__ __forceinline__ float2 weights(const float* v, float m) {
    if constexpr (E == 1) {
        const float d = fmaxf(v[0] - m, -200.f), w = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
        return make_float2(w, w * d);
    } else {
        const float2 x = weights<E / 2>(v, m), y = weights<E / 2>(v + E / 2, m);
        return make_float2(x.x + y.x, x.y + y.y);
    }
}

// A wave's statistics of its part of a chunk; mine: the lane's largest.
template <int E, int TH = STH>
__device__ __forceinline__ WaveStats wave_stats(const float (&v)[E], int c, uint32_t token, float given, float& mine) {
    mine = -INFINITY;
#pragma unroll
    for (int u = 0; u < E; u++) mine = v[u] > mine ? v[u] : mine;  // (a NaN of either kind is none)
    WaveStats w;
    w.m = over_wave(mine, max2);
    float2 s = make_float2(0.f, 0.f);
    if (fabsf(w.m) < INFINITY) {
        s = weights<E>(v, w.m);
    } else if (w.m == INFINITY) {
#pragma unroll
        for (int u = 0; u < E; u++) s.x += v[u] == INFINITY ? 1.f : 0.f;
    }
    w.s = over_wave(s.x, add2);
    w.e = over_wave(s.y, add2);
    // a larger logit is ahead, an equal one where it lies ahead
    int ahead = 0;
    const long long first = (long long)c * (TH * E), end = first + TH * E;
    if (given == -INFINITY || (token >= first && token < end)) {
        const unsigned long long key = token_key(logit_key(given), (int)token);
#pragma unroll
        for (int u = 0; u < E; u++) {
            const int i = chunk_index<E, TH>(c, threadIdx.x, u);
            ahead += token_key(logit_key(clean_logit(v[u])), i) > key;
        }
    } else if (token < first) {
#pragma unroll
        for (int u = 0; u < E; u++) ahead += v[u] > given;
    } else {
#pragma unroll
        for (int u = 0; u < E; u++) ahead += v[u] >= given;
    }
    w.ahead = over_wave(ahead, iadd2);
    return w;
}
// Sums of several of them against the largest of their maxima, in 64 bits.
struct RunStats {
    float m = -INFINITY;
    double s = 0.0, e = 0.0;
    int ahead = 0;
    // (m: at least w's)
    __device__ __forceinline__ void add(const WaveStats& w) {
        const double f = weight64(w.m, m, 1.0);
        if (f > 0.0 && w.m > -INFINITY) {
            const double d = w.m == m ? 0.0 : (double)w.m - (double)m;
            s += f * w.s;
            e += f * (w.e + d * w.s);
        }
        ahead += w.ahead;
    }
    __device__ __forceinline__ void follow(float to) {
        if (to > m) {
            const double f = weight64(m, to, 1.0);
            e = f > 0.0 ? f * (e + ((double)m - (double)to) * s) : 0.0;
            s *= f;
            m = to;
        }
    }
};

// the row's token: its logit as it is ordered (+inf of one outside the vocabulary: nothing is ahead of it)
__device__ __forceinline__ float given_logit(const LogprobArgs& a, int row, uint32_t token) {
    return token < (uint32_t)a.V ? clean_logit(a.logits[(size_t)row * a.V + token]) : INFINITY;
}
__device__ __forceinline__ uint32_t given_token(const LogprobArgs& a, int row) {
    return a.tokens ? a.tokens[row] : 0xFFFFFFFFu;
}

struct RowSums {
    float m;
    double log_s;
    __device__ __forceinline__ float logprob(float x) const {
        if (m == -INFINITY) return -INFINITY;
        return x == m ? (float)-log_s : (float)((double)x - (double)m - log_s);
    }
};
// A row's sums from those of n waves, by a wave; its outputs but the alternatives.  mine: st[lane], requested ahead.
__device__ __forceinline__ WaveStats lane_stats(const WaveStats* st, int n) {
    const int lane = threadIdx.x & 63;
    return lane < n ? st[lane] : WaveStats{-INFINITY, 0.f, 0.f, 0};
}
__device__ __forceinline__ RowSums row_sums(const LogprobArgs& a, int row, const WaveStats* st, int n,
                                            const WaveStats& mine, uint32_t token, float given) {
    const int lane = threadIdx.x & 63;
    RowSums r;
    float m = mine.m;
    for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, st[i].m);
    RunStats run;
    run.m = r.m = over_wave(m, max2);
    for (int i = lane; i < n; i += 64) run.add(i == lane ? mine : st[i]);
    const double s = wave_sum64(run.s), e = wave_sum64(run.e);
    const int ahead = over_wave(run.ahead, iadd2);
    r.log_s = log(s);
    if (lane == 0) {
        const bool known = token < (uint32_t)a.V;
        if (a.logprobs) a.logprobs[row] = known ? r.logprob(given) : -INFINITY;
        if (a.ranks) a.ranks[row] = known ? ahead : -1;
        if (a.entropies) a.entropies[row] = r.m == -INFINITY ? 0.f : (float)(r.log_s - e / s);
    }
    return r;
}

// ---- alternatives
// (of TH threads)
template <int TH>
struct TopShared {
    unsigned long long list[LIST];
    uint32_t key[TH];
    int cnt[8], wave[TH / 64], n;
};

// Of TH keys a bound that at least `need` of them, and not many more, reach; by each wave for itself.
template <int TH>
__device__ __forceinline__ uint32_t bound_of(const uint32_t* keys, int need) {
    const int lane = threadIdx.x & 63;
    uint32_t k[TH / 64], lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
    for (int u = 0; u < TH / 64; u++) {
        k[u] = keys[lane + 64 * u];
        lo = min(lo, k[u]);
        hi = max(hi, k[u]);
    }
    lo = __builtin_amdgcn_readfirstlane(over_wave(lo, umin2));
    hi = __builtin_amdgcn_readfirstlane(over_wave(hi, umax2));
    int reach = TH;
    while (lo < hi && reach > need + (need >> 2) + 4) {
        const uint32_t mid = lo + ((hi - lo) >> 1) + 1;
        int c = 0;
#pragma unroll
        for (int u = 0; u < TH / 64; u++) c += __popcll(__ballot(k[u] >= mid));
        if (c >= need) {
            lo = mid;
            reach = c;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// The alternatives of a row by search: the n-th largest key three bits at a time, then the logits above it and the
// first of those at it.  Leaves all of them in the list.
template <int TH>
__device__ void flat_tops(const LogprobArgs& a, const float* l, TopShared<TH>& sh) {
    const int tid = threadIdx.x, lane = tid & 63, V = a.V, need = a.top;
    uint32_t at = 0;
    for (int shift = 29; shift >= 0; shift = shift == 2 ? 0 : shift - 3) {
        const int digits = shift ? 8 : 4;
        if (tid < 8) sh.cnt[tid] = 0;
        __syncthreads();
        int c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int i = tid; i < V; i += TH) {
            const uint32_t k = logit_key(clean_logit(l[i]));
#pragma unroll
            for (int j = 1; j < 8; j++) c[j] += j < digits && k >= at + ((uint32_t)j << shift);
        }
#pragma unroll
        for (int j = 1; j < 8; j++) {
            const int x = over_wave(c[j], iadd2);
            if (lane == 0) atomicAdd(&sh.cnt[j], x);
        }
        __syncthreads();
        int best = 0;
#pragma unroll
        for (int j = 1; j < 8; j++)
            if (j < digits && sh.cnt[j] >= need) best = j;
        at += (uint32_t)best << shift;
        __syncthreads();
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    for (int i = tid; i < V; i += TH) {  // fewer than `need`
        const uint32_t k = logit_key(clean_logit(l[i]));
        if (k > at) sh.list[atomicAdd(&sh.n, 1)] = token_key(k, i);
    }
    __syncthreads();
    for (int base = 0; base < V; base += TH) {
        const int i = base + tid;
        const bool is = i < V && logit_key(clean_logit(l[min(i, V - 1)])) == at;
        const unsigned long long b = __ballot(is);
        if (lane == 0) sh.wave[tid >> 6] = __popcll(b);
        __syncthreads();
        int before = sh.n, all = before;
#pragma unroll
        for (int w = 0; w < TH / 64; w++) {
            before += w < tid >> 6 ? sh.wave[w] : 0;
            all += sh.wave[w];
        }
        before += __popcll(b & ((1ull << lane) - 1));
        if (is && before < need) sh.list[before] = token_key(at, i);
        __syncthreads();
        if (tid == 0) sh.n = min(all, need);
        __syncthreads();
        if (all >= need) break;
    }
}

// The alternatives from the candidates in the list (`over`: there were more than it holds, or than could be read
// again), in order; where fewer logits than that are above -inf, the first of the others behind them.
template <int TH>
__device__ void write_tops(const LogprobArgs& a, int row, const float* l, TopShared<TH>& sh, bool over, const RowSums& r) {
    const int tid = threadIdx.x;
    if (over) flat_tops(a, l, sh);
    const int n = sh.n;
    uint32_t* tokens = a.top_tokens + (size_t)row * a.top;
    float* lps = a.top_logprobs + (size_t)row * a.top;
    for (int i = tid; i < n; i += TH) {
        const unsigned long long x = sh.list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += sh.list[j] > x;
        if (rank < a.top) {
            tokens[rank] = 0xFFFFFFFFu - (uint32_t)x;
            lps[rank] = r.logprob(key_logit((uint32_t)(x >> 32)));
        }
    }
    if (n < a.top && tid < 64) {
        int at = n;
        for (int base = 0; at < a.top && base < a.V; base += 64) {
            const int i = base + tid;
            const bool none = i < a.V && clean_logit(l[min(i, a.V - 1)]) == -INFINITY;
            const unsigned long long b = __ballot(none);
            const int rank = at + __popcll(b & ((1ull << tid) - 1));
            if (none && rank < a.top) {
                tokens[rank] = i;
                lps[rank] = -INFINITY;
            }
            at += __popcll(b);
        }
    }
}

// ---- rows of up to TH * E logits: one workgroup, and with alternatives a wave more for the sums
template <int E, int TH>
__global__ __launch_bounds__(TH + 64) void logprobs_small_kernel(LogprobArgs a) {
    __shared__ TopShared<TH + 64> sh;
    __shared__ WaveStats s_st[TH / 64];
    __shared__ RowSums s_r;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const float* l = a.logits + (size_t)row * a.V;
    const uint32_t token = given_token(a, row);
    if (tid >= TH) {
        const float given = given_logit(a, row, token);
        __syncthreads();
        const RowSums r = row_sums(a, row, s_st, TH / 64, lane_stats(s_st, TH / 64), token, given);
        if (tid == TH) s_r = r;
        __syncthreads();
    } else {
        float v[E], mine;
        load_chunk<E, TH>(l, a.V, 0, v);
        const float given = given_logit(a, row, token);
        const WaveStats w = wave_stats<E, TH>(v, 0, token, given, mine);
        if (lane == 0) s_st[tid >> 6] = w;
        sh.key[tid] = logit_key(mine + 0.f);
        if (tid == 0) sh.n = 0;
        __syncthreads();
        if (a.top == 0) {  // (without the wave more)
            if (tid < 64) row_sums(a, row, s_st, TH / 64, lane_stats(s_st, TH / 64), token, given);
            return;
        }
        const uint32_t bound = max(bound_of<TH>(sh.key, a.top), KEY_NONE + 1);
        if (__any(sh.key[tid] >= bound)) {
            uint32_t key[E];
            int all = 0;
#pragma unroll
            for (int u = 0; u < E; u++) {
                key[u] = logit_key(clean_logit(v[u]));
                all += __popcll(__ballot(key[u] >= bound));
            }
            int at = 0;
            if (lane == 0) at = atomicAdd(&sh.n, all);
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int u = 0; u < E; u++) {
                const unsigned long long b = __ballot(key[u] >= bound);
                if (!b) continue;
                const int x = at + __popcll(b & ((1ull << lane) - 1));
                if (key[u] >= bound && x < LIST) sh.list[x] = token_key(key[u], chunk_index<E, TH>(0, tid, u));
                at += __popcll(b);
            }
        }
        __syncthreads();
    }
    const bool over = sh.n > LIST;
    __syncthreads();
    write_tops(a, row, l, sh, over, s_r);
}

// ---- longer rows: their splits, then a row's join
template <int E>
__global__ __launch_bounds__(STH) void logprobs_split_kernel(LogprobArgs a) {
    const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x;
    const float* l = a.logits + (size_t)row * a.V;
    const uint32_t token = given_token(a, row);
    const int chunks = (a.V + STH * E - 1) / (STH * E);
    float v[E], most;
    load_chunk<E>(l, a.V, split, v);
    const float given = given_logit(a, row, token);
    WaveStats w = wave_stats<E>(v, split, token, given, most);
    if (chunks > a.S) {  // (for all workgroups)
        RunStats run;
        run.m = w.m;
        run.add(w);
        for (int c = split + a.S; c < chunks; c += a.S) {
            float mine;
            load_chunk<E>(l, a.V, c, v);
            w = wave_stats<E>(v, c, token, given, mine);
            run.follow(w.m);
            run.add(w);
            most = fmaxf(most, mine);
        }
        w = WaveStats{run.m, (float)run.s, (float)run.e, run.ahead};
    }
    if ((tid & 63) == 0) a.stats[((size_t)row * a.S + split) * (STH / 64) + (tid >> 6)] = w;
    if (a.top) a.sub[((size_t)row * a.S + split) * STH + tid] = most;
}

__global__ __launch_bounds__(STH) void logprobs_sums_kernel(LogprobArgs a) {
    const int row = blockIdx.x * (STH / 64) + (threadIdx.x >> 6), n = a.S * (STH / 64);
    if (row >= a.rows) return;
    const WaveStats* st = a.stats + (size_t)row * n;
    const WaveStats mine = lane_stats(st, n);
    const uint32_t token = given_token(a, row);
    row_sums(a, row, st, n, mine, token, given_logit(a, row, token));
}

// A wave more than the maxima's for the sums, which nothing waits for but the log probabilities of the alternatives.
// The others keep their sub-ranges to themselves up to the candidates: two barriers.  R: maxima a thread holds, all
// requested at once.  Cycles of a row of 151,936, 20 alternatives: maxima 2,800 (a read of what another launch wrote),
// barrier 500, bound 1,600, list 800, second read 2,400, barriers 1,300, order and output 2,000: 11,500.  (20,000 with one
// list of sub-ranges by atomics, maxima requested one after another and the sums by one of these waves.)
template <int E, int R>
__global__ __launch_bounds__(JTH + 64) void logprobs_tops_kernel(LogprobArgs a) {
    __shared__ TopShared<JTH + 64> sh;
    __shared__ int s_subs[JTH / 64][SUBS];
    __shared__ RowSums s_r;
    const int row = blockIdx.x, tid = threadIdx.x, n_sub = a.S * STH, waves = a.S * (STH / 64), V = a.V;
    const float* l = a.logits + (size_t)row * V;
    if (tid >= JTH) {
        const WaveStats* st = a.stats + (size_t)row * waves;
        const WaveStats stats = lane_stats(st, waves);
        const uint32_t token = given_token(a, row);
        const float given = given_logit(a, row, token);
        __syncthreads();
        const RowSums r = row_sums(a, row, st, waves, stats, token, given);
        if (tid == JTH) s_r = r;
        __syncthreads();
    } else {
        const float* sub = a.sub + (size_t)row * n_sub;
        float x[R];
#pragma unroll
        for (int u = 0; u < R; u++) x[u] = sub[min(tid + JTH * u, n_sub - 1)];
        uint32_t mine[R], most = 0;
#pragma unroll
        for (int u = 0; u < R; u++) {
            mine[u] = tid + JTH * u < n_sub ? logit_key(x[u] + 0.f) : 0;
            most = max(most, mine[u]);
        }
        sh.key[tid] = most;
        if (tid == 0) sh.n = 0;
        __syncthreads();
        const uint32_t bound = max(bound_of<JTH>(sh.key, a.top), KEY_NONE + 1);
        const int lane = tid & 63;
        int *const subs = s_subs[tid >> 6], ns = 0;
#pragma unroll
        for (int u = 0; u < R; u++) {
            const unsigned long long b = __ballot(mine[u] >= bound);
            if (!b) continue;  // (nearly always)
            const int at = ns + __popcll(b & ((1ull << lane) - 1));
            if (mine[u] >= bound && at < SUBS) subs[at] = tid + JTH * u;
            ns += __popcll(b);
        }
        __builtin_amdgcn_wave_barrier();  // (of one wave: its writes are in order with its reads)
        const int chunks = (V + STH * E - 1) / (STH * E), per = (chunks + a.S - 1) / a.S * (E / 4);
        if (ns > SUBS && lane == 0) atomicAdd(&sh.n, LIST + 1);
        for (int w0 = 0; w0 < (ns <= SUBS ? ns * per : 0); w0 += 64) {
            const int w = w0 + lane, in = min(w, ns * per - 1), y = subs[in / per], rest = in % per;
            const int i0 = chunk_index<E>(y / STH + rest / (E / 4) * a.S, y % STH, 4 * (rest % (E / 4)));
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = l[min(i0 + k, V - 1)];
            uint32_t key[4];
            int at[4], all = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                key[k] = w == in && i0 + k < V ? logit_key(clean_logit(v[k])) : 0;
                const unsigned long long b = __ballot(key[k] >= bound);
                at[k] = all + __popcll(b & ((1ull << lane) - 1));
                all += __popcll(b);
            }
            int first = 0;
            if (lane == 0) first = atomicAdd(&sh.n, all);
            first = __builtin_amdgcn_readfirstlane(first);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (key[k] >= bound && first + at[k] < LIST) sh.list[first + at[k]] = token_key(key[k], i0 + k);
        }
        __syncthreads();
    }
    const bool over = sh.n > LIST;
    __syncthreads();
    write_tops(a, row, l, sh, over, s_r);
}

// Splits of 32 logits a thread, or of 8, which reach more CUs with fewer rows and leave less of a short row's last split
// empty, but take a row past 131,072 in turns.  Of 8 against of 32, us, 20 alternatives: 8 rows of 32,000 / 49,152 /
// 80,000 / 128,256 / 151,936 logits 8.1 / 8.2 / 9.6 / 10.2 / 11.5 against 9.5 / 8.7 / 9.6 / 9.7 / 9.7; 128 rows 11.6 /
// 12.9 / 16.5 / 20.9 / 28.9 against 12.4 / 13.2 / 15.9 / 19.4 / 20.9; 512 rows 20.3 / 28.5 / 44.4 / 64.8 / 83.8 against
// 20.8 / 25.5 / 38.3 / 58.3 / 64.3.  100,003 logits: of 32 from the first row on (9.3 against 10.0).
constexpr int WIDE = 3 << 15, NARROW = 40000, WIDE_ALL = 1 << 23;  // logits of a row, of a row, of a call
static bool wide_splits(int rows, int V) {
    return V >= WIDE || (V >= NARROW && (long long)rows * V >= WIDE_ALL);
}
static int splits_of(int rows, int V) {
    const int per = STH * (wide_splits(rows, V) ? 32 : 8);
    return std::min(SPLITS, (V + per - 1) / per);
}
// Logits of a row that one workgroup takes.  8 rows of 8,000, 20 alternatives: 7.8 us where splits take 8.3; 512 rows 10.7
// and 15.0.  (Up to 2,048 by 256 threads: 1,000 logits 4.9 where 512 take 5.2.)
constexpr int SMALL = STH * 32;

size_t token_logprobs_workspace_bytes(int rows, int V, int top) {
    if (V <= SMALL) return 16;
    auto bytes = [&](size_t n) { return n * splits_of((int)n, V) * ((STH / 64) * sizeof(WaveStats) + (top ? STH * 4 : 0)); };
    // never less than of fewer rows, whose splits may be more
    const int narrow = V >= NARROW && V < WIDE ? std::min(rows, (WIDE_ALL - 1) / V) : rows;
    return std::max(bytes(rows), bytes(narrow));
}

int launch_token_logprobs(const float* logits, int rows, int V, const uint32_t* tokens, float* logprobs, int32_t* ranks,
                          float* entropies, int top, uint32_t* top_tokens, float* top_logprobs, void* ws,
                          size_t ws_bytes, hipStream_t s) {
    QH_REQUIRE(logits && ws, QRAF_HIP_ERR_INVALID, "token_logprobs: null pointer");
    QH_REQUIRE(rows > 0 && rows <= 65535 && V > 0 && V <= 1 << 30, QRAF_HIP_ERR_INVALID,
               "token_logprobs: %d rows of %d logits", rows, V);
    QH_REQUIRE(tokens || (!logprobs && !ranks), QRAF_HIP_ERR_INVALID,
               "token_logprobs: log probabilities and ranks need tokens");
    QH_REQUIRE(top >= 0 && top <= TOP_MAX && top <= V, QRAF_HIP_ERR_INVALID,
               "token_logprobs: %d alternatives (at most %d, and the vocabulary)", top, TOP_MAX);
    QH_REQUIRE(top == 0 || (top_tokens && top_logprobs), QRAF_HIP_ERR_INVALID,
               "token_logprobs: %d alternatives need their tokens and log probabilities", top);
    QH_REQUIRE(((uintptr_t)ws & 15) == 0, QRAF_HIP_ERR_INVALID, "token_logprobs: the workspace must be 16-byte aligned");
    const size_t need = token_logprobs_workspace_bytes(rows, V, top);
    QH_REQUIRE(ws_bytes >= need, QRAF_HIP_ERR_INVALID, "token_logprobs: workspace of %zu bytes, %zu needed", ws_bytes,
               need);
    LogprobArgs a{logits, tokens, logprobs, entropies, top_logprobs, ranks, top_tokens, nullptr, nullptr, V, 1, top, rows};
    if (V <= SMALL) {
        const int more = top ? 64 : 0;
        if (V <= STH * 8) hipLaunchKernelGGL((logprobs_small_kernel<8, STH>), dim3(rows), dim3(STH + more), 0, s, a);
        else hipLaunchKernelGGL((logprobs_small_kernel<16, 512>), dim3(rows), dim3(512 + more), 0, s, a);
        QH_CHECK_HIP(hipGetLastError());
        return QRAF_HIP_OK;
    }
    a.S = splits_of(rows, V);
    a.stats = (WaveStats*)ws;
    a.sub = (float*)(a.stats + (size_t)rows * a.S * (STH / 64));
    const bool wide = wide_splits(rows, V);
    if (wide) hipLaunchKernelGGL(logprobs_split_kernel<32>, dim3(a.S, rows), dim3(STH), 0, s, a);
    else hipLaunchKernelGGL(logprobs_split_kernel<8>, dim3(a.S, rows), dim3(STH), 0, s, a);
    QH_CHECK_HIP(hipGetLastError());
    if (!top)
        hipLaunchKernelGGL(logprobs_sums_kernel, dim3((rows + STH / 64 - 1) / (STH / 64)), dim3(STH), 0, s, a);
    else {
#define QH_TOPS(Ev, Rv) hipLaunchKernelGGL((logprobs_tops_kernel<Ev, Rv>), dim3(rows), dim3(JTH + 64), 0, s, a)
        const int per = (a.S * STH + JTH - 1) / JTH;
        if (wide) {
            if (per <= 4) QH_TOPS(32, 4);
            else if (per <= 12) QH_TOPS(32, 12);
            else QH_TOPS(32, 32);
        } else {
            if (per <= 4) QH_TOPS(8, 4);
            else if (per <= 12) QH_TOPS(8, 12);
            else QH_TOPS(8, 32);
        }
#undef QH_TOPS
    }
    QH_CHECK_HIP(hipGetLastError());
    return QRAF_HIP_OK;
}

}  // namespace qraf_hip

using namespace qraf_hip;

extern "C" {

uint64_t qraf_hip_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top) {
    if (rows <= 0 || vocab <= 0 || top < 0) return 0;
    return token_logprobs_workspace_bytes(rows, vocab, top);
}

int qraf_hip_token_logprobs_dev(const float* logits, int32_t rows, int32_t vocab, const uint32_t* tokens,
                                float* logprobs, int32_t* ranks, float* entropies, int32_t top, uint32_t* top_tokens,
                                float* top_logprobs, void* workspace, uint64_t workspace_bytes, void* stream) {
    clear_error();
    return launch_token_logprobs(logits, rows, vocab, tokens, logprobs, ranks, entropies, top, top_tokens, top_logprobs,
                                 workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
