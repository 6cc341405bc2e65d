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
// found by radix select over the keys, with counts for top_k and weights for
// top_p.  Weights are summed as integers (w times a power of two that keeps the
// row's sum below 2^62, from a 64-bit exponential): integer sums do not depend
// on the order of the atomics, so results repeat bit for bit, and the border
// of a nucleus whose tokens weigh 1e-6 of the row each is the one of the sums in
// 64-bit floating point.
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

namespace qraf_hip {

constexpr int PNT = 1024;  // threads per row

// a logit as it is ordered and weighed: NaN counts as -inf, -0 as +0
__device__ __forceinline__ float clean_logit(float l) { return l == l ? l + 0.0f : -INFINITY; }

__device__ __forceinline__ uint32_t logit_key(float f) {  // a < b  <=>  key(a) < key(b)
    const uint32_t b = __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// exp((l - m) / T) in 64 bits; m is the largest logit and not -inf
__device__ __forceinline__ double weight64(float l, float m, double T) {
    if (l == m) return 1.0;
    if (l == -INFINITY || m == INFINITY) return 0.0;
    return exp(((double)l - (double)m) / T);
}

__global__ __launch_bounds__(PNT) void probs_rows_kernel(const float* __restrict__ logits, int V, float T, int cutoff,
                                                         float top_p, float* __restrict__ probs) {
    const int tid = threadIdx.x, row = blockIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* l = logits + (size_t)row * V;
    float* p = probs + (size_t)row * V;
    __shared__ float s_f[16];
    __shared__ int s_i[16];
    __shared__ unsigned long long s_hist[256];
    __shared__ unsigned long long s_sum;
    __shared__ uint32_t s_key;
    __shared__ unsigned long long s_need;
    __shared__ int s_cut, s_cnt[PNT];

    // ---- the largest logit and its first index
    float m = -INFINITY;
    int mi = V;
    for (int i = tid; i < V; i += PNT) {
        const float v = clean_logit(l[i]);
        if (v > m) {
            m = v;
            mi = i;
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float om = __shfl_xor(m, o);
        const int oi = __shfl_xor(mi, o);
        if (om > m || (om == m && oi < mi)) {
            m = om;
            mi = oi;
        }
    }
    if (lane == 0) {
        s_f[wave] = m;
        s_i[wave] = mi;
    }
    __syncthreads();
    for (int w = 0; w < 16; w++)
        if (s_f[w] > m || (s_f[w] == m && s_i[w] < mi)) {
            m = s_f[w];
            mi = s_i[w];
        }
    if (m == -INFINITY || !(T > 0.f)) {  // no token, or the first of the largest
        for (int i = tid; i < V; i += PNT) p[i] = i == mi ? 1.f : 0.f;
        return;
    }

    const double t64 = T;
    const double unit = ldexp(1.0, 62 - (32 - __clz(V)));
    auto weigh = [&](float v) { return (unsigned long long)(weight64(v, m, t64) * unit + 0.5); };

    // the kept set: keys above `key`, and of the logits at it those before index `cut`
    uint32_t key = 0;
    int cut = V;
    // among the kept logits, the largest prefix-closed set that falls short of
    // `need` (counts, or weights), as a key and the need left at it
    auto select = [&](bool by_weight, unsigned long long need) {
        uint32_t prefix = 0, mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s_hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += PNT) {
                const float v = clean_logit(l[i]);
                const uint32_t k = logit_key(v);
                if ((k & mask) != prefix || k < key || (k == key && i >= cut)) continue;
                atomicAdd(&s_hist[(k >> shift) & 255u], by_weight ? weigh(v) : 1ull);
            }
            __syncthreads();
            if (tid == 0) {
                unsigned long long acc = 0;
                int d = 255;
                for (; d > 0; d--) {
                    if (acc + s_hist[d] >= need) break;
                    acc += s_hist[d];
                }
                s_key = prefix | ((uint32_t)d << shift);
                s_need = need - acc;
            }
            __syncthreads();
            prefix = s_key;
            need = s_need;
            mask |= 255u << shift;
            __syncthreads();
        }
        // `need` more at key `prefix`: so many of the equal logits
        unsigned long long ties = need;
        if (by_weight) {
            const uint32_t b = (prefix & 0x80000000u) ? (prefix & 0x7FFFFFFFu) : ~prefix;
            const unsigned long long w = weigh(__uint_as_float(b));
            ties = w ? (need + w - 1) / w : (unsigned long long)V;
        }
        // the index behind the ties-th of them
        const int ch = (V + PNT - 1) / PNT, i0 = min(V, tid * ch), i1 = min(V, i0 + ch);
        int c = 0;
        for (int i = i0; i < i1; i++) c += logit_key(clean_logit(l[i])) == prefix;
        s_cnt[tid] = c;
        if (tid == 0) s_cut = V;
        __syncthreads();
        unsigned long long before = 0;
        for (int t = 0; t < tid; t++) before += s_cnt[t];
        if (before < ties && before + c >= ties) {
            int i = i0;
            for (; before < ties; i++) before += logit_key(clean_logit(l[i])) == prefix;
            s_cut = i;
        }
        __syncthreads();
        cut = prefix == key ? min(cut, s_cut) : s_cut;
        key = prefix;
        __syncthreads();
    };
    auto total = [&]() {  // the kept set's weight
        if (tid == 0) s_sum = 0;
        __syncthreads();
        unsigned long long z = 0;
        for (int i = tid; i < V; i += PNT) {
            const float v = clean_logit(l[i]);
            const uint32_t k = logit_key(v);
            if (k > key || (k == key && i < cut)) z += weigh(v);
        }
        atomicAdd(&s_sum, z);
        __syncthreads();
        z = s_sum;
        __syncthreads();
        return z;
    };
    if (cutoff < V) select(false, (unsigned long long)cutoff);
    unsigned long long z = total();
    if (top_p > 0.f && top_p < 1.f) {
        const double need = ceil((double)z * (double)top_p);
        select(true, max(1ull, (unsigned long long)need));
        z = total();
    }
    const double inv = unit / (double)z;
    for (int i = tid; i < V; i += PNT) {
        const float v = clean_logit(l[i]);
        const uint32_t k = logit_key(v);
        p[i] = k > key || (k == key && i < cut) ? (float)(weight64(v, m, t64) * inv) : 0.f;
    }
}

size_t sample_probs_workspace_bytes(int rows, int V) {
    (void)rows;
    (void)V;
    return 16;
}

int launch_sample_probs(float* logits, int rows, int V, const qraf_sampling_params& sp, const uint32_t* recent,
                        const int32_t* counts, int stride, float* probs, void* ws, size_t ws_bytes, hipStream_t s) {
    QH_REQUIRE(logits && probs && ws && rows > 0 && V > 0, QRAF_HIP_ERR_INVALID, "sample_probs: bad arguments");
    QH_REQUIRE(ws_bytes >= sample_probs_workspace_bytes(rows, V), QRAF_HIP_ERR_INVALID,
               "sample_probs: workspace of %zu bytes, %zu needed", ws_bytes, sample_probs_workspace_bytes(rows, V));
    QH_TRY(launch_penalty(logits, rows, V, sp.repetition_penalty, recent, counts, stride, s));
    const int cutoff = (sp.top_k > 0 && sp.top_k < V) ? sp.top_k : V;
    hipLaunchKernelGGL(probs_rows_kernel, dim3(rows), dim3(PNT), 0, s, logits, V, sp.temperature, cutoff, sp.top_p,
                       probs);
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

// weight of token t in the draw of row r
__device__ __forceinline__ double draw_weight(const VerifyArgs& a, size_t r, int t, int mode, uint32_t x) {
    const double p = a.p[r * a.V + t];
    if (mode == 0) return p;
    if (mode == 1) return (uint32_t)t == x ? 0.0 : p;
    return fmax(p - (double)a.q[r * a.V + t], 0.0);
}

__global__ __launch_bounds__(PNT) void verify_kernel(VerifyArgs a) {
    const int s = blockIdx.x, tid = threadIdx.x;
    __shared__ double s_part[PNT];
    __shared__ int s_row, s_token;
    const int r0 = max(0, min(a.row_starts[s], a.n_rows)), r1 = max(r0, min(a.row_starts[s + 1], a.n_rows));
    if (r1 == r0) {  // a sequence without rows
        if (tid == 0) a.accepted[s] = 0;
        return;
    }
    if (tid == 0) {
        int r = r0;
        for (; r < r1 - 1; r++) {
            const uint32_t x = a.draft[r];
            if (x >= (uint32_t)a.V) break;
            const double q = a.q ? (double)a.q[(size_t)r * a.V + x] : 1.0;
            if (!((double)a.u[r] * q < (double)a.p[(size_t)r * a.V + x])) break;
        }
        s_row = r;
        s_token = a.V;
    }
    __syncthreads();
    const int r = s_row;
    const uint32_t x = a.draft[r];
    int mode = r < r1 - 1 ? (a.q ? 2 : 1) : 0;
    const int ch = (a.V + PNT - 1) / PNT, i0 = min(a.V, tid * ch), i1 = min(a.V, i0 + ch);
    double all = 0.0, before = 0.0;
    for (int round = 0; round < 2; round++) {
        double w = 0.0;
        for (int i = i0; i < i1; i++) w += draw_weight(a, r, i, mode, x);
        s_part[tid] = w;
        __syncthreads();
        all = before = 0.0;
        for (int t = 0; t < PNT; t++) {
            if (t == tid) before = all;
            all += s_part[t];
        }
        __syncthreads();
        if (all > 0.0 || mode == 0) break;
        mode = 0;  // nothing left of p: the target's own distribution
    }
    // a draw outside [0, 1) (or NaN) takes the nearest inside
    const double target = (double)fminf(fmaxf(a.v[s], 0.f), 0x1.fffffep-1f) * all;
    int mine = a.V;
    double c = before;
    for (int i = i0; i < i1; i++) {
        c += draw_weight(a, r, i, mode, x);
        if (c > target) {
            mine = i;
            break;
        }
    }
    atomicMin(&s_token, mine);
    __syncthreads();
    if (tid == 0) {
        a.accepted[s] = r - r0;
        for (int i = r0; i < r; i++) a.tokens[i] = a.draft[i];
        a.tokens[r] = s_token < a.V ? (uint32_t)s_token : 0u;
        for (int i = r + 1; i < r1; i++) a.tokens[i] = 0xFFFFFFFFu;
    }
}

size_t verify_draft_workspace_bytes(int n, int V) {
    (void)n;
    (void)V;
    return 16;
}

int launch_verify_draft(const float* probs, const float* draft_probs, const uint32_t* draft_tokens,
                        const int32_t* row_starts, int n, int n_rows, int V, const float* accept_uniforms,
                        const float* pick_uniforms, int32_t* accepted, uint32_t* tokens, void* ws, size_t ws_bytes,
                        hipStream_t s) {
    QH_REQUIRE(probs && draft_tokens && row_starts && accept_uniforms && pick_uniforms && accepted && tokens && ws,
               QRAF_HIP_ERR_INVALID, "verify_draft: null pointer");
    QH_REQUIRE(n > 0 && n_rows > 0 && V > 0, QRAF_HIP_ERR_INVALID, "verify_draft: %d sequences, %d rows, vocabulary %d",
               n, n_rows, V);
    QH_REQUIRE(ws_bytes >= verify_draft_workspace_bytes(n, V), QRAF_HIP_ERR_INVALID,
               "verify_draft: workspace of %zu bytes, %zu needed", ws_bytes, verify_draft_workspace_bytes(n, V));
    const VerifyArgs a{probs, draft_probs, draft_tokens, row_starts, accept_uniforms, pick_uniforms,
                       accepted, tokens, n, n_rows, V};
    hipLaunchKernelGGL(verify_kernel, dim3(n), dim3(PNT), 0, s, a);
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
