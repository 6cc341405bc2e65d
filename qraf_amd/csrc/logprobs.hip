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
#include <math.h>

#include <algorithm>

#include "common.h"

namespace qraf_hip {

constexpr int LTH = 1024;  // threads of a row
constexpr int TOP_MAX = 64;

struct LogprobArgs {
    const float* logits;
    const uint32_t* tokens;
    float *logprobs, *entropies, *top_logprobs;
    int32_t* ranks;
    uint32_t* top_tokens;
    int V, top;
};

// tokens in their order: a is ahead of b  <=>  key(a) > key(b)
__device__ __forceinline__ unsigned long long token_key(float clean, int i) {
    return (unsigned long long)logit_key(clean) << 32 | (0xFFFFFFFFu - (uint32_t)i);
}

template <typename T, typename F>
__device__ __forceinline__ T block_all(T x, F op, T* s) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = op(x, __shfl_xor(x, o));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s[0];
    for (int w = 1; w < LTH / 64; w++) x = op(x, s[w]);
    __syncthreads();
    return x;
}

__global__ __launch_bounds__(LTH) void logprobs_row_kernel(LogprobArgs a) {
    __shared__ unsigned long long s_k[LTH / 64];
    __shared__ double s_d[LTH / 64];
    __shared__ int s_i[LTH / 64];
    const int row = blockIdx.x, tid = threadIdx.x, V = a.V;
    const float* l = a.logits + (size_t)row * V;
    auto most = [](unsigned long long x, unsigned long long y) { return max(x, y); };
    auto sum = [](double x, double y) { return x + y; };
    unsigned long long first = 0;
    for (int i = tid; i < V; i += LTH) first = max(first, token_key(clean_logit(l[i]), i));
    first = block_all(first, most, s_k);
    const float m = key_logit((uint32_t)(first >> 32));
    const uint32_t token = a.tokens ? a.tokens[row] : 0xFFFFFFFFu;
    const bool known = token < (uint32_t)V;
    const unsigned long long mine = known ? token_key(clean_logit(l[token]), (int)token) : ~0ull;
    double S = 0.0, E = 0.0;
    int ahead = 0;
    for (int i = tid; i < V; i += LTH) {
        const float x = clean_logit(l[i]), d = x == m ? 0.f : x - m, w = expf(d);
        S += w;
        E += w > 0.f ? (double)w * d : 0.0;
        ahead += token_key(x, i) > mine;
    }
    S = block_all(S, sum, s_d);
    E = block_all(E, sum, s_d);
    ahead = block_all(ahead, [](int x, int y) { return x + y; }, s_i);
    const double log_s = log(S);
    auto logprob = [&](float x) {
        if (m == -INFINITY) return -INFINITY;
        return x == m ? (float)-log_s : (float)((double)x - (double)m - log_s);
    };
    if (tid == 0) {
        if (a.tokens) {
            if (a.logprobs) a.logprobs[row] = known ? logprob(clean_logit(l[token])) : -INFINITY;
            if (a.ranks) a.ranks[row] = known ? ahead : -1;
        }
        if (a.entropies) a.entropies[row] = m == -INFINITY ? 0.f : (float)(log_s - E / S);
    }
    for (int k = 0; k < a.top; k++) {
        if (k > 0) {
            unsigned long long next = 0;
            for (int i = tid; i < V; i += LTH) {
                const unsigned long long key = token_key(clean_logit(l[i]), i);
                next = key < first ? max(next, key) : next;
            }
            first = block_all(next, most, s_k);
        }
        if (tid == 0) {
            a.top_tokens[(size_t)row * a.top + k] = 0xFFFFFFFFu - (uint32_t)first;
            a.top_logprobs[(size_t)row * a.top + k] = logprob(key_logit((uint32_t)(first >> 32)));
        }
    }
}

size_t token_logprobs_workspace_bytes(int rows, int V, int top) {
    (void)rows, (void)V, (void)top;
    return 16;
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
    const LogprobArgs a{logits, tokens, logprobs, entropies, top_logprobs, ranks, top_tokens, V, top};
    hipLaunchKernelGGL(logprobs_row_kernel, dim3(rows), dim3(LTH), 0, s, a);
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
