// Log probabilities of given tokens with the entropy of their rows' distributions and the most likely alternatives, and the
// gradient of all three.
//
// With m = max x, s = sum exp(x - m), w = sum exp(x - m) (x - m) over a row of V scores:
//   lse = m + log s,  log p = x - lse,  H = -sum p log p = log s - w / s
//   dx[v] = -p[v] (sum of the cotangents of log probabilities) - gH p[v] (log p[v] + H) + the cotangents of v's own log probabilities
//
// A token outside [0, V) marks its row as padding: results are 0 (alternatives: token -1), the row's scores are not read. Scores of
// -inf are masked: p = 0, and p log p counts as 0. Where every score of a row is -inf there is no distribution: log p = -inf, H = 0,
// gradient 0. NaN and +inf make their row NaN by themselves (+inf - +inf).
#include "common.h"

struct LogProbsParams { uint32_t first; uint32_t V, top; };

__device__ __forceinline__ uint64_t place_of(float x, uint32_t v) {
    // larger for larger scores (NaN above all), among equal ones for the smaller number; neither 0 nor all ones
    const float y = x == 0.f ? 0.f : x;                               // -0 and 0 are equal
    const uint32_t b = f2u(y), key = x != x ? 0xFFFFFFFEu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (uint64_t)key << 32 | (0xFFFFFFFFu - v);
}

__device__ __forceinline__ float block_sum(float v, float* room) {
    v = lanes_allreduce(v, 64u, [](float a, float b) { return a + b; });
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) room[threadIdx.x >> 6] = v;
    __syncthreads();
    return (room[0] + room[1]) + (room[2] + room[3]);
}

// One block per row, which reads it once for the maximum, once for the sums and once per alternative.
extern "C" __global__ __launch_bounds__(256) void log_probs(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token,
                                                            const float* logits, const uint32_t* tokens, LogProbsParams P) {
    __shared__ float room[4];
    __shared__ uint64_t keys[4];
    const uint64_t row = blockIdx.x;
    const uint32_t token = tokens[row];
    if (token >= P.V) {
        if (threadIdx.x == 0) {
            if (log_prob) log_prob[row] = 0.f;
            if (entropy) entropy[row] = 0.f;
            if (log_sum) log_sum[row] = 0.f;
        }
        if (threadIdx.x < P.top) {
            if (top_log_prob) top_log_prob[row * P.top + threadIdx.x] = 0.f;
            if (top_token) top_token[row * P.top + threadIdx.x] = -1;
        }
        return;
    }
    const float* const x = logits + row * P.V;
    float m = -INFINITY;
    for (uint32_t v = threadIdx.x; v < P.V; v += 256) m = fmaxf(m, x[v]);
    m = lanes_allreduce(m, 64u, [](float a, float b) { return fmaxf(a, b); });
    if ((threadIdx.x & 63u) == 0) room[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(room[0], room[1]), fmaxf(room[2], room[3]));
    const bool empty = m == -INFINITY;                                // (or only NaN and -inf: the sums say which)
    const float from = empty ? 0.f : m;
    float s = 0.f, w = 0.f;
    for (uint32_t v = threadIdx.x; v < P.V; v += 256) {
        const float d = x[v] - from, e = expf(d);
        s += e;
        w += e == 0.f ? 0.f : e * d;
    }
    s = block_sum(s, room); w = block_sum(w, room);
    const bool nothing = s == 0.f;
    const float lse = nothing ? -INFINITY : from + logf(s);
    if (threadIdx.x == 0) {
        if (log_prob) log_prob[row] = nothing ? -INFINITY : x[token] - lse;
        if (entropy) entropy[row] = nothing ? 0.f : logf(s) - w / s;
        if (log_sum) log_sum[row] = lse;
    }
    uint64_t below = ~0ull;
    for (uint32_t k = 0; k < P.top; ++k) {
        uint64_t best = 0;
        for (uint32_t v = threadIdx.x; v < P.V; v += 256) {
            const uint64_t key = place_of(x[v], v);
            if (key < below && key > best) best = key;
        }
        best = lanes_allreduce(best, 64u, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) keys[threadIdx.x >> 6] = best;
        __syncthreads();
        for (int i = 0; i < 4; ++i) best = keys[i] > best ? keys[i] : best;
        below = best;
        if (threadIdx.x == 0) {
            const uint32_t v = 0xFFFFFFFFu - (uint32_t)best;
            if (top_log_prob) top_log_prob[row * P.top + k] = nothing ? -INFINITY : x[v] - lse;
            if (top_token) top_token[row * P.top + k] = (int32_t)v;
        }
    }
}

// One block per row; cotangents that are null are zeros.
extern "C" __global__ __launch_bounds__(256) void log_probs_grad(float* dx, const float* logits, const uint32_t* tokens, const float* log_sum, const float* entropy,
                                                                 const float* g_log_prob, const float* g_entropy, const float* g_top, const int32_t* top_token, LogProbsParams P) {
    const uint64_t row = blockIdx.x;
    const uint32_t token = tokens[row];
    const float* const x = logits + row * P.V;
    float* const out = dx + row * P.V;
    const float lse = log_sum[row];
    if (token >= P.V || lse == -INFINITY) {
        for (uint32_t v = threadIdx.x; v < P.V; v += 256) out[v] = 0.f;
        return;
    }
    const float own = g_log_prob ? g_log_prob[row] : 0.f, gh = g_entropy ? g_entropy[row] : 0.f, H = entropy[row];
    float total = own;
    for (uint32_t k = 0; k < P.top; ++k) total += g_top[row * P.top + k];
    for (uint32_t v = threadIdx.x; v < P.V; v += 256) {
        const float lp = x[v] - lse, p = expf(lp);
        float d = p == 0.f ? 0.f : -p * (total + gh * (lp + H));
        if (v == token) d += own;
        for (uint32_t k = 0; k < P.top; ++k) if (top_token[row * P.top + k] == (int32_t)v) d += g_top[row * P.top + k];
        out[v] = d;
    }
}
