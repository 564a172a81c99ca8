// Group norm of channels-last arrays [N, S, C] with the activation behind it, and its gradient.
//
//   mean, var over the S * C / G values of one sample in one group of neighbouring channels; rstd = 1 / sqrt(var + eps)
//   hat = (x - mean) rstd,  z = hat scale + shift,  y = act(z)
//   d = g act'(z);  dshift = sum d,  dscale = sum d hat  (over samples and positions)
//   dx = rstd (d scale - mean(d scale) - hat mean(d scale hat))  (means over the group)
//
// Sums and statistics are held in 32 bits; the variance is summed from deviations from the mean, never as a difference of
// squares, so that activations far from zero keep theirs.
#include "common.h"

enum Activation : uint32_t { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2 };

struct NormParams { uint32_t first; uint32_t S, C, G, cg, act; float eps; };

__device__ __forceinline__ float act_value(float z, uint32_t act) {
    if (act == ACT_RELU) return (z > 0.f || z != z) ? z : 0.f;
    if (act == ACT_SILU) return z / (1.f + expf(-z));
    return z;
}
// g * act'(z)
__device__ __forceinline__ float act_gradient(float g, float z, uint32_t act) {
    if (act == ACT_RELU) return z > 0.f ? g : 0.f;
    if (act == ACT_SILU) { const float s = 1.f / (1.f + expf(-z)); return g * (s * (1.f + z * (1.f - s))); }
    return g;
}

// The sum over a block of 256 threads, in every thread; `room`: 4 floats of LDS that nothing else uses.
__device__ __forceinline__ float block_sum(float v, float* room) {
    v = lanes_allreduce(v, 64u, [](float a, float b) { return a + b; });
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) room[threadIdx.x >> 6] = v;
    __syncthreads();
    return (room[0] + room[1]) + (room[2] + room[3]);
}

// One block per sample and group.
extern "C" __global__ __launch_bounds__(256) void group_norm(float* y, float* mean_out, float* rstd_out, const float* x, const float* scale, const float* shift, NormParams P) {
    __shared__ float room[4];
    const uint32_t n = blockIdx.x / P.G, group = blockIdx.x % P.G;
    const uint64_t base = (uint64_t)n * P.S * P.C + group * P.cg;
    const uint64_t count = (uint64_t)P.S * P.cg;
    auto place = [&](uint64_t e) { return base + e / P.cg * P.C + e % P.cg; };
    float sum = 0.f;
    for (uint64_t e = threadIdx.x; e < count; e += 256) sum += x[place(e)];
    const float mean = block_sum(sum, room) / (float)count;
    float square = 0.f;
    for (uint64_t e = threadIdx.x; e < count; e += 256) { const float d = x[place(e)] - mean; square += d * d; }
    const float rstd = 1.f / sqrtf(block_sum(square, room) / (float)count + P.eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[blockIdx.x] = mean;
        if (rstd_out) rstd_out[blockIdx.x] = rstd;
    }
    if (y == nullptr) return;
    for (uint64_t e = threadIdx.x; e < count; e += 256) {
        const uint32_t c = group * P.cg + (uint32_t)(e % P.cg);
        y[place(e)] = act_value((x[place(e)] - mean) * rstd * scale[c] + shift[c], P.act);
    }
}

// One block per sample and group: dx, and the sample's share of dscale and dshift ([2, N, C]).
extern "C" __global__ __launch_bounds__(256) void group_norm_grad(float* dx, float* shares, const float* g, const float* x, const float* scale, const float* shift,
                                                                  const float* means, const float* rstds, NormParams P, uint32_t N) {
    __shared__ float room[4];
    const uint32_t n = blockIdx.x / P.G, group = blockIdx.x % P.G;
    const uint64_t base = (uint64_t)n * P.S * P.C + group * P.cg;
    const float mean = means[blockIdx.x], rstd = rstds[blockIdx.x];
    float first = 0.f, second = 0.f;
    for (uint32_t k = 0; k < P.cg; ++k) {
        const uint32_t c = group * P.cg + k;
        float d_sum = 0.f, dh_sum = 0.f;
        for (uint32_t s = threadIdx.x; s < P.S; s += 256) {
            const uint64_t at = base + (uint64_t)s * P.C + k;
            const float hat = (x[at] - mean) * rstd, d = act_gradient(g[at], hat * scale[c] + shift[c], P.act);
            d_sum += d; dh_sum += d * hat;
        }
        d_sum = block_sum(d_sum, room); dh_sum = block_sum(dh_sum, room);
        if (threadIdx.x == 0) { shares[(uint64_t)n * P.C + c] = dh_sum; shares[((uint64_t)N + n) * P.C + c] = d_sum; }
        first += d_sum * scale[c]; second += dh_sum * scale[c];
    }
    if (dx == nullptr) return;
    const float inverse = 1.f / ((float)P.S * (float)P.cg);
    first *= inverse; second *= inverse;
    const uint64_t count = (uint64_t)P.S * P.cg;
    for (uint64_t e = threadIdx.x; e < count; e += 256) {
        const uint64_t at = base + e / P.cg * P.C + e % P.cg;
        const uint32_t c = group * P.cg + (uint32_t)(e % P.cg);
        const float hat = (x[at] - mean) * rstd, d = act_gradient(g[at], hat * scale[c] + shift[c], P.act);
        dx[at] = rstd * (d * scale[c] - first - hat * second);
    }
}
