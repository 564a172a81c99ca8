// Linear recurrences along time over [B, T, C]: h[t] = a[t] h[t-1] + b[t], with factors a and addends b as they are, or from gates:
// a = sigmoid(gate), b = (1 - a) x. Their gradient runs the other way: with l[t] = g[t] + a[t+1] l[t+1] (g of the last step: and the
// last state's cotangent)
//   dx = l (gated: l (1 - a)),  dfactor = l h[t-1] (gated: l (h[t-1] - x) a (1 - a)),  dstate = a[first] l[first].
// From a sequence's length on steps are not taken: the state stays, and the operands are not used there.
#include "common.h"

struct RecurrenceParams { uint32_t T, C, gated, reverse; };

// sigmoid(gate) and 1 - sigmoid(gate), each rounded from the exact exponential: one of them is not the difference of the other to 1
__device__ __forceinline__ void gate_factors(float gate, float& a, float& rest) {
    const float e = expf(-fabsf(gate)), near = 1.f / (1.f + e), far = e * near;
    a = gate < 0.f ? far : near;
    rest = gate < 0.f ? near : far;
}

__device__ __forceinline__ uint32_t length_of(const int32_t* lengths, uint32_t b, uint32_t T) {
    return lengths ? (uint32_t)min((int64_t)max(lengths[b], 0), (int64_t)T) : T;
}

// A thread per channel of a sequence walks through time.
extern "C" __global__ __launch_bounds__(64) void recurrence(float* h, float* last, const float* factor, const float* x, const float* state, const int32_t* lengths, RecurrenceParams P) {
    const uint32_t c = blockIdx.x * 64u + threadIdx.x, b = blockIdx.y;
    if (c >= P.C) return;
    const uint32_t length = length_of(lengths, b, P.T);
    float now = state ? state[(uint64_t)b * P.C + c] : 0.f;
    for (uint32_t step = 0; step < P.T; ++step) {
        const uint32_t t = P.reverse ? P.T - 1u - step : step;
        const uint64_t at = ((uint64_t)b * P.T + t) * P.C + c;
        if (t < length) {
            if (P.gated) { float a, rest; gate_factors(factor[at], a, rest); now = __builtin_fmaf(a, now, rest * x[at]); }
            else now = __builtin_fmaf(factor[at], now, x[at]);
        }
        if (h) h[at] = now;
    }
    if (last) last[(uint64_t)b * P.C + c] = now;
}

extern "C" __global__ __launch_bounds__(64) void recurrence_grad(float* dfactor, float* dx, float* dstate, const float* h, const float* factor, const float* x, const float* state,
                                                                 const int32_t* lengths, const float* g, const float* g_last, RecurrenceParams P) {
    const uint32_t c = blockIdx.x * 64u + threadIdx.x, b = blockIdx.y;
    if (c >= P.C) return;
    const uint32_t length = length_of(lengths, b, P.T);
    const uint64_t base = (uint64_t)b * P.T * P.C + c;
    float l = g_last ? g_last[(uint64_t)b * P.C + c] : 0.f;
    for (uint32_t step = P.T; step-- > 0;) {
        const uint32_t t = P.reverse ? P.T - 1u - step : step;
        const uint64_t at = base + (uint64_t)t * P.C;
        if (g) l += g[at];
        float df = 0.f, db = 0.f;
        if (t < length) {
            const uint32_t previous = P.reverse ? t + 1u : t - 1u;
            const float before = step ? h[base + (uint64_t)previous * P.C] : state ? state[(uint64_t)b * P.C + c] : 0.f;
            if (P.gated) {
                float a, rest;
                gate_factors(factor[at], a, rest);
                df = l * (before - x[at]) * (a * rest); db = l * rest; l *= a;
            } else { df = l * before; db = l; l *= factor[at]; }
        }
        if (dfactor) dfactor[at] = df;
        if (dx) dx[at] = db;
    }
    if (dstate) dstate[(uint64_t)b * P.C + c] = l;
}
