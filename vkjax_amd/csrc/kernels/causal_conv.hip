// Short causal convolutions along time over [B, T, C], channel by channel, and their gradient.
//
//   z[t] = bias + sum_k w[k] row[t + k],  rows: the K - 1 inputs in front of the sequence (its state), then x;  y = z, or z sigmoid(z)
//   d[t] = g[t] act'(z[t]);  drow[t + k] += w[k] d[t];  dw[k] = sum d[t] row[t + k];  dbias = sum d[t]
// From a sequence's length on y is 0, nothing is looked at and nothing comes back. The state behind it is its last K - 1 rows.
//
// A thread has VEC channels and L steps that follow one another: it loads its rows and the K - 1 before them into registers at once (neighbouring
// threads' rows overlap by those, which the caches serve) and goes through its steps from there. The gradient needs K - 1 steps on either side and works their
// d out again. Lanes lie along channels: whole lines of 128 bytes wherever there are 32 channels. Bound by memory: 8 bytes a value, 12 with the gradient.
// 8 x 2048 x 2048, 4 taps, silu, sequences of up to 2048 steps: forward 47 us, gradient 103 and 5 for the sums (what lies inside the lengths, at 4.9 TB/s: 97 us for both). One token of 64
// sequences 3.6 us: a launch. Eight steps a thread, whose K - 1 rows in front come from the caches.
// Sums over time (dw, dbias) are those of a thread's steps, then of the threads of a block, which walks `turns` tiles of time, then of the blocks in their order by
// a second launch: no atomics.
#include "common.h"

struct CausalConvParams {
    uint32_t first;                         // (bit 31: the result is stored past the caches)
    uint32_t T, C, cstrips, ttiles, turns, log2_w, silu;
};

// (see norm.hip: five instructions, off by some 2 |z| 2^-24 of itself)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

template <int VEC> __device__ __forceinline__ void get(float (&v)[VEC], const float* p) {
    if constexpr (VEC == 4) { const f32x4 q = *reinterpret_cast<const f32x4*>(p); v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
    else v[0] = *p;
}
template <int VEC> __device__ __forceinline__ void clear(float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.f;
}
template <int VEC> __device__ __forceinline__ void put(float* p, const float (&v)[VEC], bool stream = false) {
    if constexpr (VEC == 4) {
        const f32x4 q = {v[0], v[1], v[2], v[3]};
        if (stream) __builtin_nontemporal_store(q, reinterpret_cast<f32x4*>(p)); else *reinterpret_cast<f32x4*>(p) = q;
    }
    else *p = v[0];
}

template <int K, int VEC>
struct Taps {
    float w[K][VEC], bias[VEC];
    __device__ Taps(const float* kernel, const float* bias_, uint32_t C, uint32_t c) {
#pragma unroll
        for (int k = 0; k < K; ++k) get<VEC>(w[k], kernel + (size_t)k * C + c);
        if (bias_) get<VEC>(bias, bias_ + c); else clear<VEC>(bias);
    }
    // z of the step whose rows begin at rows[0]
    __device__ void apply(float (&z)[VEC], const float (*rows)[VEC]) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            z[e] = bias[e];
#pragma unroll
            for (int k = 0; k < K; ++k) z[e] = __builtin_fmaf(w[k][e], rows[k][e], z[e]);
        }
    }
};

// A sequence's rows, as steps of time: negative ones are its state
template <int K, int VEC>
struct Rows {
    const float *x, *state;                  // of this sequence and channel
    int64_t C; int length;
    __device__ Rows(const float* x_, const float* state_, const CausalConvParams& P, uint32_t b, uint32_t c, int length_)
        : x(x_ + (int64_t)b * P.T * P.C + c), state(state_ ? state_ + (int64_t)b * (K - 1) * P.C + c : nullptr), C(P.C), length(length_) {}
    __device__ void row(float (&v)[VEC], int t) const {
        if (t >= 0 && t < length) get<VEC>(v, x + t * C);
        else if (t < 0 && state && t + K - 1 >= 0) get<VEC>(v, state + (t + K - 1) * C);
        else clear<VEC>(v);
    }
};

__device__ __forceinline__ int sequence_length(const int32_t* lengths, uint32_t b, uint32_t T) {
    return lengths ? min(max(lengths[b], 0), (int)T) : (int)T;
}

template <int K, int VEC, int L>
__device__ __forceinline__ void causal_conv_body(float* __restrict__ y, float* __restrict__ last, const float* __restrict__ x, const float* __restrict__ kernel,
                                                 const float* __restrict__ bias, const float* __restrict__ state, const int32_t* __restrict__ lengths, const CausalConvParams& P) {
    const uint32_t W = 1u << P.log2_w, G = 256u >> P.log2_w, block = xcd_contiguous_block();
    const uint32_t strip = block % P.cstrips, rest = block / P.cstrips, tile = rest % P.ttiles, b = rest / P.ttiles;
    const uint32_t c = (strip * W + (threadIdx.x & (W - 1u))) * VEC, t0 = (tile * G + (threadIdx.x >> P.log2_w)) * L;
    if (c >= P.C || t0 >= P.T) return;
    const int length = sequence_length(lengths, b, P.T);
    const Rows<K, VEC> rows(x, state, P, b, c, length);
    float win[L + K - 1][VEC];
#pragma unroll
    for (int i = 0; i < L + K - 1; ++i) rows.row(win[i], (int)t0 + i - (K - 1));
    const Taps<K, VEC> taps(kernel, bias, P.C, c);
    float* const out = y ? y + ((int64_t)b * P.T + t0) * P.C + c : nullptr;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int t = (int)t0 + i;
        if (!out || t >= (int)P.T) break;
        float z[VEC];
        clear<VEC>(z);
        if (t < length) {
            taps.apply(z, win + i);
            if (P.silu)
#pragma unroll
                for (int e = 0; e < VEC; ++e) z[e] *= sigmoid(z[e]);
        }
        put<VEC>(out + (int64_t)i * P.C, z, streams_result(P.first));
    }
    if (t0 == 0 && last)
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float v[VEC];
            rows.row(v, length + j - (K - 1));
            put<VEC>(last + ((int64_t)b * (K - 1) + j) * P.C + c, v);
        }
}

template <int K, int VEC, int L>
__device__ __forceinline__ void causal_conv_grad_body(float* __restrict__ dx, float* __restrict__ dstate, float* __restrict__ partial, const float* __restrict__ x,
                                                      const float* __restrict__ kernel, const float* __restrict__ bias, const float* __restrict__ state,
                                                      const int32_t* __restrict__ lengths, const float* __restrict__ g, const float* __restrict__ g_last, const CausalConvParams& P) {
    extern __shared__ float sums[];                                      // [G][K + 1][W VEC]
    const uint32_t W = 1u << P.log2_w, G = 256u >> P.log2_w, block = xcd_contiguous_block();
    const uint32_t strip = block % P.cstrips, rest = block / P.cstrips, chunks = (P.ttiles + P.turns - 1u) / P.turns, chunk = rest % chunks, b = rest / chunks;
    const uint32_t col = threadIdx.x & (W - 1u), group = threadIdx.x >> P.log2_w, c = (strip * W + col) * VEC;
    const int length = sequence_length(lengths, b, P.T);
    float acc[K + 1][VEC];
#pragma unroll
    for (int k = 0; k <= K; ++k) clear<VEC>(acc[k]);
    if (c < P.C) {
        const Rows<K, VEC> rows(x, state, P, b, c, length);
        const Taps<K, VEC> taps(kernel, bias, P.C, c);
        const float* const g_at = g ? g + (int64_t)b * P.T * P.C + c : nullptr;
        const float* const g_last_at = g_last ? g_last + (int64_t)b * (K - 1) * P.C + c : nullptr;
        for (uint32_t turn = 0; turn < P.turns; ++turn) {
            const uint32_t t0 = ((chunk * P.turns + turn) * G + group) * L;
            if (t0 >= P.T) break;
            float win[L + 2 * K - 2][VEC], d[L + K - 1][VEC];
#pragma unroll
            for (int i = 0; i < L + 2 * K - 2; ++i) rows.row(win[i], (int)t0 + i - (K - 1));
#pragma unroll
            for (int i = 0; i < L + K - 1; ++i)
                if (g_at && (int)t0 + i < length) get<VEC>(d[i], g_at + (int64_t)(t0 + i) * P.C); else clear<VEC>(d[i]);
            if (P.silu)
#pragma unroll
                for (int i = 0; i < L + K - 1; ++i) {
                    float z[VEC];
                    taps.apply(z, win + i);
                    // (behind the length there is no z: what its rows are there is not all there is of it)
                    if (g_at && (int)t0 + i < length)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float s = sigmoid(z[e]);
                            d[i][e] *= s * __builtin_fmaf(z[e], 1.f - s, 1.f);
                        }
                }
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int t = (int)t0 + i;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    // (a step that is not taken adds nothing, whatever the rows in front of it hold)
                    if (t < length) {
#pragma unroll
                        for (int k = 0; k < K; ++k) acc[k][e] = __builtin_fmaf(d[i][e], win[i + k][e], acc[k][e]);
                        acc[K][e] += d[i][e];
                    }
                }
                if (dx && t < (int)P.T) {
                    float v[VEC];
                    clear<VEC>(v);
                    if (t < length) {
                        if (g_last_at && t - length + K - 1 >= 0) get<VEC>(v, g_last_at + (int64_t)(t - length + K - 1) * P.C);
#pragma unroll
                        for (int j = 0; j < K; ++j)
                            if (t + j < length)
#pragma unroll
                                for (int e = 0; e < VEC; ++e) v[e] = __builtin_fmaf(taps.w[K - 1 - j][e], d[i + j][e], v[e]);
                    }
                    put<VEC>(dx + ((int64_t)b * P.T + t) * P.C + c, v, streams_result(P.first));
                }
            }
            if (t0 == 0 && dstate)
#pragma unroll
                for (int i = 0; i < K - 1; ++i) {
                    float v[VEC];
                    clear<VEC>(v);
                    if (g_last_at && i >= length) get<VEC>(v, g_last_at + (int64_t)(i - length) * P.C);
#pragma unroll
                    for (int k = 0; k <= i; ++k)
                        if (i - k < length)
#pragma unroll
                            for (int e = 0; e < VEC; ++e) v[e] = __builtin_fmaf(taps.w[k][e], d[i - k][e], v[e]);
                    put<VEC>(dstate + ((int64_t)b * (K - 1) + i) * P.C + c, v);
                }
        }
    }
    if (!partial) return;
    const uint32_t width = W * VEC;
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[(group * (K + 1) + k) * width + col * VEC + e] = acc[k][e];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < (K + 1) * width; i += 256u) {
        const uint32_t k = i / width, at = strip * width + i % width;
        float s = 0.f;
        for (uint32_t q = 0; q < G; ++q) s += sums[q * (K + 1) * width + i];
        if (at < P.C) partial[((uint64_t)rest * (K + 1) + k) * P.C + at] = s;
    }
}

#define CAUSAL_CONV(K, VEC, L)                                                                                                                             \
    extern "C" __global__ __launch_bounds__(256) void causal_conv_k##K##_v##VEC##_l##L(float* y, float* last, const float* x, const float* kernel, const float* bias, \
                                                                                       const float* state, const int32_t* lengths, CausalConvParams P) {   \
        causal_conv_body<K, VEC, L>(y, last, x, kernel, bias, state, lengths, P);                                                                          \
    }
#define CAUSAL_CONV_GRAD(K, VEC, L)                                                                                                                        \
    extern "C" __global__ __launch_bounds__(256) void causal_conv_grad_k##K##_v##VEC##_l##L(float* dx, float* dstate, float* partial, const float* x, const float* kernel, \
                                                                                            const float* bias, const float* state, const int32_t* lengths, \
                                                                                            const float* g, const float* g_last, CausalConvParams P) {     \
        causal_conv_grad_body<K, VEC, L>(dx, dstate, partial, x, kernel, bias, state, lengths, g, g_last, P);                                              \
    }
#define CAUSAL_CONV_WIDTHS(F, VEC, L) F(2, VEC, L) F(3, VEC, L) F(4, VEC, L) F(5, VEC, L) F(6, VEC, L) F(7, VEC, L) F(8, VEC, L)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV, 4, 1)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV, 1, 1)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV, 4, 8)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV, 1, 8)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV_GRAD, 4, 1)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV_GRAD, 1, 1)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV_GRAD, 4, 8)
CAUSAL_CONV_WIDTHS(CAUSAL_CONV_GRAD, 1, 8)

// dkernel [K, C] and dbias [C]: the blocks' rows of sums, added up. A block has 64 columns, its 16 waves every 16th row.
struct CausalConvSumsParams { uint32_t rows, C, taps; };
extern "C" __global__ __launch_bounds__(1024) void causal_conv_sums(float* __restrict__ dkernel, float* __restrict__ dbias, const float* __restrict__ partial, CausalConvSumsParams P) {
    __shared__ float part[16][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, columns = (P.taps + 1u) * P.C, at = blockIdx.x * 64u + lane;
    float s = 0.f;
    if (at < columns)
        for (uint32_t r = wave; r < P.rows; r += 16u) s += partial[(uint64_t)r * columns + at];
    part[wave][lane] = s;
    __syncthreads();
    if (wave != 0u || at >= columns) return;
    s = part[0][lane];
#pragma unroll
    for (int q = 1; q < 16; ++q) s += part[q][lane];
    if (at < P.taps * P.C) { if (dkernel) dkernel[at] = s; }
    else if (dbias) dbias[at - P.taps * P.C] = s;
}
