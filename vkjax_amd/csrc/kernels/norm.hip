// Group norm of channels-last arrays [N, S, C] with the activation behind it, and its gradient.
//
//   mean, var over the S * C / G values of one sample in one group of neighbouring channels; rstd = 1 / sqrt(var + eps)
//   hat = (x - mean) rstd,  z = hat scale + shift,  y = act(z)
//   d = g act'(z);  dshift = sum d,  dscale = sum d hat  (over samples and positions)
//   dx = rstd (d scale - mean(d scale) - hat mean(d scale hat))  (means over the group)
//
// Sums and statistics are held in 32 bits. The variance is never a difference of squares: a thread has mean and squared deviations of
// its own values, and those are joined by n1 (mean1 - mean)^2 terms (Chan, Golub, LeVeque), so activations far from zero keep theirs.
//
// A block owns a span of channels (whole groups, or a piece of one that is too wide for a block): V lanes of VEC channels each read a
// position's span, and 256 / V (1024 / V) positions are read side by side. A lane's channels stay the same, so what belongs to a channel
// is in registers, and reading and writing are whole lines wherever a span has 32 channels. What the positions' lanes have found meets in
// shared memory, where a few lanes per group add it up.
//   * group_norm_held: samples small enough stay in registers: one launch that reads once and writes once. Several small samples share a
//     block. 1 x 7 x 7 x 512 5 us, as long as a launch and its three round trips to memory take; 32 x 56 x 56 x 64 in 32 groups 16 us (51 MB,
//     3.2 TB/s: every block reads, waits and writes once, and there are no more blocks than CUs to take turns; by half or quarter
//     lines, 512 or 1024 threads, 15.7-17).
//   * group_norm_rows: samples of one position, several rows to a block. 8191 x 1040 in 16 groups 17 us, 4.0 TB/s; its gradient 29, 3.5: a block loads, puts its rows
//     into shared memory, waits, sums, waits and stores, with nothing of the next rows on the way. (They go through shared memory because groups of 65 channels do
//     not begin where vectors do; groups of 64 take 16.5 and 25 by the same kernels.)
//   * group_norm_wide: samples of one position with wide groups (layer norms): a block to a group, several vectors to a thread, a sum over the block
//     for the mean and one for the deviations from it. 8191 x 8192 82 us, 6.5 TB/s, its gradient 175, 4.6: every row waits for its two sums, one after
//     the other, before the next one's operands are asked for, with four waves to a SIMD; 8191 x 1021 16 and 25.
//   * group_norm_stats / _apply: the others are cut along their positions. The first launch leaves mean and squared deviations of each
//     chunk, the second joins a sample's chunks and reads x again (from the caches where they hold it). 64 x 56 x 56 x 256: 35 and 68 us, and
//     68 and 107 for the gradient's two, all at 5.8-6.1 TB/s: bound by memory, and by reading everything twice. (Each launch
//     begins where the one before it ended, for what the caches still hold.)
// The gradient has the same forms; what dscale and dshift get from a block is a row of sums per block, added up by a last launch
// (group_norm_columns) in a fixed order: no atomics.
#include "common.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));

enum Activation : uint32_t { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2 };

struct NormParams {
    uint32_t first;                         // (bit 31: the result is stored past the caches)
    uint32_t N, S, C, G, cg, act; float eps;
    uint32_t span, spans, pieces;           // channels of a block, blocks per row of channels, blocks per group where it is wider than a block (else 1)
    uint32_t V, P, M;                       // lanes per position, positions side by side (of one sample), samples side by side
    uint32_t log2_lc, log2_lq;              // lanes per group in the joining step: along its channels, along positions
    uint32_t chunks, chunk;                 // chunks of positions per sample, positions in one
};

constexpr uint32_t NOWHERE = 0x80000000u;

__device__ __forceinline__ float reciprocal(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);             // a Newton step
}
// 1 / (1 + exp(-z)) in five instructions: the exponential in base 2, whose exponent z log2(e) is rounded twice, so that it is off by some 2 |z| 2^-24 of itself,
// and the reciprocal to one unit of the last place. That is where this operator's launches have their instructions: 25 a value with the library's exponential and
// a division bounded them. (exp(-z) beyond fp32 is infinite, and its reciprocal 0.)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }
// What the activation is taken of, hat = (x - mean) rstd: rounded alike in every kernel, so that next to zero a gradient is that of the relu that the
// forward pass has taken.
__device__ __forceinline__ float z_of(float hat, float gamma, float beta) { return __builtin_fmaf(hat, gamma, beta); }
__device__ __forceinline__ float act_value(float z, uint32_t act) {
    if (act == ACT_RELU) return (z > 0.f || z != z) ? z : 0.f;
    if (act == ACT_SILU) return z * sigmoid(z);
    return z;
}
// g * act'(z)
__device__ __forceinline__ float act_gradient(float g, float z, uint32_t act) {
    if (act == ACT_RELU) return z > 0.f ? g : 0.f;
    if (act == ACT_SILU) { const float s = sigmoid(z); return g * (s * __builtin_fmaf(z, 1.f - s, 1.f)); }
    return g;
}

template <int VEC> __device__ __forceinline__ void load(float (&v)[VEC], __amdgpu_buffer_rsrc_t r, uint32_t at) {
    if constexpr (VEC == 4) { const f32x4 t = buffer_load_x4(r, at); v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; }
    else v[0] = buffer_load_x1(r, at);
}
template <int VEC> __device__ __forceinline__ void store(const float (&v)[VEC], __amdgpu_buffer_rsrc_t r, uint32_t at, bool stream) {
    if constexpr (VEC == 4) {
        const u32x4 t = u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
        if (stream) __builtin_amdgcn_raw_buffer_store_b128(t, r, at, 0, 2);
        else __builtin_amdgcn_raw_buffer_store_b128(t, r, at, 0, 0);
    } else {
        if (stream) __builtin_amdgcn_raw_buffer_store_b32(f2u(v[0]), r, at, 0, 2);
        else __builtin_amdgcn_raw_buffer_store_b32(f2u(v[0]), r, at, 0, 0);
    }
}

extern __shared__ __attribute__((aligned(16))) float room[];

// to[0 .. VEC) = v in shared memory; whole vectors lie at multiples of 16 bytes
template <int VEC> __device__ __forceinline__ void put(float* to, const float (&v)[VEC]) {
    if constexpr (VEC == 4) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
    else to[0] = v[0];
}


// A span of channels and this thread's part of it.
template <int VEC>
struct Span {
    uint32_t c0, width, groups, g0;         // first channel, channels, whole groups in it (1 of a piece), its first group
    uint32_t col, p, c;                     // this thread's lane within a position, its place among the positions, its first channel
    __device__ Span(const NormParams& P, uint32_t number) {
        if (P.pieces == 1u) {
            c0 = number * P.span; width = min(P.span, P.C - c0);
            groups = width / P.cg; g0 = c0 / P.cg;
        } else {
            const uint32_t piece = number % P.pieces;
            g0 = number / P.pieces; groups = 1u;
            c0 = g0 * P.cg + piece * P.span; width = min(P.span, P.cg - piece * P.span);
        }
        p = threadIdx.x / P.V; col = threadIdx.x - p * P.V;
        c = c0 + col * VEC;
    }
    __device__ bool owns() const { return col * VEC < width; }
    __device__ uint32_t group_of(const NormParams& P, int j) const { return P.pieces == 1u ? (col * VEC + j) / P.cg : 0u; }      // within the span
};

// Goes through the entries of every group in shared memory, a few lanes to a group: entry.add for each, entry.join across the lanes, a second
// round where entry.again(), and done(sample, group, whether this lane reports it, entry). Entries lie at (sample * P + position's lane) * span + channel.
template <class Entry, class Done>
__device__ __forceinline__ void for_groups(const NormParams& P, uint32_t groups, uint32_t channels_per_group, uint32_t samples, Entry entry, Done done) {
    const uint32_t log2_lanes = P.log2_lc + P.log2_lq, lanes = 1u << log2_lanes, lane = threadIdx.x & (lanes - 1u);
    const uint32_t lc = lane & ((1u << P.log2_lc) - 1u), lq = lane >> P.log2_lc, sets = blockDim.x >> log2_lanes;
    const uint32_t all = groups * samples;
    for (uint32_t at = threadIdx.x >> log2_lanes; at - (threadIdx.x >> log2_lanes) < all; at += sets) {      // (every lane goes round as often: lanes meet below)
        const bool use = at < all;
        const uint32_t m = use ? at / groups : 0u, g = use ? at - m * groups : 0u;
        entry.start();
        if (use)
            for (uint32_t ch = lc; ch < channels_per_group; ch += 1u << P.log2_lc) {
#pragma unroll 4
                for (uint32_t q = lq; q < P.P; q += 1u << P.log2_lq) entry.add((m * P.P + q) * P.span + g * channels_per_group + ch, q, g * channels_per_group + ch);
            }
        entry.join(lanes);
        if (use && entry.again())
            for (uint32_t ch = lc; ch < channels_per_group; ch += 1u << P.log2_lc) {
#pragma unroll 4
                for (uint32_t q = lq; q < P.P; q += 1u << P.log2_lq) entry.add_again((m * P.P + q) * P.span + g * channels_per_group + ch, q);
            }
        entry.join_again(lanes);
        if (use) done(m, g, lane == 0u, entry);
    }
}

__device__ __forceinline__ float add_lanes(float v, uint32_t lanes) { return lanes_allreduce(v, lanes, [](float a, float b) { return a + b; }); }

// Mean and squared deviations of a group from the sums and squared deviations of (thread, channel): `count(q)` values each.
template <class Count>
struct JoinStats {
    const float *sums, *squares;
    Count count;
    float total, sum, mean, square;
    __device__ void start() { total = sum = square = 0.f; mean = 0.f; }
    __device__ void add(uint32_t at, uint32_t q, uint32_t) { sum += sums[at]; total += count(q); }
    __device__ void join(uint32_t lanes) { sum = add_lanes(sum, lanes); total = add_lanes(total, lanes); mean = sum / total; }
    __device__ bool again() const { return true; }
    __device__ void add_again(uint32_t at, uint32_t q) {
        const float n = count(q), d = n > 0.f ? __builtin_fmaf(sums[at], reciprocal(n), -mean) : 0.f;
        square += __builtin_fmaf(n * d, d, squares[at]);
    }
    __device__ void join_again(uint32_t lanes) { square = add_lanes(square, lanes); }
};
// The sums of scale * first and scale * second over a group.
struct JoinSums {
    const float *first, *second, *scale;       // (scale: of the span's first channel)
    float a, b;
    __device__ void start() { a = b = 0.f; }
    __device__ void add(uint32_t at, uint32_t, uint32_t channel) { const float s = scale[channel]; a = __builtin_fmaf(s, first[at], a); b = __builtin_fmaf(s, second[at], b); }
    __device__ void join(uint32_t lanes) { a = add_lanes(a, lanes); b = add_lanes(b, lanes); }
    __device__ bool again() const { return false; }
    __device__ void add_again(uint32_t, uint32_t) {}
    __device__ void join_again(uint32_t) {}
};

// A block's row of sums per channel, over `rows` entries of each in shared memory, a few lanes to a channel.
__device__ __forceinline__ void write_channel_sums(const float* firsts, const float* seconds, uint32_t rows, uint32_t stride, uint32_t width, float* to_first, float* to_second) {
    const uint32_t log2_lanes = min(31u - (uint32_t)__clz((int)min(max(blockDim.x / width, 1u), 64u)), 31u - (uint32_t)__clz((int)rows)), lanes = 1u << log2_lanes;
    const uint32_t lane = threadIdx.x & (lanes - 1u);
    for (uint32_t base = 0; base < width; base += blockDim.x >> log2_lanes) {      // (every lane goes round as often: lanes meet below)
        const uint32_t ch = base + (threadIdx.x >> log2_lanes);
        float a = 0.f, b = 0.f;
        if (ch < width)
            for (uint32_t k = lane; k < rows; k += lanes) { a += firsts[k * stride + ch]; b += seconds[k * stride + ch]; }
        a = add_lanes(a, lanes); b = add_lanes(b, lanes);
        if (ch < width && lane == 0u) { to_first[ch] = a; to_second[ch] = b; }
    }
}

// How many of `count` positions the lane q of `side` side by side has.
__device__ __forceinline__ uint32_t share_of(uint32_t count, uint32_t q, uint32_t side) { return count > q ? (count - q - 1u) / side + 1u : 0u; }

// ---------------------------------------------------------------------------------------------- samples that stay in registers

template <int VEC, int K>
__device__ __forceinline__ void held_body(float* y, float* means, float* rstds, const float* x, const float* scale, const float* shift, const NormParams& P) {
    const uint32_t block = xcd_contiguous_block();                       // neighbouring spans share lines: on one XCD, one fetch
    const Span<VEC> span(P, block % P.spans);
    const uint32_t n0 = block / P.spans * P.M, m = span.p / P.P, q = span.p - m * P.P;
    const bool use = m < P.M && n0 + m < P.N && span.owns();
    const uint64_t base = (uint64_t)n0 * P.S * P.C + span.c0;
    const uint32_t bytes = ((min(P.M, P.N - n0) * P.S - 1u) * P.C + span.width) * 4u;
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(x + base, bytes);
    const uint32_t first = ((m * P.S + q) * P.C + span.col * VEC) * 4u, step = P.P * P.C * 4u;
    const uint32_t mine = use ? share_of(P.S, q, P.P) : 0u;
    float v[K][VEC];
#pragma unroll
    for (int i = 0; i < K; ++i) load<VEC>(v[i], x_rsrc, (uint32_t)i < mine ? first + i * step : NOWHERE);
    float gamma[VEC], beta[VEC];
    {
        const __amdgpu_buffer_rsrc_t a = make_rsrc(scale + span.c0, span.width * 4u), b = make_rsrc(shift + span.c0, span.width * 4u);
        load<VEC>(gamma, a, span.owns() ? span.col * VEC * 4u : NOWHERE);
        load<VEC>(beta, b, span.owns() ? span.col * VEC * 4u : NOWHERE);
    }
    const uint32_t entries = P.M * P.P * P.span, groups_at_most = P.span / P.cg * P.M;
    float* const sums = room, * const squares = room + entries, * const mean_of = room + 2u * entries, * const rstd_of = mean_of + groups_at_most;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        float sum = 0.f, square = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) sum += v[i][j];                      // (beyond the sample: zeros)
        const float mean = sum / (float)max(mine, 1u);
#pragma unroll
        for (int i = 0; i < K; ++i) { const float d = (uint32_t)i < mine ? v[i][j] - mean : 0.f; square = __builtin_fmaf(d, d, square); }
        if (m < P.M && span.col * VEC + j < P.span) { sums[span.p * P.span + span.col * VEC + j] = sum; squares[span.p * P.span + span.col * VEC + j] = square; }
    }
    __syncthreads();
    const uint32_t each = P.S / P.P, more = P.S % P.P;
    auto count = [&](uint32_t lane_q) { return (float)(each + (lane_q < more ? 1u : 0u)); };
    JoinStats<decltype(count)> join{sums, squares, count};
    for_groups(P, span.groups, P.cg, P.M, join, [&](uint32_t sample, uint32_t g, bool reports, const JoinStats<decltype(count)>& found) {
        if (!reports) return;
        const float rstd = 1.f / sqrtf(found.square / found.total + P.eps);
        mean_of[sample * span.groups + g] = found.mean; rstd_of[sample * span.groups + g] = rstd;
        if (n0 + sample < P.N) {
            const uint64_t at = (uint64_t)(n0 + sample) * P.G + span.g0 + g;
            if (means) means[at] = found.mean;
            if (rstds) rstds[at] = rstd;
        }
    });
    __syncthreads();
    if (!use || y == nullptr) return;
    const bool stream = streams_result(P.first);
    const __amdgpu_buffer_rsrc_t y_rsrc = make_rsrc(y + base, bytes);
    float mean[VEC], rstd[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const uint32_t g = m * span.groups + span.group_of(P, j);
        mean[j] = mean_of[g]; rstd[j] = rstd_of[g];
    }
#pragma unroll
    for (int i = 0; i < K; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = act_value(z_of((v[i][j] - mean[j]) * rstd[j], gamma[j], beta[j]), P.act);
        store<VEC>(v[i], y_rsrc, (uint32_t)i < mine ? first + i * step : NOWHERE, stream);
    }
}

// The gradient of samples that stay in registers. Blocks take one set of samples after the other; the row of sums for dscale and dshift of
// a block is written at its end.
template <int VEC, int K>
__device__ __forceinline__ void held_grad_body(float* dx, float* dscale_rows, float* dshift_rows, const float* gs, const float* x, const float* scale, const float* shift,
                                               const float* means, const float* rstds, const NormParams& P) {
    const uint32_t block = xcd_contiguous_block();
    const Span<VEC> span(P, block % P.spans);
    const uint32_t m = span.p / P.P, q = span.p - m * P.P, entries = P.M * P.P * P.span, sets = (P.N - 1u) / P.M + 1u, row = block / P.spans, rows = gridDim.x / P.spans;
    float* const firsts = room, * const seconds = room + entries, * const a_of = room + 2u * entries, * const b_of = a_of + P.span / P.cg * P.M;
    float gamma[VEC], beta[VEC], d_total[VEC], dh_total[VEC];
    {
        const __amdgpu_buffer_rsrc_t a = make_rsrc(scale + span.c0, span.width * 4u), b = make_rsrc(shift + span.c0, span.width * 4u);
        load<VEC>(gamma, a, span.owns() ? span.col * VEC * 4u : NOWHERE);
        load<VEC>(beta, b, span.owns() ? span.col * VEC * 4u : NOWHERE);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { d_total[j] = 0.f; dh_total[j] = 0.f; }
    const float inverse = 1.f / ((float)P.S * (float)P.cg);
    const bool stream = streams_result(P.first);
    for (uint32_t set = row; set < sets; set += rows) {
        const uint32_t n0 = set * P.M;
        const bool use = m < P.M && n0 + m < P.N && span.owns();
        const uint64_t base = (uint64_t)n0 * P.S * P.C + span.c0;
        const uint32_t bytes = ((min(P.M, P.N - n0) * P.S - 1u) * P.C + span.width) * 4u;
        const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(x + base, bytes), g_rsrc = make_rsrc(gs + base, bytes);
        const uint32_t first = ((m * P.S + q) * P.C + span.col * VEC) * 4u, step = P.P * P.C * 4u;
        const uint32_t mine = use ? share_of(P.S, q, P.P) : 0u;
        float v[K][VEC], d[K][VEC], mean[VEC], rstd[VEC], A[VEC], B[VEC];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            load<VEC>(v[i], x_rsrc, (uint32_t)i < mine ? first + i * step : NOWHERE);
            load<VEC>(d[i], g_rsrc, (uint32_t)i < mine ? first + i * step : NOWHERE);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const uint64_t at = (uint64_t)(n0 + m) * P.G + span.g0 + span.group_of(P, j);
            mean[j] = use && span.col * VEC + j < span.width ? means[at] : 0.f; rstd[j] = use && span.col * VEC + j < span.width ? rstds[at] : 0.f;
            A[j] = 0.f; B[j] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] = (v[i][j] - mean[j]) * rstd[j];
                d[i][j] = act_gradient(d[i][j], z_of(v[i][j], gamma[j], beta[j]), P.act);
                d[i][j] = (uint32_t)i < mine ? d[i][j] : 0.f; v[i][j] = (uint32_t)i < mine ? v[i][j] : 0.f;
                A[j] += d[i][j]; B[j] = __builtin_fmaf(d[i][j], v[i][j], B[j]);
            }
        __syncthreads();                                                 // (what the set before has left has been read)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (m < P.M && span.col * VEC + j < P.span) { firsts[span.p * P.span + span.col * VEC + j] = A[j]; seconds[span.p * P.span + span.col * VEC + j] = B[j]; }
            d_total[j] += A[j]; dh_total[j] += B[j];
        }
        if (dx == nullptr) continue;
        __syncthreads();
        JoinSums join{firsts, seconds, scale + span.c0};
        for_groups(P, span.groups, P.cg, P.M, join, [&](uint32_t sample, uint32_t g, bool reports, const JoinSums& found) {
            if (reports) { a_of[sample * span.groups + g] = found.a * inverse; b_of[sample * span.groups + g] = found.b * inverse; }
        });
        __syncthreads();
        const __amdgpu_buffer_rsrc_t dx_rsrc = make_rsrc(dx + base, bytes);
        float a[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const uint32_t g = m * span.groups + span.group_of(P, j);
            a[j] = use && span.col * VEC + j < span.width ? a_of[g] : 0.f; b[j] = use && span.col * VEC + j < span.width ? b_of[g] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < K; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = rstd[j] * (__builtin_fmaf(d[i][j], gamma[j], -a[j]) - v[i][j] * b[j]);
            store<VEC>(v[i], dx_rsrc, (uint32_t)i < mine ? first + i * step : NOWHERE, stream);
        }
    }
    // the block's sums per channel, over its positions' and samples' lanes
    __syncthreads();
    const uint32_t all = P.M * P.P;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (span.p < all && span.col * VEC + j < P.span) { firsts[span.p * P.span + span.col * VEC + j] = d_total[j]; seconds[span.p * P.span + span.col * VEC + j] = dh_total[j]; }
    __syncthreads();
    const uint64_t to = (uint64_t)row * P.C + span.c0;
    write_channel_sums(firsts, seconds, all, P.span, span.width, dshift_rows + to, dscale_rows + to);
}

// ---------------------------------------------------------------------------------------------- single positions

// Samples of one position: rows of C values. A thread has the same channels of K rows, P rows apart; all of a block's rows and groups are joined
// together from shared memory, where channels of a group need not be those of whole vectors (65 channels to a group: 4 to a lane).

// done(row, group, lane 0 of the group's, first of its values in shared memory, how many lanes): lanes of one group go through its channels.
template <class Done>
__device__ __forceinline__ void for_row_groups(const NormParams& P, uint32_t groups, uint32_t rows, Done done) {
    const uint32_t lanes = 1u << P.log2_lc, lane = threadIdx.x & (lanes - 1u), sets = blockDim.x >> P.log2_lc, all = groups * rows, start = threadIdx.x >> P.log2_lc;
    for (uint32_t at = start; at - start < all; at += sets) {             // (every lane goes round as often: lanes meet in `done`)
        const bool use = at < all;
        const uint32_t m = use ? at / groups : 0u, g = use ? at - m * groups : 0u;
        done(m, g, use && lane == 0u, m * P.span + g * P.cg, lane, lanes);
    }
}

// The groups of a vector's channels: two at most, since groups of one channel have the kernels with one channel per lane.
template <int VEC>
struct TwoGroups {
    uint32_t first, last, from;                  // channels from `from` on belong to `last`
    __device__ TwoGroups(const NormParams& P, const Span<VEC>& span) {
        first = span.owns() ? span.group_of(P, 0) : 0u; last = span.owns() ? span.group_of(P, VEC - 1) : 0u;
        from = last * P.cg - span.col * VEC;
    }
    __device__ float pick(int j, float a, float b) const { return VEC > 1 && first != last && (uint32_t)j >= from ? b : a; }
};

// Mean and squared deviations of values[lane], values[lane + lanes] .. (`count` in all), by the lanes together. A lane goes through its values once: with
// s = sum (x - k), q = sum (x - k)^2 of its n values, k the first of them, their squared deviations are q - s^2 / n. k being one of them, q is at most n times
// that difference, whose error is then at most n u of itself: with at most some 64 values a lane that is a sum's own error. Lanes are joined by their means.
__device__ __forceinline__ void row_stats(const float* values, uint32_t count, uint32_t lane, uint32_t lanes, float inverse, float& mean, float& square) {
    const float k = lane < count ? values[lane] : 0.f;
    float s = 0.f, q = 0.f;
    uint32_t i = lane + lanes;
    for (; i + 3u * lanes < count; i += 4u * lanes) {
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = values[i + e * lanes] - k;
#pragma unroll
        for (int e = 0; e < 4; ++e) { s += d[e]; q = __builtin_fmaf(d[e], d[e], q); }
    }
    for (; i < count; i += lanes) { const float d = values[i] - k; s += d; q = __builtin_fmaf(d, d, q); }
    const float n = lane < count ? (float)((count - lane - 1u) / lanes + 1u) : 0.f, own = n > 0.f ? __builtin_fmaf(s, reciprocal(n), k) : 0.f;
    mean = add_lanes(own * n, lanes) * inverse;
    const float d = own - mean;
    square = n > 0.f ? fmaxf(__builtin_fmaf(-s * reciprocal(n), s, q), 0.f) : 0.f;
    square = s != s ? s : square;                                         // (a maximum would lose a NaN)
    square = add_lanes(__builtin_fmaf(n * d, d, square), lanes);
}
__device__ __forceinline__ float row_sum(const float* values, uint32_t count, uint32_t lane, uint32_t lanes) {
    float s[2] = {0.f, 0.f};
    uint32_t i = lane;
    for (; i + 3u * lanes < count; i += 4u * lanes) {
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = values[i + e * lanes];
        s[0] += d[0] + d[1]; s[1] += d[2] + d[3];
    }
    for (; i < count; i += lanes) s[0] += values[i];
    return add_lanes(s[0] + s[1], lanes);
}

template <int VEC, int K>
__device__ __forceinline__ void rows_body(float* y, float* means, float* rstds, const float* x, const float* scale, const float* shift, const NormParams& P) {
    const uint32_t block = xcd_contiguous_block();
    const Span<VEC> span(P, block % P.spans);
    const uint32_t n0 = block / P.spans * P.M, here = min(P.M, P.N - n0), side = P.M / K;
    const bool use = span.p < side && span.owns();
    const uint64_t base = (uint64_t)n0 * P.C + span.c0;
    const uint32_t bytes = ((here - 1u) * P.C + span.width) * 4u;
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(x + base, bytes);
    float v[K][VEC], gamma[VEC], beta[VEC];
    auto at = [&](int i) { const uint32_t m = span.p + i * side; return use && m < here ? (m * P.C + span.col * VEC) * 4u : NOWHERE; };
#pragma unroll
    for (int i = 0; i < K; ++i) load<VEC>(v[i], x_rsrc, at(i));
    {
        const __amdgpu_buffer_rsrc_t a = make_rsrc(scale + span.c0, span.width * 4u), b = make_rsrc(shift + span.c0, span.width * 4u);
        load<VEC>(gamma, a, span.owns() ? span.col * VEC * 4u : NOWHERE);
        load<VEC>(beta, b, span.owns() ? span.col * VEC * 4u : NOWHERE);
    }
    float* const values = room;
    f32x2* const stats_of = reinterpret_cast<f32x2*>(room + ((P.M * P.span + 1u) & ~1u));      // (pairs lie at even words)
#pragma unroll
    for (int i = 0; i < K; ++i) if (use) put<VEC>(values + (span.p + i * side) * P.span + span.col * VEC, v[i]);
    __syncthreads();
    const float inverse = 1.f / (float)P.cg;
    for_row_groups(P, span.groups, here, [&](uint32_t m, uint32_t g, bool reports, uint32_t first, uint32_t lane, uint32_t lanes) {
        float mean, square;
        row_stats(values + first, P.cg, lane, lanes, inverse, mean, square);
        if (!reports) return;
        const float rstd = 1.f / sqrtf(square * inverse + P.eps);
        stats_of[m * span.groups + g] = f32x2{mean, rstd};
        const uint64_t to = (uint64_t)(n0 + m) * P.G + span.g0 + g;
        if (means) means[to] = mean;
        if (rstds) rstds[to] = rstd;
    });
    __syncthreads();
    if (!use || y == nullptr) return;
    const bool stream = streams_result(P.first);
    const __amdgpu_buffer_rsrc_t y_rsrc = make_rsrc(y + base, bytes);
    const TwoGroups<VEC> two(P, span);
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const uint32_t m = span.p + i * side;
        const f32x2* const from = stats_of + (m < here ? m * span.groups : 0u);
        const f32x2 a = from[two.first], b = from[two.last];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = act_value(z_of((v[i][j] - two.pick(j, a.x, b.x)) * two.pick(j, a.y, b.y), gamma[j], beta[j]), P.act);
        store<VEC>(v[i], y_rsrc, at(i), stream);
    }
}

template <int VEC, int K>
__device__ __forceinline__ void rows_grad_body(float* dx, float* dscale_rows, float* dshift_rows, const float* gs, const float* x, const float* scale, const float* shift,
                                               const float* means, const float* rstds, const NormParams& P) {
    const uint32_t block = xcd_contiguous_block();
    const Span<VEC> span(P, block % P.spans);
    const uint32_t side = P.M / K, sets = (P.N - 1u) / P.M + 1u, row = block / P.spans, rows = gridDim.x / P.spans;
    const bool use = span.p < side && span.owns();
    float* const firsts = room, * const seconds = room + P.M * P.span;
    f32x2* const stats_of = reinterpret_cast<f32x2*>(seconds + P.M * P.span), * const sums_of = stats_of + P.span / P.cg * P.M;
    float gamma[VEC], beta[VEC], d_total[VEC], dh_total[VEC];
    const TwoGroups<VEC> two(P, span);
    {
        const __amdgpu_buffer_rsrc_t a = make_rsrc(scale + span.c0, span.width * 4u), b = make_rsrc(shift + span.c0, span.width * 4u);
        load<VEC>(gamma, a, span.owns() ? span.col * VEC * 4u : NOWHERE);
        load<VEC>(beta, b, span.owns() ? span.col * VEC * 4u : NOWHERE);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { d_total[j] = 0.f; dh_total[j] = 0.f; }
    const float inverse = 1.f / (float)P.cg;
    const bool stream = streams_result(P.first);
    for (uint32_t set = row; set < sets; set += rows) {
        const uint32_t n0 = set * P.M, here = min(P.M, P.N - n0);
        const uint64_t base = (uint64_t)n0 * P.C + span.c0;
        const uint32_t bytes = ((here - 1u) * P.C + span.width) * 4u;
        const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(x + base, bytes), g_rsrc = make_rsrc(gs + base, bytes);
        float v[K][VEC], d[K][VEC];
        auto there = [&](int i) { return use && span.p + i * side < here; };
        auto at = [&](int i) { return there(i) ? ((span.p + i * side) * P.C + span.col * VEC) * 4u : NOWHERE; };
#pragma unroll
        for (int i = 0; i < K; ++i) { load<VEC>(v[i], x_rsrc, at(i)); load<VEC>(d[i], g_rsrc, at(i)); }
        // the statistics of these rows, by way of shared memory
        __syncthreads();                                                 // (what the set before has left has been read)
        for (uint32_t e = threadIdx.x; e < P.M * span.groups; e += blockDim.x) {
            const uint32_t m = e / span.groups, g = e - m * span.groups;
            const uint64_t from = (uint64_t)(n0 + m) * P.G + span.g0 + g;
            stats_of[e] = m < here ? f32x2{means[from], rstds[from]} : f32x2{0.f, 0.f};
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const f32x2* const from = stats_of + (use ? (span.p + i * side) * span.groups : 0u);
            const f32x2 a = from[two.first], b = from[two.last];
            float product[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] = there(i) ? (v[i][j] - two.pick(j, a.x, b.x)) * two.pick(j, a.y, b.y) : 0.f;
                d[i][j] = there(i) ? act_gradient(d[i][j], z_of(v[i][j], gamma[j], beta[j]), P.act) : 0.f;
                d_total[j] += d[i][j]; dh_total[j] = __builtin_fmaf(d[i][j], v[i][j], dh_total[j]);
                d[i][j] *= gamma[j];
                product[j] = d[i][j] * v[i][j];
            }
            if (use) {
                put<VEC>(firsts + (span.p + i * side) * P.span + span.col * VEC, d[i]);
                put<VEC>(seconds + (span.p + i * side) * P.span + span.col * VEC, product);
            }
        }
        if (dx == nullptr) continue;
        __syncthreads();
        for_row_groups(P, span.groups, here, [&](uint32_t m, uint32_t g, bool reports, uint32_t first, uint32_t lane, uint32_t lanes) {
            const float a = row_sum(firsts + first, P.cg, lane, lanes), b = row_sum(seconds + first, P.cg, lane, lanes);
            if (reports) sums_of[m * span.groups + g] = f32x2{a * inverse, b * inverse};
        });
        __syncthreads();
        const __amdgpu_buffer_rsrc_t dx_rsrc = make_rsrc(dx + base, bytes);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const uint32_t row0 = use ? (span.p + i * side) * span.groups : 0u;
            const f32x2 a = sums_of[row0 + two.first], b = sums_of[row0 + two.last];
            const float ra = stats_of[row0 + two.first].y, rb = stats_of[row0 + two.last].y;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = two.pick(j, ra, rb) * (d[i][j] - two.pick(j, a.x, b.x) - v[i][j] * two.pick(j, a.y, b.y));
            store<VEC>(v[i], dx_rsrc, at(i), stream);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VEC; ++j) if (use) { firsts[span.p * P.span + span.col * VEC + j] = d_total[j]; seconds[span.p * P.span + span.col * VEC + j] = dh_total[j]; }
    __syncthreads();
    const uint64_t to = (uint64_t)row * P.C + span.c0;
    write_channel_sums(firsts, seconds, side, P.span, span.width, dshift_rows + to, dscale_rows + to);
}

// ---------------------------------------------------------------------------------------------- single positions, wide groups

// Samples of one position with wide groups: a block to a group of a row, K vectors of it to a thread.

// The sum of v over the block, in every thread. `parts`: 16 floats of shared memory for this sum alone.
__device__ __forceinline__ float block_sum(float v, float* parts) {
    v = add_lanes(v, 64u);
    const uint32_t waves = blockDim.x >> 6;
    if ((threadIdx.x & 63u) == 0u) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    return add_lanes((threadIdx.x & 15u) < waves ? parts[threadIdx.x & 15u] : 0.f, 16u);
}

template <int VEC, int K>
struct Wide {
    uint32_t g, cg, lane0;                       // the group, its channels, this thread's first
    __device__ Wide(const NormParams& P, uint32_t group) : g(group), cg(P.cg), lane0(threadIdx.x * VEC) {}
    __device__ uint32_t channel(int i) const { return lane0 + (uint32_t)i * blockDim.x * VEC; }      // (whole vectors: VEC divides cg)
    __device__ bool there(int i) const { return channel(i) < cg; }
    __device__ uint32_t at(int i) const { return there(i) ? channel(i) * 4u : NOWHERE; }
    __device__ __amdgpu_buffer_rsrc_t of_row(const float* p, const NormParams& P, uint32_t n) const { return make_rsrc(p + (uint64_t)n * P.C + (uint64_t)g * cg, cg * 4u); }
    __device__ __amdgpu_buffer_rsrc_t of_channels(const float* p) const { return make_rsrc(p + (uint64_t)g * cg, cg * 4u); }
};

template <int VEC, int K>
__device__ __forceinline__ void wide_body(float* y, float* means, float* rstds, const float* x, const float* scale, const float* shift, const NormParams& P) {
    __shared__ float parts[2][16];
    const uint32_t n = blockIdx.x / P.G;
    const Wide<VEC, K> wide(P, blockIdx.x - n * P.G);
    const __amdgpu_buffer_rsrc_t x_rsrc = wide.of_row(x, P, n);
    float v[K][VEC], sum = 0.f, square = 0.f;
#pragma unroll
    for (int i = 0; i < K; ++i) load<VEC>(v[i], x_rsrc, wide.at(i));
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += v[i][j];                     // (beyond the group: zeros)
    const float inverse = 1.f / (float)wide.cg, mean = block_sum(sum, parts[0]) * inverse;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) { const float d = wide.there(i) ? v[i][j] - mean : 0.f; square = __builtin_fmaf(d, d, square); }
    const float rstd = 1.f / sqrtf(block_sum(square, parts[1]) * inverse + P.eps);
    if (threadIdx.x == 0u) {
        if (means) means[(uint64_t)n * P.G + wide.g] = mean;
        if (rstds) rstds[(uint64_t)n * P.G + wide.g] = rstd;
    }
    if (y == nullptr) return;
    const bool stream = streams_result(P.first);
    const __amdgpu_buffer_rsrc_t y_rsrc = wide.of_row(y, P, n), gammas = wide.of_channels(scale), betas = wide.of_channels(shift);
#pragma unroll
    for (int i = 0; i < K; ++i) {
        float gamma[VEC], beta[VEC];
        load<VEC>(gamma, gammas, wide.at(i)); load<VEC>(beta, betas, wide.at(i));
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = act_value(z_of((v[i][j] - mean) * rstd, gamma[j], beta[j]), P.act);
        store<VEC>(v[i], y_rsrc, wide.at(i), stream);
    }
}

// Its gradient: a block takes one row after the other, gridDim.x / G rows apart, and keeps what they add to its channels' dscale and dshift.
template <int VEC, int K>
__device__ __forceinline__ void wide_grad_body(float* dx, float* dscale_rows, float* dshift_rows, const float* gs, const float* x, const float* scale, const float* shift,
                                               const float* means, const float* rstds, const NormParams& P) {
    __shared__ float parts[4][16];
    const uint32_t row = blockIdx.x / P.G, rows = gridDim.x / P.G;
    const Wide<VEC, K> wide(P, blockIdx.x - row * P.G);
    const __amdgpu_buffer_rsrc_t gammas = wide.of_channels(scale), betas = wide.of_channels(shift);
    const float inverse = 1.f / (float)wide.cg;
    const bool stream = streams_result(P.first);
    float d_total[K][VEC], dh_total[K][VEC];
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) { d_total[i][j] = 0.f; dh_total[i][j] = 0.f; }
    uint32_t turn = 0;                                                    // (two rows' sums in turn: a wave may be one row ahead of another)
    for (uint32_t n = row; n < P.N; n += rows, turn ^= 2u) {
        const __amdgpu_buffer_rsrc_t x_rsrc = wide.of_row(x, P, n), g_rsrc = wide.of_row(gs, P, n);
        const float mean = means[(uint64_t)n * P.G + wide.g], rstd = rstds[(uint64_t)n * P.G + wide.g];
        float v[K][VEC], d[K][VEC], a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) { load<VEC>(v[i], x_rsrc, wide.at(i)); load<VEC>(d[i], g_rsrc, wide.at(i)); }
#pragma unroll
        for (int i = 0; i < K; ++i) {
            float gamma[VEC], beta[VEC];
            load<VEC>(gamma, gammas, wide.at(i)); load<VEC>(beta, betas, wide.at(i));
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] = wide.there(i) ? (v[i][j] - mean) * rstd : 0.f;
                d[i][j] = wide.there(i) ? act_gradient(d[i][j], z_of(v[i][j], gamma[j], beta[j]), P.act) : 0.f;
                d_total[i][j] += d[i][j]; dh_total[i][j] = __builtin_fmaf(d[i][j], v[i][j], dh_total[i][j]);
                d[i][j] *= gamma[j];
                a += d[i][j]; b = __builtin_fmaf(d[i][j], v[i][j], b);
            }
        }
        if (dx == nullptr) continue;
        a = block_sum(a, parts[turn]) * inverse; b = block_sum(b, parts[turn + 1u]) * inverse;
        const __amdgpu_buffer_rsrc_t dx_rsrc = wide.of_row(dx, P, n);
#pragma unroll
        for (int i = 0; i < K; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = rstd * (d[i][j] - a - v[i][j] * b);
            store<VEC>(v[i], dx_rsrc, wide.at(i), stream);
        }
    }
    const uint64_t to = (uint64_t)row * P.C;
    const __amdgpu_buffer_rsrc_t first = wide.of_channels(dshift_rows + to), second = wide.of_channels(dscale_rows + to);
#pragma unroll
    for (int i = 0; i < K; ++i) { store<VEC>(d_total[i], first, wide.at(i), false); store<VEC>(dh_total[i], second, wide.at(i), false); }
}

// ---------------------------------------------------------------------------------------------- samples in chunks

// Which chunk of which sample and span a block has.
struct Chunk {
    uint32_t number, n, from, count, chunk;
    // `last_first`: in the opposite order. What a launch reads that another one has read just before is taken from its end: that is what the 256 MB
    // behind the L2s still hold.
    __device__ Chunk(const NormParams& P, bool last_first) {
        const uint32_t block = last_first ? gridDim.x - 1u - blockIdx.x : blockIdx.x;
        number = block % P.spans;
        const uint32_t rest = block / P.spans;
        chunk = rest % P.chunks; n = rest / P.chunks;
        from = chunk * P.chunk; count = min(P.chunk, P.S - from);
    }
};

// U positions of a chunk in flight at a time: step(values, how many of the U are there)
template <int VEC, int U, class Step>
__device__ __forceinline__ void walk(const NormParams& P, const Span<VEC>& span, const Chunk& chunk, const float* x, Step step) {
    const uint32_t mine = span.p < P.P && span.owns() ? share_of(chunk.count, span.p, P.P) : 0u;
    const uint64_t base = ((uint64_t)chunk.n * P.S + chunk.from) * P.C + span.c0;
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(x + base, ((chunk.count - 1u) * P.C + span.width) * 4u);
    for (uint32_t i = 0; i < mine; i += U) {
        float v[U][VEC];
#pragma unroll
        for (int k = 0; k < U; ++k) load<VEC>(v[k], rsrc, i + k < mine ? ((span.p + (i + k) * P.P) * P.C + span.col * VEC) * 4u : NOWHERE);
        step(v, min(mine - i, (uint32_t)U), i);
    }
}

template <int VEC>
__device__ __forceinline__ void stats_body(float* partial, const float* x, const NormParams& P) {
    const Chunk chunk(P, false);
    const Span<VEC> span(P, chunk.number);
    constexpr int U = 8;
    float mean[VEC], square[VEC], n = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { mean[j] = 0.f; square[j] = 0.f; }
    walk<VEC, U>(P, span, chunk, x, [&](const float (&v)[U][VEC], uint32_t here, uint32_t) {
        // mean and squared deviations of these, joined with those before
        const float count = (float)here, inverse = 1.f / count, share = count / (n + count), both = n * share;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float sum = 0.f, sq = 0.f;
#pragma unroll
            for (int k = 0; k < U; ++k) sum += v[k][j];
            const float m = sum * inverse;
#pragma unroll
            for (int k = 0; k < U; ++k) { const float d = (uint32_t)k < here ? v[k][j] - m : 0.f; sq = __builtin_fmaf(d, d, sq); }
            const float d = m - mean[j];
            square[j] += __builtin_fmaf(d * d, both, sq);
            mean[j] = __builtin_fmaf(d, share, mean[j]);
        }
        n += count;
    });
    const uint32_t entries = P.P * P.span;
    float* const sums = room, * const squares = room + entries;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (span.p < P.P && span.col * VEC + j < P.span) { sums[span.p * P.span + span.col * VEC + j] = mean[j] * n; squares[span.p * P.span + span.col * VEC + j] = square[j]; }
    __syncthreads();
    const uint32_t each = chunk.count / P.P, more = chunk.count % P.P;
    auto count = [&](uint32_t q) { return (float)(each + (q < more ? 1u : 0u)); };
    JoinStats<decltype(count)> join{sums, squares, count};
    const uint32_t piece = P.pieces == 1u ? 0u : chunk.number % P.pieces;
    for_groups(P, span.groups, P.pieces == 1u ? P.cg : span.width, 1u, join, [&](uint32_t, uint32_t g, bool reports, const JoinStats<decltype(count)>& found) {
        if (!reports) return;
        float* const to = partial + 2u * ((((uint64_t)chunk.n * P.G + span.g0 + g) * P.pieces + piece) * P.chunks + chunk.chunk);
        to[0] = found.mean; to[1] = found.square;
    });
}

// Joins what the chunks and pieces of the groups of a span have left, a few lanes to a group: all groups at once, but no more than eight parts to a lane, which it
// reads together (2 x 1196 x 256 in 64 groups, 75 chunks, forward and gradient: a wave to a group 54 us, so 33). `use(group, mean or first sum, deviations or second sum)` in the lane that reports.
// STATS: means and squared deviations; else two sums.
template <bool STATS, int VEC, class Use>
__device__ __forceinline__ void join_chunks(const NormParams& P, const Span<VEC>& span, uint32_t n, const float* partial, Use use) {
    constexpr uint32_t HELD = 8;
    const uint32_t parts = P.chunks * P.pieces, groups = max(P.span / P.cg, 1u);
    auto log2_below = [](uint32_t v) { return 31u - (uint32_t)__clz((int)v); };
    const uint32_t log2_lanes = min(6u, max(log2_below(max(blockDim.x / groups, 1u)), log2_below(2u * ((parts - 1u) / HELD) + 1u))), lanes = 1u << log2_lanes;
    const uint32_t lane = threadIdx.x & (lanes - 1u), sets = blockDim.x >> log2_lanes;
    const uint32_t start = threadIdx.x >> log2_lanes;
    for (uint32_t g = start; g - start < span.groups; g += sets) {
        const bool there = g < span.groups;
        const f32x2* const from = reinterpret_cast<const f32x2*>(partial) + ((uint64_t)n * P.G + span.g0 + (there ? g : 0u)) * parts;
        auto count = [&](uint32_t k) {
            const uint32_t piece = k / P.chunks, c = k - piece * P.chunks;
            const uint32_t channels = P.pieces == 1u ? P.cg : min(P.span, P.cg - piece * P.span);
            return (float)min(P.chunk, P.S - c * P.chunk) * (float)channels;
        };
        float a = 0.f, b = 0.f, total = 0.f;
        auto first = [&](f32x2 part, uint32_t k) {
            if constexpr (STATS) { const float c = count(k); a = __builtin_fmaf(part.x, c, a); total += c; }
            else { a += part.x; b += part.y; }
        };
        auto second = [&](f32x2 part, uint32_t k) { const float d = part.x - a; b += __builtin_fmaf(count(k) * d, d, part.y); };
        if (parts <= HELD * lanes) {
            f32x2 mine[HELD];
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) mine[i] = i * lanes + lane < parts ? from[i * lanes + lane] : f32x2{0.f, 0.f};
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) if (i * lanes + lane < parts) first(mine[i], i * lanes + lane);
            a = add_lanes(a, lanes);
            if constexpr (STATS) {
                a /= add_lanes(total, lanes);
#pragma unroll
                for (uint32_t i = 0; i < HELD; ++i) if (i * lanes + lane < parts) second(mine[i], i * lanes + lane);
            }
        } else {
            for (uint32_t k = lane; k < parts; k += lanes) first(from[k], k);
            a = add_lanes(a, lanes);
            if constexpr (STATS) {
                a /= add_lanes(total, lanes);
                for (uint32_t k = lane; k < parts; k += lanes) second(from[k], k);
            }
        }
        b = add_lanes(b, lanes);
        if (there && lane == 0u) use(g, a, b);
    }
}

template <int VEC>
__device__ __forceinline__ void apply_body(float* y, float* means, float* rstds, const float* partial, const float* x, const float* scale, const float* shift, const NormParams& P) {
    const Chunk chunk(P, true);
    const Span<VEC> span(P, chunk.number);
    float* const mean_of = room, * const rstd_of = room + max(P.span / P.cg, 1u);
    const float inverse = 1.f / ((float)P.S * (float)P.cg);
    join_chunks<true>(P, span, chunk.n, partial, [&](uint32_t g, float mean, float square) {
        const float rstd = 1.f / sqrtf(square * inverse + P.eps);
        mean_of[g] = mean; rstd_of[g] = rstd;
        if (chunk.chunk == 0u && (P.pieces == 1u || chunk.number % P.pieces == 0u)) {
            const uint64_t at = (uint64_t)chunk.n * P.G + span.g0 + g;
            if (means) means[at] = mean;
            if (rstds) rstds[at] = rstd;
        }
    });
    __syncthreads();
    if (y == nullptr || !span.owns()) return;
    float mean[VEC], rstd[VEC], gamma[VEC], beta[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const uint32_t g = span.group_of(P, j);
        mean[j] = mean_of[g]; rstd[j] = rstd_of[g]; gamma[j] = scale[span.c + j]; beta[j] = shift[span.c + j];
    }
    const bool stream = streams_result(P.first);
    const uint64_t base = ((uint64_t)chunk.n * P.S + chunk.from) * P.C + span.c0;
    const __amdgpu_buffer_rsrc_t y_rsrc = make_rsrc(y + base, ((chunk.count - 1u) * P.C + span.width) * 4u);
    constexpr int U = 8;
    walk<VEC, U>(P, span, chunk, x, [&](float (&v)[U][VEC], uint32_t here, uint32_t i) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[k][j] = act_value(z_of((v[k][j] - mean[j]) * rstd[j], gamma[j], beta[j]), P.act);
            store<VEC>(v[k], y_rsrc, (uint32_t)k < here ? ((span.p + (i + k) * P.P) * P.C + span.col * VEC) * 4u : NOWHERE, stream);
        }
    });
}

// hat and d of U positions of x and g: step(hat, d, how many, the first one's number)
template <int VEC, int U, class Step>
__device__ __forceinline__ void walk_gradient(const NormParams& P, const Span<VEC>& span, const Chunk& chunk, const float* gs, const float* x, const float* scale, const float* shift,
                                              const float* means, const float* rstds, float (&rstd)[VEC], float (&gamma)[VEC], Step step) {
    const bool owns = span.p < P.P && span.owns();
    float mean[VEC], beta[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const uint64_t at = (uint64_t)chunk.n * P.G + span.g0 + span.group_of(P, j);
        mean[j] = owns ? means[at] : 0.f; rstd[j] = owns ? rstds[at] : 0.f;
        gamma[j] = owns ? scale[span.c + j] : 0.f; beta[j] = owns ? shift[span.c + j] : 0.f;
    }
    const uint32_t mine = owns ? share_of(chunk.count, span.p, P.P) : 0u;
    const uint64_t base = ((uint64_t)chunk.n * P.S + chunk.from) * P.C + span.c0;
    const uint32_t bytes = ((chunk.count - 1u) * P.C + span.width) * 4u;
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(x + base, bytes), g_rsrc = make_rsrc(gs + base, bytes);
    for (uint32_t i = 0; i < mine; i += U) {
        float v[U][VEC], d[U][VEC];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint32_t at = i + k < mine ? ((span.p + (i + k) * P.P) * P.C + span.col * VEC) * 4u : NOWHERE;
            load<VEC>(v[k], x_rsrc, at); load<VEC>(d[k], g_rsrc, at);
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[k][j] = (v[k][j] - mean[j]) * rstd[j];
                d[k][j] = act_gradient(d[k][j], z_of(v[k][j], gamma[j], beta[j]), P.act);
            }
        step(v, d, min(mine - i, (uint32_t)U), i);
    }
}

// A block takes one sample after the other, as many apart as there are blocks for each chunk and span (of most sizes: one), and leaves one row of sums for dscale
// and dshift of all of them. (A row for each of many samples of few positions would be as large as the samples.)
template <int VEC>
__device__ __forceinline__ void grad_sums_body(float* partial, float* dscale_rows, float* dshift_rows, const float* gs, const float* x, const float* scale, const float* shift,
                                               const float* means, const float* rstds, const NormParams& P) {
    Chunk chunk(P, false);
    const Span<VEC> span(P, chunk.number);
    constexpr int U = 4;
    const uint32_t first_n = chunk.n, side = gridDim.x / (P.spans * P.chunks), entries = P.P * P.span;
    float* const firsts = room, * const seconds = room + entries;
    const uint32_t piece = P.pieces == 1u ? 0u : chunk.number % P.pieces;
    auto leave = [&](const float (&a)[VEC], const float (&b)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (span.p < P.P && span.col * VEC + j < P.span) { firsts[span.p * P.span + span.col * VEC + j] = a[j]; seconds[span.p * P.span + span.col * VEC + j] = b[j]; }
        __syncthreads();
    };
    float rstd[VEC], gamma[VEC], A_total[VEC], B_total[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { A_total[j] = 0.f; B_total[j] = 0.f; }
    for (; chunk.n < P.N; chunk.n += side) {
        float A[VEC], B[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { A[j] = 0.f; B[j] = 0.f; }
        walk_gradient<VEC, U>(P, span, chunk, gs, x, scale, shift, means, rstds, rstd, gamma, [&](const float (&hat)[U][VEC], const float (&d)[U][VEC], uint32_t here, uint32_t) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float a = 0.f, b = 0.f;
#pragma unroll
                for (int k = 0; k < U; ++k) { const float dk = (uint32_t)k < here ? d[k][j] : 0.f; a += dk; b = (uint32_t)k < here ? __builtin_fmaf(dk, hat[k][j], b) : b; }
                A[j] += a; B[j] += b;
            }
        });
        if (chunk.n != first_n) __syncthreads();                          // (what the sample before has left has been read)
        leave(A, B);
        JoinSums join{firsts, seconds, scale + span.c0};
        for_groups(P, span.groups, P.pieces == 1u ? P.cg : span.width, 1u, join, [&](uint32_t, uint32_t g, bool reports, const JoinSums& found) {
            if (!reports) return;
            float* const to = partial + 2u * ((((uint64_t)chunk.n * P.G + span.g0 + g) * P.pieces + piece) * P.chunks + chunk.chunk);
            to[0] = found.a; to[1] = found.b;
        });
#pragma unroll
        for (int j = 0; j < VEC; ++j) { A_total[j] += A[j]; B_total[j] += B[j]; }
    }
    if (first_n + side < P.N) {                                           // (else they are there)
        __syncthreads();
        leave(A_total, B_total);
    }
    const uint64_t to = ((uint64_t)first_n * P.chunks + chunk.chunk) * P.C + span.c0;
    write_channel_sums(firsts, seconds, P.P, P.span, span.width, dshift_rows + to, dscale_rows + to);
}

template <int VEC>
__device__ __forceinline__ void grad_apply_body(float* dx, const float* partial, const float* gs, const float* x, const float* scale, const float* shift, const float* means,
                                                const float* rstds, const NormParams& P) {
    const Chunk chunk(P, true);
    const Span<VEC> span(P, chunk.number);
    float* const a_of = room, * const b_of = room + max(P.span / P.cg, 1u);
    const float inverse = 1.f / ((float)P.S * (float)P.cg);
    join_chunks<false>(P, span, chunk.n, partial, [&](uint32_t g, float a, float b) { a_of[g] = a * inverse; b_of[g] = b * inverse; });
    __syncthreads();
    if (!span.owns()) return;
    float rstd[VEC], gamma[VEC], a[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { const uint32_t g = span.group_of(P, j); a[j] = a_of[g]; b[j] = b_of[g]; }
    const bool stream = streams_result(P.first);
    const uint64_t base = ((uint64_t)chunk.n * P.S + chunk.from) * P.C + span.c0;
    const __amdgpu_buffer_rsrc_t dx_rsrc = make_rsrc(dx + base, ((chunk.count - 1u) * P.C + span.width) * 4u);
    constexpr int U = 4;
    walk_gradient<VEC, U>(P, span, chunk, gs, x, scale, shift, means, rstds, rstd, gamma, [&](float (&hat)[U][VEC], const float (&d)[U][VEC], uint32_t here, uint32_t i) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) hat[k][j] = rstd[j] * (__builtin_fmaf(d[k][j], gamma[j], -a[j]) - hat[k][j] * b[j]);
            store<VEC>(hat[k], dx_rsrc, (uint32_t)k < here ? ((span.p + (i + k) * P.P) * P.C + span.col * VEC) * 4u : NOWHERE, stream);
        }
    });
}

// ---------------------------------------------------------------------------------------------- kernels

#define HELD(VEC, K, THREADS)                                                                                                                                       \
    extern "C" __global__ __launch_bounds__(THREADS) void group_norm_held_v##VEC##_k##K##_t##THREADS(float* y, float* means, float* rstds, const float* x,          \
                                                                                                     const float* scale, const float* shift, NormParams P) {        \
        held_body<VEC, K>(y, means, rstds, x, scale, shift, P);                                                                                                     \
    }
#define HELD_GRAD(VEC, K, THREADS)                                                                                                                                  \
    extern "C" __global__ __launch_bounds__(THREADS) void group_norm_held_grad_v##VEC##_k##K##_t##THREADS(float* dx, float* dscale_rows, float* dshift_rows,        \
            const float* g, const float* x, const float* scale, const float* shift, const float* means, const float* rstds, NormParams P) {                         \
        held_grad_body<VEC, K>(dx, dscale_rows, dshift_rows, g, x, scale, shift, means, rstds, P);                                                                  \
    }
#define ROWS(VEC, K, THREADS)                                                                                                                                       \
    extern "C" __global__ __launch_bounds__(THREADS) void group_norm_rows_v##VEC##_k##K##_t##THREADS(float* y, float* means, float* rstds, const float* x,          \
                                                                                                     const float* scale, const float* shift, NormParams P) {        \
        rows_body<VEC, K>(y, means, rstds, x, scale, shift, P);                                                                                                     \
    }
#define ROWS_GRAD(VEC, K, THREADS)                                                                                                                                  \
    extern "C" __global__ __launch_bounds__(THREADS) void group_norm_rows_grad_v##VEC##_k##K##_t##THREADS(float* dx, float* dscale_rows, float* dshift_rows,        \
            const float* g, const float* x, const float* scale, const float* shift, const float* means, const float* rstds, NormParams P) {                         \
        rows_grad_body<VEC, K>(dx, dscale_rows, dshift_rows, g, x, scale, shift, means, rstds, P);                                                                  \
    }
#define CHUNKED(VEC)                                                                                                                                                \
    extern "C" __global__ __launch_bounds__(256) void group_norm_stats_v##VEC(float* partial, const float* x, NormParams P) { stats_body<VEC>(partial, x, P); }     \
    extern "C" __global__ __launch_bounds__(256) void group_norm_apply_v##VEC(float* y, float* means, float* rstds, const float* partial, const float* x,           \
                                                                              const float* scale, const float* shift, NormParams P) {                               \
        apply_body<VEC>(y, means, rstds, partial, x, scale, shift, P);                                                                                              \
    }                                                                                                                                                               \
    extern "C" __global__ __launch_bounds__(256) void group_norm_grad_sums_v##VEC(float* partial, float* dscale_rows, float* dshift_rows, const float* g,           \
            const float* x, const float* scale, const float* shift, const float* means, const float* rstds, NormParams P) {                                         \
        grad_sums_body<VEC>(partial, dscale_rows, dshift_rows, g, x, scale, shift, means, rstds, P);                                                                \
    }                                                                                                                                                               \
    extern "C" __global__ __launch_bounds__(256) void group_norm_grad_apply_v##VEC(float* dx, const float* partial, const float* g, const float* x,                 \
            const float* scale, const float* shift, const float* means, const float* rstds, NormParams P) {                                                         \
        grad_apply_body<VEC>(dx, partial, g, x, scale, shift, means, rstds, P);                                                                                     \
    }
HELD(4, 4, 256)  HELD(4, 16, 256)  HELD(4, 4, 1024)  HELD(4, 16, 1024)  HELD(1, 4, 256)  HELD(1, 16, 256)  HELD(1, 8, 1024)
HELD_GRAD(4, 2, 256)  HELD_GRAD(4, 8, 256)  HELD_GRAD(4, 2, 1024)  HELD_GRAD(4, 4, 1024)  HELD_GRAD(1, 4, 256)  HELD_GRAD(1, 16, 256)  HELD_GRAD(1, 4, 1024)
ROWS(4, 1, 256)  ROWS(4, 2, 256)  ROWS(4, 4, 256)
ROWS(1, 1, 256)  ROWS(1, 4, 256)  ROWS(1, 8, 256)
ROWS_GRAD(4, 1, 256)  ROWS_GRAD(4, 2, 256)
ROWS_GRAD(1, 1, 256)  ROWS_GRAD(1, 4, 256)  ROWS_GRAD(1, 8, 256)
#define WIDE(VEC, K, THREADS)                                                                                                                                       \
    extern "C" __global__ __launch_bounds__(THREADS) void group_norm_wide_v##VEC##_k##K##_t##THREADS(float* y, float* means, float* rstds, const float* x,          \
                                                                                                     const float* scale, const float* shift, NormParams P) {        \
        wide_body<VEC, K>(y, means, rstds, x, scale, shift, P);                                                                                                     \
    }
#define WIDE_GRAD(VEC, K, THREADS)                                                                                                                                  \
    extern "C" __global__ __launch_bounds__(THREADS) void group_norm_wide_grad_v##VEC##_k##K##_t##THREADS(float* dx, float* dscale_rows, float* dshift_rows,        \
            const float* g, const float* x, const float* scale, const float* shift, const float* means, const float* rstds, NormParams P) {                         \
        wide_grad_body<VEC, K>(dx, dscale_rows, dshift_rows, g, x, scale, shift, means, rstds, P);                                                                  \
    }
WIDE(4, 2, 256)  WIDE(4, 8, 256)  WIDE(4, 8, 1024)  WIDE(1, 4, 256)  WIDE(1, 8, 256)  WIDE(1, 8, 1024)
WIDE_GRAD(4, 2, 256)  WIDE_GRAD(4, 4, 256)  WIDE_GRAD(4, 4, 512)  WIDE_GRAD(4, 4, 1024)  WIDE_GRAD(1, 4, 256)  WIDE_GRAD(1, 8, 256)  WIDE_GRAD(1, 8, 1024)
CHUNKED(4)
CHUNKED(1)

// Sums of the columns of two arrays [rows, C]: 32 columns to a block, and 32 lanes that take every 32nd row of them each. (1024 rows of 256: 64 columns to a
// block 10 us, 32 6: a launch of few blocks, bound by how many loads a lane has behind one another.)
extern "C" __global__ __launch_bounds__(1024) void group_norm_columns(float* first, float* second, const float* first_rows, const float* second_rows, uint32_t rows, uint32_t C) {
    __shared__ float parts[32][33];
    const uint32_t blocks = (C + 31u) / 32u, lane = threadIdx.x & 31u, side = threadIdx.x >> 5, c = blockIdx.x % blocks * 32u + lane;
    const bool other = blockIdx.x >= blocks;
    const float* const from = other ? second_rows : first_rows;
    float* const to = other ? second : first;
    if (to == nullptr) return;
    float sums[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) sums[k] = 0.f;
    if (c < C) {
        uint32_t r = side;
        for (; r + 224u < rows; r += 256u)
#pragma unroll
            for (int k = 0; k < 8; ++k) sums[k] += from[(uint64_t)(r + 32u * k) * C + c];
        for (; r < rows; r += 32u) sums[0] += from[(uint64_t)r * C + c];
    }
    parts[side][lane] = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
    __syncthreads();
    // a half wave to a column
    float total = parts[lane][side];
    total = lanes_allreduce(total, 32u, [](float a, float b) { return a + b; });
    const uint32_t column = blockIdx.x % blocks * 32u + side;
    if (lane == 0u && column < C) to[column] = total;
}
