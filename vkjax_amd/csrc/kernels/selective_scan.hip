// Selective state spaces along time over [B, T, C] with N states per channel, and their gradient.
//
//   dt = softplus(delta + bias) (or delta),  f[n] = exp(dt A[c, n]),  h[n] = f[n] h[n] + dt x b[t, n]
//   seen = sum_n c[t, n] h[n] + D x,  y = seen silu(gate)
//   gy = g silu(gate);  the adjoint runs the other way: l[n] = gy c[t, n] + f[t + 1, n] l[n] (behind the last step: the last state's cotangent)
//   e[n] = l f h[t - 1];  ddt = sum_n e A + x sum_n l b;  dx = dt sum_n l b + D gy;  db = sum over channels of l dt x;  dc = sum over channels of gy h
//   dA = sum e dt;  dD = sum gy x;  ddelta = ddt sigmoid(delta + bias);  dbias = sum ddelta;  dgate = g seen silu'(gate);  dstate = f l at the first step
// From a sequence's length on the state stays (dt = 0) and y is 0; nothing is looked at there and nothing comes back.
//
// A block has 64 channels, a lane of each of its M waves one of them and NS of its states in registers, so b and c, which all channels of a sequence share, come
// from shared memory, a vector for all lanes. What a step needs once per channel (dt, the gates, loads and stores) is shared out: of every 8 steps a wave prepares 8 / M and puts them into shared memory, all waves go
// through the 8 steps with their states and leave their parts of the sums over n there, and the wave that has prepared a step adds those up and stores its results. Bound by the
// vector instructions: an exponential takes the time of four of them, a state and step that of eight, in the gradient 27.
// 1 x 16384 x 2048 x 16 states: 122 us for the chunks' states and 177 for the scan (537 million exponentials each, which alone take 60 us: 16 cycles for a wave's 64), 5 between them; the
// arrays alone are 110 us. 4 x 2048 x 2048 x 16 with its gradient: 60 + 111 forward, 67 + 282 + 17 backward. b and c through shared memory, eight steps at a time: read as scalars they took
// 603 us of the former in all.
// A block goes through its steps one after the other; where batch and channels are too few to fill the machine, time is cut into chunks: a first launch leaves each chunk's
// sum of dt (the product of its factors is exp(A sum dt)) and its state from zero, a second one follows those along the chunks, and the third has the state in front of
// each chunk. The gradient's adjoint goes the same way from the last chunk on.
// The forward pass of a gradient keeps the state in front of every 8 steps; the gradient works the 8 states out again, in registers, and goes back over them.
// Sums over channels (db, dc) go through the lanes of a wave by halving (a step of a butterfly leaves each lane half of the values), then through a launch that adds up blocks in
// their order; sums over time (dA, dD, dbias) stay in a lane and are added up the same way. No atomics. All sums and states are fp32.
#include "common.h"

constexpr int KEPT = 8;                          // steps between two kept states

struct ScanParams {
    uint32_t first;                              // (bit 31: the result is stored past the caches)
    uint32_t B, T, C, N, strips, chunks, chunk, softplus;         // strips of 64 channels; steps of a chunk (a multiple of KEPT)
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
// a as the factor of an exponent of 2, one that is infinite as the largest number, whose product with a width of zero (of a step that is not taken) is zero
__device__ __forceinline__ float factor_of(float a) {
    const float v = a * LOG2E;
    return __builtin_fabsf(v) == __builtin_inff() ? __builtin_copysignf(3.4028234e38f, v) : v;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp2_of(z * -LOG2E)); }        // (see norm.hip)
// log(1 + exp(v)) = max(v, 0) + log(1 + q), q = exp(-|v|) in (0, 1]: the logarithm as 2 atanh(s), s = q / (2 + q) <= 1/3, by its series up to s^15 (the rest is below 2e-9 of it),
// so that it keeps its bits also where q is small.
__device__ __forceinline__ float softplus_of(float v) {
    const float q = exp2_of(-__builtin_fabsf(v) * LOG2E), d = 2.f + q, r0 = __builtin_amdgcn_rcpf(d);
    const float s = q * __builtin_fmaf(__builtin_fmaf(-d, r0, 1.f), r0, r0), s2 = s * s;
    float p = 1.f / 15.f;
    p = __builtin_fmaf(p, s2, 1.f / 13.f); p = __builtin_fmaf(p, s2, 1.f / 11.f); p = __builtin_fmaf(p, s2, 1.f / 9.f);
    p = __builtin_fmaf(p, s2, 1.f / 7.f);  p = __builtin_fmaf(p, s2, 1.f / 5.f);  p = __builtin_fmaf(p, s2, 1.f / 3.f);
    p = __builtin_fmaf(p, s2, 1.f);
    const float w = __builtin_fmaf(2.f * s, p, fmaxf(v, 0.f));
    return v != v ? v : w;
}
__device__ __forceinline__ float width_of(float delta, float bias, uint32_t softplus) { return softplus ? softplus_of(delta + bias) : delta + bias; }
__device__ __forceinline__ int sequence_length(const int32_t* lengths, uint32_t b, uint32_t T) {
    return lengths ? min(max(lengths[b], 0), (int)T) : (int)T;
}
template <bool B> struct Whole { static constexpr bool value = B; };
#define STEP_FENCE() __builtin_amdgcn_sched_barrier(0)

// Where a wave is: a strip of channels of one sequence, a chunk of its time, NS of the states. Lanes behind the last channel work on that one again and store nothing.
template <int NS, int M>
struct Place {
    static constexpr int OWN = KEPT / M;         // steps that a wave prepares: wave * OWN ..
    uint32_t b, chunk, strip, lane, wave, c, n0; bool there; int length, begin, end, stop;        // end: of the chunk; steps are taken up to stop
    __device__ Place(const ScanParams& P, const int32_t* lengths) {
        const uint32_t block = xcd_contiguous_block(), rest = block / P.strips;
        lane = threadIdx.x & 63u; wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        strip = block % P.strips; chunk = rest % P.chunks; b = rest / P.chunks;
        n0 = wave * NS;
        there = strip * 64u + lane < P.C; c = min(strip * 64u + lane, P.C - 1u);
        length = sequence_length(lengths, b, P.T);
        begin = (int)(chunk * P.chunk); end = min(begin + (int)P.chunk, (int)P.T); stop = min(end, length);
    }
    // a step's row of an array [B, T, C] (where it begins is the wave's, so that a lane's part of an address is its channel)
    template <class V> __device__ V* row(V* p, const ScanParams& P, int t) const { return p + ((int64_t)b * P.T + t) * P.C; }
    // state i's row in [chunk or kept number][B][N][C]
    template <class V> __device__ V* held(V* p, const ScanParams& P, uint32_t number, int i) const { return p + (((int64_t)number * P.B + b) * P.N + n0 + i) * P.C; }
    __device__ int64_t state(const ScanParams& P, int i) const { return ((int64_t)b * P.C + c) * P.N + n0 + i; }
    __device__ bool has(const ScanParams& P, int i) const { return n0 + i < P.N; }
    __device__ int own(int q) const { return (int)wave * OWN + q; }
    // This thread's element of the eight steps' values from [B, T, N], as they lie in shared memory, [step][NS * M]: zeros for states that there are not. TAKEN_ONLY: and for steps that are not taken,
    // whose width of zero times an infinite value of the last one would be NaN (where they are not gone through, that one again)
    static constexpr int STAGED = KEPT * NS * M;
    template <bool TAKEN_ONLY> __device__ float staged(const float* __restrict__ p, const ScanParams& P, int t0) const {
        const uint32_t s = threadIdx.x / (uint32_t)(NS * M), n = threadIdx.x % (uint32_t)(NS * M);
        const bool has = threadIdx.x < (uint32_t)STAGED && n < P.N;
        if constexpr (TAKEN_ONLY) return has && t0 + (int)s < stop ? p[((int64_t)b * P.T + t0 + (int)s) * P.N + n] : 0.f;
        return has ? p[((int64_t)b * P.T + min(t0 + (int)s, stop - 1)) * P.N + n] : 0.f;
    }
    __device__ void stage(float (&rows)[KEPT][NS * M], float v) const { if (threadIdx.x < (uint32_t)STAGED) (&rows[0][0])[threadIdx.x] = v; }
    // ... and from there to the registers of the wave that has these states
    __device__ void maps(float (&v)[NS], const float (&rows)[KEPT][NS * M], int s) const {
#pragma unroll
        for (int i = 0; i < NS; i += 4) {
            const f32x4 q = *reinterpret_cast<const f32x4*>(&rows[s][n0 + i]);
            v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
        }
    }
    __device__ void factors(float (&a2)[NS], const float* __restrict__ a, const ScanParams& P) const {
#pragma unroll
        for (int i = 0; i < NS; ++i) a2[i] = has(P, i) ? factor_of(a[(int64_t)c * P.N + n0 + i]) : 0.f;
    }
    // behind a wave's writes to shared memory, in front of other waves' reads (of one wave: nothing to wait for but its own writes)
    __device__ static void meet() { if constexpr (M > 1) __syncthreads(); else __builtin_amdgcn_wave_barrier(); }
};

// ---- a chunk's sum of dt, and its state from zero
template <int NS, int M>
__device__ __forceinline__ void scan_chunk_body(float* __restrict__ sums, float* __restrict__ states, const float* __restrict__ x, const float* __restrict__ delta, const float* __restrict__ a,
                                                const float* __restrict__ bmap, const float* __restrict__ bias, const int32_t* __restrict__ lengths, const ScanParams& P) {
    __shared__ float prepared[2][2][KEPT][64];                       // [turn's parity][dt, dt x][step][lane]
    __shared__ __attribute__((aligned(16))) float map[2][KEPT][NS * M];
    const Place<NS, M> at(P, lengths);
    float a2[NS], h[NS] = {}, sum = 0.f, mapped;
    at.factors(a2, a, P);
    const float add = bias ? bias[at.c] : 0.f;
    float xs[at.OWN], ds[at.OWN];
    auto request = [&](int t0) {
#pragma unroll
        for (int q = 0; q < at.OWN; ++q) {
            const int t = min(t0 + at.own(q), at.stop - 1);
            xs[q] = at.row(x, P, t)[at.c]; ds[q] = at.row(delta, P, t)[at.c];
        }
        mapped = at.template staged<true>(bmap, P, t0);
    };
    if (at.begin < at.stop) request(at.begin);
    int parity = 0;
    for (int t0 = at.begin; t0 < at.stop; t0 += KEPT, parity ^= 1) {
#pragma unroll
        for (int q = 0; q < at.OWN; ++q) {
            const bool taken = t0 + at.own(q) < at.stop;
            const float w = width_of(ds[q], add, P.softplus);
            prepared[parity][0][at.own(q)][at.lane] = taken ? w : 0.f;
            prepared[parity][1][at.own(q)][at.lane] = taken ? w * xs[q] : 0.f;
        }
        at.stage(map[parity], mapped);
        if (t0 + KEPT < at.stop) request(t0 + KEPT);
        at.meet();
        float dt[KEPT], u[KEPT], bs[NS], next[NS];
#pragma unroll
        for (int s = 0; s < KEPT; ++s) { dt[s] = prepared[parity][0][s][at.lane]; u[s] = prepared[parity][1][s][at.lane]; }
        at.maps(next, map[parity], 0);
#pragma unroll
        for (int s = 0; s < KEPT; ++s) {
#pragma unroll
            for (int i = 0; i < NS; ++i) bs[i] = next[i];
            if (s + 1 < KEPT) at.maps(next, map[parity], s + 1);
            sum += dt[s];
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = __builtin_fmaf(exp2_of(a2[i] * dt[s]), h[i], u[s] * bs[i]);
            STEP_FENCE();
        }
    }
    if (!at.there) return;
    if (at.wave == 0u) sums[((int64_t)at.chunk * P.B + at.b) * P.C + at.c] = sum;
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if (at.has(P, i)) at.held(states, P, at.chunk, i)[at.c] = h[i];
}

// ---- the state in front of every chunk, in the place of its state from zero; the same for the adjoint from the last chunk on. A block has 64
// (sequence, state, channel) and up to 16 waves, of which each composes eight chunks to a map, h -> product h + own; what lies in front of its first chunk follows from the waves' maps in front of
// it. (Chunk by chunk in one wave, loads wait for one another: 191 chunks took 50 us.)
struct ScanJoinParams { uint32_t first, B, C, N, chunks, back; };
extern "C" __global__ __launch_bounds__(1024) void selective_scan_join(float* __restrict__ states, const float* __restrict__ sums, const float* __restrict__ a,
                                                                       const float* __restrict__ initial, ScanJoinParams P) {
    constexpr uint32_t EACH = 8u;
    __shared__ float maps[2][16][2][64];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t all = P.B * P.N * P.C, place = blockIdx.x * 64u + lane, id = min(place, all - 1u), c = id % P.C, rest = id / P.C, n = rest % P.N, b = rest / P.N;
    const float a2 = factor_of(a[(int64_t)c * P.N + n]);
    const int64_t at = ((int64_t)b * P.C + c) * P.N + n, each = (int64_t)P.B * P.N * P.C, first = ((int64_t)b * P.N + n) * P.C + c;
    const int64_t s_each = (int64_t)P.B * P.C, s_first = (int64_t)b * P.C + c;
    float h = initial ? initial[at] : 0.f;
    for (uint32_t k0 = 0, turn = 0; k0 < P.chunks; k0 += EACH * waves, turn ^= 1u) {
        const uint32_t mine = k0 + EACH * wave;
        auto number = [&](uint32_t k) { return P.back ? P.chunks - 1u - k : k; };
        float own[EACH], factor[EACH], product = 1.f, sum = 0.f;
#pragma unroll
        for (uint32_t q = 0; q < EACH; ++q) {
            const uint32_t k = number(min(mine + q, P.chunks - 1u));
            own[q] = states[first + k * each]; factor[q] = sums[s_first + k * s_each];
        }
#pragma unroll
        for (uint32_t q = 0; q < EACH; ++q) {
            const bool there = mine + q < P.chunks;
            factor[q] = there ? exp2_of(a2 * factor[q]) : 1.f;
            own[q] = there ? own[q] : 0.f;
            product *= factor[q];
            sum = __builtin_fmaf(factor[q], sum, own[q]);
        }
        maps[turn][wave][0][lane] = product; maps[turn][wave][1][lane] = sum;
        __syncthreads();
        float mine_h = h;
        for (uint32_t w = 0; w < waves; ++w) {
            if (w == wave) mine_h = h;
            h = __builtin_fmaf(maps[turn][w][0][lane], h, maps[turn][w][1][lane]);
        }
#pragma unroll
        for (uint32_t q = 0; q < EACH; ++q) {
            if (mine + q < P.chunks && place < all) states[first + number(mine + q) * each] = mine_h;
            mine_h = __builtin_fmaf(factor[q], mine_h, own[q]);
        }
    }
}

// ---- the scan itself, a chunk from the state in front of it
template <int NS, int M>
__device__ __forceinline__ void scan_body(float* __restrict__ y, float* __restrict__ last, float* __restrict__ kept, const float* __restrict__ x, const float* __restrict__ delta,
                                          const float* __restrict__ a, const float* __restrict__ bmap, const float* __restrict__ cmap, const float* __restrict__ through,
                                          const float* __restrict__ gate, const float* __restrict__ state, const int32_t* __restrict__ lengths, const float* __restrict__ bias,
                                          const float* __restrict__ states, const ScanParams& P) {
    __shared__ float prepared[2][KEPT][64], parts[M][KEPT][64];      // [dt, dt x][step][lane], sums over a wave's states
    __shared__ __attribute__((aligned(16))) float map[2][KEPT][NS * M];
    const Place<NS, M> at(P, lengths);
    float a2[NS], h[NS], mapped[2];
    at.factors(a2, a, P);
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = !at.has(P, i) ? 0.f : states ? at.held(states, P, at.chunk, i)[at.c] : state ? state[at.state(P, i)] : 0.f;
    const float add = bias ? bias[at.c] : 0.f, D = through ? through[at.c] : 0.f;
    const bool stream = streams_result(P.first);
    float xs[at.OWN], ds[at.OWN], gs[at.OWN];
    auto request = [&](int t0) {
#pragma unroll
        for (int q = 0; q < at.OWN; ++q) {
            const int t = min(t0 + at.own(q), at.stop - 1);
            xs[q] = at.row(x, P, t)[at.c]; ds[q] = at.row(delta, P, t)[at.c];
            if (gate) gs[q] = at.row(gate, P, t)[at.c];
        }
        mapped[0] = at.template staged<false>(bmap, P, t0); mapped[1] = at.template staged<false>(cmap, P, t0);
    };
    if (at.begin < at.stop) request(at.begin);
    for (int t0 = at.begin; t0 < at.end; t0 += KEPT) {
        if (kept && at.there)
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (at.has(P, i)) at.held(kept, P, (uint32_t)t0 / KEPT, i)[at.c] = h[i];
        float ys[at.OWN], open[at.OWN];
        if (t0 < at.stop) {
#pragma unroll
            for (int q = 0; q < at.OWN; ++q) {
                const bool taken = t0 + at.own(q) < at.stop;
                const float w = width_of(ds[q], add, P.softplus);
                prepared[0][at.own(q)][at.lane] = taken ? w : 0.f;
                prepared[1][at.own(q)][at.lane] = taken ? w * xs[q] : 0.f;
                ys[q] = D * xs[q];
                open[q] = gate ? gs[q] * sigmoid(gs[q]) : 1.f;
            }
            at.stage(map[0], mapped[0]); at.stage(map[1], mapped[1]);
            if (t0 + KEPT < at.stop) request(t0 + KEPT);
            at.meet();
            float dt[KEPT], u[KEPT], bs[NS], cs[NS], next_b[NS], next_c[NS];
#pragma unroll
            for (int s = 0; s < KEPT; ++s) { dt[s] = prepared[0][s][at.lane]; u[s] = prepared[1][s][at.lane]; }
            at.maps(next_b, map[0], 0);
            at.maps(next_c, map[1], 0);
            // (steps behind the last are nobody's: a single one would take the time of eight. Whole turns have a loop of their own, which knows of none: 177 us of a prompt, not 184)
            const int count = at.stop - t0;
            auto steps = [&](auto whole) {
#pragma unroll
            for (int s = 0; s < KEPT; ++s) {
                if (!decltype(whole)::value && s >= count) break;
#pragma unroll
                for (int i = 0; i < NS; ++i) { bs[i] = next_b[i]; cs[i] = next_c[i]; }
                if (s + 1 < KEPT) { at.maps(next_b, map[0], s + 1); at.maps(next_c, map[1], s + 1); }
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    h[i] = __builtin_fmaf(exp2_of(a2[i] * dt[s]), h[i], u[s] * bs[i]);
                    sum = __builtin_fmaf(cs[i], h[i], sum);
                }
                parts[at.wave][s][at.lane] = sum;
                STEP_FENCE();
            }
            };
            if (count >= KEPT) steps(Whole<true>{}); else steps(Whole<false>{});
            at.meet();
#pragma unroll
            for (int q = 0; q < at.OWN; ++q) {
                float sum = parts[0][at.own(q)][at.lane];
#pragma unroll
                for (int w = 1; w < M; ++w) sum += parts[w][at.own(q)][at.lane];
                ys[q] = (through ? ys[q] + sum : sum) * open[q];
            }
        }
        if (y && at.there)
#pragma unroll
            for (int q = 0; q < at.OWN; ++q) {
                const int t = t0 + at.own(q);
                if (t >= at.end) continue;
                const float v = t < at.stop ? ys[q] : 0.f;
                if (stream) __builtin_nontemporal_store(v, at.row(y, P, t) + at.c); else at.row(y, P, t)[at.c] = v;
            }
    }
    if (last && at.there && at.chunk == P.chunks - 1u)
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (at.has(P, i)) last[at.state(P, i)] = h[i];
}

// ---- one step of every sequence: four states to a lane, the states read and written once
struct ScanStepParams { uint32_t first, B, C, N, log2_lanes, softplus, pad; };
extern "C" __global__ __launch_bounds__(256) void selective_scan_step(float* __restrict__ y, float* __restrict__ last, const float* __restrict__ x, const float* __restrict__ delta,
                                                                      const float* __restrict__ a, const float* __restrict__ bmap, const float* __restrict__ cmap,
                                                                      const float* __restrict__ through, const float* __restrict__ gate, const float* __restrict__ state,
                                                                      const int32_t* __restrict__ lengths, const float* __restrict__ bias, ScanStepParams P) {
    const uint64_t id = (uint64_t)blockIdx.x * 256u + threadIdx.x, row = id >> P.log2_lanes;
    const uint32_t lanes = 1u << P.log2_lanes, n0 = ((uint32_t)id & (lanes - 1u)) * 4u;
    const bool there = row < (uint64_t)P.B * P.C;
    const uint64_t r = there ? row : 0;
    const uint32_t b = (uint32_t)(r / P.C), c = (uint32_t)(r - (uint64_t)b * P.C);
    const bool taken = !lengths || lengths[b] > 0, vectors = (P.N & 3u) == 0u;
    auto four = [&](const float* p) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (!p || n0 >= P.N) return v;
        if (vectors) return *reinterpret_cast<const f32x4*>(p + n0);
#pragma unroll
        for (int i = 0; i < 4; ++i) if (n0 + i < P.N) v[i] = p[n0 + i];
        return v;
    };
    f32x4 h = four(state ? state + r * P.N : nullptr);
    float out = 0.f;
    if (taken) {
        const f32x4 as = four(a + (uint64_t)c * P.N), bs = four(bmap + (uint64_t)b * P.N), cs = four(cmap + (uint64_t)b * P.N);
        const float xv = x[r], dt = width_of(delta[r], bias ? bias[c] : 0.f, P.softplus), u = dt * xv;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = __builtin_fmaf(exp2_of(factor_of(as[i]) * dt), h[i], u * bs[i]);
            sum = __builtin_fmaf(cs[i], h[i], sum);
        }
        out = sum;
    }
    out = lanes_allreduce(out, lanes, [](float p, float q) { return p + q; });
    if (!there) return;
    if (y && n0 == 0u) {
        if (taken) {
            if (through) out += through[c] * x[r];
            if (gate) out *= gate[r] * sigmoid(gate[r]);
        }
        y[r] = taken ? out : 0.f;
    }
    if (last && n0 < P.N) {
        if (vectors) *reinterpret_cast<f32x4*>(last + r * P.N + n0) = h;
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) if (n0 + i < P.N) last[r * P.N + n0 + i] = h[i];
    }
}

// ---- the adjoint of a chunk from zero
template <int NS, int M>
__device__ __forceinline__ void scan_grad_chunk_body(float* __restrict__ sums, float* __restrict__ states, const float* __restrict__ delta, const float* __restrict__ a, const float* __restrict__ cmap,
                                                     const float* __restrict__ gate, const float* __restrict__ bias, const int32_t* __restrict__ lengths, const float* __restrict__ g,
                                                     const ScanParams& P) {
    __shared__ float prepared[2][2][KEPT][64];                       // [turn's parity][dt, gy][step][lane]
    __shared__ __attribute__((aligned(16))) float map[2][KEPT][NS * M];
    const Place<NS, M> at(P, lengths);
    float a2[NS], l[NS] = {}, sum = 0.f, mapped;
    at.factors(a2, a, P);
    const float add = bias ? bias[at.c] : 0.f;
    const int turns = at.begin < at.stop ? (at.stop - at.begin + KEPT - 1) / KEPT : 0;
    float ds[at.OWN], gs[at.OWN], gates[at.OWN];
    auto request = [&](int t0) {
#pragma unroll
        for (int q = 0; q < at.OWN; ++q) {
            const int t = min(t0 + at.own(q), at.stop - 1);
            ds[q] = at.row(delta, P, t)[at.c]; gs[q] = g ? at.row(g, P, t)[at.c] : 0.f;
            if (gate) gates[q] = at.row(gate, P, t)[at.c];
        }
        mapped = at.template staged<true>(cmap, P, t0);
    };
    if (turns) request(at.begin + (turns - 1) * KEPT);
    for (int turn = turns - 1; turn >= 0; --turn) {
        const int t0 = at.begin + turn * KEPT, parity = turn & 1;
#pragma unroll
        for (int q = 0; q < at.OWN; ++q) {
            const bool taken = t0 + at.own(q) < at.stop;
            prepared[parity][0][at.own(q)][at.lane] = taken ? width_of(ds[q], add, P.softplus) : 0.f;
            prepared[parity][1][at.own(q)][at.lane] = taken ? (gate ? gs[q] * (gates[q] * sigmoid(gates[q])) : gs[q]) : 0.f;
        }
        at.stage(map[parity], mapped);
        if (turn > 0) request(t0 - KEPT);
        at.meet();
        float dt[KEPT], gy[KEPT], cs[NS], next[NS];
#pragma unroll
        for (int s = 0; s < KEPT; ++s) { dt[s] = prepared[parity][0][s][at.lane]; gy[s] = prepared[parity][1][s][at.lane]; }
        at.maps(next, map[parity], KEPT - 1);
#pragma unroll
        for (int s = KEPT - 1; s >= 0; --s) {
#pragma unroll
            for (int i = 0; i < NS; ++i) cs[i] = next[i];
            if (s > 0) at.maps(next, map[parity], s - 1);
            sum += dt[s];
#pragma unroll
            for (int i = 0; i < NS; ++i) l[i] = exp2_of(a2[i] * dt[s]) * __builtin_fmaf(gy[s], cs[i], l[i]);
            STEP_FENCE();
        }
    }
    if (!at.there) return;
    if (at.wave == 0u) sums[((int64_t)at.chunk * P.B + at.b) * P.C + at.c] = sum;
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if (at.has(P, i)) at.held(states, P, at.chunk, i)[at.c] = l[i];
}

// Sums over a wave's channels of eight values per lane (of eight states, or of two steps' four): a step of the butterfly leaves a lane half of them, then the eight lanes that have the
// same one add up. A lane has value lane / 8 in the end; of those that have it the first stores it.
__device__ __forceinline__ float over_channels(float (&v)[8]) {
    // (in the lower half of the lanes both halves' v[i], in the upper one v[i + 4])
#pragma unroll
    for (int i = 0; i < 4; ++i) { const auto r = __builtin_amdgcn_permlane32_swap(f2u(v[i]), f2u(v[i + 4]), false, false); v[i] = u2f(r[0]) + u2f(r[1]); }
#pragma unroll
    for (int i = 0; i < 2; ++i) { const auto r = __builtin_amdgcn_permlane16_swap(f2u(v[i]), f2u(v[i + 2]), false, false); v[i] = u2f(r[0]) + u2f(r[1]); }
    const bool upper = (threadIdx.x & 8u) != 0u;
    float s = (upper ? v[1] : v[0]) + lane_xor<8>(upper ? v[0] : v[1]);
    s += lane_xor<4>(s);
    s += lane_xor<2>(s);
    return s + lane_xor<1>(s);
}

// ---- the gradient of a chunk; what the adjoint comes to in front of the first one is the initial state's cotangent
template <int NS, int M>
__device__ __forceinline__ void scan_grad_body(float* __restrict__ dx, float* __restrict__ ddelta, float* __restrict__ dgate, float* __restrict__ dstate, float* __restrict__ maps, float* __restrict__ channel_sums,
                                               const float* __restrict__ x, const float* __restrict__ delta, const float* __restrict__ a, const float* __restrict__ bmap,
                                               const float* __restrict__ cmap, const float* __restrict__ through, const float* __restrict__ gate, const int32_t* __restrict__ lengths,
                                               const float* __restrict__ bias, const float* __restrict__ kept, const float* __restrict__ g, const float* __restrict__ g_last,
                                               const float* __restrict__ adjoints, const ScanParams& P) {
    // [dt, x, gy][step][lane]; a wave's sums over its states [seen, l b, e A][step][lane]; its sums over channels [db, dc][step][state]
    __shared__ float prepared[3][KEPT][64], parts[M][3][KEPT][64], mapped[2][KEPT][NS * M];
    __shared__ __attribute__((aligned(16))) float map[2][KEPT][NS * M];
    const Place<NS, M> at(P, lengths);
    constexpr int AT_ONCE = 8 / NS;                  // steps whose sums over channels go together
    const uint32_t over = at.lane >> 3;              // the value of those that a lane has
    const bool over_stores = (at.lane & 7u) == 0u;
    float a2[NS], l[NS], da[NS] = {}, dD = 0.f, dbias = 0.f;
    at.factors(a2, a, P);
#pragma unroll
    for (int i = 0; i < NS; ++i) l[i] = !at.has(P, i) ? 0.f : adjoints ? at.held(adjoints, P, at.chunk, i)[at.c] : g_last ? g_last[at.state(P, i)] : 0.f;
    const float add = bias ? bias[at.c] : 0.f, D = through ? through[at.c] : 0.f;
    const int turns = (at.end - at.begin + KEPT - 1) / KEPT;
    const bool stream = streams_result(P.first);
    float rx[at.OWN], rd[at.OWN], rg[at.OWN], rz[at.OWN], rh[NS], rmap[2];
    auto request = [&](int t0) {
#pragma unroll
        for (int q = 0; q < at.OWN; ++q) {
            const int t = min(t0 + at.own(q), at.stop - 1);
            rx[q] = at.row(x, P, t)[at.c]; rd[q] = at.row(delta, P, t)[at.c]; rg[q] = g ? at.row(g, P, t)[at.c] : 0.f;
            if (gate) rz[q] = at.row(gate, P, t)[at.c];
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) rh[i] = at.has(P, i) ? at.held(kept, P, (uint32_t)t0 / KEPT, i)[at.c] : 0.f;
        rmap[0] = at.template staged<(AT_ONCE > 1)>(bmap, P, t0); rmap[1] = at.template staged<(AT_ONCE > 1)>(cmap, P, t0);
    };
    bool requested = false;
    for (int turn = turns - 1; turn >= 0; --turn) {
        const int t0 = at.begin + turn * KEPT;
        float vx[at.OWN], vd[at.OWN], vz[at.OWN];
        if (t0 < at.stop) {
            if (!requested) { request(t0); requested = true; }
            float own_dt[at.OWN], own_x[at.OWN], own_gy[at.OWN], slope[at.OWN], dgs[at.OWN];
#pragma unroll
            for (int q = 0; q < at.OWN; ++q) {
                // (lanes behind the last channel have no part in the sums over channels)
                const bool taken = t0 + at.own(q) < at.stop && at.there;
                const float v = rd[q] + add, gv = taken ? rg[q] : 0.f, z = gate ? rz[q] : 0.f, open = gate ? sigmoid(z) : 1.f;
                own_dt[q] = taken ? (P.softplus ? softplus_of(v) : v) : 0.f;
                own_x[q]  = taken ? rx[q] : 0.f;
                own_gy[q] = taken ? (gate ? gv * (z * open) : gv) : 0.f;
                slope[q]  = P.softplus ? sigmoid(v) : 1.f;
                dgs[q]    = gv * (open * __builtin_fmaf(z, 1.f - open, 1.f));
                prepared[0][at.own(q)][at.lane] = own_dt[q];
                prepared[1][at.own(q)][at.lane] = own_x[q];
                prepared[2][at.own(q)][at.lane] = own_gy[q];
            }
            float h[NS], before[KEPT][NS];
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = rh[i];
            at.stage(map[0], rmap[0]); at.stage(map[1], rmap[1]);
            if (turn > 0) request(t0 - KEPT);
            at.meet();
            // (a step's dt, x, gy and maps, and those of the step behind it: all eight's would take the registers of a third wave)
            float dt, xs, gy, bs[NS], cs[NS], next_dt, next_x, next_gy, next_b[NS], next_c[NS];
            auto next = [&](int s) {
                next_dt = prepared[0][s][at.lane]; next_x = prepared[1][s][at.lane]; next_gy = prepared[2][s][at.lane];
                at.maps(next_b, map[0], s); at.maps(next_c, map[1], s);
            };
            auto take = [&] {
                dt = next_dt; xs = next_x; gy = next_gy;
#pragma unroll
                for (int i = 0; i < NS; ++i) { bs[i] = next_b[i]; cs[i] = next_c[i]; }
            };
            next(0);
            const int count = at.stop - t0;
#pragma unroll
            for (int s0 = 0; s0 < KEPT; s0 += AT_ONCE) {
                if (s0 >= count) break;
                float part[8];
#pragma unroll
                for (int g = 0; g < AT_ONCE; ++g) {
                    const int s = s0 + g;
                    take();
                    if (s + 1 < KEPT) next(s + 1);
                    const float u = dt * xs;
                    float seen = 0.f;
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        before[s][i] = h[i];
                        h[i] = __builtin_fmaf(exp2_of(a2[i] * dt), h[i], u * bs[i]);
                        part[g * NS + i] = gy * h[i];
                        seen = __builtin_fmaf(cs[i], h[i], seen);
                    }
                    parts[at.wave][0][s][at.lane] = seen;
                }
                const float sum = over_channels(part);
                if (over_stores) mapped[1][s0 + over / NS][at.n0 + over % NS] = sum;
                STEP_FENCE();
            }
            next(min(count, KEPT) - 1 | (AT_ONCE - 1));
#pragma unroll
            for (int s0 = KEPT - AT_ONCE; s0 >= 0; s0 -= AT_ONCE) {
                if (s0 >= count) continue;
                float part[8];
#pragma unroll
                for (int g = AT_ONCE - 1; g >= 0; --g) {
                    const int s = s0 + g;
                    take();
                    if (s > 0) next(s - 1);
                    const float u = dt * xs;
                    float lb = 0.f, ea = 0.f;
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        l[i] = __builtin_fmaf(gy, cs[i], l[i]);
                        lb = __builtin_fmaf(l[i], bs[i], lb);
                        part[g * NS + i] = l[i] * u;
                        l[i] *= exp2_of(a2[i] * dt);
                        const float e = l[i] * before[s][i];
                        ea = __builtin_fmaf(e, a2[i], ea);
                        da[i] = __builtin_fmaf(e, dt, da[i]);
                    }
                    parts[at.wave][1][s][at.lane] = lb;
                    parts[at.wave][2][s][at.lane] = ea;
                }
                const float sum = over_channels(part);
                if (over_stores) mapped[0][s0 + over / NS][at.n0 + over % NS] = sum;
                STEP_FENCE();
            }
            at.meet();
#pragma unroll
            for (int q = 0; q < at.OWN; ++q) {
                const int s = at.own(q);
                float seen = gate ? parts[0][0][s][at.lane] : 0.f, lb = parts[0][1][s][at.lane], ea = parts[0][2][s][at.lane];
#pragma unroll
                for (int w = 1; w < M; ++w) {
                    if (gate) seen += parts[w][0][s][at.lane];
                    lb += parts[w][1][s][at.lane]; ea += parts[w][2][s][at.lane];
                }
                vd[q] = __builtin_fmaf(ea, LN2, lb * own_x[q]) * slope[q];
                vx[q] = __builtin_fmaf(lb, own_dt[q], D * own_gy[q]);
                vz[q] = dgs[q] * __builtin_fmaf(D, own_x[q], seen);
                // (steps that are not taken have no part in the sums)
                if (t0 + s < at.stop) { dD = __builtin_fmaf(own_gy[q], own_x[q], dD); dbias += vd[q]; }
            }
        }
        if (at.there)
#pragma unroll
            for (int q = 0; q < at.OWN; ++q) {
                const int t = t0 + at.own(q);
                if (t >= at.end) continue;
                const bool taken = t < at.stop;
                auto put = [&](float* p, float v) {
                    if (!p) return;
                    if (stream) __builtin_nontemporal_store(taken ? v : 0.f, at.row(p, P, t) + at.c); else at.row(p, P, t)[at.c] = taken ? v : 0.f;
                };
                put(dx, vx[q]); put(ddelta, vd[q]); put(dgate, vz[q]);
            }
        // [strip][B][T][2 N]
        for (uint32_t i = threadIdx.x; i < KEPT * 2u * P.N; i += 64u * M) {
            const uint32_t s = i / (2u * P.N), n = i - s * 2u * P.N;
            const int t = t0 + (int)s;
            if (t >= at.end) break;
            maps[(((uint64_t)at.strip * P.B + at.b) * P.T + (uint32_t)t) * 2u * P.N + n] = t >= at.stop ? 0.f : n < P.N ? mapped[0][s][n] : mapped[1][s][n - P.N];
        }
        // (what is read here is written again behind the next meeting, what the next turn writes in front of that was read in front of the last one)
    }
    // [B chunks][N + 2][C]
    prepared[0][at.wave][at.lane] = dD;
    prepared[1][at.wave][at.lane] = dbias;
    at.meet();
    if (!at.there) return;
    if (dstate && at.chunk == 0u)
#pragma unroll
        for (int i = 0; i < NS; ++i) if (at.has(P, i)) dstate[at.state(P, i)] = l[i];
    float* const row = channel_sums + ((uint64_t)at.b * P.chunks + at.chunk) * (P.N + 2u) * P.C + at.c;
#pragma unroll
    for (int i = 0; i < NS; ++i) if (at.has(P, i)) row[(uint64_t)(at.n0 + i) * P.C] = da[i];
    if (at.wave != 0u) return;
#pragma unroll
    for (int w = 1; w < M; ++w) { dD += prepared[0][w][at.lane]; dbias += prepared[1][w][at.lane]; }
    row[(uint64_t)P.N * P.C] = dD; row[(uint64_t)(P.N + 1u) * P.C] = dbias;
}

#define SELECTIVE_SCAN(NS, M)                                                                                                                                                      \
    extern "C" __global__ __launch_bounds__(64 * M) void selective_scan_chunk_n##NS##_m##M(float* sums, float* states, const float* x, const float* delta, const float* a, const float* bmap, \
                                                                                           const float* bias, const int32_t* lengths, ScanParams P) {                              \
        scan_chunk_body<NS, M>(sums, states, x, delta, a, bmap, bias, lengths, P);                                                                                                 \
    }                                                                                                                                                                              \
    extern "C" __global__ __launch_bounds__(64 * M, NS == 8 ? 4 : 1) void selective_scan_n##NS##_m##M(float* y, float* last, float* kept, const float* x, const float* delta, const float* a,       \
                                                                                     const float* bmap, const float* cmap, const float* through, const float* gate,                \
                                                                                     const float* state, const int32_t* lengths, const float* bias, const float* states,           \
                                                                                     ScanParams P) {                                                                               \
        scan_body<NS, M>(y, last, kept, x, delta, a, bmap, cmap, through, gate, state, lengths, bias, states, P);                                                                  \
    }                                                                                                                                                                              \
    extern "C" __global__ __launch_bounds__(64 * M) void selective_scan_grad_chunk_n##NS##_m##M(float* sums, float* states, const float* delta, const float* a, const float* cmap, \
                                                                                                const float* gate, const float* bias, const int32_t* lengths, const float* g,      \
                                                                                                ScanParams P) {                                                                    \
        scan_grad_chunk_body<NS, M>(sums, states, delta, a, cmap, gate, bias, lengths, g, P);                                                                                      \
    }                                                                                                                                                                              \
    extern "C" __global__ __launch_bounds__(64 * M, NS == 8 || M == 1 ? 2 : M == 8 ? 4 : 3) void selective_scan_grad_n##NS##_m##M(float* dx, float* ddelta, float* dgate, float* dstate, float* maps, float* channel_sums, const float* x, \
                                                                                          const float* delta, const float* a, const float* bmap, const float* cmap,                \
                                                                                          const float* through, const float* gate, const int32_t* lengths, const float* bias,      \
                                                                                          const float* kept, const float* g, const float* g_last, const float* adjoints,           \
                                                                                          ScanParams P) {                                                                          \
        scan_grad_body<NS, M>(dx, ddelta, dgate, dstate, maps, channel_sums, x, delta, a, bmap, cmap, through, gate, lengths, bias, kept, g, g_last, adjoints, P);                         \
    }
SELECTIVE_SCAN(4, 1)
SELECTIVE_SCAN(4, 2)
SELECTIVE_SCAN(4, 4)
SELECTIVE_SCAN(4, 8)
SELECTIVE_SCAN(8, 8)

// What blocks have found, added up in their order: [strips][B T][2 N] to db and dc [B T, N], and [rows][N + 2][C] to dA [C, N], dD and dbias [C]. The first `map_blocks`
// blocks have 1024 elements of the former each, the others 64 columns of the latter, their 16 waves every 16th row.
struct ScanSumsParams { uint32_t first, rows, C, N, strips, steps, map_blocks; };
extern "C" __global__ __launch_bounds__(1024) void selective_scan_sums(float* __restrict__ da, float* __restrict__ db, float* __restrict__ dc, float* __restrict__ dD, float* __restrict__ dbias,
                                                                       const float* __restrict__ maps, const float* __restrict__ channel_sums, ScanSumsParams P) {
    __shared__ float part[16][64];
    if (blockIdx.x < P.map_blocks) {
        const uint64_t at = (uint64_t)blockIdx.x * 1024u + threadIdx.x, all = (uint64_t)P.steps * 2u * P.N;
        if (at >= all) return;
        float s = maps[at];
        for (uint32_t k = 1; k < P.strips; ++k) s += maps[k * all + at];
        const uint64_t step = at / (2u * P.N);
        const uint32_t n = (uint32_t)(at - step * 2u * P.N);
        if (n < P.N) { if (db) db[step * P.N + n] = s; }
        else if (dc) dc[step * P.N + n - P.N] = s;
        return;
    }
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, columns = (P.N + 2u) * P.C, at = (blockIdx.x - P.map_blocks) * 64u + lane;
    float s = 0.f;
    if (at < columns)
        for (uint32_t r = wave; r < P.rows; r += 16u) s += channel_sums[(uint64_t)r * columns + at];
    part[wave][lane] = s;
    __syncthreads();
    if (wave != 0u || at >= columns) return;
    s = part[0][lane];
#pragma unroll
    for (int q = 1; q < 16; ++q) s += part[q][lane];
    const uint32_t n = at / P.C, c = at - n * P.C;
    if (n < P.N) { if (da) da[(uint64_t)c * P.N + n] = s; }
    else if (n == P.N) { if (dD) dD[c] = s; }
    else if (dbias) dbias[c] = s;
}
