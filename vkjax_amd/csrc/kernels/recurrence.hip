// Linear recurrences along time over [B, T, C]: h[t] = a[t] h[t-1] + b[t], with factors a and addends b as they are, or from gates:
// a = sigmoid(gate), b = (1 - a) x. Their gradient runs the other way: with l[t] = g[t] + a[t+1] l[t+1] (at the last step: the last
// state's cotangent in the place of the second term)
//   dx = l (gated: l (1 - a)),  dfactor = l h[t-1] (gated: l (h[t-1] - x) a (1 - a)),  dstate = a[first] l[first].
// From a sequence's length on steps are not taken: the state stays (a = 1, b = 0), and the operands are not used there.
//
// One pass over the data. A block takes a tile: W lanes of VEC channels each, and 256 / W groups of L steps that follow one another.
// A thread reads its L steps into registers and composes them to one map h -> A h + H; maps compose to maps
// (A2 (A1 h + H1) + H2), so a scan across the lanes of a wave and the four waves tells every thread the map in front of its own
// steps. What is still missing is the state in front of the tile; with it a thread goes through its steps once more, from
// registers, and stores. Groups of 16 lanes x 4 channels read whole 256-byte pieces of every step, 16 KB per wave in flight.
//
// The state in front of a tile (where time has more than one): tiles hand it on within the launch. A tile publishes its map (A, H) as
// soon as it has it, and the state behind it as soon as it knows that; it looks at the WINDOW tiles before it until one of them
// shows its state and all after that one their maps, then applies those maps in turn. Every tile applies the same maps to the same
// states in the same order, whatever it finds published, so the results do not depend on the order in which blocks run.
//   * The wait ends: tiles are numbered in the order in which their blocks start (a ticket), a tile looks at earlier ones only, and
//     the first tile without a state finds its predecessor's. So the earliest one always gets on, and then the next.
//   * A channel's word, 64 bits stored at once: H above, A below, with the lowest bit of A (a rounding of 2^-23 of A, for the tile's
//     own use too) telling launches apart: its value alternates from launch to launch, and every launch writes every word. A state
//     is marked by a NaN of its own in the place of A. No fence is needed, since a word holds all that is read, and nothing has to be
//     cleared: the tickets count on through the launches, so their quotient is the launch's number.
// Measured against the alternatives in this file's history: see the figures at the kernels.
#include "common.h"

struct RecurrenceParams {
    uint32_t first;                      // (bit 31: the result is stored past the caches)
    uint32_t T, C, cstrips, strips, log2_w, reverse;
};

constexpr uint32_t THREADS = 256, WINDOW = 16, CHAIN_CHANNELS = 64;
constexpr uint32_t STATE_MARK = 0x7FC01230u, MAP_NAN = 0x7FE00000u;

// sigmoid(gate) and 1 - sigmoid(gate), each rounded from the exponential: neither is the difference of the other to 1
__device__ __forceinline__ void gate_factors(float gate, float& a, float& rest) {
    const float e = expf(-fabsf(gate)), d = 1.f + e;                     // d in [1, 2]
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);                // a Newton step: the reciprocal's error squared
    const float far = e * r;
    a = gate < 0.f ? far : r;
    rest = gate < 0.f ? r : far;
}

__device__ __forceinline__ uint32_t length_of(const int32_t* lengths, uint32_t b, uint32_t T) {
    return lengths ? (uint32_t)min((int64_t)max(lengths[b], 0), (int64_t)T) : T;
}

template <int VEC> __device__ __forceinline__ void load(float (&v)[VEC], __amdgpu_buffer_rsrc_t r, uint32_t at) {
    if constexpr (VEC == 4) { const f32x4 t = buffer_load_x4(r, at); v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; }
    else v[0] = buffer_load_x1(r, at);
}
template <int VEC> __device__ __forceinline__ void store(const float (&v)[VEC], __amdgpu_buffer_rsrc_t r, uint32_t at, bool stream = false) {
    if constexpr (VEC == 4) {
        const u32x4 t = u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
        if (stream) __builtin_amdgcn_raw_buffer_store_b128(t, r, at, 0, 2);
        else __builtin_amdgcn_raw_buffer_store_b128(t, r, at, 0, 0);
    } else {
        if (stream) __builtin_amdgcn_raw_buffer_store_b32(f2u(v[0]), r, at, 0, 2);
        else __builtin_amdgcn_raw_buffer_store_b32(f2u(v[0]), r, at, 0, 0);
    }
}

constexpr uint32_t NOWHERE = 0x80000000u;

// Where a block's tile lies. `s` counts steps in the direction of the scan.
template <int VEC, int L, bool CHAIN>
struct Tile {
    uint32_t W, G, col, group;                   // lanes per step, groups of L steps, this thread's place
    uint32_t b, c0, k, n;                        // sequence, first channel, number along time, steps in it
    uint32_t tlow, T, C, length, strips, strip, tag;
    bool back;                                   // the scan runs from the last time to the first
    unsigned long long* words;

    __device__ Tile(const RecurrenceParams& P, const int32_t* lengths, unsigned long long* chain, bool back_) : T(P.T), C(P.C), strips(P.strips), back(back_) {
        __shared__ unsigned long long ticket;
        W = 1u << P.log2_w; G = THREADS >> P.log2_w;
        col = threadIdx.x & (W - 1u); group = threadIdx.x >> P.log2_w;
        uint32_t tile = blockIdx.x;
        tag = 0; words = nullptr;
        if constexpr (CHAIN) {
            if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(chain, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            const unsigned long long t = ticket;
            const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)t), hi = __builtin_amdgcn_readfirstlane((uint32_t)(t >> 32));
            const unsigned long long mine = (unsigned long long)hi << 32 | lo, launch = mine / gridDim.x;
            tile = (uint32_t)(mine - launch * gridDim.x);
            tag = (uint32_t)(launch + 1ull) & 1u;                          // (the first launch's words are odd: memory starts as zeros)
            words = chain + 8;                                             // behind the ticket's line
        }
        k = tile / P.strips; strip = tile % P.strips;
        b = strip / P.cstrips; c0 = (strip % P.cstrips) * W * VEC;
        n = min(G * L, T - k * (G * L));
        tlow = back ? T - k * (G * L) - n : k * (G * L);
        length = length_of(lengths, b, T);
    }
    __device__ uint32_t row(uint32_t i) const { const uint32_t s = group * L + i; return back ? n - 1u - s : s; }       // of step i, from tlow on
    __device__ bool valid(uint32_t i) const { return group * L + i < n && c0 + col * VEC < C; }
    __device__ bool inside(uint32_t i) const { return valid(i) && tlow + row(i) < length; }
    __device__ uint32_t at(uint32_t i, bool take) const { return take ? (row(i) * C + col * VEC) * 4u : NOWHERE; }
    // a descriptor of the tile's part of an array [B, T, C], `shift` steps away (nothing where the array is null)
    __device__ __amdgpu_buffer_rsrc_t rsrc(const float* p, int shift = 0) const {
        return make_rsrc(p + (((int64_t)b * T + tlow + shift) * C + c0), p ? (n * C + min(C - c0, W * VEC)) * 4u : 0u);
    }
    // the same of an array [B, C]; its element of this thread
    __device__ __amdgpu_buffer_rsrc_t state_rsrc(const float* p) const { return make_rsrc(p + ((int64_t)b * C + c0), p ? min(C - c0, W * VEC) * 4u : 0u); }
    __device__ uint32_t state_at() const { return c0 + col * VEC < C ? col * VEC * 4u : NOWHERE; }

    // In: the map of this thread's steps. Out: the state in front of them, given the one in front of the first tile.
    __device__ void state_before(float (&A)[VEC], float (&H)[VEC], const float (&initial)[VEC], float (&now)[VEC]) {
        __shared__ float parts[4][64][2 * VEC];
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        for (uint32_t off = W; off < 64u; off <<= 1) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float pa = __shfl_up(A[j], off), ph = __shfl_up(H[j], off);
                if (lane >= off) { H[j] = __builtin_fmaf(A[j], ph, H[j]); A[j] *= pa; }
            }
        }
        const uint32_t w = min(W, 64u);
        if (lane >= 64u - w)
#pragma unroll
            for (int j = 0; j < VEC; ++j) { parts[wave][lane - (64u - w)][j] = A[j]; parts[wave][lane - (64u - w)][VEC + j] = H[j]; }
        float before_a[VEC], before_h[VEC];                               // the map of the wave's groups before this one
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float pa = __shfl_up(A[j], w), ph = __shfl_up(H[j], w);
            before_a[j] = lane < w ? 1.f : pa; before_h[j] = lane < w ? 0.f : ph;
        }
        __syncthreads();
        const uint32_t stride = W <= 64u ? 1u : W >> 6, at = lane & (w - 1u);
        float fa[VEC], fh[VEC];                                           // the map of the waves before this one
#pragma unroll
        for (int j = 0; j < VEC; ++j) { fa[j] = 1.f; fh[j] = 0.f; }
        for (uint32_t p = wave % stride; p < wave; p += stride)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float pa = parts[p][at][j], ph = parts[p][at][VEC + j];
                fh[j] = __builtin_fmaf(pa, fh[j], ph); fa[j] *= pa;
            }
        float s[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = initial[j];
        if constexpr (CHAIN) state_of_tile(parts, initial, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) now[j] = __builtin_fmaf(before_a[j], __builtin_fmaf(fa[j], s[j], fh[j]), before_h[j]);
    }

    // The state in front of this tile, from the tiles before it; publishes this one's map and state.
    __device__ void state_of_tile(const float (&parts)[4][64][2 * VEC], const float (&initial)[VEC], float (&s)[VEC]) {
        __shared__ unsigned long long window[WINDOW][CHAIN_CHANNELS];
        __shared__ float front[CHAIN_CHANNELS];
        const uint32_t channels = W * VEC;
        const bool lead = group == 0u;                                    // the threads that follow the chain: the first group
        unsigned long long* const own = words + ((uint64_t)k * strips + strip) * channels + col * VEC;
        float ta[VEC], th[VEC];
        if (lead) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                ta[j] = 1.f; th[j] = 0.f;
                for (uint32_t p = 0; p < 4u; ++p) { const float pa = parts[p][col][j], ph = parts[p][col][VEC + j]; th[j] = __builtin_fmaf(pa, th[j], ph); ta[j] *= pa; }
                // A with its lowest bit cleared, rounded to nearest, ties to even: an error of up to 2^-23 of it once per tile, as much as two of the tile's
                // own multiplications
                const uint32_t bits = f2u(ta[j]), even = ta[j] != ta[j] ? MAP_NAN : (bits + ((bits >> 1) & 1u)) & ~1u;
                ta[j] = u2f(even);
                __hip_atomic_store(own + j, (unsigned long long)f2u(th[j]) << 32 | even | tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (k > 0u) {
            for (;;) {
                for (uint32_t e = group; e < WINDOW; e += G) {
                    const int p = (int)(k + e) - (int)WINDOW;             // (tile -1: what the sequence starts with)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        unsigned long long word = p == -1 ? (unsigned long long)f2u(initial[j]) << 32 | STATE_MARK | tag : (unsigned long long)(tag ^ 1u);
                        if (p >= 0) word = __hip_atomic_load(words + ((uint64_t)p * strips + strip) * channels + col * VEC + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        window[e][col * VEC + j] = word;
                    }
                }
                __syncthreads();
                bool known = true;
                if (lead) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        bool found = false;
                        for (uint32_t e = 0; e < WINDOW; ++e) {
                            const unsigned long long word = window[e][col * VEC + j];
                            const uint32_t low = (uint32_t)word;
                            const float value = u2f((uint32_t)(word >> 32));
                            const bool current = (low & 1u) == tag, is_state = (low & ~1u) == STATE_MARK;
                            s[j] = is_state ? value : __builtin_fmaf(u2f(low & ~1u), s[j], value);
                            found = current && (is_state || found);
                        }
                        known = known && found;
                    }
                }
                if (!__syncthreads_or(!known)) break;
                __builtin_amdgcn_s_sleep(1);
            }
        }
        if (lead) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float behind = __builtin_fmaf(ta[j], s[j], th[j]);
                __hip_atomic_store(own + j, (unsigned long long)f2u(behind) << 32 | STATE_MARK | tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                front[col * VEC + j] = s[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = front[col * VEC + j];
    }
    __device__ bool at_the_end() const { return (uint64_t)(k + 1u) * (G * L) >= T && group == G - 1u; }
};

template <int VEC, int L, bool GATED, bool CHAIN>
__device__ __forceinline__ void recurrence_body(float* h, float* last, const float* factor, const float* x, const float* state, const int32_t* lengths, unsigned long long* chain,
                                                const RecurrenceParams& P) {
    Tile<VEC, L, CHAIN> tile(P, lengths, chain, P.reverse != 0u);
    const __amdgpu_buffer_rsrc_t f_rsrc = tile.rsrc(factor), x_rsrc = tile.rsrc(x);
    float a[L][VEC], b[L][VEC], A[VEC], H[VEC], initial[VEC], now[VEC];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const uint32_t at = tile.at(i, tile.inside(i));
        load<VEC>(a[i], f_rsrc, at);
        load<VEC>(b[i], x_rsrc, at);
    }
    load<VEC>(initial, tile.state_rsrc(state), tile.state_at());
#pragma unroll
    for (int j = 0; j < VEC; ++j) { A[j] = 1.f; H[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const bool inside = tile.inside(i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (GATED) {
                float factor_here, rest;
                gate_factors(a[i][j], factor_here, rest);
                a[i][j] = factor_here; b[i][j] *= rest;
            }
            a[i][j] = inside ? a[i][j] : 1.f; b[i][j] = inside ? b[i][j] : 0.f;
            H[j] = __builtin_fmaf(a[i][j], H[j], b[i][j]); A[j] *= a[i][j];
        }
    }
    tile.state_before(A, H, initial, now);
    const __amdgpu_buffer_rsrc_t h_rsrc = tile.rsrc(h);
    const bool stream = streams_result(P.first);
#pragma unroll
    for (int i = 0; i < L; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) now[j] = __builtin_fmaf(a[i][j], now[j], b[i][j]);
        store<VEC>(now, h_rsrc, tile.at(i, tile.valid(i)), stream);
    }
    if (tile.at_the_end()) store<VEC>(now, tile.state_rsrc(last), tile.state_at());
}

template <int VEC, int L, bool GATED, bool CHAIN>
__device__ __forceinline__ void recurrence_grad_body(float* dfactor, float* dx, float* dstate, const float* h, const float* factor, const float* x, const float* state,
                                                     const int32_t* lengths, const float* g, const float* g_last, unsigned long long* chain, const RecurrenceParams& P) {
    Tile<VEC, L, CHAIN> tile(P, lengths, chain, P.reverse == 0u);
    const __amdgpu_buffer_rsrc_t f_rsrc = tile.rsrc(factor), x_rsrc = tile.rsrc(GATED ? x : nullptr), g_rsrc = tile.rsrc(g), h_rsrc = tile.rsrc(h, P.reverse ? 1 : -1);
    float gs[L][VEC], a[L][VEC], before[L][VEC], rest[GATED ? L : 1][VEC], A[VEC], H[VEC], initial[VEC], now[VEC];
    const uint32_t start = P.reverse ? P.T - 1u : 0u;                    // the time of the recurrence's first step
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const bool inside = tile.inside(i), first = tile.tlow + tile.row(i) == start;
        load<VEC>(gs[i], g_rsrc, tile.at(i, tile.valid(i)));
        load<VEC>(a[i], f_rsrc, tile.at(i, inside));
        load<VEC>(before[i], h_rsrc, tile.at(i, inside && !first));
        if constexpr (GATED) load<VEC>(rest[i], x_rsrc, tile.at(i, inside));
        if (first && state) load<VEC>(before[i], tile.state_rsrc(state), inside ? tile.state_at() : NOWHERE);
    }
    load<VEC>(initial, tile.state_rsrc(g_last), tile.state_at());
#pragma unroll
    for (int j = 0; j < VEC; ++j) { A[j] = 1.f; H[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const bool inside = tile.inside(i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (GATED) {
                before[i][j] -= rest[i][j];
                float factor_here, rest_here;
                gate_factors(a[i][j], factor_here, rest_here);
                a[i][j] = factor_here; rest[i][j] = rest_here;
            }
            a[i][j] = inside ? a[i][j] : 1.f;
            H[j] = a[i][j] * (H[j] + gs[i][j]); A[j] *= a[i][j];
        }
    }
    tile.state_before(A, H, initial, now);
    const __amdgpu_buffer_rsrc_t df_rsrc = tile.rsrc(dfactor), dx_rsrc = tile.rsrc(dx);
    const bool stream = streams_result(P.first);
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const bool inside = tile.inside(i);
        float df[VEC], db[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float l = now[j] + gs[i][j];
            if constexpr (GATED) { df[j] = l * before[i][j] * (a[i][j] * rest[i][j]); db[j] = l * rest[i][j]; }
            else { df[j] = l * before[i][j]; db[j] = l; }
            df[j] = inside ? df[j] : 0.f; db[j] = inside ? db[j] : 0.f;
            now[j] = a[i][j] * l;
        }
        const uint32_t at = tile.at(i, tile.valid(i));
        store<VEC>(df, df_rsrc, at, stream);
        store<VEC>(db, dx_rsrc, at, stream);
    }
    if (tile.at_the_end()) store<VEC>(now, tile.state_rsrc(dstate), tile.state_at());
}

// Names: _v<channels per lane>_l<steps per thread>, _gated, _chain (more tiles than one along time)
#define RECURRENCE(name, VEC, L, GATED, CHAIN)                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void recurrence_##name(float* h, float* last, const float* factor, const float* x, const float* state, \
                                                                        const int32_t* lengths, unsigned long long* chain, RecurrenceParams P) {        \
        recurrence_body<VEC, L, GATED, CHAIN>(h, last, factor, x, state, lengths, chain, P);                                                            \
    }
#define RECURRENCE_GRAD(name, VEC, L, GATED, CHAIN)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void recurrence_grad_##name(float* dfactor, float* dx, float* dstate, const float* h, const float* factor, \
            const float* x, const float* state, const int32_t* lengths, const float* g, const float* g_last, unsigned long long* chain, RecurrenceParams P) { \
        recurrence_grad_body<VEC, L, GATED, CHAIN>(dfactor, dx, dstate, h, factor, x, state, lengths, g, g_last, chain, P);                             \
    }
#define RECURRENCE_VARIANTS(KERNEL, LONG4, LONG1)                                                                   \
    KERNEL(v4_l1, 4, 1, false, false)            KERNEL(v4_l1_gated, 4, 1, true, false)                             \
    KERNEL(v4, 4, LONG4, false, false)           KERNEL(v4_gated, 4, LONG4, true, false)                            \
    KERNEL(v4_chain, 4, LONG4, false, true)      KERNEL(v4_gated_chain, 4, LONG4, true, true)                       \
    KERNEL(v1_l1, 1, 1, false, false)            KERNEL(v1_l1_gated, 1, 1, true, false)                             \
    KERNEL(v1, 1, LONG1, false, false)           KERNEL(v1_gated, 1, LONG1, true, false)                            \
    KERNEL(v1_chain, 1, LONG1, false, true)      KERNEL(v1_gated_chain, 1, LONG1, true, true)
RECURRENCE_VARIANTS(RECURRENCE, 8, 16)
RECURRENCE_VARIANTS(RECURRENCE_GRAD, 4, 8)
