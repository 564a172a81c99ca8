// Linear recurrences along time over [B, T, C]: h[t] = a[t] h[t-1] + b[t], with factors a and addends b as they are, or from gates:
// a = sigmoid(gate), b = (1 - a) x. Their gradient runs the other way: with l[t] = g[t] + a[t+1] l[t+1] (at the last step: the last
// state's cotangent in the place of the second term)
//   dx = l (gated: l (1 - a)),  dfactor = l h[t-1] (gated: l (h[t-1] - x) a (1 - a)),  dstate = a[first] l[first].
// From a sequence's length on steps are not taken: the state stays (a = 1, b = 0), and the operands are not used there.
//
// One pass over the data. A block takes a tile: W lanes of VEC channels each, and 256 / W groups of L steps that follow one another.
// A thread reads its L steps into registers and composes them to one map h -> A h + H; maps compose to maps
// (A2 (A1 h + H1) + H2), so a scan across the lanes of a wave and the four waves tells every thread the map in front of its own
// steps. What is still missing is the state in front of the tile (below: single-pass scans with look-back, as published for prefix sums);
// with it a thread goes through its steps once more, from registers, and stores. Groups of 8 lanes x 4 channels read whole lines of 128 bytes of every step, 32 KB per wave in flight.
//
// The state in front of a tile (where time has more than one): tiles hand it on within the launch. A tile publishes its map (A, H) as
// soon as it has it, and the state behind it as soon as it knows that; it looks at the WINDOW tiles before it until one of them
// shows its state and all after that one their maps, then applies those maps in turn. Every tile applies the same maps to the same
// states in the same order, whatever it finds published, so the results do not depend on the order in which blocks run.
//   * A map's factor is a product of up to 512 steps' and may fall out of fp32's range where the state times each of them in turn would not: at 16 steps a thread, six
//     products across a wave, four waves and 16 tiles an error of up to 2^-150 each, 2^-144 of the state in all.
//   * The wait ends: tiles are numbered in the order in which their blocks start (a ticket), a tile looks at earlier ones only, and
//     the first tile without a state finds its predecessor's. So the earliest one always gets on, and then the next.
//   * There are eight lines of tickets, one for every eighth block: drawn from one alone, they follow one another some 10 ns apart (3 x 1021 x
//     333 11 us instead of 8). A line has neighbouring strips, an eighth of all, or, where they come out even, of every sequence's, so that
//     different lengths keep all lines busy (8 x 2048 x 2048 with ragged lengths, forward and gradient 222 -> 207 us). Every eighth block is on
//     one XCD: where rows are no multiple of 128 bytes, neighbouring strips share lines of memory, which are fetched once there. (15933 steps
//     of 1976 channels, factors as they are, 100 -> 90 us, the gradient 226 -> 207, and 142 with parts of lines stored through the
//     caches, which put them together.) No result depends on where blocks run.
//   * A channel's word, 64 bits stored at once: H above, A below, with the lowest bit of A (a rounding of 2^-23 of A, for the tile's
//     own use too) telling launches apart: its value alternates from launch to launch, and every launch writes every word. A state
//     is marked by a NaN of its own in the place of A. No fence is needed, since a word holds all that is read, and nothing has to be
//     cleared: the tickets count on through the launches, so their quotient is the launch's number.
// What bounds it: memory, with two waves per SIMD; while a tile waits for its state the other block of its CU loads. 65536 steps of 1024
// channels (805 MB) 150 us, 5.3 TB/s, where a large copy by a library reaches 5.1-5.5; 8 x 2048 x 2048 with ragged lengths 67-74 us, and
// its gradient 138-143 us (716 MB); single steps of 64 x 2048 3 us, a launch. Smaller tiles have more words to look at and more ends to wait for: 8 steps per thread 160 us, 4 steps
// 250. Strips of 64 channels 10-15 % slower (fewer chains side by side), of 16 20 % (half lines). Blocks that draw a tile ahead and
// load it while they wait hold up the tiles behind it: 265 us.
#include "common.h"

struct RecurrenceParams {
    uint32_t first;                      // (bit 31: the result is stored past the caches)
    uint32_t T, C, cstrips, strips, tiles;
    uint32_t lines, of_each;             // lines of tickets, and whether each has a part of every sequence's strips
    uint32_t log2_w, reverse;
};

constexpr uint32_t THREADS = 256, WINDOW = 16, CHAIN_CHANNELS = 32, LINES = 8;
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
    // (past the caches: nothing is read twice. 3 % of a launch)
    if constexpr (VEC == 4) {
        const f32x4 t = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 2));
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    }
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

    bool there;                                  // (a block beyond the last tile has none)

    __device__ Tile(const RecurrenceParams& P, const int32_t* lengths, unsigned long long* chain, bool back_) : T(P.T), C(P.C), strips(P.strips), back(back_), there(true) {
        __shared__ unsigned long long ticket;
        W = 1u << P.log2_w; G = THREADS >> P.log2_w;
        col = threadIdx.x & (W - 1u); group = threadIdx.x >> P.log2_w;
        tag = 0; words = nullptr; k = 0;
        strip = blockIdx.x;
        if constexpr (CHAIN) {
            const uint32_t line = blockIdx.x & (P.lines - 1u), per = gridDim.x / P.lines;
            const uint32_t all = P.of_each ? P.cstrips : P.strips, s0 = all * line / P.lines, neighbours = all * (line + 1u) / P.lines - s0;
            const uint32_t mine = P.of_each ? P.strips / P.cstrips * neighbours : neighbours;
            if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(chain + line * 8u, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            const unsigned long long t = ticket;
            const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)t), hi = __builtin_amdgcn_readfirstlane((uint32_t)(t >> 32));
            const unsigned long long number = (unsigned long long)hi << 32 | lo, launch = number / per;
            const uint32_t tile = (uint32_t)(number - launch * per);
            tag = (uint32_t)(launch + 1ull) & 1u;                          // (the first launch's words are odd: memory starts as zeros)
            words = chain + LINES * 8u;                                    // behind the tickets, a line each
            there = tile < mine * P.tiles;
            k = tile / mine;
            const uint32_t at = tile - k * mine, sequence = at / neighbours;      // (0 where a line's strips are not of every sequence)
            strip = sequence * P.cstrips + s0 + (at - sequence * neighbours);
        }
        b = strip / P.cstrips; c0 = (strip % P.cstrips) * W * VEC;
        n = min(G * L, T - k * (G * L));
        tlow = back ? T - k * (G * L) - n : k * (G * L);
        length = there ? length_of(lengths, b, T) : 0u;
    }
    __device__ uint32_t row(uint32_t i) const { const uint32_t s = group * L + i; return back ? n - 1u - s : s; }       // of step i, from tlow on
    __device__ bool valid(uint32_t i) const { return group * L + i < n && c0 + col * VEC < C; }
    __device__ bool inside(uint32_t i) const { return valid(i) && tlow + row(i) < length; }
    __device__ uint32_t at(uint32_t i, bool take) const { return take ? (row(i) * C + col * VEC) * 4u : NOWHERE; }
    // a descriptor of the tile's part of an array [B, T, C], `shift` steps away (nothing where the array is null): it ends behind the last
    // step's channels, in front of NOWHERE
    __device__ __amdgpu_buffer_rsrc_t rsrc(const float* p, int shift = 0) const {
        return make_rsrc(p + (((int64_t)b * T + tlow + shift) * C + c0), p ? ((n - 1u) * C + min(C - c0, W * VEC)) * 4u : 0u);
    }
    // the same of an array [B, C]; its element of this thread
    __device__ __amdgpu_buffer_rsrc_t state_rsrc(const float* p) const { return make_rsrc(p + ((int64_t)b * C + c0), p ? min(C - c0, W * VEC) * 4u : 0u); }
    __device__ uint32_t state_at() const { return c0 + col * VEC < C ? col * VEC * 4u : NOWHERE; }

    // In: the map of this thread's steps. Out: the state in front of them, given the one in front of the first tile.
    __device__ void state_before(float (&A)[VEC], float (&H)[VEC], const float* initial_states, float (&now)[VEC]) {
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
        if constexpr (CHAIN) state_of_tile(parts, initial_states, s);
        else load<VEC>(s, state_rsrc(initial_states), state_at());
#pragma unroll
        for (int j = 0; j < VEC; ++j) now[j] = __builtin_fmaf(before_a[j], __builtin_fmaf(fa[j], s[j], fh[j]), before_h[j]);
    }

    // The state in front of this tile, from the tiles before it; publishes this one's map and state. The first wave does it, a lane per channel and half of
    // the window: the halves' words are all in flight together, the second half's lanes go on from the state that the first one's have found.
    __device__ void state_of_tile(const float (&parts)[4][64][2 * VEC], const float* initial_states, float (&s)[VEC]) {
        __shared__ float front[CHAIN_CHANNELS];
        const uint32_t channels = W * VEC;
        if (threadIdx.x < 64u) {
            constexpr int HALF = WINDOW / 2;
            const uint32_t channel = threadIdx.x & (CHAIN_CHANNELS - 1u), from = channel / VEC, j = channel % VEC;
            const bool second = threadIdx.x >= CHAIN_CHANNELS, use = channel < channels;
            unsigned long long* const mine = words + (uint64_t)strip * channels + (use ? channel : 0u);
            const uint64_t step = (uint64_t)strips * channels;               // to the next tile's word
            float a = 1.f, h = 0.f;
            for (uint32_t p = 0; p < 4u; ++p) { const float pa = parts[p][use ? from : 0u][j], ph = parts[p][use ? from : 0u][VEC + j]; h = __builtin_fmaf(pa, h, ph); a *= pa; }
            // A with its lowest bit cleared, rounded to nearest, ties to even: an error of up to 2^-23 of it once per tile, as much as two of the tile's
            // own multiplications
            const uint32_t bits = f2u(a), even = a != a ? MAP_NAN : (bits + ((bits >> 1) & 1u)) & ~1u;
            a = u2f(even);
            if (use && !second) __hip_atomic_store(mine + k * step, (unsigned long long)f2u(h) << 32 | even | tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const float initial = buffer_load_x1(state_rsrc(initial_states), use && c0 + channel < C ? channel * 4u : NOWHERE);
            float state = initial;
            if (k > 0u) {
                const int e0 = (int)k - (int)WINDOW + (second ? HALF : 0);    // this lane's first tile (tile -1: what the sequence starts with)
                for (;;) {
                    unsigned long long word[HALF];
#pragma unroll
                    for (int e = 0; e < HALF; ++e) {
                        word[e] = e0 + e == -1 ? (unsigned long long)f2u(initial) << 32 | STATE_MARK | tag : (unsigned long long)(tag ^ 1u);
                        if (e0 + e >= 0) word[e] = __hip_atomic_load(mine + (uint64_t)(e0 + e) * step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                    bool found = false;
                    auto follow = [&]() {
#pragma unroll
                        for (int e = 0; e < HALF; ++e) {
                            const uint32_t low = (uint32_t)word[e];
                            const float value = u2f((uint32_t)(word[e] >> 32));
                            const bool is_state = (low & ~1u) == STATE_MARK;
                            state = is_state ? value : __builtin_fmaf(u2f(low & ~1u), state, value);
                            found = (low & 1u) == tag && (is_state || found);
                        }
                    };
                    follow();
                    const float state_before = __shfl(state, channel);          // (of the first half)
                    const bool found_before = __shfl((int)found, channel) != 0;
                    if (second) { state = state_before; found = found_before; follow(); }
                    if (__builtin_amdgcn_ballot_w64(second && use && !found) == 0ull) break;
                    __builtin_amdgcn_s_sleep(1);
                }
            }
            if (second || k == 0u) {
                if (use && second) __hip_atomic_store(mine + k * step, (unsigned long long)f2u(__builtin_fmaf(a, state, h)) << 32 | STATE_MARK | tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (use) front[channel] = state;
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
    if (CHAIN && !tile.there) return;
    const __amdgpu_buffer_rsrc_t f_rsrc = tile.rsrc(factor), x_rsrc = tile.rsrc(x);
    float a[L][VEC], b[L][VEC], A[VEC], H[VEC], now[VEC];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const uint32_t at = tile.at(i, tile.inside(i));
        load<VEC>(a[i], f_rsrc, at);
        load<VEC>(b[i], x_rsrc, at);
    }
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
    tile.state_before(A, H, state, now);
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
    if (CHAIN && !tile.there) return;
    const __amdgpu_buffer_rsrc_t f_rsrc = tile.rsrc(factor), x_rsrc = tile.rsrc(GATED ? x : nullptr), g_rsrc = tile.rsrc(g), h_rsrc = tile.rsrc(h, P.reverse ? 1 : -1);
    float gs[L][VEC], a[L][VEC], before[L][VEC], rest[GATED ? L : 1][VEC], A[VEC], H[VEC], now[VEC];
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
    tile.state_before(A, H, g_last, now);
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

// Names: _v<channels per lane>_l<steps per thread>, _gated, _chain (more tiles than one along time). Several numbers of steps, so that tiles need not reach far
// beyond the last step.
#define RECURRENCE(name, VEC, L, GATED, CHAIN)                                                                                                          \
    extern "C" __global__ __launch_bounds__(256, 2) void recurrence_##name(float* h, float* last, const float* factor, const float* x, const float* state, \
                                                                        const int32_t* lengths, unsigned long long* chain, RecurrenceParams P) {        \
        recurrence_body<VEC, L, GATED, CHAIN>(h, last, factor, x, state, lengths, chain, P);                                                            \
    }
#define RECURRENCE_GRAD(name, VEC, L, GATED, CHAIN)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256, 2) void recurrence_grad_##name(float* dfactor, float* dx, float* dstate, const float* h, const float* factor, \
            const float* x, const float* state, const int32_t* lengths, const float* g, const float* g_last, unsigned long long* chain, RecurrenceParams P) { \
        recurrence_grad_body<VEC, L, GATED, CHAIN>(dfactor, dx, dstate, h, factor, x, state, lengths, g, g_last, chain, P);                             \
    }
#define RECURRENCE_VARIANTS(KERNEL, VEC, L)                                                                          \
    KERNEL(v##VEC##_l##L, VEC, L, false, false)            KERNEL(v##VEC##_l##L##_gated, VEC, L, true, false)
#define RECURRENCE_CHAINS(KERNEL, VEC, L)                                                                            \
    KERNEL(v##VEC##_l##L##_chain, VEC, L, false, true)     KERNEL(v##VEC##_l##L##_gated_chain, VEC, L, true, true)
RECURRENCE_VARIANTS(RECURRENCE, 4, 1)  RECURRENCE_VARIANTS(RECURRENCE, 4, 4)  RECURRENCE_VARIANTS(RECURRENCE, 4, 8)  RECURRENCE_VARIANTS(RECURRENCE, 4, 16)
RECURRENCE_VARIANTS(RECURRENCE, 1, 1)  RECURRENCE_VARIANTS(RECURRENCE, 1, 4)  RECURRENCE_VARIANTS(RECURRENCE, 1, 16)
RECURRENCE_CHAINS(RECURRENCE, 4, 8)    RECURRENCE_CHAINS(RECURRENCE, 4, 16)   RECURRENCE_CHAINS(RECURRENCE, 1, 16)
RECURRENCE_VARIANTS(RECURRENCE_GRAD, 4, 1)  RECURRENCE_VARIANTS(RECURRENCE_GRAD, 4, 3)  RECURRENCE_VARIANTS(RECURRENCE_GRAD, 4, 6)  RECURRENCE_VARIANTS(RECURRENCE_GRAD, 4, 8)
RECURRENCE_VARIANTS(RECURRENCE_GRAD, 1, 1)  RECURRENCE_VARIANTS(RECURRENCE_GRAD, 1, 4)  RECURRENCE_VARIANTS(RECURRENCE_GRAD, 1, 8)
RECURRENCE_CHAINS(RECURRENCE_GRAD, 4, 4)    RECURRENCE_CHAINS(RECURRENCE_GRAD, 4, 6)    RECURRENCE_CHAINS(RECURRENCE_GRAD, 1, 8)
