// Products of fp32 matrices on the fp16 matrix cores (v_mfma_f32_32x32x16_f16) with the accuracy of fp32 products, between operands that have been taken apart
// beforehand.
//
// A number x of an operand, scaled by a power of two so that the operand's largest is below 2^15, is hi + 2^-11 lo: hi its nearest fp16 (11 bits), lo the nearest fp16 of what is
// left times 2^11, which has its 11 bits too wherever x is not below 2^-28 of the largest; so x is off by at most 2^-22 of itself, or by 2^-51 of the largest. A product of two such
// numbers is taken as hi.hi + 2^-11 (hi.lo + lo.hi), each exact in fp32; the two kinds are summed in fp32 accumulators of their own, which meet in the end, and
// lo.lo, below 2^-22 of the product, is left out. Three matrix instructions instead of one, at 16 times the rate of the fp32 ones. What is lost per product (root mean square
// 2^-24) is less than what the roundings of a sum of 64 terms are; a sum is rounded after every 16 terms, where the fp32 instructions round after every second one.
// An operand that is infinite or NaN makes its row of the result NaN.
//
// A taken-apart operand is laid out as the lanes of a wave want it: [block of 32 rows][step of 16 k][hi, lo][lane] x 8 fp16; lane l has row l % 32, and with h = l / 32 its
// element 4 i + j is k = 8 i + 4 h + j of the step. That is the order in which a lane has the rows of a 32 x 32 block of a result (register 4 i + j of a half of the block is row
// 8 i + 4 h + j), so a result becomes an operand that is contracted over its rows without leaving its lanes. Rows and k beyond the end are zeros; k comes in pairs of steps.
// The same operand also serves products that are contracted over its rows (TURNED): 32 rows are a pair of steps then, 16 k are half of a block, and the lanes get theirs by reads of shared
// memory that transpose 4 rows x 16 columns (ds_read_b64_tr_b16: of 16 lanes, lane 4 a + b asks for 4 numbers of row a, and lane r is given column r of the four rows).
//
// PLAIN operands are for numbers that are too far apart for a scale, and for infinities and NaN: in the same places lie the upper and the lower halves of the numbers' own 32 bits. The same tiles, reads
// and epilogues serve them; a step puts the halves together again and multiplies by v_mfma_f32_32x32x2_f32 (element e of both operands' lanes: two k), whose sums are `large`.
// Log probabilities of 4096 x 1024 x 32000 with their gradient take 9400 us so, 3400 taken apart; 128 x 1024 x 32000 forward 175 and 108. (That a launch can do either costs it 1 to 2 us where it takes 70
// to 90, and nothing that can be measured where it takes 400.)
#pragma once
#include "common.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float    f32x2 __attribute__((ext_vector_type(2)));

constexpr float HALF_REST = 0x1p11f;                     // what a lo part is scaled by
constexpr int   HALF_TOP  = 14;                          // an operand's largest number is scaled to [2^14, 2^15)

// The parts of two neighbouring numbers (scaled already), the first in the low halves
__device__ __forceinline__ void half_parts(float a, float b, uint32_t& hi, uint32_t& lo) {
    const f16x2 h = __builtin_convertvector((f32x2{a, b}), f16x2);
    const f32x2 w = __builtin_convertvector(h, f32x2);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{(a - w.x) * HALF_REST, (b - w.y) * HALF_REST}), f16x2));
}
// ... and their own bits' halves, of a plain operand
__device__ __forceinline__ void plain_parts(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = f2u(a) >> 16 | (f2u(b) & 0xFFFF0000u);
    lo = (f2u(a) & 0xFFFFu) | f2u(b) << 16;
}
// The power of two that an operand with this largest magnitude is scaled by (within what fp32 has both ways: an operand that has nothing beyond 2^-106 is scaled to less)
__device__ __forceinline__ int half_scale(float largest) {
    const int e = (int)(f2u(largest) >> 23) - 127;
    return min(HALF_TOP - e, 120);
}
__device__ __forceinline__ float power_of_two(int e) { return u2f((uint32_t)(127 + e) << 23); }          // (-126 <= e <= 127)

// ---- the product of a tile: four waves, two by two, of T x T blocks of 32 x 32 each. Pairs of steps (32 k) of both operands go straight from memory into one of STAGES buffers in
// shared memory while the waves work on another one.
//   T = 2, STAGES = 2   tiles of 128, 64 KB, two blocks to a CU: for what fills the machine. 8192^3 354 to 378 TFLOP/s of fp32 products (an fp32 library product 153, a third of an fp16 one
//                       381). Bound by power: the matrix cores are busy 57 % of the time at 1.73 GHz, 54 % at 1.96 for 4096^3.
//   T = 1, STAGES = 4   tiles of 64, 64 KB, two blocks to a CU: few tiles, whose time is that of a pair of steps after the other: 0.38 us each, of 128 0.68
//   T = 1, STAGES = 2   the same, 32 KB, four blocks to a CU: between the two
// (Tiles of 128 with four buffers and a block to a CU: 0.76 us a pair.)
// Few tiles, or those left behind whole rounds of the machine, share a tile's contraction among `slices` blocks: they leave their sums in memory, and the one that arrives last adds them
// in the order of the slices. Nobody waits for another block.
template <int T> struct HalfTileOf {
    static constexpr int SIDE = 64 * T;
    typedef u32x4 Stage[2][2 * T][2][2][64];             // [operand][block of 32 rows][step][hi, lo][lane]
    static constexpr uint32_t PITCH = SIDE + 4;          // words of a row of results in shared memory: lanes that read vectors of neighbouring rows meet no bank twice
    typedef uint32_t Turned[SIDE][PITCH];
};
template <int T, int STAGES> union HalfShared { typename HalfTileOf<T>::Stage stages[STAGES]; typename HalfTileOf<T>::Turned turned; uint32_t arrived; };

struct HalfOperand {
    const u32x4* parts;
    uint32_t blocks, stride, first;                      // blocks of 32 rows, steps of 16 k per block, and the step at which the contraction starts (even)
};
// (TURNED: blocks of 32 of what is a result's row or column, the steps of a block of 32 of what is contracted, and where the contraction starts, in steps of 16)
enum HalfTurned { TURNED_NONE, TURNED_A, TURNED_B };

template <int T> struct HalfSums { f32x16 large[T][T], small[T][T]; };      // of a wave's blocks of 32 x 32: hi.hi, and the others times 2^11

// A turned operand's half block [32 rows of it][16 k] lies in shared memory with a row's two lanes side by side, every other half block shifted by half of the banks: the reads that turn it
// take two half blocks' rows v .. v + 3, which are all banks once.
__device__ __forceinline__ uint32_t half_turned_place(uint32_t row, uint32_t h, uint32_t half_block) { return (2u * row + h) ^ (half_block << 3); }

template <int T, HalfTurned TURNED>
__device__ __forceinline__ void half_request(typename HalfTileOf<T>::Stage& to, const HalfOperand& a, const HalfOperand& b, uint32_t m, uint32_t n, uint32_t step) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t u = 0; u < T; ++u) {
        // a block of 32 rows of either operand (behind the last one, that one again: its results are nobody's)
        const uint32_t unit = wave * T + u, of_b = unit / (2u * T), block = unit % (2u * T);
        const HalfOperand& o = of_b ? b : a;
        const uint32_t at = min((of_b ? n : m) * (2u * T) + block, o.blocks - 1u);
        const bool turned = TURNED != TURNED_NONE && of_b == (TURNED == TURNED_B ? 1u : 0u);
        const u32x4* const from = o.parts + (turned ? (uint64_t)((o.first + step) / 2u) * o.stride + 2u * at : (uint64_t)at * o.stride + o.first + step) * 128u;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // (the lane whose numbers belong at place `lane`)
            const uint32_t place = lane ^ ((uint32_t)(q >> 1) << 3), source = turned ? (place >> 1) + 32u * (place & 1u) : lane;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + 64 * q + source), (__attribute__((address_space(3))) void*)&to[of_b][block][q >> 1][q & 1][0], 16, 0, 0);
        }
    }
}
// What a wave needs of a step of 16 k: its blocks' parts
template <int T, HalfTurned TURNED> struct HalfStep {
    f16x8 a[T][2], b[T][2];
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef u32x4 Block[2][2][64];
    // rows 16 s .. 16 s + 15 of a turned block, as the operand of a step: lane l has column l % 32, rows 8 i + 4 h + j
    __device__ __forceinline__ static f16x8 turned(const Block& from, int s, int t) {
        const uint32_t lane = threadIdx.x & 63u, half_block = lane >> 4 & 1u, row = 4u * (lane >> 5) + (lane >> 2 & 3u), column = lane & 3u;
        const uint32_t place = half_turned_place(row, column & 1u, half_block);
        const __attribute__((address_space(3))) char* const at = (const __attribute__((address_space(3))) char*)&from[0][0][0] + half_block * 2048u + place * 16u + (column >> 1) * 8u + s * 512u + t * 1024u;
        const s16x4 low  = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 256u));
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ void read(const typename HalfTileOf<T>::Stage& from, int s) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, wm = wave >> 1, wn = wave & 1u;
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                a[i][t] = TURNED == TURNED_A ? turned(from[0][T * wm + i], s, t) : __builtin_bit_cast(f16x8, from[0][T * wm + i][s][t][lane]);
                b[i][t] = TURNED == TURNED_B ? turned(from[1][T * wn + i], s, t) : __builtin_bit_cast(f16x8, from[1][T * wn + i][s][t][lane]);
            }
    }
    // number e of a lane's eight of a plain operand
    __device__ __forceinline__ static float plain(const f16x8 (&parts)[2], int e) {
        const uint32_t hi = __builtin_bit_cast(u32x4, parts[0])[e >> 1], lo = __builtin_bit_cast(u32x4, parts[1])[e >> 1];
        return u2f(e & 1 ? (hi & 0xFFFF0000u) | lo >> 16 : hi << 16 | (lo & 0xFFFFu));
    }
    template <bool PLAIN> __device__ __forceinline__ void multiply(HalfSums<T>& sums) const {
        if constexpr (PLAIN) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < T; ++i)
#pragma unroll
                    for (int j = 0; j < T; ++j) sums.large[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(plain(a[i], e), plain(b[j], e), sums.large[i][j], 0, 0, 0);
            return;
        }
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j) {
                sums.small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][0], b[j][1], sums.small[i][j], 0, 0, 0);
                sums.large[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][0], b[j][0], sums.large[i][j], 0, 0, 0);
                sums.small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][1], b[j][0], sums.small[i][j], 0, 0, 0);
            }
    }
};
// All but the last N loads of this wave have arrived (lgkmcnt and expcnt as they are)
template <int N> __device__ __forceinline__ void loads_left() { __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | 15 << 8 | (N >> 4) << 14); }
__device__ __forceinline__ void in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); asm volatile("" ::: "memory"); }
#define HALF_FENCE() __builtin_amdgcn_sched_barrier(0)

template <bool B> struct HalfPlain { static constexpr bool value = B; };
// The sums of tile (m, n) over `pairs` pairs of steps from pair `begin` on. With more than two buffers a wave has the parts of the next step in registers before it
// multiplies those of this one: the barrier in front of a pair stands between the two steps of the pair before.
// EITHER: operands that are plain where *plain says so, which is read while the first pairs are on their way.
template <int T, int STAGES, HalfTurned TURNED = TURNED_NONE, bool EITHER = false>
__device__ __forceinline__ void half_product(HalfSums<T>& sums, HalfShared<T, STAGES>& shared, const HalfOperand& a, const HalfOperand& b, uint32_t m, uint32_t n, uint32_t begin, uint32_t pairs,
                                             const int32_t* plain = nullptr) {
    static_assert(STAGES == 2 || STAGES == 4, "as many pairs are on their way as meet() counts");
    constexpr int LOADS = 4 * T;                         // of a wave per stage
    if (pairs == 0u) return;                             // (a slice of nothing)
    uint32_t asked = 0u;                                 // pairs that have been requested
    auto request = [&](uint32_t at) { half_request<T, TURNED>(shared.stages[at], a, b, m, n, 2u * (begin + asked)); ++asked; };
    // pair p has arrived, for all waves (those asked for behind it may be on their way); and all have read what they wanted of the pair before the last
    auto meet = [&](uint32_t p) {
        const uint32_t behind = asked - 1u - p;
        if (STAGES > 2 && behind >= 2u) loads_left<2 * LOADS>(); else if (STAGES > 2 && behind == 1u) loads_left<LOADS>(); else loads_left<0>();
        in_order();
        __builtin_amdgcn_s_barrier();
        in_order();
    };
#pragma unroll
    for (uint32_t p = 0; p < STAGES - 1; ++p)
        if (p < pairs) request(p);
    auto multiply = [&](auto kind) {
        constexpr bool PLAIN = decltype(kind)::value;
        uint32_t at = 0u;
        if constexpr (STAGES == 2) {
            for (uint32_t p = 0; p < pairs; ++p) {
                meet(p);
                if (asked < pairs) request(at ^ 1u);
                HalfStep<T, TURNED> step;
                step.read(shared.stages[at], 0);
                step.template multiply<PLAIN>(sums);
                step.read(shared.stages[at], 1);
                step.template multiply<PLAIN>(sums);
                at ^= 1u;
            }
        } else {
            HalfStep<T, TURNED> first, second;
            meet(0u);
            if (asked < pairs) request(STAGES - 1u);
            first.read(shared.stages[0], 0);
            for (uint32_t p = 0; p < pairs; ++p) {
                second.read(shared.stages[at], 1);
                HALF_FENCE();
                first.template multiply<PLAIN>(sums);
                HALF_FENCE();
                const uint32_t next = at + 1u == STAGES ? 0u : at + 1u;
                if (p + 1u < pairs) {
                    meet(p + 1u);
                    // (in the place of pair p - 1; reads of pair p may still be on their way)
                    if (p > 0u && asked < pairs) request(at == 0u ? STAGES - 1u : at - 1u);
                    first.read(shared.stages[next], 0);
                }
                HALF_FENCE();
                second.template multiply<PLAIN>(sums);
                HALF_FENCE();
                at = next;
            }
        }
    };
    // (the branch is the whole launch's)
    if constexpr (EITHER) { if (__builtin_amdgcn_readfirstlane(*plain)) multiply(HalfPlain<true>{}); else multiply(HalfPlain<false>{}); }
    else multiply(HalfPlain<false>{});
    __syncthreads();
}

// Consecutive blocks go to the 8 XCDs in turn; each works through a contiguous range of the numbers
__device__ __forceinline__ uint32_t half_turn(uint32_t block, uint32_t blocks) {
    const uint32_t per = blocks / 8u;
    return per > 0u && block < per * 8u ? (block & 7u) * per + (block >> 3) : block;
}
// What a block of a launch does: the first `whole` tiles by a block each, the contraction of every one behind them by `slices` blocks
struct HalfShares { uint32_t whole, slices; };
__device__ __forceinline__ void half_work(uint32_t block, const HalfShares& P, uint32_t pairs, uint32_t& tile, uint32_t& slice, uint32_t& begin, uint32_t& end) {
    tile = half_turn(block, P.whole); slice = 0u; begin = 0u; end = pairs;
    if (block < P.whole) return;
    const uint32_t rest = half_turn(block - P.whole, gridDim.x - P.whole);
    tile = P.whole + rest / P.slices; slice = rest % P.slices;
    begin = (uint32_t)((uint64_t)pairs * slice / P.slices); end = (uint32_t)((uint64_t)pairs * (slice + 1u) / P.slices);
}
// The sums of a tile behind the whole ones: true in the block that has all of them (in `large`, both kinds)
template <int T, int STAGES>
__device__ __forceinline__ bool half_join(HalfSums<T>& sums, HalfShared<T, STAGES>& shared, float* partial, uint32_t* arrivals, uint32_t tile, uint32_t slice, const HalfShares& P) {
    if (tile < P.whole || P.slices == 1u) return true;
    constexpr uint32_t BYTES = HalfTileOf<T>::SIDE * HalfTileOf<T>::SIDE * 4u;
    const uint32_t mine = tile - P.whole, tid = threadIdx.x;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(reinterpret_cast<char*>(partial) + (uint64_t)mine * P.slices * BYTES, P.slices * BYTES);
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) sums.large[i][j][k] = __builtin_fmaf(sums.small[i][j][k], 1.f / HALF_REST, sums.large[i][j][k]);
    // Stored from where they are and stay: a buffer store of 16 bytes whose offset is a scalar register still reads its first word, for the last quarter of a row's lanes, while the instruction
    // behind it runs, and the compiler lets that one write the register (values of another part of the tile were found in their place).
    HALF_FENCE();
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = {sums.large[i][j][4 * q], sums.large[i][j][4 * q + 1], sums.large[i][j][4 * q + 2], sums.large[i][j][4 * q + 3]};
                // (past the L2, which is not the other XCDs')
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, tid * 16u, slice * BYTES + (uint32_t)((i * T + j) * 4 + q) * 4096u, 16);
            }
    HALF_FENCE();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // the stores have reached memory
    HALF_FENCE();
    __syncthreads();
    if (tid == 0u) {
        const uint32_t n = __hip_atomic_fetch_add(arrivals + mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (n + 1u == P.slices) __hip_atomic_store(arrivals + mine, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // (for the next launch)
        shared.arrived = n;
    }
    __syncthreads();
    const bool last = __builtin_amdgcn_readfirstlane(shared.arrived) + 1u == P.slices;
    __syncthreads();
    if (!last) return false;
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j) { sums.large[i][j] = f32x16{}; sums.small[i][j] = f32x16{}; }
#pragma nounroll
    for (uint32_t s = 0; s < P.slices; ++s)
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, tid * 16u, s * BYTES + (uint32_t)((i * T + j) * 4 + q) * 4096u, 16));
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums.large[i][j][4 * q + e] += v[e];
                }
    return true;
}
// A result
template <int T> __device__ __forceinline__ float half_sum(const HalfSums<T>& sums, int i, int j, int k) { return __builtin_fmaf(sums.small[i][j][k], 1.f / HALF_REST, sums.large[i][j][k]); }

// Tiles in strips of 8 columns of tiles, row by row of a strip, so that blocks that run together share rows and columns in an XCD's L2
__device__ __forceinline__ void half_tile(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t& m, uint32_t& n) {
    const uint32_t strip = id / (8u * tiles_m), width = min(8u, tiles_n - 8u * strip), at = id - strip * 8u * tiles_m;
    m = at / width; n = 8u * strip + at - m * width;
}

// ---- a tile of a result as an operand of products that follow: contracted over its rows, as the lanes have it (`by_column`: its index is the column), or over its columns (`by_row`),
// turned in shared memory. value(block of rows i, of columns j, register, row, column) is what is taken apart, scaled (PLAIN: as it is); it is zero behind the result's last row and column.
struct HalfTarget { u32x4* parts; uint32_t blocks, steps, block, step; };      // blocks of 32 of its index, steps of 16 k per block (all of them); where this tile's begin

template <int T, bool PLAIN = false, class F>
__device__ __forceinline__ void half_store(typename HalfTileOf<T>::Turned& turned, const HalfTarget& by_column, const HalfTarget& by_row, F value) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, wm = wave >> 1, wn = wave & 1u;
#pragma unroll
    for (int j = 0; j < T; ++j) {
        const uint32_t column = (wn * T + j) * 32u + (lane & 31u), block = by_column.block + wn * T + j;
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const uint32_t row0 = (wm * T + i) * 32u + 4u * (lane >> 5);
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t row = row0 + 8u * (k >> 1) + 2u * (k & 1);
                const float one = value(i, j, 2 * k, row, column), two = value(i, j, 2 * k + 1, row + 1u, column);
                if constexpr (PLAIN) plain_parts(one, two, hi[k], lo[k]); else half_parts(one, two, hi[k], lo[k]);
            }
            if (by_column.parts && block < by_column.blocks)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t step = by_column.step + (wm * T + i) * 2u + s;
                    if (step < by_column.steps) {
                        u32x4* const to = by_column.parts + ((uint64_t)block * by_column.steps + step) * 128u + lane;
                        to[0]  = u32x4{hi[4 * s], hi[4 * s + 1], hi[4 * s + 2], hi[4 * s + 3]};
                        to[64] = u32x4{lo[4 * s], lo[4 * s + 1], lo[4 * s + 2], lo[4 * s + 3]};
                    }
                }
            if (by_row.parts)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const uint32_t h = k & 1 ? hi[k >> 1] >> 16 : hi[k >> 1] & 0xFFFFu, l = k & 1 ? lo[k >> 1] & 0xFFFF0000u : lo[k >> 1] << 16;
                    turned[row0 + 8u * (k >> 2) + (k & 3)][column] = h | l;
                }
        }
    }
    if (!by_row.parts) return;
    __syncthreads();
    // of the tile's 2 T blocks of 32 rows with 4 T steps of 16 columns a quarter to a wave
#pragma unroll
    for (uint32_t q = 0; q < 2u * T * T; ++q) {
        const uint32_t item = wave * (2u * T * T) + q, rb = item / (4u * T), s = item % (4u * T);
        if (by_row.step + s >= by_row.steps || by_row.block + rb >= by_row.blocks) continue;
        const uint32_t* const row = &turned[rb * 32u + (lane & 31u)][0];
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const u32x4 t = *reinterpret_cast<const u32x4*>(row + 16u * s + 8u * e + 4u * (lane >> 5));
            hi[2 * e] = (t.x & 0xFFFFu) | t.y << 16; hi[2 * e + 1] = (t.z & 0xFFFFu) | t.w << 16;
            lo[2 * e] = t.x >> 16 | (t.y & 0xFFFF0000u); lo[2 * e + 1] = t.z >> 16 | (t.w & 0xFFFF0000u);
        }
        u32x4* const to = by_row.parts + ((uint64_t)(by_row.block + rb) * by_row.steps + by_row.step + s) * 128u + lane;
        to[0] = hi; to[64] = lo;
    }
}
