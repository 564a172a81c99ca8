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
// The power of two that an operand with this largest magnitude is scaled by (within what fp32 has both ways: an operand that has nothing beyond 2^-106 is scaled to less)
__device__ __forceinline__ int half_scale(float largest) {
    const int e = (int)(f2u(largest) >> 23) - 127;
    return min(HALF_TOP - e, 120);
}
__device__ __forceinline__ float power_of_two(int e) { return u2f((uint32_t)(127 + e) << 23); }          // (-126 <= e <= 127)

// ---- the product of a tile of 128 x 128: four waves, 64 x 64 each. A pair of steps (32 k) of both operands, 32 KB, goes straight from memory into one of two buffers in shared
// memory while the waves work on the other one; two blocks to a CU.
constexpr int HALF_TILE = 128;
typedef u32x4 HalfStage[2][4][2][2][64];                 // [operand][block of 32 rows][step][hi, lo][lane]

struct HalfOperand {
    const u32x4* parts;
    uint32_t blocks, stride, first;                      // blocks of 32 rows, steps of 16 k per block, and the step at which the contraction starts (even)
};

struct HalfSums { f32x16 large[2][2], small[2][2]; };    // of a wave's 2 x 2 blocks of 32 x 32: hi.hi, and the others times 2^11

__device__ __forceinline__ void half_request(HalfStage& to, const HalfOperand& a, const HalfOperand& b, uint32_t block_a, uint32_t block_b, uint32_t step) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    // a wave brings a block of 32 rows of either operand (behind the last one, that one again: its results are nobody's)
    const u32x4* const from_a = a.parts + ((uint64_t)min(block_a + wave, a.blocks - 1u) * a.stride + a.first + step) * 128u + lane;
    const u32x4* const from_b = b.parts + ((uint64_t)min(block_b + wave, b.blocks - 1u) * b.stride + b.first + step) * 128u + lane;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from_a + 64 * q), (__attribute__((address_space(3))) void*)&to[0][wave][q >> 1][q & 1][0], 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from_b + 64 * q), (__attribute__((address_space(3))) void*)&to[1][wave][q >> 1][q & 1][0], 16, 0, 0);
    }
}
__device__ __forceinline__ void half_multiply(HalfSums& sums, const HalfStage& from) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, wm = wave >> 1, wn = wave & 1u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        f16x8 a[2][2], b[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                a[i][t] = __builtin_bit_cast(f16x8, from[0][2 * wm + i][s][t][lane]);
                b[i][t] = __builtin_bit_cast(f16x8, from[1][2 * wn + i][s][t][lane]);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sums.small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][0], b[j][1], sums.small[i][j], 0, 0, 0);
                sums.large[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][0], b[j][0], sums.large[i][j], 0, 0, 0);
                sums.small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][1], b[j][0], sums.small[i][j], 0, 0, 0);
            }
    }
}
// The sums of tile (m, n) over `pairs` pairs of steps from pair `begin` on
__device__ __forceinline__ void half_product(HalfSums& sums, HalfStage (&stages)[2], const HalfOperand& a, const HalfOperand& b, uint32_t m, uint32_t n, uint32_t begin, uint32_t pairs) {
    half_request(stages[0], a, b, 4u * m, 4u * n, 2u * begin);
    __syncthreads();
    for (uint32_t p = 0; p < pairs; ++p) {
        if (p + 1u < pairs) half_request(stages[(p + 1u) & 1u], a, b, 4u * m, 4u * n, 2u * (begin + p + 1u));
        half_multiply(sums, stages[p & 1u]);
        __syncthreads();
    }
}
// Consecutive blocks go to the 8 XCDs in turn; each works through a contiguous range of the tiles, in strips of 8 columns of tiles, row by row of a strip, so that the blocks of an
// XCD that run together share rows and columns in its L2.
__device__ __forceinline__ void half_tile_of(uint32_t block, uint32_t blocks, uint32_t tiles_m, uint32_t tiles_n, uint32_t& m, uint32_t& n) {
    const uint32_t per = blocks / 8u, id = per > 0u && block < per * 8u ? (block & 7u) * per + (block >> 3) : block;
    const uint32_t strip = id / (8u * tiles_m), width = min(8u, tiles_n - 8u * strip), at = id - strip * 8u * tiles_m;
    m = at / width; n = 8u * strip + at - m * width;
}

// ---- a tile of a result as an operand of products that follow: contracted over its rows, as the lanes have it (`by_column`: its index is the column), or over its columns (`by_row`),
// turned in shared memory. value(block of rows i, of columns j, register, row, column) is what is taken apart, scaled; it is zero behind the result's last row and column.
constexpr uint32_t HALF_PITCH = 132u;                    // words of a row in shared memory: lanes that read vectors of neighbouring rows meet no bank twice
typedef uint32_t HalfTurned[HALF_TILE][HALF_PITCH];
union HalfShared { HalfStage stages[2]; HalfTurned turned; };

struct HalfTarget { u32x4* parts; uint32_t blocks, steps, block, step; };      // blocks of 32 of its index, steps of 16 k per block (all of them); where this tile's begin

template <class F>
__device__ __forceinline__ void half_store(HalfTurned& turned, const HalfTarget& by_column, const HalfTarget& by_row, F value) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, wm = wave >> 1, wn = wave & 1u;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t column = wn * 64u + 32u * j + (lane & 31u), block = by_column.block + wn * 2u + j;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t row0 = wm * 64u + 32u * i + 4u * (lane >> 5);
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t row = row0 + 8u * (k >> 1) + 2u * (k & 1);
                half_parts(value(i, j, 2 * k, row, column), value(i, j, 2 * k + 1, row + 1u, column), hi[k], lo[k]);
            }
            if (by_column.parts && block < by_column.blocks)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t step = by_column.step + wm * 4u + 2u * i + s;
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
    // wave: a block of 32 rows, the tile's eight steps of 16 columns
    const uint32_t block = by_row.block + wave;
    const uint32_t* const row = &turned[wave * 32u + (lane & 31u)][0];
    if (block >= by_row.blocks) return;
#pragma unroll
    for (uint32_t s = 0; s < 8u; ++s) {
        if (by_row.step + s >= by_row.steps) break;
        u32x4 hi, lo;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const u32x4 t = *reinterpret_cast<const u32x4*>(row + 16u * s + 8u * q + 4u * (lane >> 5));
            hi[2 * q] = (t.x & 0xFFFFu) | t.y << 16; hi[2 * q + 1] = (t.z & 0xFFFFu) | t.w << 16;
            lo[2 * q] = t.x >> 16 | (t.y & 0xFFFF0000u); lo[2 * q + 1] = t.z >> 16 | (t.w & 0xFFFF0000u);
        }
        u32x4* const to = by_row.parts + ((uint64_t)block * by_row.steps + by_row.step + s) * 128u + lane;
        to[0] = hi; to[64] = lo;
    }
}
