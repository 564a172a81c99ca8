// Matrices with their singular values brought towards 1 by a polynomial: X = x / (|x| + eps) (Frobenius norm, per matrix), then `steps` times
//   A = X X^T,  B = a I + b A + c A A,  X <- B X          (of the wide way round: a matrix with more rows than columns is transposed)
// so that every singular value s becomes a s + b s^3 + c s^5. Products are those of half_product.h, between operands that never leave their taken-apart form: a product's tile
// turns its results into an operand, X into one contracted over its columns (turned in shared memory), which B X reads turned again (contracted over rows). A and B are symmetric:
// of their tiles only those on and above the diagonal are computed, and stored both ways. Only A is kept as fp32 too, since b A is a term of B. X has 22 bits between the steps; no
// operand's magnitude depends on the data beyond |x|, since a singular value's bound follows from the polynomial alone, so scales are known to the host.
// Matrices of a stack lie side by side in every launch.
// Bound by the matrix cores' power where a matrix fills the machine: 4096 x 4096 takes 211 us for a square, 260 for the polynomial (whose epilogue reads the square), 375 for B X (367 TFLOP/s of fp32
// products), 4.4 ms for five steps, of which the products alone at that rate are 3.6. 12 of 512 x 512: 13 to 18 us a launch, whose contraction of 512 is 16 pairs of steps behind one another.
#include "half_product.h"

typedef f32x4 f32x4_anywhere __attribute__((aligned(4)));

struct SquaresParams { uint32_t blocks, pad; uint64_t n; };
// [matrix][block]: sums of squares
extern "C" __global__ __launch_bounds__(256) void orthogonal_squares(float* __restrict__ sums, const float* __restrict__ x, SquaresParams P) {
    __shared__ float part[4];
    const uint32_t matrix = blockIdx.x / P.blocks, block = blockIdx.x % P.blocks;
    const float* const from = x + matrix * P.n;
    const uint64_t stride = (uint64_t)P.blocks * 256u;
    float s[4] = {};
    // (vectors wherever every matrix begins at one)
    const uint64_t vectors = (P.n & 3u) == 0u ? P.n / 4u : 0u;
    uint64_t at = (uint64_t)block * 256u + threadIdx.x;
    for (; at < vectors; at += 4u * stride) {
        f32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = at + k * stride < vectors ? reinterpret_cast<const f32x4*>(from)[at + k * stride] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(v[k][e], v[k][e], s[e]);
    }
    for (at = 4u * vectors + (uint64_t)block * 256u + threadIdx.x; at < P.n; at += stride) s[0] = __builtin_fmaf(from[at], from[at], s[0]);
    float t = (s[0] + s[1]) + (s[2] + s[3]);
    wave_butterfly([&](auto step) { t += lane_xor<decltype(step)::value>(t); });
    if ((threadIdx.x & 63u) == 0u) part[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0u) sums[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X taken apart, contracted over its columns [rows][columns]. A wave takes up to `each` steps of a block of 32.
struct OrthogonalPackParams {
    uint32_t matrices, R, C, sum_blocks, each, blocks;                                   // blocks of 256 threads, per matrix
    uint64_t sr, sc;                                                                     // element strides of row and column
    float eps; int32_t scale;
};
extern "C" __global__ __launch_bounds__(256) void orthogonal_pack(u32x4* __restrict__ by_row, const float* __restrict__ x, const float* __restrict__ sums, OrthogonalPackParams P) {
    __shared__ float part[4];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t matrix = blockIdx.x / P.blocks, block = blockIdx.x - matrix * P.blocks;
    float t = 0.f;
    for (uint32_t k = threadIdx.x; k < P.sum_blocks; k += 256u) t += sums[(uint64_t)matrix * P.sum_blocks + k];
    wave_butterfly([&](auto step) { t += lane_xor<decltype(step)::value>(t); });
    if (lane == 0u) part[wave] = t;
    __syncthreads();
    const float norm = __builtin_sqrtf((part[0] + part[1]) + (part[2] + part[3])) + P.eps, up = power_of_two(P.scale);
    const uint32_t I = P.R, K = P.C, steps = 2u * ((K + 31u) / 32u), each = P.each;
    const uint64_t si = P.sr, sk = P.sc;
    const uint32_t groups = (steps + each - 1u) / each, all = block * 4u + wave, blocks32 = (I + 31u) / 32u;
    const bool along_k = sk == 1u;
    const uint32_t rb = along_k ? all / groups : all % blocks32, group = along_k ? all % groups : all / blocks32;
    if (rb >= blocks32 || group >= groups) return;
    const uint32_t i = rb * 32u + (lane & 31u), h4 = 4u * (lane >> 5);
    const float* const from = x + (uint64_t)matrix * P.R * P.C + (uint64_t)min(i, I - 1u) * si;
    u32x4* const to = by_row + ((uint64_t)matrix * blocks32 + rb) * steps * 128u + lane;
    // (the operands of four steps at once)
    constexpr int AT_ONCE = 4;
    const uint32_t end = min(steps, (group + 1u) * each);
    for (uint32_t s0 = group * each; s0 < end; s0 += AT_ONCE) {
        float v[AT_ONCE][8];
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t k = (s0 + t) * 16u + h4 + 8u * q;
                if (along_k && k + 4u <= K && i < I) {
                    const f32x4 w = *reinterpret_cast<const f32x4_anywhere*>(from + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[t][4 * q + e] = w[e];
                } else
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[t][4 * q + e] = i < I && k + e < K ? from[(uint64_t)(k + e) * sk] : 0.f;
            }
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t) {
            if (s0 + t >= end) break;
            u32x4 hi, lo;
#pragma unroll
            for (int q = 0; q < 4; ++q) { uint32_t a, b; half_parts(v[t][2 * q] / norm * up, v[t][2 * q + 1] / norm * up, a, b); hi[q] = a; lo[q] = b; }
            to[(s0 + t) * 128u] = hi; to[(s0 + t) * 128u + 64u] = lo;
        }
    }
}

// What a launch of products computes
enum OrthogonalKind : uint32_t { SQUARE = 0, POLYNOMIAL = 1, NEXT = 2, LAST = 3 };
struct OrthogonalParams {
    uint32_t kind, M, N, K, tiles_m, tiles_n, tiles;     // tiles of a matrix: those on and above the diagonal of a square
    int32_t scale_a, scale_b, scale_out;
    float a, b, c; uint32_t whole, slices, pad;          // (HalfShares)
    uint64_t sr, sc;                                     // the last result's element strides
};
// (kinds in templates: their epilogues share no registers)
template <uint32_t KIND, int T, int STAGES, bool SHARED>
__device__ __forceinline__ void orthogonal_body(u32x4* __restrict__ by_column, u32x4* __restrict__ by_row, float* __restrict__ out, float* __restrict__ partial, uint32_t* __restrict__ arrivals,
                                                const u32x4* __restrict__ a, const u32x4* __restrict__ b, const float* __restrict__ square, const OrthogonalParams& P) {
    __shared__ HalfShared<T, STAGES> shared;
    constexpr bool SYMMETRIC = KIND == SQUARE || KIND == POLYNOMIAL;
    constexpr uint32_t SIDE = 64u * T;
    const uint32_t steps_k = 2u * ((P.K + 31u) / 32u), blocks_m = (P.M + 31u) / 32u, blocks_n = (P.N + 31u) / 32u, steps_m = 2u * blocks_m, steps_n = 2u * blocks_n;
    uint32_t tile, slice, begin, end, m, n;
    half_work(blockIdx.x, HalfShares{P.whole, P.slices}, steps_k / 2u, tile, slice, begin, end);
    const uint32_t matrix = tile / P.tiles, at = tile - matrix * P.tiles;
    if constexpr (SYMMETRIC) {
        // column by column of the triangle: n (n + 1) / 2 tiles in front of column n
        n = (uint32_t)((__builtin_sqrtf(8.f * (float)at + 1.f) - 1.f) * 0.5f);
        while ((n + 1u) * (n + 2u) / 2u <= at) ++n;
        while (n * (n + 1u) / 2u > at) --n;
        m = at - n * (n + 1u) / 2u;
    } else half_tile(at, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    const HalfOperand left{a + (uint64_t)matrix * blocks_m * steps_k * 128u, blocks_m, steps_k, 0u};
    if constexpr (SYMMETRIC) half_product<T, STAGES>(acc, shared, left, HalfOperand{b + (uint64_t)matrix * blocks_n * steps_k * 128u, blocks_n, steps_k, 0u}, m, n, begin, end - begin);
    else half_product<T, STAGES, TURNED_B>(acc, shared, left, HalfOperand{b + (uint64_t)matrix * (steps_k / 2u) * steps_n * 128u, blocks_n, steps_n, 0u}, m, n, begin, end - begin);
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, HalfShares{P.whole, P.slices})) return;
    const float down = power_of_two(-P.scale_a) * power_of_two(-P.scale_b), up = power_of_two(P.scale_out);
    const uint32_t row0 = m * SIDE, column0 = n * SIDE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t lane_row = row0 + (wave >> 1) * 32u * T + 4u * (lane >> 5), lane_column = column0 + (wave & 1u) * 32u * T + (lane & 31u);
    const uint64_t each = (uint64_t)matrix * P.M * P.N;
    if constexpr (KIND == LAST) {
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const uint32_t row = lane_row + 32u * i + 8u * (k >> 2) + (k & 3), column = lane_column + 32u * j;
                    if (row < P.M && column < P.N) out[each + row * P.sr + column * P.sc] = half_sum(acc, i, j, k) * down;
                }
        return;
    }
    // (all at once, in front of the stores)
    f32x16 squares[T][T] = {};
    if constexpr (KIND == POLYNOMIAL)
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const uint32_t row = min(lane_row + 32u * i + 8u * (k >> 2) + (k & 3), P.M - 1u), column = min(lane_column + 32u * j, P.N - 1u);
                    squares[i][j][k] = square[each + (uint64_t)row * P.N + column];
                }
    const HalfTarget columns{SYMMETRIC ? by_column + (uint64_t)matrix * blocks_n * steps_m * 128u : nullptr, blocks_n, steps_m, n * 2u * T, m * 4u * T};
    // (a tile on the diagonal of a square is its own mirror image)
    const HalfTarget rows{SYMMETRIC && m == n ? nullptr : by_row + (uint64_t)matrix * blocks_m * steps_n * 128u, blocks_m, steps_n, m * 2u * T, n * 4u * T};
    half_store<T>(shared.turned, columns, rows, [&](int i, int j, int k, uint32_t row, uint32_t column) {
        row += row0; column += column0;
        if (row >= P.M || column >= P.N) return 0.f;
        float v = half_sum(acc, i, j, k) * down;
        if constexpr (KIND == SQUARE) out[each + (uint64_t)row * P.N + column] = v;
        if constexpr (KIND == POLYNOMIAL) v = __builtin_fmaf(P.c, v, __builtin_fmaf(P.b, squares[i][j][k], row == column ? P.a : 0.f));
        return v * up;
    });
}
#define ORTHOGONAL(NAME, KIND, SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void orthogonal_##NAME##SUFFIX(u32x4* by_column, u32x4* by_row, float* out, float* partial, uint32_t* arrivals, \
                                                                                        const u32x4* a, const u32x4* b, const float* square, OrthogonalParams P) {    \
        orthogonal_body<KIND, T, STAGES, SHARED>(by_column, by_row, out, partial, arrivals, a, b, square, P);                                                         \
    }
#define ORTHOGONAL_KINDS(SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                           \
    ORTHOGONAL(square, SQUARE, SUFFIX, T, STAGES, BLOCKS, SHARED) ORTHOGONAL(polynomial, POLYNOMIAL, SUFFIX, T, STAGES, BLOCKS, SHARED)                               \
    ORTHOGONAL(next, NEXT, SUFFIX, T, STAGES, BLOCKS, SHARED) ORTHOGONAL(last, LAST, SUFFIX, T, STAGES, BLOCKS, SHARED)
// (contractions that are not shared have kernels of their own: what adds slices up costs registers, 372 -> 400 us for 4096^3)
ORTHOGONAL_KINDS(_128, 2, 2, 2, false)
ORTHOGONAL_KINDS(_128_shared, 2, 2, 2, true)
ORTHOGONAL_KINDS(_64, 1, 4, 2, false)
// (of the others half_plan shares none: their contractions are as long as the matrix has rows, and where that is long there are tiles enough)
ORTHOGONAL(square, SQUARE, _64_shared, 1, 4, 2, true)
ORTHOGONAL_KINDS(_64_many, 1, 2, 4, false)
ORTHOGONAL_KINDS(_64_many_shared, 1, 2, 4, true)
