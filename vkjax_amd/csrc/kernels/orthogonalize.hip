// Matrices with their singular values brought towards 1 by a polynomial: X = x / (|x| + eps) (Frobenius norm, per matrix), then `steps` times
//   A = X X^T,  B = a I + b A + c A A,  X <- B X          (of the wide way round: a matrix with more rows than columns is transposed)
// so that every singular value s becomes a s + b s^3 + c s^5. Products are those of half_product.h, between operands that never leave their taken-apart form: a product's tile
// turns its results into an operand, X into one contracted over its columns (turned in shared memory), which B X reads turned again (contracted over rows). A and B are symmetric:
// of their tiles only those on and above the diagonal are computed, and stored both ways. Only A is kept as fp32 too, since b A is a term of B. X has 22 bits between the steps; no
// operand's magnitude depends on the data beyond |x|, since a singular value's bound follows from the polynomial alone, so scales are known to the host - but for a matrix that eps leaves small: X is
// scaled by 2^small more then, small by how far |x| / (|x| + eps) is below 1, less `grown`, what the steps in front may have made of it.
// Matrices of a stack lie side by side in every launch.
// Bound by the matrix cores' power where a matrix fills the machine: 4096 x 4096 takes 212 us for a square, 257 for the polynomial (whose epilogue reads the square), 380 for B X (362 TFLOP/s of fp32
// products), 4.45 ms for five steps, of which the products alone at that rate are 3.6. 12 of 512 x 512: 13 to 18 us a launch, whose contraction of 512 is 16 pairs of steps behind one another.
#include "half_product.h"

typedef f32x4 f32x4_anywhere __attribute__((aligned(4)));

__device__ __forceinline__ double wave_sum(double t) {
    wave_butterfly([&](auto step) { t += __builtin_bit_cast(double, lane_xor<decltype(step)::value>(__builtin_bit_cast(uint64_t, t))); });
    return t;
}
struct SquaresParams { uint32_t blocks, pad; uint64_t n; };
// [matrix][block]: sums of squares, in fp64, whose range has the squares of all fp32 numbers (and whose rate leaves the launch to memory)
extern "C" __global__ __launch_bounds__(256) void orthogonal_squares(double* __restrict__ sums, const float* __restrict__ x, SquaresParams P) {
    __shared__ double part[4];
    const uint32_t matrix = blockIdx.x / P.blocks, block = blockIdx.x % P.blocks;
    const float* const from = x + matrix * P.n;
    const uint64_t stride = (uint64_t)P.blocks * 256u;
    double s[4] = {};
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
            for (int e = 0; e < 4; ++e) s[e] = __builtin_fma((double)v[k][e], (double)v[k][e], s[e]);
    }
    for (at = 4u * vectors + (uint64_t)block * 256u + threadIdx.x; at < P.n; at += stride) s[0] = __builtin_fma((double)from[at], (double)from[at], s[0]);
    const double t = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
    if ((threadIdx.x & 63u) == 0u) part[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0u) sums[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X taken apart, contracted over its columns [rows][columns]. A wave takes up to `each` steps of a block of 32.
struct OrthogonalPackParams {
    uint32_t matrices, R, C, sum_blocks, each, blocks;                                   // blocks of 256 threads, per matrix
    uint64_t sr, sc;                                                                     // element strides of row and column
    float eps; int32_t scale; uint32_t grown, pad;
};
__device__ __forceinline__ int exponent_of(double v) { return (int)(__builtin_bit_cast(uint64_t, v) >> 52 & 0x7FFu) - 1023; }
__device__ __forceinline__ int more_scale(uint32_t small, uint32_t grown) { return (int)(small > grown ? small - grown : 0u); }
extern "C" __global__ __launch_bounds__(256) void orthogonal_pack(u32x4* __restrict__ by_row, uint32_t* __restrict__ smalls, const float* __restrict__ x, const double* __restrict__ sums, OrthogonalPackParams P) {
    __shared__ double part[4];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t matrix = blockIdx.x / P.blocks, block = blockIdx.x - matrix * P.blocks;
    double t = 0.0;
    for (uint32_t k = threadIdx.x; k < P.sum_blocks; k += 256u) t += sums[(uint64_t)matrix * P.sum_blocks + k];
    t = wave_sum(t);
    if (lane == 0u) part[wave] = t;
    __syncthreads();
    // the norm as a number between 1 and 2 and a power of two, which fp32's range need not have (one that is not finite makes all of its matrix NaN)
    const double own_norm = __builtin_sqrt((part[0] + part[1]) + (part[2] + part[3])), all_norm = own_norm + (double)P.eps;
    // (a matrix of zeros has no exponent)
    const uint32_t small = own_norm > 0.0 ? (uint32_t)(exponent_of(all_norm) - exponent_of(own_norm)) : 0u;
    if (block == 0u && threadIdx.x == 0u) smalls[matrix] = small;
    const int up = P.scale + more_scale(small, P.grown) - exponent_of(all_norm);
    const float norm = all_norm < __builtin_inf() ? (float)__builtin_bit_cast(double, (__builtin_bit_cast(uint64_t, all_norm) & 0xFFFFFFFFFFFFFull) | 1023ull << 52) : __builtin_nanf("");
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
            for (int q = 0; q < 4; ++q) { uint32_t a, b; half_parts(__builtin_amdgcn_ldexpf(v[t][2 * q] / norm, up), __builtin_amdgcn_ldexpf(v[t][2 * q + 1] / norm, up), a, b); hi[q] = a; lo[q] = b; }
            to[(s0 + t) * 128u] = hi; to[(s0 + t) * 128u + 64u] = lo;
        }
    }
}

// What a launch of products computes
enum OrthogonalKind : uint32_t { SQUARE = 0, POLYNOMIAL = 1, NEXT = 2, LAST = 3 };
struct OrthogonalParams {
    uint32_t kind, M, N, K, tiles_m, tiles_n, tiles;     // tiles of a matrix: those on and above the diagonal of a square
    int32_t scale_a, scale_b, scale_out;
    float a, b, c; uint32_t whole, slices;               // (HalfShares)
    uint32_t grown, grown_next, pad;
    uint64_t sr, sc;                                     // the last result's element strides
};
// (kinds in templates: their epilogues share no registers)
template <uint32_t KIND, int T, int STAGES, bool SHARED>
__device__ __forceinline__ void orthogonal_body(u32x4* __restrict__ by_column, u32x4* __restrict__ by_row, float* __restrict__ out, float* __restrict__ partial, uint32_t* __restrict__ arrivals,
                                                const u32x4* __restrict__ a, const u32x4* __restrict__ b, const float* __restrict__ square, const uint32_t* __restrict__ smalls, const OrthogonalParams& P) {
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
    // (both operands' scales at once: their factors' product may be below what fp32 has where a result is not; X's own is what the matrix has more)
    const int more = KIND == POLYNOMIAL ? 0 : more_scale(smalls[matrix], P.grown);
    const int down = -(P.scale_a + P.scale_b) - (KIND == SQUARE ? 2 : 1) * more, up = P.scale_out + (KIND == NEXT ? more_scale(smalls[matrix], P.grown_next) : 0);
    auto result = [&](int i, int j, int k) { return __builtin_amdgcn_ldexpf(half_sum(acc, i, j, k), down); };
    const uint32_t row0 = m * SIDE, column0 = n * SIDE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t lane_row = row0 + (wave >> 1) * 32u * T + 4u * (lane >> 5), lane_column = column0 + (wave & 1u) * 32u * T + (lane & 31u);
    const uint64_t each = (uint64_t)matrix * P.M * P.N;
    if constexpr (KIND == LAST) {
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int k0 = 0; k0 < 16; k0 += 4) {
                    // (four rows that are neighbours, in memory too where the matrix is tall)
                    const uint32_t row = lane_row + 32u * i + 2u * k0, column = lane_column + 32u * j;
                    float* const to = out + each + row * P.sr + column * P.sc;
                    if (column >= P.N) continue;
                    if (P.sr == 1u && row + 4u <= P.M)
                        *reinterpret_cast<f32x4_anywhere*>(to) = f32x4{result(i, j, k0), result(i, j, k0 + 1), result(i, j, k0 + 2), result(i, j, k0 + 3)};
                    else
#pragma unroll
                        for (uint32_t e = 0; e < 4u; ++e) if (row + e < P.M) to[e * P.sr] = result(i, j, k0 + e);
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
        if constexpr (KIND == NEXT) return __builtin_amdgcn_ldexpf(half_sum(acc, i, j, k), down + up);
        float v = result(i, j, k);
        if constexpr (KIND == SQUARE) out[each + (uint64_t)row * P.N + column] = v;
        if constexpr (KIND == POLYNOMIAL) v = __builtin_fmaf(P.c, v, __builtin_fmaf(P.b, squares[i][j][k], row == column ? P.a : 0.f));
        return __builtin_amdgcn_ldexpf(v, up);
    });
}
#define ORTHOGONAL(NAME, KIND, SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void orthogonal_##NAME##SUFFIX(u32x4* by_column, u32x4* by_row, float* out, float* partial, uint32_t* arrivals, \
                                                                                        const u32x4* a, const u32x4* b, const float* square, const uint32_t* smalls,  \
                                                                                        OrthogonalParams P) {                                                         \
        orthogonal_body<KIND, T, STAGES, SHARED>(by_column, by_row, out, partial, arrivals, a, b, square, smalls, P);                                                 \
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

// ---- few rows (4 to 64 of the wide way round). All of the polynomials are functions of G = X X^T, so that G alone goes through the steps, G <- B G B, P <- B P, by a block per matrix, and X only
// through the first product and the last, P X. That is three launches instead of two and three for every step. G starts in fp64, from products that are exact there, and stays in it (v_mfma_f64_16x16x4):
// a small singular value s is there as s^2, and what fp32 would lose of that beside the largest is what decides its polynomial. P X is a product of fp32 numbers.
// (Errors of G grow with the small eigenvalues and are not made good by a product X X^T in every step: for as many steps as leave them below 2^-24, six with a = 3.44, 18 with 1.5.)
// Lanes of the instruction: operands row (column) l % 16 and k = l / 16, results row 4 q + l / 16, column l % 16. Symmetric matrices have their blocks on and above the diagonal computed.
typedef double f64x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t SMALL = 64u, SMALL_BLOCKS = 10u;
__device__ __forceinline__ uint32_t upper_block(uint32_t i, uint32_t j) { return j * (j + 1u) / 2u + i; }

struct GramParams { uint32_t R, C, slices, each; uint64_t sr, sc; };        // each: columns of a slice, a multiple of 64
// [matrix][slice][upper block][q][lane]
extern "C" __global__ __launch_bounds__(256) void orthogonal_gram(double* __restrict__ sums, const float* __restrict__ x, GramParams P) {
    __shared__ double met[3][SMALL_BLOCKS][4][64];
    const uint32_t matrix = blockIdx.x / P.slices, slice = blockIdx.x % P.slices, lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t blocks = (P.R + 15u) / 16u, row = lane & 15u, quarter = lane >> 4, end = min(P.C, (slice + 1u) * P.each);
    const float* const from = x + (uint64_t)matrix * P.R * P.C;
    const bool along = P.sc == 1u;
    f64x4 acc[SMALL_BLOCKS] = {};
    float next[4][4];
    // 16 columns: four to a lane's vector where they are neighbours, every fourth one otherwise
    auto request = [&](uint32_t c0) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            if (i >= blocks) continue;
            const float* const at = from + min(16u * i + row, P.R - 1u) * P.sr;
            if (along && c0 + 16u <= P.C) {
                const f32x4 v = *reinterpret_cast<const f32x4_anywhere*>(at + c0 + 4u * quarter);
#pragma unroll
                for (int e = 0; e < 4; ++e) next[i][e] = v[e];
            } else
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) next[i][e] = at[min(c0 + (along ? 4u * quarter + e : 4u * e + quarter), P.C - 1u) * P.sc];
        }
    };
    uint32_t c0 = slice * P.each + 16u * wave;
    if (c0 < end) request(c0);
    for (; c0 < end; c0 += 64u) {
        double v[4][4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                const uint32_t c = c0 + (along ? 4u * quarter + e : 4u * e + quarter);
                v[i][e] = i < blocks && 16u * i + row < P.R && c < end ? (double)next[i][e] : 0.0;
            }
        if (c0 + 64u < end) request(c0 + 64u);
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j)
#pragma unroll
            for (uint32_t i = 0; i <= j; ++i)
                if (j < blocks)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[upper_block(i, j)] = __builtin_amdgcn_mfma_f64_16x16x4f64(v[i][e], v[j][e], acc[upper_block(i, j)], 0, 0, 0);
    }
    if (wave > 0u)
#pragma unroll
        for (uint32_t b = 0; b < SMALL_BLOCKS; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q) met[wave - 1u][b][q][lane] = acc[b][q];
    __syncthreads();
    if (wave > 0u) return;
    const uint32_t upper = blocks * (blocks + 1u) / 2u;
    double* const to = sums + (uint64_t)blockIdx.x * upper * 256u + lane;
#pragma unroll
    for (uint32_t b = 0; b < SMALL_BLOCKS; ++b)
        if (b < upper)
#pragma unroll
        for (int q = 0; q < 4; ++q) to[(b * 4u + q) * 64u] = ((acc[b][q] + met[0][b][q][lane]) + met[1][b][q][lane]) + met[2][b][q][lane];
}

struct SmallParams { uint32_t R, slices, steps; float a, b, c, eps; uint32_t pad; };
// P / (|x| + eps) of every matrix, fp32, [S][S] for its rows in whole blocks of 16, zeros behind the last. Up to 16 waves, so that a SIMD has others to multiply for while one waits for shared memory (with four,
// a block to each SIMD's one wave, five steps of 64 x 64 took 56 us, not 36); waves and shared memory as the matrix wants them, so that a CU has several small ones. Rows of S + 2 doubles: 16 rows'
// pairs of words lie in different banks.
extern "C" __global__ __launch_bounds__(1024) void orthogonal_small(float* __restrict__ polynomials, const double* __restrict__ sums, SmallParams P) {
    extern __shared__ double memory[];                          // G, B, P
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, blocks = (P.R + 15u) / 16u, upper = blocks * (blocks + 1u) / 2u;
    const uint32_t S = 16u * blocks, pitch = S + 2u;
    double* const G = memory, * const B = G + S * pitch, * const Q = B + S * pitch;
    // element q of this lane of an upper block, and its mirror image
    auto block_of = [&](uint32_t number, uint32_t& i, uint32_t& j) { j = number < 1u ? 0u : number < 3u ? 1u : number < 6u ? 2u : 3u; i = number - j * (j + 1u) / 2u; };
    auto put = [&](double* m, uint32_t i, uint32_t j, const f64x4& v) {
#pragma unroll
        for (uint32_t q = 0; q < 4u; ++q) {
            const uint32_t r = 16u * i + 4u * q + (lane >> 4), c = 16u * j + (lane & 15u);
            m[r * pitch + c] = v[q];
            if (i != j) m[c * pitch + r] = v[q];
        }
    };
    // block (i, j) of the product of two symmetric matrices
    auto product = [&](const double* m, const double* n, uint32_t i, uint32_t j) {
        f64x4 s = {0.0, 0.0, 0.0, 0.0};
        const double* const a = m + (16u * i + (lane & 15u)) * pitch + (lane >> 4);
        const double* const b = n + (16u * j + (lane & 15u)) * pitch + (lane >> 4);
#pragma unroll 2
        for (uint32_t k = 0; k < 16u * blocks; k += 16u)
#pragma unroll
            for (uint32_t e = 0; e < 16u; e += 4u) s = __builtin_amdgcn_mfma_f64_16x16x4f64(a[k + e], b[k + e], s, 0, 0, 0);
        return s;
    };
    for (uint32_t number = wave; number < upper; number += waves) {
        uint32_t i, j;
        block_of(number, i, j);
        const double* const from = sums + ((uint64_t)blockIdx.x * P.slices * upper + number) * 256u + lane;
        f64x4 s = {0.0, 0.0, 0.0, 0.0};
        for (uint32_t k = 0; k < P.slices; k += 4u) {
            f64x4 v[4];
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u)
#pragma unroll
                for (uint32_t q = 0; q < 4u; ++q) v[u][q] = from[(uint64_t)min(k + u, P.slices - 1u) * upper * 256u + q * 64u];
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u)
                if (k + u < P.slices)
#pragma unroll
                    for (uint32_t q = 0; q < 4u; ++q) s[q] += v[u][q];
        }
        put(G, i, j, s);
    }
    __syncthreads();
    double squares = 0.0;
    for (uint32_t k = 0; k < P.R; ++k) squares += G[k * pitch + k];
    const double norm = __builtin_sqrt(squares) + (double)P.eps, down = 1.0 / (norm * norm);
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < S * S; k += blockDim.x) G[k / S * pitch + k % S] *= down;
    __syncthreads();
    uint32_t i, j;
    block_of(min(wave, upper - 1u), i, j);
    for (uint32_t step = 0; step < P.steps; ++step) {
        // B = a I + b G + c G G
        if (wave < upper) {
            f64x4 s = product(G, G, i, j);
#pragma unroll
            for (uint32_t q = 0; q < 4u; ++q) {
                const uint32_t r = 16u * i + 4u * q + (lane >> 4), c = 16u * j + (lane & 15u);
                s[q] = (double)P.c * s[q] + (double)P.b * G[r * pitch + c] + (r == c ? (double)P.a : 0.0);
            }
            put(B, i, j, s);
        }
        __syncthreads();
        // P <- P B and G <- G B, then G <- G B once more; of the blocks of both (P's first), two at most to a wave
        const bool last = step + 1u == P.steps;
        const uint32_t units = last ? upper : 2u * upper;
        f64x4 found[2];
        auto unit = [&](uint32_t u, auto f) {
            if (u >= units) return;
            uint32_t bi, bj;
            block_of(u < upper ? u : u - upper, bi, bj);
            f(u < upper, bi, bj);
        };
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u)
            unit(wave + waves * u, [&](bool of_p, uint32_t bi, uint32_t bj) {
                if (of_p && step == 0u) {
#pragma unroll
                    for (uint32_t q = 0; q < 4u; ++q) found[u][q] = B[(16u * bi + 4u * q + (lane >> 4)) * pitch + 16u * bj + (lane & 15u)];
                } else found[u] = product(of_p ? Q : G, B, bi, bj);
            });
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u) unit(wave + waves * u, [&](bool of_p, uint32_t bi, uint32_t bj) { put(of_p ? Q : G, bi, bj, found[u]); });
        __syncthreads();
        if (last) break;
        if (wave < upper) found[0] = product(G, B, i, j);
        __syncthreads();
        if (wave < upper) put(G, i, j, found[0]);
        __syncthreads();
    }
    for (uint32_t k = threadIdx.x; k < S * S; k += blockDim.x) {
        const uint32_t r = k / S, c = k % S;
        polynomials[(uint64_t)blockIdx.x * S * S + k] = r < P.R && c < P.R ? (float)(Q[r * pitch + c] / norm) : 0.f;
    }
}

// P x, with the fp32 matrix instructions: a wave has up to 32 rows of the result and 32 of its columns, which are a lane each where x is [R][C] (four to a lane: a lone wave's products take 4 us,
// not one, and large matrices gain nothing), and a row each where it lies the other way round.
struct ApplyParams { uint32_t R, C, tasks, blocks; };                       // tasks of a matrix, one a wave; blocks of four waves a matrix
template <bool WIDE, int ROWS>
__device__ __forceinline__ void orthogonal_apply_body(float* __restrict__ out, const float* __restrict__ x, const float* __restrict__ polynomials, const ApplyParams& P) {
    __shared__ float poly[SMALL][SMALL];
    constexpr uint32_t HALVES = ROWS == 64 ? 2u : 1u;
    const uint32_t matrix = blockIdx.x / P.blocks, task = (blockIdx.x % P.blocks) * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t half = threadIdx.x >> 5 & 1u, l32 = threadIdx.x & 31u, r0 = task % HALVES * 32u, c0 = task / HALVES * 32u, c = min(c0 + l32, P.C - 1u);
    const uint64_t first = (uint64_t)matrix * P.R * P.C;
    // (columns and rows behind the end are the last ones again; what is stored twice is the same)
    float v[ROWS / 2];
    if constexpr (WIDE) {
#pragma unroll
        for (uint32_t k = 0; k < ROWS / 2; ++k) v[k] = x[first + (uint64_t)min(2u * k + half, P.R - 1u) * P.C + c];
    } else
#pragma unroll
        for (uint32_t k = 0; k < ROWS / 8; ++k) {
            const f32x4 t = *reinterpret_cast<const f32x4_anywhere*>(x + first + (uint64_t)c * P.R + min(8u * k + 4u * half, P.R - 4u));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * k + e] = t[e];
        }
    const uint32_t S = (P.R + 15u) / 16u * 16u;
    const float* const from = polynomials + (uint64_t)matrix * S * S;
    constexpr uint32_t VECTORS = (ROWS < 32 ? 32 : ROWS) / 4;
#pragma unroll
    for (uint32_t k0 = 0; k0 < ROWS * VECTORS; k0 += 256u) {
        const uint32_t k = k0 + threadIdx.x, r = k / VECTORS, at = k % VECTORS * 4u;
        const f32x4 p = *reinterpret_cast<const f32x4*>(from + min(r, S - 1u) * S + min(at, S - 4u));
        if (k < ROWS * VECTORS) *reinterpret_cast<f32x4*>(&poly[r][at]) = r < S && at < S ? p : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
    if (task >= P.tasks || r0 >= P.R) return;
    f32x16 acc = {};
#pragma unroll
    for (uint32_t k = 0; k < ROWS / 2; ++k) {
        if constexpr (WIDE) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(poly[2u * k + half][r0 + l32], v[k], acc, 0, 0, 0);      // (behind the last row: zeros, times x's last row again)
        else {
            const uint32_t wanted = 8u * (k / 4u) + 4u * half, at = min(wanted, P.R - 4u) + k % 4u;
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(at >= wanted ? v[k] : 0.f, poly[at][r0 + l32], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const uint32_t r = 8u * (q >> 2) + 4u * half + (q & 3);
        if constexpr (WIDE) { if (r0 + r < P.R) out[first + (uint64_t)(r0 + r) * P.C + c] = acc[q]; }
        else if (c0 + r < P.C && r0 + l32 < P.R) out[first + (uint64_t)(c0 + r) * P.R + r0 + l32] = acc[q];
    }
}
#define ORTHOGONAL_APPLY(NAME, WIDE, ROWS)                                                                                                                            \
    extern "C" __global__ __launch_bounds__(256) void orthogonal_apply_##NAME##_##ROWS(float* out, const float* x, const float* polynomials, ApplyParams P) {         \
        orthogonal_apply_body<WIDE, ROWS>(out, x, polynomials, P);                                                                                                    \
    }
ORTHOGONAL_APPLY(wide, true, 16)
ORTHOGONAL_APPLY(wide, true, 32)
ORTHOGONAL_APPLY(wide, true, 64)
ORTHOGONAL_APPLY(tall, false, 16)
ORTHOGONAL_APPLY(tall, false, 32)
ORTHOGONAL_APPLY(tall, false, 64)
