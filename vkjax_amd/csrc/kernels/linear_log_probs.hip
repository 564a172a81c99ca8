// Log probabilities of given tokens under softmax(x W), without keeping the scores x W, and their gradient.
//
//   s[r, v] = sum_h x[r, h] W[h, v];  peak = max_v s,  total = sum_v exp(s - peak);  log_sum = peak + log(total),  log_prob = s[r, token] - log_sum
//   ds = g_lp [v = token] + (g_ls - g_lp) p,  p = exp(s - peak) / total;  dx = ds W^T,  dW = x^T ds
// A row whose token lies outside the vocabulary is padding: zeros, x is not looked at there, no gradient.
//
// Products are those of half_product.h: x and W are taken apart first (the largest magnitudes, for their scales, then the parts; numbers that are too far apart for that stay as they are), then
//   * forward: a product whose rows are the vocabulary and whose columns are the rows of x, so that a lane has 32 scores of one row; a tile of 128 tokens leaves each row's peak and
//     sum, a last launch joins the tiles. 4096 x 1024 x 32000: the product as fast as one that keeps its scores, and nothing of 0.5 GB is written.
//   * backward, in pieces of the vocabulary: the same product again, whose lanes turn scores into q = ds / m, |q| <= 2, with m = max(|g_lp|, |g_ls - g_lp|) of the row, and store q as an operand
//     (4 bytes a score of a piece). dx = q W^T reads q as it is and the forward pass's W turned, dW = x^T ds reads q turned (half_product.h), so neither is laid out twice; the rows' m is a factor
//     of dx's rows, and of the x that dW is made of. (Taken apart both ways, W and q: 321 x 500 x 50001 490 us, not 424, 172 x 1400 x 46807 880, not 733, 4096 x 1024 x 32000 3500, not 3340.)
// 4096 x 1024 x 32000 with its gradient: 745 us the scores (360 TFLOP/s of fp32 products), 780 q, 790 each dx and dW (the floor of 268 GFLOP each at 378 TFLOP/s is 710 us), 100 us to take
// operands apart. Bound by the matrix cores' power; with few rows by the weights' bytes.
// Up to 64 rows take the fp32 matrix instructions (RowsProduct), which read W as it is, once forward and once for dx: bound by memory. The scores of so few rows are kept for the gradient.
#include "half_product.h"

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int Q_SCALE = 13;                              // |q| <= 2

__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * LOG2E); }
// (two operands' scales at once: one after the other, a factor beyond fp32's range would meet a number that is inside it in the end)
__device__ __forceinline__ float scaled(float v, int e) { return __builtin_amdgcn_ldexpf(v, e); }
__device__ __forceinline__ bool is_token(int32_t t, uint32_t V) { return (uint32_t)t < V; }
typedef f32x4 f32x4_anywhere __attribute__((aligned(4)));

// (NaN counts as infinite)
__device__ __forceinline__ float magnitude(float v) { const float a = __builtin_fabsf(v); return a < __builtin_inff() ? a : __builtin_inff(); }
__device__ __forceinline__ float wave_largest(float v) {
    wave_butterfly([&](auto s) { v = fmaxf(v, lane_xor<decltype(s)::value>(v)); });
    return v;
}

// ---- the largest magnitudes of W, of x and of m x, one of each per block: [weight_blocks] then pairs [row_blocks]; a row's (m, (g_ls - g_lp) / m, g_lp / m)
struct LargestParams { uint32_t first, rows, H, V, weight_blocks, row_blocks; };
extern "C" __global__ __launch_bounds__(256) void linear_largest(float* __restrict__ largest, float* __restrict__ factors, const float* __restrict__ x, const float* __restrict__ w,
                                                                 const int32_t* __restrict__ tokens, const float* __restrict__ g_log_probs, const float* __restrict__ g_log_sums, LargestParams P) {
    __shared__ float part[2][4];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    float one = 0.f, two = 0.f;
    if (blockIdx.x < P.weight_blocks) {
        const uint64_t n = (uint64_t)P.H * P.V, stride = (uint64_t)P.weight_blocks * 1024u, at0 = (uint64_t)blockIdx.x * 1024u + threadIdx.x * 4u;
        uint64_t at = at0;
        for (; at + 3u * stride + 4u <= n; at += 4u * stride) {
            f32x4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const f32x4*>(w + at + k * stride);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) one = fmaxf(one, magnitude(v[k][e]));
        }
        for (; at < n; at += stride)
            for (uint32_t e = 0; e < 4u; ++e) if (at + e < n) one = fmaxf(one, magnitude(w[at + e]));
    } else
        for (uint32_t r = (blockIdx.x - P.weight_blocks) * 4u + wave; r < P.rows; r += P.row_blocks * 4u) {
            const bool given = is_token(tokens[r], P.V);
            const float lp = given && g_log_probs ? g_log_probs[r] : 0.f, all = (given && g_log_sums ? g_log_sums[r] : 0.f) - lp;
            // (a cotangent that is not finite is a factor of its row by itself)
            const float most = fmaxf(__builtin_fabsf(lp), __builtin_fabsf(all)), m = lp != lp || all != all ? __builtin_nanf("") : most;
            if (factors && lane == 0u) {
                const bool plain = m > 0.f && m < __builtin_inff();
                factors[3u * r] = m; factors[3u * r + 1u] = plain ? all / m : 0.f; factors[3u * r + 2u] = plain ? lp / m : 0.f;
            }
            float row = 0.f;
            const float* const from = x + (uint64_t)r * P.H;
            if (given) {
                uint32_t h = 4u * lane;
                for (; h + 4u <= P.H; h += 256u) {
                    const f32x4 v = *reinterpret_cast<const f32x4_anywhere*>(from + h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) row = fmaxf(row, magnitude(v[e]));
                }
                for (uint32_t e = 0; e < 4u; ++e) if (h + e < P.H) row = fmaxf(row, magnitude(from[h + e]));
            }
            const float scaled_row = row * m;
            one = fmaxf(one, row); two = fmaxf(two, scaled_row < __builtin_inff() ? scaled_row : 0.f);           // (what is not finite has no part in a scale)
        }
    one = wave_largest(one); two = wave_largest(two);
    if (lane == 0u) { part[0][wave] = one; part[1][wave] = two; }
    __syncthreads();
    if (threadIdx.x != 0u) return;
    one = fmaxf(fmaxf(part[0][0], part[0][1]), fmaxf(part[0][2], part[0][3]));
    two = fmaxf(fmaxf(part[1][0], part[1][1]), fmaxf(part[1][2], part[1][3]));
    if (blockIdx.x < P.weight_blocks) largest[blockIdx.x] = one;
    else { const uint32_t at = P.weight_blocks + 2u * (blockIdx.x - P.weight_blocks); largest[at] = one; largest[at + 1u] = two; }
}

// ---- operands taken apart (half_product.h), or plain ones. A taken-apart number is off by 2^-51 of its operand's largest (or 2^-22 of itself), so a score by up to 2^-50 H times the largest
// magnitudes of x and W: where that is above 2^-24, half a step of a number between 1 and 2, or a number is not finite, the operands are plain, and with them x and q of the gradient. A row of x that is
// 10^20 times as large as the others, or a token that is masked by a weight of -10^30, leaves the other rows and tokens what they are by themselves.
// `scales`: of the kinds of operands, and whether they are plain. (`given`: the scales of the forward pass, where its operands are taken as they are.)
constexpr int PLAIN = 3;
__device__ __forceinline__ bool too_far_apart(float largest_w, float largest_x, uint32_t H) { return !(largest_w * largest_x * (float)H <= 0x1p26f); }

// What element (i, k) of an operand is: W or x as they lie, x only of rows that are given, or with the rows' factors.
enum PackKind : uint32_t { PACK_WEIGHTS = 0, PACK_ROWS = 1, PACK_SCALED = 2 };
struct PackJob { uint32_t blocks, I, K, stride, kind, steps; uint64_t si, sk; };      // blocks of 256 threads; steps of 16 k; element strides of i and k; `stride`: steps that a wave takes
struct PackParams { uint32_t weight_blocks, row_blocks, V, H; PackJob jobs[3]; };
struct PackOuts { void* parts[3]; };
extern "C" __global__ __launch_bounds__(256) void linear_pack(PackOuts outs, int32_t* __restrict__ scales, const float* __restrict__ x, const float* __restrict__ w,
                                                              const int32_t* __restrict__ tokens, const float* __restrict__ largest, const float* __restrict__ factors,
                                                              const int32_t* __restrict__ given, PackParams P) {
    __shared__ float part[3][4];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t block = blockIdx.x, job = 0u;
    while (job < 2u && block >= P.jobs[job].blocks) block -= P.jobs[job++].blocks;
    const PackJob J = P.jobs[job];
    // the operands' scales, of their blocks' largest magnitudes
    const bool weights = J.kind == PACK_WEIGHTS;
    float most[3] = {};
    for (uint32_t k = threadIdx.x; k < P.weight_blocks; k += 256u) most[0] = fmaxf(most[0], largest[k]);
    for (uint32_t k = threadIdx.x; k < P.row_blocks; k += 256u)
#pragma unroll
        for (uint32_t kind = 1; kind < 3u; ++kind) most[kind] = fmaxf(most[kind], largest[P.weight_blocks + 2u * k + kind - 1u]);
#pragma unroll
    for (int kind = 0; kind < 3; ++kind) {
        most[kind] = wave_largest(most[kind]);
        if (lane == 0u) part[kind][wave] = most[kind];
    }
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 3; ++kind) most[kind] = fmaxf(fmaxf(part[kind][0], part[kind][1]), fmaxf(part[kind][2], part[kind][3]));
    const bool plain = given ? given[PLAIN] != 0 : too_far_apart(most[PACK_WEIGHTS], most[PACK_ROWS], P.H);
    const int e = plain ? 0 : half_scale(weights ? most[PACK_WEIGHTS] : J.kind == PACK_ROWS ? most[PACK_ROWS] : most[PACK_SCALED]);
    if (block == 0u && threadIdx.x == 0u) { scales[J.kind] = e; if (job == 0u) scales[PLAIN] = plain; }
    const float up = power_of_two(e);
    // waves beside one another along the side that is contiguous in memory
    const uint32_t groups = (J.steps + J.stride - 1u) / J.stride, all = block * 4u + wave, rows32 = (J.I + 31u) / 32u;
    const bool along_k = J.sk == 1u;
    const uint32_t rb = along_k ? all / groups : all % rows32, group = along_k ? all % groups : all / rows32;
    if (rb >= rows32 || group >= groups) return;
    const uint32_t i = rb * 32u + (lane & 31u), h4 = 4u * (lane >> 5);
    const float* const from = (weights ? w : x) + (uint64_t)min(i, J.I - 1u) * J.si;
    bool there = i < J.I;
    if (J.kind == PACK_ROWS) there = there && is_token(tokens[min(i, J.I - 1u)], P.V);
    // (the operands of four steps at once)
    constexpr int AT_ONCE = 4;
    const uint32_t end = min(J.steps, (group + 1u) * J.stride);
    u32x4* const to = reinterpret_cast<u32x4*>(outs.parts[job]) + (uint64_t)rb * J.steps * 128u + lane;
    for (uint32_t s0 = group * J.stride; s0 < end; s0 += AT_ONCE) {
        float v[AT_ONCE][8];
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t k = (s0 + t) * 16u + h4 + 8u * q;
                if (along_k && k + 4u <= J.K && there) {
                    const f32x4 f = *reinterpret_cast<const f32x4_anywhere*>(from + k);
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) v[t][4 * q + e4] = f[e4];
                } else
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) v[t][4 * q + e4] = there && k + e4 < J.K ? from[(uint64_t)(k + e4) * J.sk] : 0.f;
            }
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t) {
            if (s0 + t >= end) break;
            if (J.kind == PACK_SCALED)
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint32_t k = (s0 + t) * 16u + h4 + 8u * (q >> 2) + (q & 3);
                    const float m = k < J.K ? factors[3u * k] : 0.f;
                    v[t][q] = m == 0.f ? 0.f : plain ? v[t][q] : v[t][q] * m;           // (a row without a cotangent has none, whatever its x is)
                }
            u32x4 hi, lo;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t a, b;
                if (plain) plain_parts(v[t][2 * q], v[t][2 * q + 1], a, b); else half_parts(v[t][2 * q] * up, v[t][2 * q + 1] * up, a, b);
                hi[q] = a; lo[q] = b;
            }
            to[(s0 + t) * 128u] = hi; to[(s0 + t) * 128u + 64u] = lo;
        }
    }
}

// ---- forward: a tile's peak and sum per row of x, [tile of tokens][rows]
struct ScoresParams { uint32_t rows, V, pairs, steps_w, steps_x, tiles_m, tiles_n, blocks_w, blocks_x, tile0, Vp, whole, slices; };

__device__ __forceinline__ HalfOperand operand_of(const u32x4* parts, uint32_t blocks, uint32_t stride, uint32_t first = 0) { return HalfOperand{parts, blocks, stride, first}; }
__device__ __forceinline__ float over_halves_max(float v) { return fmaxf(v, lane_xor<32>(v)); }
__device__ __forceinline__ float over_halves_sum(float v) { return v + lane_xor<32>(v); }

template <int T, int STAGES, bool SHARED>
__device__ __forceinline__ void linear_scores_body(float* __restrict__ peaks, float* __restrict__ sums, float* __restrict__ of_token, float* __restrict__ partial, uint32_t* __restrict__ arrivals,
                                                   const u32x4* __restrict__ w, const u32x4* __restrict__ x, const int32_t* __restrict__ tokens, const int32_t* __restrict__ scales,
                                                   const ScoresParams& P) {
    constexpr uint32_t SIDE = HalfTileOf<T>::SIDE;
    __shared__ HalfShared<T, STAGES> shared;
    uint32_t m, n, tile, slice, begin, end;
    half_work(blockIdx.x, HalfShares{P.whole, P.slices}, P.pairs, tile, slice, begin, end);
    half_tile(tile, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    half_product<T, STAGES, TURNED_NONE, true>(acc, shared, operand_of(w, P.blocks_w, P.steps_w), operand_of(x, P.blocks_x, P.steps_x), m, n, begin, end - begin, scales + PLAIN);
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, HalfShares{P.whole, P.slices})) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, wm = wave >> 1, wn = wave & 1u;
    const int down = -(scales[PACK_WEIGHTS] + scales[PACK_ROWS]);
    float (*const met)[SIDE][2] = reinterpret_cast<float (*)[SIDE][2]>(&shared.stages[0]);  // [wm][column][peak, sum]
    const uint32_t v0 = m * SIDE + wm * 32u * T + 4u * (lane >> 5);
#pragma unroll
    for (int j = 0; j < T; ++j) {
        const uint32_t column = (wn * T + j) * 32u + (lane & 31u), r = n * SIDE + column;
        const int32_t token = r < P.rows ? tokens[r] : -1;
        float peak = -__builtin_inff(), sum = 0.f, mine = 0.f;
        bool has = false;
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const uint32_t v = v0 + 32u * i + 8u * (q >> 2) + (q & 3);
                float s = scaled(half_sum(acc, i, j, q), down);
                if (v == (uint32_t)token) { mine = s; has = true; }
                s = v < P.V ? s : -__builtin_inff();
                acc.large[i][j][q] = s;
                peak = fmaxf(peak, s);
            }
        if (has && is_token(token, P.V)) of_token[r] = mine;
        peak = over_halves_max(peak);
        const float base = peak == -__builtin_inff() ? 0.f : peak;
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) sum += exp_of(acc.large[i][j][q] - base);
        sum = over_halves_sum(sum);
        if (lane < 32u) { met[wm][column][0] = peak; met[wm][column][1] = sum; }
    }
    __syncthreads();
    if (threadIdx.x < SIDE) {
        const uint32_t r = n * SIDE + threadIdx.x;
        const float p0 = met[0][threadIdx.x][0], p1 = met[1][threadIdx.x][0], peak = fmaxf(p0, p1), base = peak == -__builtin_inff() ? 0.f : peak;
        if (r < P.rows) {
            peaks[(uint64_t)m * P.rows + r] = peak;
            sums[(uint64_t)m * P.rows + r]  = met[0][threadIdx.x][1] * exp_of(p0 - base) + met[1][threadIdx.x][1] * exp_of(p1 - base);
        }
    }
}
#define LINEAR_SCORES(SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                                \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void linear_scores##SUFFIX(float* peaks, float* sums, float* of_token, float* partial, uint32_t* arrivals,     \
                                                                                    const u32x4* w, const u32x4* x, const int32_t* tokens, const int32_t* scales,       \
                                                                                    ScoresParams P) {                                                                   \
        linear_scores_body<T, STAGES, SHARED>(peaks, sums, of_token, partial, arrivals, w, x, tokens, scales, P);                                                       \
    }
// (the kernels of half_product.h, by suffix)
#define LINEAR_KERNELS(F) F(_128, 2, 2, 2, false) F(_128_shared, 2, 2, 2, true) F(_64, 1, 4, 2, false) F(_64_shared, 1, 4, 2, true) F(_64_many, 1, 2, 4, false) F(_64_many_shared, 1, 2, 4, true)
LINEAR_KERNELS(LINEAR_SCORES)

// A row's tiles joined. A block has R rows (a power of two up to 64): 1024 / R lanes to a row, which take tiles in turn, eight at a time, and meet by butterflies and in shared memory.
struct JoinParams { uint32_t log2_rows, rows, V, tiles; };
struct PeakSum {
    float peak, sum;
    __device__ __forceinline__ void add(float p, float s) {
        const float next = fmaxf(peak, p), base = next == -__builtin_inff() ? 0.f : next;
        sum = sum * exp_of(peak - base) + s * exp_of(p - base);
        peak = next;
    }
};
extern "C" __global__ __launch_bounds__(1024) void linear_join(float* __restrict__ log_probs, float* __restrict__ log_sums, float* __restrict__ row_peaks, float* __restrict__ row_totals,
                                                               const float* __restrict__ peaks, const float* __restrict__ sums, const float* __restrict__ of_token,
                                                               const int32_t* __restrict__ tokens, JoinParams P) {
    __shared__ float met[16][64][2];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, R = 1u << P.log2_rows, row = lane & (R - 1u), r = blockIdx.x * R + row, at = min(r, P.rows - 1u);
    const uint32_t groups = 1024u >> P.log2_rows, group = threadIdx.x >> P.log2_rows;
    PeakSum all = {-__builtin_inff(), 0.f};
    for (uint32_t t0 = group; t0 < P.tiles; t0 += 8u * groups) {
        float p[8], s[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) {
            const bool has = t0 + k * groups < P.tiles;
            const uint64_t from = (uint64_t)min(t0 + k * groups, P.tiles - 1u) * P.rows + at;
            const float pk = peaks[from], sk = sums[from];
            p[k] = has ? pk : -__builtin_inff(); s[k] = has ? sk : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) all.add(p[k], s[k]);
    }
    wave_butterfly([&](auto step) {
        constexpr int S = decltype(step)::value;
        const float p = lane_xor<S>(all.peak), s = lane_xor<S>(all.sum);
        if ((uint32_t)S >= R) all.add(p, s);
    });
    met[wave][lane][0] = all.peak; met[wave][lane][1] = all.sum;
    __syncthreads();
    if (wave != 0u || lane >= R || r >= P.rows) return;
#pragma unroll
    for (int q = 1; q < 16; ++q) all.add(met[q][lane][0], met[q][lane][1]);
    const bool given = is_token(tokens[r], P.V);
    const float log_total = __builtin_amdgcn_logf(all.sum) * LN2;
    if (log_probs) log_probs[r] = given ? (of_token[r] - all.peak) - log_total : 0.f;
    if (log_sums)  log_sums[r]  = given ? all.peak + log_total : 0.f;
    if (row_peaks)  row_peaks[r]  = given ? all.peak : 0.f;
    if (row_totals) row_totals[r] = given ? all.sum : 1.f;
}

// ---- up to 32 NT rows: out[m, r] = sum_k A[m, k] b[r, k] with fp32 matrix instructions, A as it lies (its columns along M: [K][M], or along K: [M][K]) and read once, b [rows][K].
// v_mfma_f32_32x32x2_f32: lane l has row l % 32 of a block of 32 and k = l / 32; which m a lane's row is, and in which order k comes, follows from how A lies. A block has 128 m, its waves
// parts of k, a wave's loads are a step ahead of its products, or three.
//   * along M: four neighbouring m to a lane's vector, 8 k of 128 m a step;
//   * along K: 32 k of 128 m a step, loaded in whole lines and turned in the wave's own part of shared memory, whose vectors of a row are exchanged so that 8 rows of one column lie in
//     different banks. (Loaded as the instruction has them, 64 bytes of a row to a lane, lines were fetched several times: 53 x 776 x 112111 took 269 us, 1.3 TB/s.)
// Bound by memory up to 32 rows (15 x 1973 x 128040: 200 us, 5 TB/s along M, 270 along K), and by memory and the products alike at 64 (64 x 4096 x 32000: 168 us, of which either takes 107 alone).
// Blocks of four waves, two a CU, hide one another's ends: with eight waves to a block 14 x 47 x 107245 took 31 us, not 19, and 32 x 896 x 83954 93 us, not 76.
template <bool ALONG_M, int NT> struct RowsProduct {
    // blocks of 32 m: two where A is turned for 64 rows, so that two blocks of waves are there too (with four, whose sums leave room for one, 53 x 776 x 112111 takes 200 us, not 157)
    static constexpr int WAVES = 4, MB = !ALONG_M && NT == 2 ? 2 : 4;
    static constexpr uint32_t TILE = 32u * MB;
    union Shared { f32x4 turned[ALONG_M ? 1 : WAVES][MB][32][8]; f32x4 met[WAVES / 2][NT * MB * 4][64]; };
    f32x16 acc[MB][NT];

    static __device__ __forceinline__ uint32_t lane() { return threadIdx.x & 63u; }
    static __device__ __forceinline__ f32x4 load(const float* at) { return *reinterpret_cast<const f32x4_anywhere*>(at); }
    // over the k of groups [all_begin, all_end); `there`: rows that are padding are zeros, whatever b holds. M and K are 4 at least: vectors that would end behind the last m or k are moved to
    // the left, and the k's that come twice by that are zeros, of b and of A (whose infinities would be NaN otherwise). (So nothing is loaded behind a branch: with one the loads of a last group waited for one another, 25 us of a block's 84 at
    // 15 x 1973 x 128040.)
    __device__ __forceinline__ void multiply(Shared& shared, const float* __restrict__ a, const float* __restrict__ b, uint32_t m0, uint32_t M, uint32_t K, const uint32_t (&r_at)[NT],
                                             const bool (&there)[NT], uint32_t all_begin, uint32_t all_end) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane() >> 5, l32 = lane() & 31u;
        const uint32_t groups = all_end - all_begin, begin = all_begin + groups * wave / WAVES, end = all_begin + groups * (wave + 1u) / WAVES;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f32x16{};
        auto of_row = [&](int j, uint32_t k) { return load(b + (uint64_t)r_at[j] * K + min(k, K - 4u)); };
        auto is_own = [&](uint32_t k, uint32_t e) { return min(k, K - 4u) + e >= k; };
        auto own = [&](f32x4 v, int j, uint32_t k) {
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) v[e] = there[j] && is_own(k, e) ? v[e] : 0.f;
            return v;
        };
        if constexpr (ALONG_M) {
            // (lanes behind the last m read the last ones again)
            const uint32_t m_at = min(m0 + 4u * l32, M - 4u);
            constexpr uint32_t DEPTH = 4u;
            f32x4 as[DEPTH][4], bs[DEPTH][NT];
            auto request = [&](f32x4 (&av)[4], f32x4 (&bv)[NT], uint32_t g) {
                const uint32_t k0 = g * 8u + 4u * half, k = min(k0, K - 4u);
#pragma unroll
                for (int q = 0; q < 4; ++q) av[q] = load(a + (uint64_t)(k + q) * M + m_at);
#pragma unroll
                for (int j = 0; j < NT; ++j) bv[j] = of_row(j, k0);
            };
            auto products = [&](const f32x4 (&av)[4], f32x4 (&bv)[NT], uint32_t g) {
#pragma unroll
                for (int j = 0; j < NT; ++j) bv[j] = own(bv[j], j, g * 8u + 4u * half);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(av[q][i], bv[j][q], acc[i][j], 0, 0, 0);
            };
#pragma unroll
            for (uint32_t k = 0; k < DEPTH - 1u; ++k) if (begin + k < end) request(as[k], bs[k], begin + k);
            // (steps that request others without a test first: behind one, a wait for a step's loads is one for later steps' too)
            uint32_t g = begin;
            for (; g + 2u * DEPTH - 2u < end; g += DEPTH)
#pragma unroll
                for (uint32_t k = 0; k < DEPTH; ++k) {
                    request(as[(k + DEPTH - 1u) % DEPTH], bs[(k + DEPTH - 1u) % DEPTH], g + k + DEPTH - 1u);
                    __builtin_amdgcn_sched_barrier(0);
                    products(as[k], bs[k], g + k);
                    __builtin_amdgcn_sched_barrier(0);
                }
            for (; g < end; g += DEPTH)
#pragma unroll
                for (uint32_t k = 0; k < DEPTH; ++k) {
                    if (g + k + DEPTH - 1u < end) request(as[(k + DEPTH - 1u) % DEPTH], bs[(k + DEPTH - 1u) % DEPTH], g + k + DEPTH - 1u);
                    if (g + k >= end) continue;
                    if ((g + k + 1u) * 8u > K)
#pragma unroll
                        for (uint32_t q = 0; q < 4u; ++q) if (!is_own((g + k) * 8u + 4u * half, q)) as[k][q] = f32x4{0.f, 0.f, 0.f, 0.f};
                    products(as[k], bs[k], g + k);
                }
        } else {
            f32x4 (&turned)[MB][32][8] = shared.turned[wave];
            const uint32_t row8 = lane() >> 3, column = lane() & 7u;
            f32x4 next[MB][4], bs[NT][4];
            auto request = [&](uint32_t g) {
                // (rows behind the last m are the last one again; 8 rows of fewer than 2^27 elements are 32 bits of bytes)
                const uint32_t at = 4u * min(g * 32u + 4u * column, K - 4u);
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t first = min(m0 + 32u * i + 8u * t, M - 1u);
                        next[i][t] = load(reinterpret_cast<const float*>(reinterpret_cast<const char*>(a + (uint64_t)first * K) + (uint64_t)(min(row8, M - 1u - first) * K * 4u) + at));
                    }
            };
            auto request_rows = [&](uint32_t g) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) bs[j][c] = of_row(j, g * 32u + 16u * half + 4u * c);
            };
            if (begin < end) { request(begin); request_rows(begin); }
            for (uint32_t g = begin; g < end; ++g) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if ((g + 1u) * 32u > K)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (uint32_t e = 0; e < 4u; ++e) next[i][t][e] = is_own(g * 32u + 4u * column, e) ? next[i][t][e] : 0.f;
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int t = 0; t < 4; ++t) turned[i][8 * t + row8][column ^ row8] = next[i][t];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                f32x4 now[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) now[j][c] = own(bs[j][c], j, g * 32u + 16u * half + 4u * c);
                if (g + 1u < end) { request(g + 1u); request_rows(g + 1u); }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    f32x4 av[MB];
#pragma unroll
                    for (int i = 0; i < MB; ++i) av[i] = turned[i][l32][(4u * half + c) ^ (l32 & 7u)];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int i = 0; i < MB; ++i)
#pragma unroll
                            for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(av[i][q], now[j][c][q], acc[i][j], 0, 0, 0);
                }
            }
            __syncthreads();                       // (the same memory follows)
        }
        // the waves' sums, the upper half of them to the lower half, until the first has all
#pragma unroll
        for (uint32_t half_of = WAVES / 2; half_of > 0u; half_of >>= 1) {
            if (wave >= half_of && wave < 2u * half_of)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            shared.met[wave - half_of][(i * NT + j) * 4 + q][lane()] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            __syncthreads();
            if (wave < half_of)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const f32x4 t = shared.met[wave][(i * NT + j) * 4 + q][lane()];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += t[e];
                        }
            __syncthreads();
        }
    }
    // the m of element q of block i. (Of a vector that was moved to the left to stay inside, those that are this lane's own: others are M)
    static __device__ __forceinline__ uint32_t m_of(uint32_t m0, uint32_t M, int i, int q) {
        const uint32_t row = 8u * (q >> 2) + 4u * (lane() >> 5) + (q & 3);
        if constexpr (!ALONG_M) return m0 + 32u * i + row;
        const uint32_t first = m0 + 4u * row, m = min(first, M - 4u) + i;
        return m >= first ? m : M;
    }
    // to out[r][m], of columns r = 32 j + l % 32 < rows
    __device__ __forceinline__ void store(float* __restrict__ out, uint32_t m0, uint32_t M, uint32_t rows) const {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint32_t r = 32u * j + (lane() & 31u);
            if (r >= rows) continue;
            float* const to = out + (uint64_t)r * M;
#pragma unroll
            for (int p = 0; p < 4 * MB; ++p) {             // four neighbours: of one row of a block along K, of the four blocks along M
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) if constexpr (ALONG_M) v[e] = acc[e][j][p]; else v[e] = acc[p >> 2][j][4 * (p & 3) + e];
                const uint32_t m = ALONG_M ? m0 + 4u * (8u * (p >> 2) + 4u * (lane() >> 5) + (p & 3)) : m0 + 32u * (p >> 2) + 8u * (p & 3) + 4u * (lane() >> 5);
                if (m + 4u <= M) *reinterpret_cast<f32x4_anywhere*>(to + m) = v;
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t at = m_of(m0, M, ALONG_M ? e : p >> 2, ALONG_M ? p : 4 * (p & 3) + e);
                        if (at < M) to[at] = v[e];
                    }
            }
        }
    }
};

struct LinearRowsParams { uint32_t rows, H, V, slices; };
template <int NT> __device__ __forceinline__ void rows_there(uint32_t (&r_at)[NT], bool (&there)[NT], const int32_t* __restrict__ tokens, const LinearRowsParams& P) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t r = 32u * j + (threadIdx.x & 31u);
        r_at[j] = min(r, P.rows - 1u);
        there[j] = r < P.rows && is_token(tokens[r_at[j]], P.V);
    }
}

// forward: 128 tokens' scores, their peak and sum per row; the scores [rows][V] themselves for a gradient. Where tiles are few, the features in slices, whose sums go to [slice][rows][V]
template <bool ALONG, int NT>
__device__ __forceinline__ void scores_rows_body(float* __restrict__ peaks, float* __restrict__ sums, float* __restrict__ of_token, float* __restrict__ scores, const float* __restrict__ x,
                                                 const float* __restrict__ w, const int32_t* __restrict__ tokens, const LinearRowsParams& P) {
    using Product = RowsProduct<ALONG, NT>;
    __shared__ typename Product::Shared shared;
    const uint32_t lane = threadIdx.x & 63u, tiles = (P.V + Product::TILE - 1u) / Product::TILE, v0 = blockIdx.x % tiles * Product::TILE, slice = blockIdx.x / tiles;
    constexpr uint32_t GROUP = ALONG ? 8u : 32u;
    const uint32_t groups = (P.H + GROUP - 1u) / GROUP;
    uint32_t r_at[NT];
    bool there[NT];
    rows_there<NT>(r_at, there, tokens, P);
    Product product;
    product.multiply(shared, w, x, v0, P.V, P.H, r_at, there, (uint32_t)((uint64_t)groups * slice / P.slices), (uint32_t)((uint64_t)groups * (slice + 1u) / P.slices));
    if (threadIdx.x >= 64u) return;
    if (scores) product.store(scores + (uint64_t)slice * P.rows * P.V, v0, P.V, P.rows);
    if (!peaks) return;
    // a lane has 16 MB scores of a row
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t r = 32u * j + (lane & 31u);
        const int32_t token = r < P.rows ? tokens[r] : -1;
        float peak = -__builtin_inff(), sum = 0.f, mine = 0.f;
        bool has = false;
#pragma unroll
        for (int i = 0; i < Product::MB; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const uint32_t v = Product::m_of(v0, P.V, i, q);
                float s = product.acc[i][j][q];
                if (v == (uint32_t)token) { mine = s; has = true; }
                product.acc[i][j][q] = s = v < P.V ? s : -__builtin_inff();
                peak = fmaxf(peak, s);
            }
        if (has && is_token(token, P.V)) of_token[r] = mine;
        peak = over_halves_max(peak);
        const float base = peak == -__builtin_inff() ? 0.f : peak;
#pragma unroll
        for (int i = 0; i < Product::MB; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) sum += exp_of(product.acc[i][j][q] - base);
        sum = over_halves_sum(sum);
        if (lane < 32u && r < P.rows) { peaks[(uint64_t)blockIdx.x * P.rows + r] = peak; sums[(uint64_t)blockIdx.x * P.rows + r] = sum; }
    }
}

// ... added up: 1024 tokens of a row, their peak and sum, the scores for a gradient
extern "C" __global__ __launch_bounds__(256) void linear_rows_sum(float* __restrict__ peaks, float* __restrict__ sums, float* __restrict__ of_token, float* __restrict__ scores,
                                                                  const float* __restrict__ parts, const int32_t* __restrict__ tokens, LinearRowsParams P) {
    __shared__ float met[2][4];
    const uint32_t r = blockIdx.y, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, v0 = blockIdx.x * 1024u + threadIdx.x;
    const int32_t token = tokens[r];
    const uint64_t row = (uint64_t)r * P.V, each = (uint64_t)P.rows * P.V;
    float s[4] = {}, peak = -__builtin_inff();
    for (uint32_t k = 0; k < P.slices; ++k)
#pragma unroll
        for (uint32_t q = 0; q < 4u; ++q) s[q] += parts[k * each + row + min(v0 + 256u * q, P.V - 1u)];
#pragma unroll
    for (uint32_t q = 0; q < 4u; ++q) {
        const uint32_t v = v0 + 256u * q;
        if (v >= P.V) { s[q] = -__builtin_inff(); continue; }
        if (scores) scores[row + v] = s[q];
        if (of_token && v == (uint32_t)token) of_token[r] = s[q];
        peak = fmaxf(peak, s[q]);
    }
    if (!peaks) return;
    peak = wave_largest(peak);
    if (lane == 0u) met[0][wave] = peak;
    __syncthreads();
    peak = fmaxf(fmaxf(met[0][0], met[0][1]), fmaxf(met[0][2], met[0][3]));
    const float base = peak == -__builtin_inff() ? 0.f : peak;
    float sum = (exp_of(s[0] - base) + exp_of(s[1] - base)) + (exp_of(s[2] - base) + exp_of(s[3] - base));
    wave_butterfly([&](auto step) { sum += lane_xor<decltype(step)::value>(sum); });
    if (lane == 0u) met[1][wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0u) {
        peaks[(uint64_t)blockIdx.x * P.rows + r] = peak;
        sums[(uint64_t)blockIdx.x * P.rows + r]  = (met[1][0] + met[1][1]) + (met[1][2] + met[1][3]);
    }
}

// backward: ds [rows][V] from the scores, zeros for padding
extern "C" __global__ __launch_bounds__(256) void linear_rows_ds(float* __restrict__ ds, const float* __restrict__ scores, const int32_t* __restrict__ tokens, const float* __restrict__ row_peaks,
                                                                 const float* __restrict__ row_totals, const float* __restrict__ g_log_probs, const float* __restrict__ g_log_sums, LinearRowsParams P) {
    const uint32_t r = blockIdx.y;
    const int32_t token = tokens[r];
    const bool given = is_token(token, P.V);
    const float one = g_log_probs ? g_log_probs[r] : 0.f, part = ((g_log_sums ? g_log_sums[r] : 0.f) - one) / row_totals[r], peak = row_peaks[r];
    const uint64_t row = (uint64_t)r * P.V;
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t v = (blockIdx.x * 4u + k) * 256u + threadIdx.x;
        if (v < P.V) ds[row + v] = given ? part * exp_of(scores[row + v] - peak) + (v == (uint32_t)token ? one : 0.f) : 0.f;
    }
}

// dx = ds W^T: blocks of 128 features by slices of the vocabulary, a slice's sums to [slice][rows][H]; padding gets zeros whatever W holds
template <bool ALONG, int NT>
__device__ __forceinline__ void rows_dx_body(float* __restrict__ dx, const float* __restrict__ ds, const float* __restrict__ w, const int32_t* __restrict__ tokens, const LinearRowsParams& P) {
    using Product = RowsProduct<ALONG, NT>;
    __shared__ typename Product::Shared shared;
    const uint32_t tiles = (P.H + Product::TILE - 1u) / Product::TILE, h0 = blockIdx.x % tiles * Product::TILE, slice = blockIdx.x / tiles, group = ALONG ? 8u : 32u, groups = (P.V + group - 1u) / group;
    uint32_t r_at[NT];
    bool there[NT];
    rows_there<NT>(r_at, there, tokens, P);
    Product product;
    product.multiply(shared, w, ds, h0, P.H, P.V, r_at, there, (uint32_t)((uint64_t)groups * slice / P.slices), (uint32_t)((uint64_t)groups * (slice + 1u) / P.slices));
    if (threadIdx.x >= 64u) return;
#pragma unroll
    for (int j = 0; j < NT; ++j)
        if (!there[j])
#pragma unroll
            for (int i = 0; i < Product::MB; ++i) product.acc[i][j] = f32x16{};
    product.store(dx + (uint64_t)slice * P.rows * P.H, h0, P.H, P.rows);
}

// dW[m, n] = sum_r a[r, m] b[r, n], of x and ds or the other way round as dW lies: a wave has 128 n, for which it holds b, and goes through its share of m, 32 at a time; four neighbouring n
// are a lane's. Bound by the writing of dW (64 rows: as much by the products).
struct OuterParams { uint32_t rows, M, N, V, steps, tiles_n, tasks, pad; };
// (ROWS: 8, 16, 32 or 64. Everything is loaded without a branch, and whole steps are stored without one: a wait for a step's loads would be one for the stores too.)
template <int ROWS>
__device__ __forceinline__ void rows_dw_body(float* __restrict__ dw, const float* __restrict__ a, const float* __restrict__ b, const int32_t* __restrict__ tokens, const OuterParams& P) {
    constexpr int STEPS = ROWS / 2;
    const uint32_t task = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = threadIdx.x >> 5 & 1u, l32 = threadIdx.x & 31u;
    if (task >= P.tasks) return;
    // (vectors and rows behind the end are the last ones again, and write the same values once more)
    const uint32_t n = min(task % P.tiles_n * 128u + 4u * l32, P.N - 4u), first = task / P.tiles_n * P.steps * 32u, m_end = min(P.M, first + P.steps * 32u);
    f32x4 held[STEPS];
    uint32_t there = 0;                            // bit k: this lane's row of step k, 2 k + half, is not padding
#pragma unroll
    for (uint32_t k = 0; k < STEPS; ++k) {
        const uint32_t r = 2u * k + half, at = min(r, P.rows - 1u);
        const int32_t token = tokens[at];
        there |= (uint32_t)((r < P.rows) & is_token(token, P.V)) << k;
        held[k] = *reinterpret_cast<const f32x4_anywhere*>(b + (uint64_t)at * P.N + n);
    }
#pragma unroll
    for (uint32_t k = 0; k < STEPS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) held[k][e] = there >> k & 1u ? held[k][e] : 0.f;
    float next[STEPS];
    auto request = [&](uint32_t m0) {
        const float* const from = a + min(m0 + l32, P.M - 1u);
#pragma unroll
        for (uint32_t k = 0; k < STEPS; ++k) next[k] = from[(uint64_t)min(2u * k + half, P.rows - 1u) * P.M];
    };
    auto step = [&](uint32_t m0, bool whole) {
        float now[STEPS];
#pragma unroll
        for (uint32_t k = 0; k < STEPS; ++k) now[k] = there >> k & 1u ? next[k] : 0.f;
        if (m0 + 32u < m_end) request(m0 + 32u);
        f32x16 acc[4] = {};
#pragma unroll
        for (uint32_t k = 0; k < STEPS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(now[k], held[k][i], acc[i], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const uint32_t to = m0 + 8u * (q >> 2) + 4u * half + (q & 3);
            if (whole || to < P.M) *reinterpret_cast<f32x4_anywhere*>(dw + (uint64_t)to * P.N + n) = f32x4{acc[0][q], acc[1][q], acc[2][q], acc[3][q]};
        }
    };
    request(first);
    uint32_t m0 = first;
    for (; m0 + 32u <= m_end; m0 += 32u) step(m0, true);
    if (m0 < m_end) step(m0, false);
}
#define ROWS_KERNELS(NAME, ALONG_V, NT)                                                                                                                            \
    extern "C" __global__ __launch_bounds__(256, 2) void linear_scores_rows_##NAME(float* peaks, float* sums, float* of_token, float* scores, const float* x,      \
                                                                                   const float* w, const int32_t* tokens, LinearRowsParams P) {                    \
        scores_rows_body<ALONG_V, NT>(peaks, sums, of_token, scores, x, w, tokens, P);                                                                             \
    }                                                                                                                                                              \
    extern "C" __global__ __launch_bounds__(256, 2) void linear_rows_dx_##NAME(float* dx, const float* ds, const float* w, const int32_t* tokens, LinearRowsParams P) { \
        rows_dx_body<!ALONG_V, NT>(dx, ds, w, tokens, P);                                                                                                          \
    }
ROWS_KERNELS(v_32, true, 1)
ROWS_KERNELS(v_64, true, 2)
ROWS_KERNELS(h_32, false, 1)
ROWS_KERNELS(h_64, false, 2)
#define ROWS_DW(ROWS) extern "C" __global__ __launch_bounds__(256) void linear_rows_dw_##ROWS(float* dw, const float* a, const float* b, const int32_t* tokens, OuterParams P) { \
        rows_dw_body<ROWS>(dw, a, b, tokens, P);                                                                                                                   \
    }
ROWS_DW(8)
ROWS_DW(16)
ROWS_DW(32)
ROWS_DW(64)

// ---- backward: a piece's q as an operand [rows][tokens], which dx is contracted over the tokens of, and dW, turned, over the rows
template <int T, int STAGES, bool SHARED>
__device__ __forceinline__ void linear_q_body(u32x4* __restrict__ by_row, float* __restrict__ partial, uint32_t* __restrict__ arrivals, const u32x4* __restrict__ w,
                                              const u32x4* __restrict__ x, const int32_t* __restrict__ tokens, const int32_t* __restrict__ scales, const float* __restrict__ row_peaks,
                                              const float* __restrict__ row_totals, const float* __restrict__ factors, const ScoresParams& P) {
    constexpr uint32_t SIDE = HalfTileOf<T>::SIDE;
    __shared__ HalfShared<T, STAGES> shared;
    uint32_t m, n, tile, slice, begin, end;
    half_work(blockIdx.x, HalfShares{P.whole, P.slices}, P.pairs, tile, slice, begin, end);
    half_tile(tile, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    half_product<T, STAGES, TURNED_NONE, true>(acc, shared, operand_of(w, P.blocks_w, P.steps_w), operand_of(x, P.blocks_x, P.steps_x), P.tile0 + m, n, begin, end - begin, scales + PLAIN);
    const bool plain = scales[PLAIN] != 0;
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, HalfShares{P.whole, P.slices})) return;
    const int down = -(scales[PACK_WEIGHTS] + scales[PACK_ROWS]);
    const uint32_t lane = threadIdx.x & 63u, wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 1u, v0 = (P.tile0 + m) * SIDE;
    // of this lane's columns
    bool given[T];
    uint32_t token[T];
    float peak[T], part[T], one[T];
#pragma unroll
    for (int j = 0; j < T; ++j) {
        const uint32_t r = n * SIDE + (wn * T + j) * 32u + (lane & 31u), at = min(r, P.rows - 1u);
        given[j] = r < P.rows && is_token(tokens[at], P.V);
        token[j] = given[j] ? (uint32_t)tokens[at] : 0xFFFFFFFFu;
        // (plain: ds itself, the rows' m has no part in the products)
        const float up = plain ? factors[3u * at] : power_of_two(Q_SCALE);
        peak[j] = row_peaks[at]; one[j] = factors[3u * at + 2u] * up; part[j] = factors[3u * at + 1u] * up / row_totals[at];
    }
    const HalfTarget to{by_row, P.blocks_x, P.Vp / 16u, n * 2u * T, m * 4u * T}, none{nullptr, 0u, 0u, 0u, 0u};
    auto q_of = [&](int i, int j, int k, uint32_t row, uint32_t) {
        const uint32_t v = v0 + row;
        const float s = scaled(half_sum(acc, i, j, k), down);
        const float q = part[j] * exp_of(s - peak[j]) + (v == token[j] ? one[j] : 0.f);
        return given[j] && v < P.V ? q : 0.f;
    };
    if (plain) half_store<T, true>(shared.turned, to, none, q_of); else half_store<T>(shared.turned, to, none, q_of);
}
#define LINEAR_Q(SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                                     \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void linear_q##SUFFIX(u32x4* by_row, float* partial, uint32_t* arrivals, const u32x4* w,      \
                                                                               const u32x4* x, const int32_t* tokens, const int32_t* scales, const float* row_peaks,    \
                                                                               const float* row_totals, const float* factors, ScoresParams P) {                         \
        linear_q_body<T, STAGES, SHARED>(by_row, partial, arrivals, w, x, tokens, scales, row_peaks, row_totals, factors, P);                                 \
    }
LINEAR_KERNELS(LINEAR_Q)

// ---- a product of two operands, one of them turned, to fp32 [M, N], rows by a factor each (every third word), added to what is there or in its place; not SHARED: a slice of the contraction to an array of its own
struct ProductParams {
    uint32_t M, N, tiles_m, tiles_n, pairs, blocks_a, blocks_b, steps_a, steps_b, first_a, first_b, add;
    int32_t scale_a, scale_b;                            // the kind of operand whose scale it is, or -1: q
    uint32_t whole, slices;                              // (HalfShares)
    uint64_t ld, slice;                                  // elements from a row of the result to the next, from a slice's result to the next one's
};
template <int T, int STAGES, bool SHARED, HalfTurned TURNED>
__device__ __forceinline__ void linear_product_body(float* __restrict__ out, float* __restrict__ partial, uint32_t* __restrict__ arrivals, const u32x4* __restrict__ a, const u32x4* __restrict__ b,
                                                    const int32_t* __restrict__ scales_a, const int32_t* __restrict__ scales_b, const float* __restrict__ factors, const ProductParams& P) {
    __shared__ HalfShared<T, STAGES> shared;
    uint32_t m, n, tile, slice, begin, end;
    half_work(blockIdx.x, HalfShares{P.whole, P.slices}, P.pairs, tile, slice, begin, end);
    half_tile(tile, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    const int32_t* const kind = (scales_a ? scales_a : scales_b) + PLAIN;
    half_product<T, STAGES, TURNED, true>(acc, shared, operand_of(a, P.blocks_a, P.steps_a, P.first_a), operand_of(b, P.blocks_b, P.steps_b, P.first_b), m, n, begin, end - begin, kind);
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, HalfShares{P.whole, P.slices})) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t lane_row = (m * 2u + (wave >> 1)) * 32u * T + 4u * (lane >> 5), lane_column = (n * 2u + (wave & 1u)) * 32u * T + (lane & 31u);
    const bool plain = *kind != 0;
    const int q_scale = plain ? 0 : Q_SCALE, down = -(P.scale_a < 0 ? q_scale : scales_a[P.scale_a]) - (P.scale_b < 0 ? q_scale : scales_b[P.scale_b]);
    float* const to = out + (SHARED ? 0u : P.slice * slice);
#pragma unroll
    for (int i = 0; i < T; ++i) {
        // (what is there is asked for at once, in front of the stores)
        float before[T][16] = {};
        if (P.add)
#pragma unroll
            for (int q = 0; q < 16; ++q)
#pragma unroll
                for (int j = 0; j < T; ++j) {
                    const uint32_t row = lane_row + 32u * i + 8u * (q >> 2) + (q & 3), column = lane_column + 32u * j;
                    if (row < P.M && column < P.N) before[j][q] = to[P.ld * row + column];
                }
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const uint32_t row = lane_row + 32u * i + 8u * (q >> 2) + (q & 3);
            if (row >= P.M) continue;
            const float f = factors ? factors[3u * row] : 1.f;
#pragma unroll
            for (int j = 0; j < T; ++j) {
                const uint32_t column = lane_column + 32u * j;
                if (column >= P.N) continue;
                float s = scaled(half_sum(acc, i, j, q), down);
                if (factors) s = f == 0.f ? 0.f : plain ? s : s * f;
                to[P.ld * row + column] = s + before[j][q];
            }
        }
    }
}
#define LINEAR_PRODUCT_OF(NAME, TURNED, T, STAGES, BLOCKS, SHARED)                                                                                                      \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void linear_product_##NAME(float* out, float* partial, uint32_t* arrivals, const u32x4* a, const u32x4* b,     \
                                                                                    const int32_t* scales_a, const int32_t* scales_b, const float* factors, ProductParams P) { \
        linear_product_body<T, STAGES, SHARED, TURNED>(out, partial, arrivals, a, b, scales_a, scales_b, factors, P);                                                     \
    }
#define LINEAR_PRODUCT(SUFFIX, T, STAGES, BLOCKS, SHARED) \
    LINEAR_PRODUCT_OF(a##SUFFIX, TURNED_A, T, STAGES, BLOCKS, SHARED) LINEAR_PRODUCT_OF(b##SUFFIX, TURNED_B, T, STAGES, BLOCKS, SHARED)
LINEAR_KERNELS(LINEAR_PRODUCT)

// ---- the slices of a contraction added up; with few elements by four waves, a quarter of the slices each
struct SumParams { uint32_t parts, pad; uint64_t n; };
__device__ __forceinline__ float sum_of(const float* __restrict__ parts, uint64_t at, uint64_t n, uint32_t begin, uint32_t end) {
    float s = 0.f;
    for (uint32_t k0 = begin; k0 < end; k0 += 8u) {
        float v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) v[k] = k0 + k < end ? parts[(k0 + k) * n + at] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[k];
    }
    return s;
}
extern "C" __global__ __launch_bounds__(256) void linear_sum(float* __restrict__ out, const float* __restrict__ parts, SumParams P) {
    const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (at < P.n) out[at] = sum_of(parts, at, P.n, 0u, P.parts);
}
extern "C" __global__ __launch_bounds__(256) void linear_sum_few(float* __restrict__ out, const float* __restrict__ parts, SumParams P) {
    __shared__ float met[4][64];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint64_t at = (uint64_t)blockIdx.x * 64u + lane;
    met[wave][lane] = at < P.n ? sum_of(parts, at, P.n, P.parts * wave / 4u, P.parts * (wave + 1u) / 4u) : 0.f;
    __syncthreads();
    if (wave == 0u && at < P.n) out[at] = (met[0][lane] + met[1][lane]) + (met[2][lane] + met[3][lane]);
}
