// Log probabilities of given tokens under softmax(x W), without keeping the scores x W, and their gradient.
//
//   s[r, v] = sum_h x[r, h] W[h, v];  peak = max_v s,  total = sum_v exp(s - peak);  log_sum = peak + log(total),  log_prob = s[r, token] - log_sum
//   ds = g_lp [v = token] + (g_ls - g_lp) p,  p = exp(s - peak) / total;  dx = ds W^T,  dW = x^T ds
// A row whose token lies outside the vocabulary is padding: zeros, x is not looked at there, no gradient.
//
// Products are those of half_product.h: x and W are taken apart first (the largest magnitudes, for their scales, then the parts), then
//   * forward: a product whose rows are the vocabulary and whose columns are the rows of x, so that a lane has 32 scores of one row; a tile of 128 tokens leaves each row's peak and
//     sum, a last launch joins the tiles. 4096 x 1024 x 32000: the product as fast as one that keeps its scores, and nothing of 0.5 GB is written.
//   * backward, in pieces of the vocabulary: the same product again, whose lanes turn scores into q = ds / m, |q| <= 2, with m = max(|g_lp|, |g_ls - g_lp|) of the row, and lay q out as an
//     operand of both products that follow, contracted over the vocabulary (the lanes have it like that) and over the rows (turned in shared memory). q takes 8 bytes a score of one
//     piece; the rows' m is a factor of dx's rows, and of the x that dW is made of.
// Up to 64 rows take the fp32 matrix instructions (linear_scores_rows), which read W once, as it is: bound by memory.
#include "half_product.h"

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int Q_SCALE = 13;                              // |q| <= 2

__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * LOG2E); }
__device__ __forceinline__ bool is_token(int32_t t, uint32_t V) { return (uint32_t)t < V; }
typedef f32x4 f32x4_anywhere __attribute__((aligned(4)));

// A finite number's magnitude (others have no part in a scale)
__device__ __forceinline__ float magnitude(float v) { const float a = __builtin_fabsf(v); return a < __builtin_inff() ? a : 0.f; }
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
            one = fmaxf(one, row); two = fmaxf(two, magnitude(row * m));
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

// ---- operands taken apart (half_product.h). What element (i, k) of an operand is: W or x as they lie, x only of rows that are given, or with the rows' factors.
enum PackKind : uint32_t { PACK_WEIGHTS = 0, PACK_ROWS = 1, PACK_SCALED = 2 };
struct PackJob { uint32_t blocks, I, K, stride, kind, steps; uint64_t si, sk; };      // blocks of 256 threads; steps of 16 k; element strides of i and k; `stride`: steps that a wave takes
struct PackParams { uint32_t weight_blocks, row_blocks, V, pad; PackJob jobs[4]; };
struct PackOuts { u32x4* parts[4]; };
extern "C" __global__ __launch_bounds__(256) void linear_pack(PackOuts outs, int32_t* __restrict__ scales, const float* __restrict__ x, const float* __restrict__ w,
                                                              const int32_t* __restrict__ tokens, const float* __restrict__ largest, const float* __restrict__ factors,
                                                              const int32_t* __restrict__ known, PackParams P) {
    __shared__ float part[4];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t block = blockIdx.x, job = 0u;
    while (job < 3u && block >= P.jobs[job].blocks) block -= P.jobs[job++].blocks;
    const PackJob J = P.jobs[job];
    // the operand's scale, of its blocks' largest magnitudes, or the weights' that is known
    const bool weights = J.kind == PACK_WEIGHTS;
    float most = 0.f;
    for (uint32_t k = threadIdx.x; k < (weights ? P.weight_blocks : P.row_blocks); k += 256u)
        most = fmaxf(most, weights ? largest[k] : largest[P.weight_blocks + 2u * k + (J.kind == PACK_SCALED ? 1u : 0u)]);
    most = wave_largest(most);
    if (lane == 0u) part[wave] = most;
    __syncthreads();
    const int e = weights && known ? known[PACK_WEIGHTS] : half_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    if (block == 0u && threadIdx.x == 0u) scales[J.kind] = e;
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
    u32x4* const to = outs.parts[job] + (uint64_t)rb * J.steps * 128u + lane;
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
                    v[t][q] = m == 0.f ? 0.f : v[t][q] * m;           // (a row without a cotangent has none, whatever its x is)
                }
            u32x4 hi, lo;
#pragma unroll
            for (int q = 0; q < 4; ++q) { uint32_t a, b; half_parts(v[t][2 * q] * up, v[t][2 * q + 1] * up, a, b); hi[q] = a; lo[q] = b; }
            to[(s0 + t) * 128u] = hi; to[(s0 + t) * 128u + 64u] = lo;
        }
    }
}

// ---- forward: a tile's peak and sum per row of x, [tile of tokens][rows]
struct ScoresParams { uint32_t rows, V, pairs, steps_w, steps_x, tiles_m, tiles_n, blocks_w, blocks_x, tile0, Vp; HalfShares shares; };

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
    half_work(blockIdx.x, P.shares, P.pairs, tile, slice, begin, end);
    half_tile(tile, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    half_product<T, STAGES>(acc, shared, operand_of(w, P.blocks_w, P.steps_w), operand_of(x, P.blocks_x, P.steps_x), m, n, begin, end - begin);
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, P.shares)) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, wm = wave >> 1, wn = wave & 1u;
    const float down_w = power_of_two(-scales[PACK_WEIGHTS]), down_x = power_of_two(-scales[PACK_ROWS]);
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
                float s = half_sum(acc, i, j, q) * down_w * down_x;
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

// ---- up to 32 NT rows: a block has 128 tokens, its waves parts of the contraction; W is read once. v_mfma_f32_32x32x2_f32: lane l has row l % 32 of a block of 32 and k = l / 32.
// Which token a lane's row is, and in which order k comes, follows from how W lies: four neighbouring tokens to a lane's vector (ALONG_V), or 16 neighbouring h.
struct RowsParams { uint32_t rows, H, V, pad; };
template <bool ALONG_V, int NT>
__device__ __forceinline__ void scores_rows_body(float* __restrict__ peaks, float* __restrict__ sums, float* __restrict__ of_token, const float* __restrict__ x, const float* __restrict__ w,
                                                 const int32_t* __restrict__ tokens, const RowsParams& P) {
    constexpr int WAVES = 8;
    __shared__ f32x4 met[WAVES / 2][NT * 16][64];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l32 = lane & 31u, v0 = blockIdx.x * 128u;
    // groups of 8 (ALONG_V) or 32 h, to the waves in turn by contiguous ranges
    constexpr uint32_t GROUP = ALONG_V ? 8u : 32u;
    const uint32_t groups = (P.H + GROUP - 1u) / GROUP, begin = groups * wave / WAVES, end = groups * (wave + 1u) / WAVES;
    f32x16 acc[4][NT] = {};
    // (lanes behind the last token or row read the last ones again)
    const uint32_t v_at = ALONG_V ? min(v0 + 4u * l32, P.V - 4u) : 0u;
    uint32_t r_at[NT];
    bool r_there[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t r = 32u * j + l32;
        r_at[j] = min(r, P.rows - 1u);
        r_there[j] = r < P.rows && is_token(tokens[r_at[j]], P.V);
    }
    auto four = [&](const float* row, uint32_t h, bool there) {
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
        if (!there) return t;
        if (h + 4u <= P.H) return (f32x4)*reinterpret_cast<const f32x4_anywhere*>(row + h);
#pragma unroll
        for (int q = 0; q < 4; ++q) if (h + q < P.H) t[q] = row[h + q];
        return t;
    };
    if constexpr (ALONG_V) {
        // (DEPTH - 1 groups are on their way while one is multiplied)
        constexpr uint32_t DEPTH = 4u;
        f32x4 ws[DEPTH][4], xs[DEPTH][NT];
        auto request = [&](f32x4 (&wv)[4], f32x4 (&xv)[NT], uint32_t g) {
            const uint32_t h0 = g * 8u + 4u * half;
#pragma unroll
            for (int q = 0; q < 4; ++q) wv[q] = *reinterpret_cast<const f32x4_anywhere*>(w + (uint64_t)min(h0 + q, P.H - 1u) * P.V + v_at);
#pragma unroll
            for (int j = 0; j < NT; ++j) xv[j] = four(x + (uint64_t)r_at[j] * P.H, h0, r_there[j]);
        };
        auto multiply = [&](const f32x4 (&wv)[4], const f32x4 (&xv)[NT]) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(wv[q][i], xv[j][q], acc[i][j], 0, 0, 0);
        };
#pragma unroll
        for (uint32_t k = 0; k < DEPTH - 1u; ++k) if (begin + k < end) request(ws[k], xs[k], begin + k);
        for (uint32_t g = begin; g < end; g += DEPTH)
#pragma unroll
            for (uint32_t k = 0; k < DEPTH; ++k) {
                if (g + k + DEPTH - 1u < end) request(ws[(k + DEPTH - 1u) % DEPTH], xs[(k + DEPTH - 1u) % DEPTH], g + k + DEPTH - 1u);
                if (g + k < end) multiply(ws[k], xs[k]);
            }
    } else {
        for (uint32_t g = begin; g < end; ++g) {
            const uint32_t h0 = g * 32u + 16u * half;
            f32x4 wv[4][4], xv[NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) wv[i][q] = four(w + (uint64_t)min(v0 + 32u * i + l32, P.V - 1u) * P.H, h0 + 4u * q, true);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) xv[j][q] = four(x + (uint64_t)r_at[j] * P.H, h0 + 4u * q, r_there[j]);
#pragma unroll
            for (int q = 0; q < 16; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(wv[i][q >> 2][q & 3], xv[j][q >> 2][q & 3], acc[i][j], 0, 0, 0);
        }
    }
    // the waves' sums, the upper half of them to the lower half, three times
#pragma unroll
    for (uint32_t half_of = WAVES / 2; half_of > 0u; half_of >>= 1) {
        if (wave >= half_of && wave < 2u * half_of)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) met[wave - half_of][(i * NT + j) * 4 + q][lane] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __syncthreads();
        if (wave < half_of)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 t = met[wave][(i * NT + j) * 4 + q][lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += t[e];
                    }
        __syncthreads();
    }
    if (wave != 0u) return;
    // a lane has 64 scores of a row
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t r = 32u * j + l32;
        const int32_t token = r < P.rows ? tokens[r] : -1;
        float peak = -__builtin_inff(), sum = 0.f;
        const auto token_of = [&](int i, int q) -> uint32_t {
            const uint32_t row = 8u * (q >> 2) + 4u * half + (q & 3);
            if constexpr (!ALONG_V) return v0 + 32u * i + row;
            // (of a vector that was moved to the left to stay inside, the tokens that are this block's and lane's own)
            const uint32_t first = v0 + 4u * row, v = min(first, P.V - 4u) + i;
            return v >= first ? v : P.V;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const uint32_t v = token_of(i, q);
                if (v == (uint32_t)token && v < P.V) of_token[r] = acc[i][j][q];
                acc[i][j][q] = v < P.V ? acc[i][j][q] : -__builtin_inff();
                peak = fmaxf(peak, acc[i][j][q]);
            }
        peak = over_halves_max(peak);
        const float base = peak == -__builtin_inff() ? 0.f : peak;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) sum += exp_of(acc[i][j][q] - base);
        sum = over_halves_sum(sum);
        if (lane < 32u && r < P.rows) { peaks[(uint64_t)blockIdx.x * P.rows + r] = peak; sums[(uint64_t)blockIdx.x * P.rows + r] = sum; }
    }
}
#define SCORES_ROWS(NAME, ALONG_V, NT)                                                                                                                             \
    extern "C" __global__ __launch_bounds__(512) void linear_scores_rows_##NAME(float* peaks, float* sums, float* of_token, const float* x, const float* w,        \
                                                                                const int32_t* tokens, RowsParams P) {                                             \
        scores_rows_body<ALONG_V, NT>(peaks, sums, of_token, x, w, tokens, P);                                                                                     \
    }
SCORES_ROWS(v_32, true, 1)
SCORES_ROWS(v_64, true, 2)
SCORES_ROWS(h_32, false, 1)
SCORES_ROWS(h_64, false, 2)

// ---- backward: a piece's q, as operands contracted over the vocabulary [rows][tokens] and over the rows [tokens][rows]
template <int T, int STAGES, bool SHARED>
__device__ __forceinline__ void linear_q_body(u32x4* __restrict__ by_row, u32x4* __restrict__ by_token, float* __restrict__ partial, uint32_t* __restrict__ arrivals, const u32x4* __restrict__ w,
                                              const u32x4* __restrict__ x, const int32_t* __restrict__ tokens, const int32_t* __restrict__ scales, const float* __restrict__ row_peaks,
                                              const float* __restrict__ row_totals, const float* __restrict__ factors, const ScoresParams& P) {
    constexpr uint32_t SIDE = HalfTileOf<T>::SIDE;
    __shared__ HalfShared<T, STAGES> shared;
    uint32_t m, n, tile, slice, begin, end;
    half_work(blockIdx.x, P.shares, P.pairs, tile, slice, begin, end);
    half_tile(tile, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    half_product<T, STAGES>(acc, shared, operand_of(w, P.blocks_w, P.steps_w), operand_of(x, P.blocks_x, P.steps_x), P.tile0 + m, n, begin, end - begin);
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, P.shares)) return;
    const float down_w = power_of_two(-scales[PACK_WEIGHTS]), down_x = power_of_two(-scales[PACK_ROWS]), up = power_of_two(Q_SCALE);
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
        peak[j] = row_peaks[at]; one[j] = factors[3u * at + 2u] * up; part[j] = factors[3u * at + 1u] * up / row_totals[at];
    }
    half_store<T>(shared.turned, HalfTarget{by_row, P.blocks_x, P.Vp / 16u, n * 2u * T, m * 4u * T}, HalfTarget{by_token, P.Vp / 32u, P.blocks_x * 2u, m * 2u * T, n * 4u * T},
                  [&](int i, int j, int k, uint32_t row, uint32_t) {
        const uint32_t v = v0 + row;
        const float s = half_sum(acc, i, j, k) * down_w * down_x;
        const float q = part[j] * exp_of(s - peak[j]) + (v == token[j] ? one[j] : 0.f);
        return given[j] && v < P.V ? q : 0.f;
    });
}
#define LINEAR_Q(SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                                     \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void linear_q##SUFFIX(u32x4* by_row, u32x4* by_token, float* partial, uint32_t* arrivals, const u32x4* w,      \
                                                                               const u32x4* x, const int32_t* tokens, const int32_t* scales, const float* row_peaks,    \
                                                                               const float* row_totals, const float* factors, ScoresParams P) {                         \
        linear_q_body<T, STAGES, SHARED>(by_row, by_token, partial, arrivals, w, x, tokens, scales, row_peaks, row_totals, factors, P);                                 \
    }
LINEAR_KERNELS(LINEAR_Q)

// ---- a product of two operands to fp32 [M, N], rows by a factor each (every third word), added to what is there or in its place; not SHARED: a slice of the contraction to an array of its own
struct ProductParams {
    uint32_t M, N, tiles_m, tiles_n, pairs, blocks_a, blocks_b, steps_a, steps_b, first_a, first_b, add;
    int32_t scale_a, scale_b;                            // the kind of operand whose scale it is, or -1: q
    HalfShares shares;
    uint64_t ld, slice;                                  // elements from a row of the result to the next, from a slice's result to the next one's
};
template <int T, int STAGES, bool SHARED>
__device__ __forceinline__ void linear_product_body(float* __restrict__ out, float* __restrict__ partial, uint32_t* __restrict__ arrivals, const u32x4* __restrict__ a, const u32x4* __restrict__ b,
                                                    const int32_t* __restrict__ scales, const float* __restrict__ factors, const ProductParams& P) {
    __shared__ HalfShared<T, STAGES> shared;
    uint32_t m, n, tile, slice, begin, end;
    half_work(blockIdx.x, P.shares, P.pairs, tile, slice, begin, end);
    half_tile(tile, P.tiles_m, P.tiles_n, m, n);
    HalfSums<T> acc = {};
    half_product<T, STAGES>(acc, shared, operand_of(a, P.blocks_a, P.steps_a, P.first_a), operand_of(b, P.blocks_b, P.steps_b, P.first_b), m, n, begin, end - begin);
    if constexpr (SHARED) if (!half_join<T, STAGES>(acc, shared, partial, arrivals, tile, slice, P.shares)) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t lane_row = (m * 2u + (wave >> 1)) * 32u * T + 4u * (lane >> 5), lane_column = (n * 2u + (wave & 1u)) * 32u * T + (lane & 31u);
    const float down = power_of_two(-(P.scale_a < 0 ? Q_SCALE : scales[P.scale_a])), down_b = power_of_two(-(P.scale_b < 0 ? Q_SCALE : scales[P.scale_b]));
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
                float s = half_sum(acc, i, j, q) * down * down_b;
                if (factors) s = f == 0.f ? 0.f : s * f;
                to[P.ld * row + column] = s + before[j][q];
            }
        }
    }
}
#define LINEAR_PRODUCT(SUFFIX, T, STAGES, BLOCKS, SHARED)                                                                                                               \
    extern "C" __global__ __launch_bounds__(256, BLOCKS) void linear_product##SUFFIX(float* out, float* partial, uint32_t* arrivals, const u32x4* a, const u32x4* b,    \
                                                                                     const int32_t* scales, const float* factors, ProductParams P) {                    \
        linear_product_body<T, STAGES, SHARED>(out, partial, arrivals, a, b, scales, factors, P);                                                                       \
    }
LINEAR_KERNELS(LINEAR_PRODUCT)

struct SumParams { uint32_t parts, pad; uint64_t n; };
extern "C" __global__ __launch_bounds__(256) void linear_sum(float* __restrict__ out, const float* __restrict__ parts, SumParams P) {
    const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (at >= P.n) return;
    float s = 0.f;
    for (uint32_t k0 = 0; k0 < P.parts; k0 += 8u) {
        float v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) v[k] = k0 + k < P.parts ? parts[(k0 + k) * P.n + at] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[k];
    }
    out[at] = s;
}
