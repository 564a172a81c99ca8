// Log probabilities of given tokens with the entropy of their rows' distributions and the most likely alternatives, and the
// gradient of all three.
//
// With m = max x, s = sum exp(x - m), w = sum exp(x - m) (x - m) over a row of V scores:
//   lse = m + log s,  log p = x - lse,  H = -sum p log p = log s - w / s
//   dx[v] = -p[v] (sum of the cotangents of log probabilities) - gH p[v] (log p[v] + H) + the cotangents of v's own log probabilities
//
// A token outside [0, V) marks its row as padding: results are 0 (alternatives: token -1), the row's scores are not read. Scores of
// -inf are masked: p = 0, and p log p counts as 0. Where every score of a row is -inf there is no distribution: log p = -inf, H = 0,
// gradient 0. NaN and +inf make their row NaN by themselves (+inf - +inf).
//
// A row is read once. A wave takes 1024 scores at a time, 16 per lane in vectors of 16 bytes (of memory: a row that starts inside a vector has its first
// scores in that one, the others' are masked). Every lane keeps a maximum and the two sums relative to it, changed when the maximum does,
// once per 16 scores; lanes, waves and slices of a row are joined the same way.
//
// The alternatives: the k-th largest of the 64 lanes' maxima is no larger than the k-th largest score, so of the first 1024 scores only what is larger, and as
// many equal ones as are missing, can be among the k largest: a few more than k scores, whose places are then counted. From then on only
// scores above the k-th so far are looked at: one comparison per lane and 16 scores, and rarely more. They gather in a list of 64, which
// is cut to k again when it is full. Where more stand out at once than the list holds, the largest are taken one by one.
#include "common.h"

struct LogProbsParams {
    uint32_t first;
    uint32_t rows, V, top;
    uint32_t slices, slice;                      // blocks per row, vectors of a row to a wave
    uint32_t log2_lanes;                         // lanes per row, where a wave has several rows
};

constexpr uint32_t NOWHERE = 0x80000000u;
constexpr uint32_t LIST = 64;
constexpr int NV = 4;                            // vectors per lane at a time
constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.4426950408889634f;

// Sums of a row's exponentials relative to a maximum (LOWEST where there is no score but -inf).
struct Sums {
    float m, s, w;
    __device__ __forceinline__ void start() { m = LOWEST; s = 0.f; w = 0.f; }
    // relative to `to`, which is no smaller. (The difference is bounded: infinity times a sum of 0 would be NaN.)
    __device__ __forceinline__ void move(float to) {
        const float d = fmaxf(m - to, -1e30f), f = __builtin_amdgcn_exp2f(d * LOG2E);
        w = f * __builtin_fmaf(d, s, w); s *= f; m = to;
    }
    // exp(x - m) in base 2, its exponent rounded twice: off by some 2 |x - m| 2^-24 of itself, which counts as little as the term does. (The maximum keeps 0 times
    // -inf out of w; a NaN stays in the exponential.)
    __device__ __forceinline__ void add(float x) {
        const float d = x - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
        s += e; w = __builtin_fmaf(e, fmaxf(d, -1e30f), w);
    }
    __device__ __forceinline__ void join(Sums other) { const float to = fmaxf(m, other.m); move(to); other.move(to); s += other.s; w += other.w; }
    __device__ __forceinline__ void join_lanes(uint32_t lanes) {
        const float to = lanes_allreduce(m, lanes, [](float a, float b) { return fmaxf(a, b); });
        move(to);
        s = lanes_allreduce(s, lanes, [](float a, float b) { return a + b; });
        w = lanes_allreduce(w, lanes, [](float a, float b) { return a + b; });
    }
    __device__ __forceinline__ bool nothing() const { return s == 0.f; }
    __device__ __forceinline__ float log_sum() const { return nothing() ? -INFINITY : m + logf(s); }
    __device__ __forceinline__ float entropy() const { return nothing() ? 0.f : logf(s) - w / s; }
    __device__ __forceinline__ float log_prob(float x) const { return nothing() ? -INFINITY : (x - m) - logf(s); }
};

// Larger for larger scores, NaN above all; -0 and 0 are equal. Neither 0 nor all ones.
__device__ __forceinline__ uint32_t score_key(float x) {
    const uint32_t b = f2u(x + 0.f);
    return x != x ? 0xFFFFFFFEu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t key) { return key == 0xFFFFFFFEu ? u2f(0x7FC00000u) : u2f((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key); }
// Among equal scores larger for the smaller token.
__device__ __forceinline__ uint64_t place_key(float x, uint32_t token) { return (uint64_t)score_key(x) << 32 | (0xFFFFFFFFu - token); }
__device__ __forceinline__ uint32_t place_token(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u)); }
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// put(place, key) for the `top` largest of `count` keys in shared memory, each lane having keys lane, lane + 64 ..: as many are larger as its place says.
template <class Put>
__device__ __forceinline__ void rank(const uint64_t* keys, uint32_t count, uint32_t top, Put put) {
    for (uint32_t at = 0; at < count; at += 64u) {
        const uint32_t mine = at + __lane_id();
        const uint64_t key = mine < count ? keys[mine] : 0ull;
        uint32_t place = 0;
        for (uint32_t i = 0; i < count; ++i) place += keys[i] > key;
        if (mine < count && place < top) put(place, key);
    }
}

// The k-th largest of the lanes' values (k <= 64): bit by bit, by how many lanes are no smaller.
__device__ __forceinline__ float kth_largest(float lane_value, uint32_t k) {
    const uint32_t key = score_key(lane_value);
    uint32_t found = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t with = found | 1u << bit;
        if ((uint32_t)__popcll(__builtin_amdgcn_ballot_w64(key >= with)) >= k) found = with;
    }
    return key_score(found);
}

// The list of a wave's candidates in shared memory.
struct Candidates {
    uint64_t* keys;                              // LIST of them
    uint32_t count, top;
    float bar;                                   // the k-th largest so far: later scores count where they are larger

    // cuts the list to the `top` largest, in order
    __device__ __forceinline__ void cut() {
        wave_fence();
        const uint32_t lane = __lane_id();
        const uint64_t key = lane < count ? keys[lane] : 0ull;
        uint32_t place = 0;
        for (uint32_t i = 0; i < count; ++i) place += keys[i] > key;
        wave_fence();
        if (lane < count && place < top) keys[place] = key;
        wave_fence();
        count = min(count, top);
        bar = key_score((uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(keys[top - 1u] >> 32)));
    }
    // Takes from 64 x 4 NV scores, whose places rise with vector, lane and element, what may be among the largest; `token(i, j)` is a score's token and
    // valid(i, j) whether it is one. `best`: the lane's largest.
    template <class Token, class Valid>
    __device__ __forceinline__ void take(const float (&v)[NV][4], float best, Token token, Valid valid) {
        const bool fresh = count == 0u;
        if (!fresh && __builtin_amdgcn_ballot_w64(!(best <= bar)) == 0ull) return;
        // (a lane's largest is a number; NaNs pass the comparisons below)
        float above = fresh ? kth_largest(best, top) : bar;
        for (;;) {
            uint32_t n = count;
            bool fits = true;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = !(v[i][j] <= above);
                    const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
                    if (mask != 0ull) {
                        const uint32_t many = (uint32_t)__popcll(mask);
                        fits = fits && n + many <= LIST;
                        if (fits && in) keys[n + lanes_below(mask)] = place_key(v[i][j], token(i, j));
                        n += many;
                    }
                }
            if (fits) { count = n; break; }
            if (fresh || count == top) {                                  // more than the list holds: one by one
                one_by_one(v, token, valid);
                return;
            }
            cut();
            above = bar;
        }
        if (fresh && count < top) {                                       // as many equal ones as are missing, the first ones
            uint32_t need = top - count;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (need == 0u) break;
                uint32_t before = 0, all = 0;
                bool is[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    is[j] = v[i][j] == above && valid(i, j);
                    const uint64_t mask = __builtin_amdgcn_ballot_w64(is[j]);
                    before += lanes_below(mask); all += (uint32_t)__popcll(mask);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (is[j] && before < need) keys[count + before] = place_key(v[i][j], token(i, j));
                    before += is[j];
                }
                const uint32_t taken = min(all, need);
                count += taken; need -= taken;
            }
        }
        if (fresh) {
            if (count >= top) cut();
            else { wave_fence(); bar = -INFINITY; }                       // (fewer scores than alternatives: the slice is short)
        } else if (count > LIST - 16u) cut();
    }
    // The `top` largest of the list, which is at its length after a cut or empty, and these scores.
    template <class Token, class Valid>
    __device__ __forceinline__ void one_by_one(const float (&v)[NV][4], Token token, Valid valid) {
        const uint32_t lane = __lane_id();
        wave_fence();
        const uint64_t old = lane < count ? keys[lane] : 0ull;
        uint64_t below = ~0ull;
        uint32_t n = 0;
        for (; n < top; ++n) {
            uint64_t best = old < below ? old : 0ull;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t key = valid(i, j) ? place_key(v[i][j], token(i, j)) : 0ull;
                    if (key < below && key > best) best = key;
                }
            best = lanes_allreduce(best, 64u, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
            if (best == 0ull) break;
            below = best;
            if (lane == 0u) keys[n] = best;
        }
        wave_fence();
        count = n;
        bar = n == top ? key_score((uint32_t)(below >> 32)) : -INFINITY;
    }
};

struct Results { float *log_prob, *entropy, *log_sum, *top_log_prob; int32_t* top_token; };

__device__ __forceinline__ void write_padding(const Results& to, uint64_t row, uint32_t lane, uint32_t lanes, uint32_t top) {
    if (lane == 0u) {
        if (to.log_prob) to.log_prob[row] = 0.f;
        if (to.entropy) to.entropy[row] = 0.f;
        if (to.log_sum) to.log_sum[row] = 0.f;
    }
    for (uint32_t k = lane; k < top; k += lanes) {
        if (to.top_log_prob) to.top_log_prob[row * top + k] = 0.f;
        if (to.top_token) to.top_token[row * top + k] = -1;
    }
}
__device__ __forceinline__ void write_sums(const Results& to, uint64_t row, const Sums& sums, float score) {
    if (to.log_prob) to.log_prob[row] = sums.log_prob(score);
    if (to.entropy) to.entropy[row] = sums.entropy();
    if (to.log_sum) to.log_sum[row] = sums.log_sum();
}
__device__ __forceinline__ void write_alternative(const Results& to, uint64_t row, uint32_t top, uint32_t place, uint64_t key, const Sums& sums) {
    if (to.top_log_prob) to.top_log_prob[row * top + place] = sums.log_prob(key_score((uint32_t)(key >> 32)));
    if (to.top_token) to.top_token[row * top + place] = (int32_t)place_token(key);
}

// A wave's part of a row: vectors [q0, q1) of it, a vector being 16 aligned bytes.
template <class Take>
__device__ __forceinline__ void read_row(const float* logits, uint64_t row, uint32_t V, uint32_t q0, uint32_t q1, Sums& sums, Take take) {
    const uint64_t start = row * V;
    const uint32_t lead = (uint32_t)start & 3u, lane = __lane_id();       // scores of other rows in the first vector
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(logits + (start - lead), (lead + V) * 4u);
    f32x4 next[NV];
    auto fetch = [&](uint32_t q) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t at = q + i * 64u + lane;
            next[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at < q1 ? at * 16u : NOWHERE, 0, 0));
        }
    };
    fetch(q0);
    for (uint32_t q = q0; q < q1; q += NV * 64u) {
        float v[NV][4];
#pragma unroll
        for (int i = 0; i < NV; ++i) { v[i][0] = next[i].x; v[i][1] = next[i].y; v[i][2] = next[i].z; v[i][3] = next[i].w; }
        if (q + NV * 64u < q1) fetch(q + NV * 64u);
        auto token = [&](int i, int j) { return (q + i * 64u + lane) * 4u + j - lead; };
        auto valid = [&](int i, int j) { return q + i * 64u + lane < q1 && token(i, j) < V; };      // (before the row: far above V)
        if (q == 0u || q + NV * 64u >= q1)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = valid(i, j) ? v[i][j] : -INFINITY;
        float best = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) best = fmaxf(best, v[i][j]);
        sums.move(fmaxf(sums.m, best));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums.add(v[i][j]);
        take(v, best, token, valid);
    }
}

// A row to a wave.
extern "C" __global__ __launch_bounds__(256) void log_probs_wave(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token,
                                                                 const float* logits, const uint32_t* tokens, LogProbsParams P) {
    __shared__ uint64_t lists[4][LIST];
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token};
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t row = (uint64_t)blockIdx.x * 4u + wave;
    if (row >= P.rows) return;
    const uint32_t token = __builtin_amdgcn_readfirstlane(tokens[row]);
    if (token >= P.V) { write_padding(to, row, lane, 64u, P.top); return; }
    const float score = logits[row * P.V + token];
    Sums sums; sums.start();
    Candidates found{lists[wave], 0u, P.top, 0.f};
    const uint32_t vectors = ((uint32_t)(row * P.V) & 3u) + P.V + 3u >> 2;
    read_row(logits, row, P.V, 0u, vectors, sums, [&](const float (&v)[NV][4], float best, auto token_of, auto valid) { if (P.top != 0u) found.take(v, best, token_of, valid); });
    sums.join_lanes(64u);
    if (lane == 0u) write_sums(to, row, sums, score);
    if (P.top == 0u) return;
    wave_fence();
    rank(found.keys, found.count, P.top, [&](uint32_t place, uint64_t key) { write_alternative(to, row, P.top, place, key, sums); });
}

// A row, or a slice of one, to a block of four waves. With slices: sums and candidates go to `parts` ([rows, slices, 4] floats: m, s, w) and
// `keys` ([rows, slices, top]) for log_probs_join.
extern "C" __global__ __launch_bounds__(256) void log_probs_block(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token, float* parts, uint64_t* keys,
                                                                  const float* logits, const uint32_t* tokens, LogProbsParams P) {
    __shared__ uint64_t lists[4 * LIST];
    __shared__ Sums of_wave[4];
    __shared__ uint32_t counts[4];
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token};
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, slice = blockIdx.x % P.slices;
    const uint64_t row = blockIdx.x / P.slices;
    const uint32_t token = __builtin_amdgcn_readfirstlane(tokens[row]);
    if (token >= P.V) {
        if (P.slices == 1u && wave == 0u) write_padding(to, row, lane, 64u, P.top);
        return;                                                           // (the whole block)
    }
    const float score = logits[row * P.V + token];
    const uint32_t vectors = ((uint32_t)(row * P.V) & 3u) + P.V + 3u >> 2, q0 = min((slice * 4u + wave) * P.slice, vectors), q1 = min(q0 + P.slice, vectors);
    Sums sums; sums.start();
    Candidates found{lists + wave * LIST, 0u, P.top, 0.f};
    if (q0 < q1) read_row(logits, row, P.V, q0, q1, sums, [&](const float (&v)[NV][4], float best, auto token_of, auto valid) { if (P.top != 0u) found.take(v, best, token_of, valid); });
    sums.join_lanes(64u);
    if (P.top != 0u && found.count > P.top) found.cut();
    if (lane == 0u) { of_wave[wave] = sums; counts[wave] = found.count; }
    __syncthreads();
    if (wave != 0u) return;
#pragma unroll
    for (int k = 1; k < 4; ++k) sums.join(of_wave[k]);
    if (P.slices == 1u) {
        if (lane == 0u) write_sums(to, row, sums, score);
    } else if (lane < 3u) parts[(row * P.slices + slice) * 4u + lane] = lane == 0u ? sums.m : lane == 1u ? sums.s : sums.w;
    if (P.top == 0u) return;
    // the four lists behind one another
    uint32_t count = counts[0];
#pragma unroll
    for (uint32_t k = 1; k < 4u; ++k) {
        const uint64_t key = lists[k * LIST + min(lane, LIST - 1u)];
        wave_fence();
        if (lane < counts[k]) lists[count + lane] = key;
        wave_fence();
        count += counts[k];
    }
    if (P.slices == 1u) rank(lists, count, P.top, [&](uint32_t place, uint64_t key) { write_alternative(to, row, P.top, place, key, sums); });
    else {
        uint64_t* const out = keys + (row * P.slices + slice) * P.top;
        if (count < P.top) for (uint32_t k = count + lane; k < P.top; k += 64u) out[k] = 0ull;      // (a slice of fewer scores)
        rank(lists, count, P.top, [&](uint32_t place, uint64_t key) { out[place] = key; });
    }
}

// Joins the slices of a row: a wave to a row.
extern "C" __global__ __launch_bounds__(64) void log_probs_join(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token, const float* parts,
                                                                const uint64_t* keys, const float* logits, const uint32_t* tokens, LogProbsParams P) {
    extern __shared__ uint64_t all[];                                     // slices * top of them
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token};
    const uint32_t lane = threadIdx.x;
    const uint64_t row = blockIdx.x;
    const uint32_t token = __builtin_amdgcn_readfirstlane(tokens[row]);
    if (token >= P.V) { write_padding(to, row, lane, 64u, P.top); return; }
    const float score = logits[row * P.V + token];
    Sums sums; sums.start();
    for (uint32_t k = lane; k < P.slices; k += 64u) {
        const float* const part = parts + (row * P.slices + k) * 4u;
        sums.join(Sums{part[0], part[1], part[2]});
    }
    sums.join_lanes(64u);
    if (lane == 0u) write_sums(to, row, sums, score);
    if (P.top == 0u) return;
    // only what is no smaller than the k-th largest of the lanes' largest can be among the k largest
    const uint32_t count = P.slices * P.top;
    const uint64_t* const from = keys + row * count;
    uint64_t best = 0ull;
    for (uint32_t k = lane; k < count; k += 64u) { const uint64_t key = from[k]; best = key > best ? key : best; }
    uint64_t least = 0ull;
#pragma unroll 8
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t with = least | 1ull << bit;
        if ((uint32_t)__popcll(__builtin_amdgcn_ballot_w64(best >= with)) >= P.top) least = with;
    }
    uint32_t n = 0;
    for (uint32_t k = 0; k < count; k += 64u) {
        const uint64_t key = k + lane < count ? from[k + lane] : 0ull;
        const bool in = key >= least && key != 0ull;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
        if (in) all[n + lanes_below(mask)] = key;
        n += (uint32_t)__popcll(mask);
    }
    wave_fence();
    rank(all, n, P.top, [&](uint32_t place, uint64_t key) { write_alternative(to, row, P.top, place, key, sums); });
}

// Short rows: 2^log2_lanes lanes to a row, a vector to a lane, and several rows to a wave. The alternatives one by one.
extern "C" __global__ __launch_bounds__(256) void log_probs_short(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token,
                                                                  const float* logits, const uint32_t* tokens, LogProbsParams P) {
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token};
    const uint32_t lanes = 1u << P.log2_lanes, lane = threadIdx.x & (lanes - 1u);
    const uint64_t row = ((uint64_t)blockIdx.x * 256u + threadIdx.x) >> P.log2_lanes;
    const bool there = row < P.rows;
    const uint32_t token = there ? tokens[row] : 0xFFFFFFFFu;
    const bool given = token < P.V;
    const uint64_t start = row * P.V;
    const uint32_t lead = (uint32_t)start & 3u;
    const float* const x = logits + start;
    const float score = given ? x[token] : 0.f;
    float v[4], best = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = -INFINITY;
    auto at = [&](int j) { return lane * 4u + j - lead; };                // (before the row: far above V)
    if (given) {
        if (lane * 4u >= lead && lane * 4u + 4u <= lead + P.V) { const f32x4 t = *reinterpret_cast<const f32x4*>(logits + (start - lead) + lane * 4u); v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; }
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) if (at(j) < P.V) v[j] = x[at(j)];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) best = fmaxf(best, v[j]);
    Sums sums; sums.start();
    sums.move(fmaxf(sums.m, best));
#pragma unroll
    for (int j = 0; j < 4; ++j) sums.add(v[j]);
    sums.join_lanes(lanes);
    if (there && !given) write_padding(to, row, lane, lanes, P.top);
    if (given && lane == 0u) write_sums(to, row, sums, score);
    uint64_t below = ~0ull;
    for (uint32_t k = 0; k < P.top; ++k) {
        uint64_t key = 0ull;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t mine = at(j) < P.V ? place_key(v[j], at(j)) : 0ull;
            if (mine < below && mine > key) key = mine;
        }
        key = lanes_allreduce(key, lanes, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        below = key;
        if (given && lane == (k & (lanes - 1u))) write_alternative(to, row, P.top, k, key, sums);
    }
}

// ---------------------------------------------------------------------------------------------- gradient

// One read and one write per score: blocks of 256 lanes x 4 NV scores of a row. Cotangents that are null are zeros. The tokens whose own log probabilities have
// cotangents are done once more behind the block's other stores: a score's value anew, and all its cotangents in one fixed order.
template <bool ENTROPY>
__device__ __forceinline__ float grad_of(float x, float lse, float total, float gh, float H) {
    const float lp = x - lse;
    // exp(lp): base 2, with the part of the exponent that its rounding loses
    const float t = lp * LOG2E, lost = __builtin_fmaf(lp, LOG2E, -t);
    float p = __builtin_amdgcn_exp2f(t);
    p = lp > -3e38f ? __builtin_fmaf(p, lost * 0.6931471805599453f, p) : p;
    const float d = ENTROPY ? __builtin_fmaf(gh, fmaxf(lp, -1e30f) + H, total) : total;
    return p == 0.f ? 0.f : -p * d;
}

extern "C" __global__ __launch_bounds__(256) void log_probs_grad(float* dx, const float* logits, const uint32_t* tokens, const float* log_sum, const float* entropy,
                                                                 const float* g_log_prob, const float* g_entropy, const float* g_top, const int32_t* top_token, LogProbsParams P) {
    const uint32_t slice = blockIdx.x % P.slices;
    const uint64_t row = blockIdx.x / P.slices, start = row * P.V;
    const uint32_t lead = (uint32_t)start & 3u, vectors = lead + P.V + 3u >> 2;
    const uint32_t q0 = slice * P.slice, q1 = min(q0 + P.slice, vectors);
    const uint32_t token = tokens[row];
    const float lse = log_sum[row];
    const bool nothing = token >= P.V || lse == -INFINITY;
    const bool stream = streams_result(P.first);
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(logits + (start - lead), nothing ? 0u : (lead + P.V) * 4u), d_rsrc = make_rsrc(dx + (start - lead), (lead + P.V) * 4u);
    const float own = g_log_prob ? g_log_prob[row] : 0.f, gh = g_entropy ? g_entropy[row] : 0.f, H = entropy[row];
    float total = own;
    for (uint32_t k = 0; k < P.top; ++k) total += g_top[row * P.top + k];
    for (uint32_t q = q0 + threadIdx.x; q < q1; q += 256u * NV) {
        f32x4 v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, q + i * 256u < q1 ? (q + i * 256u) * 16u : NOWHERE, 0, 0));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t at = q + i * 256u;
            f32x4 d;
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = nothing ? 0.f : gh == 0.f ? grad_of<false>(v[i][j], lse, total, gh, H) : grad_of<true>(v[i][j], lse, total, gh, H);
            if (at >= q1) continue;
            if (at * 4u >= lead && at * 4u + 4u <= lead + P.V) {
                const u32x4 t = u32x4{f2u(d[0]), f2u(d[1]), f2u(d[2]), f2u(d[3])};
                if (stream) __builtin_amdgcn_raw_buffer_store_b128(t, d_rsrc, at * 16u, 0, 2);
                else __builtin_amdgcn_raw_buffer_store_b128(t, d_rsrc, at * 16u, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (at * 4u + j - lead < P.V) dx[start + (at * 4u + j - lead)] = d[j];
            }
        }
    }
    if (nothing) return;
    __syncthreads();
    // thread k < top: alternative k, thread `top`: the given token; in the block that has its score
    const uint32_t k = threadIdx.x;
    if (k > P.top) return;
    const uint32_t mine = k < P.top ? (uint32_t)top_token[row * P.top + k] : token, vector = mine + lead >> 2;
    if (mine >= P.V || vector < q0 || vector >= q1) return;
    float d = grad_of<true>(logits[start + mine], lse, total, gh, H);
    if (mine == token) d += own;
    for (uint32_t i = 0; i < P.top; ++i) if ((uint32_t)top_token[row * P.top + i] == mine) d += g_top[row * P.top + i];
    dx[start + mine] = d;
}
