// Log probabilities of given tokens with the entropy of their rows' distributions and the most likely alternatives, and the
// gradient of all three.
//
// With m = max x, s = sum exp(x - m), w = sum exp(x - m) (x - m) over a row of V scores:
//   lse = m + log s,  log p = x - lse,  H = -sum p log p = log s - w / s
//   dx[v] = -p[v] (sum of the cotangents of log probabilities) - gH p[v] (log p[v] + H) + the cotangents of v's own log probabilities
//
// log p is the difference to the maximum less log s. What the gradient gets of a row is lse, rounded, and the rest that its rounding lost: at scores around
// 10^4 half a step of lse would be 5 10^-4 of every p of the row, and where all of them are the type's lowest value lse alone is one of them, and p 1.
//
// A token outside [0, V) marks its row as padding: results are 0 (alternatives: token -1), the row's scores are not read. Scores of
// -inf are masked: p = 0, and p log p counts as 0. Where every score of a row is -inf there is no distribution: log p = -inf, H = 0,
// gradient 0. NaN and +inf make their row NaN by themselves (+inf - +inf).
//
// A row is read once. A wave takes 1024 scores at a time, 16 per lane in vectors of 16 bytes (of memory: a row that starts inside a vector has its first
// scores in that one, the others' are masked). Every lane keeps a maximum and the two sums relative to it, changed when the maximum does,
// once per 16 scores; lanes, waves and slices of a row are joined the same way.
//
// The alternatives: with the lanes in k groups or more, the smallest of the groups' maxima is no larger than the k-th largest score: a bar, found in six steps
// and raised by a few bisections where many lanes pass it. Of the first 1024 scores only what reaches the bar can be among the k largest: a few more than k
// scores, which go into a list. From then on only scores above the bar are looked at: one comparison per lane and 16 scores, and rarely
// more. The list is cut to k scores, and the bar raised, when it is long. Where more stand out at once than the list holds, a bisection of their
// keys raises the bar; only where that many are equal, the largest are taken one by one, 60 us of a wave's time. (Without the bisection one wave in a hundred
// came to that, and the launch waited for it: 32 of 1024 x 4092 82 us instead of 23.) Places in the list are counted once, at the end.
//
// What bounds it: without alternatives, memory (65536 rows of 1000 39 us, 6.8 TB/s; 4096 of 32000 89 us, 5.9; its gradient 172 us, 5.9). With them, the
// instructions that look for them: 5 of 65536 x 1000 54 us, 20 63; 20 of 4096 x 32000 120. (Rows a few to a wave, the next one's scores asked for ahead, need
// 131 registers or memory for them: 88 us instead of 54.) A few rows of 32000 are cut into slices of 4000, a block each, and joined by a second launch: 8 rows
// with 20 alternatives 7.8 + 4.3 us, without 3.4 + 2.6: one wave's chain of steps each, which nothing else hides.
#include "common.h"

struct LogProbsParams {
    uint32_t first;                              // (the gradient: the rows, and in bit 31 whether the result is stored past the caches)
    uint32_t rows, V, top;
    uint32_t slices, slice;                      // blocks per row, vectors of a row to a wave
    uint32_t log2_lanes;                         // lanes per row, where a wave has several rows
};

constexpr uint32_t NOWHERE = 0x80000000u;
constexpr uint32_t LIST = 128;
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
};
// What a row's sums say. (The logarithm once: it is as many instructions as ten scores.)
struct Distribution {
    float m, log_s, entropy;
    bool nothing;
    __device__ __forceinline__ explicit Distribution(const Sums& sums) : m(sums.m), nothing(sums.s == 0.f) {
        log_s = logf(sums.s);
        entropy = nothing ? 0.f : log_s - sums.w / sums.s;
    }
    __device__ __forceinline__ float log_sum() const { return nothing ? -INFINITY : m + log_s; }
    // what the rounding of log_sum has lost, exactly (Knuth's sum of two numbers)
    __device__ __forceinline__ float log_sum_rest() const {
        const float sum = m + log_s, second = sum - m;
        return nothing ? 0.f : (m - (sum - second)) + (log_s - second);
    }
    __device__ __forceinline__ float log_prob(float x) const { return nothing ? -INFINITY : (x - m) - log_s; }
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

__device__ __forceinline__ uint64_t of_lane(uint64_t v, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), (int)lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, (int)lane);
}
// The places of keys, of which a lane has numbers lane, lane + 64 .., `count` of them among the first `end` numbers (the others are zeros): how many are larger, by
// the scores alone, four from shared memory at a time, unless some of these are equal; then places are no permutation, which their sum tells. `scores`: 64 N words
// of shared memory.
template <int N>
__device__ __forceinline__ void places_of(const uint64_t (&keys)[N], uint32_t end, uint32_t count, uint32_t* scores, uint32_t (&places)[N]) {
    const uint32_t lane = __lane_id();
    uint32_t sum = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) { scores[k * 64 + lane] = (uint32_t)(keys[k] >> 32); places[k] = 0u; }
    wave_fence();
    for (uint32_t at = 0; at < end; at += 4u) {
        const u32x4 others = *reinterpret_cast<const u32x4*>(scores + at);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t own = (uint32_t)(keys[k] >> 32);
            places[k] += others.x > own; places[k] += others.y > own; places[k] += others.z > own; places[k] += others.w > own;
        }
    }
    wave_fence();
#pragma unroll
    for (int k = 0; k < N; ++k) sum += keys[k] != 0ull ? places[k] : 0u;
    if (lanes_allreduce(sum, 64u, [](uint32_t a, uint32_t b) { return a + b; }) == count * (count - 1u) / 2u) return;
#pragma unroll
    for (int k = 0; k < N; ++k) places[k] = 0u;
#pragma unroll
    for (int m = 0; m < N; ++m)
#pragma nounroll
        for (uint32_t i = 0; i < 64u && m * 64u + i < end; ++i) {
            const uint64_t other = of_lane(keys[m], i);
#pragma unroll
            for (int k = 0; k < N; ++k) places[k] += other > keys[k];
        }
}
// A value that at least k (up to 32) of the lanes' values reach, and not many more: of 2^n >= k groups of lanes the smallest maximum, raised by bisection.
__device__ __forceinline__ float bar_of(float lane_value, uint32_t k) {
    const uint32_t group = 64u >> (32u - (uint32_t)__clz((int)k - 1));    // lanes to a group (k = 1: all)
    float bar = lane_value, most = lane_value;
    wave_butterfly([&](auto step) {                                       // from the widest step: the lanes of a group lie group's number apart
        constexpr int S = decltype(step)::value;
        const float other = lane_xor<S>(bar);
        bar = (uint32_t)S >= 64u / group ? fmaxf(bar, other) : fminf(bar, other);
        most = fmaxf(most, lane_xor<S>(most));
    });
    for (int i = 0; i < 8; ++i) {
        if ((uint32_t)__popcll(__builtin_amdgcn_ballot_w64(lane_value >= bar)) <= k + (k >> 2) + 2u) break;
        const float between = __builtin_fmaf(0.5f, bar, 0.5f * most);
        const bool enough = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(lane_value >= between)) >= k;
        bar = enough ? between : bar; most = enough ? most : between;
    }
    return bar;
}

__device__ __forceinline__ float wave_max(float v) { return lanes_allreduce(v, 64u, [](float a, float b) { return fmaxf(a, b); }); }

// The k-th largest of the lanes' values, bit by bit, by how many lanes are no smaller.
__device__ __forceinline__ float kth_largest(float lane_value, uint32_t k) {
    const uint32_t key = score_key(lane_value);
    uint32_t found = 0;
#pragma nounroll
    for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1)
        if ((uint32_t)__popcll(__builtin_amdgcn_ballot_w64(key >= (found | bit))) >= k) found |= bit;
    return key_score(found);
}
// The largest value smaller than x (x finite or +inf).
__device__ __forceinline__ float below(float x) {
    const uint32_t b = f2u(x);
    return x == 0.f ? u2f(0x80000001u) : u2f(x > 0.f ? b - 1u : b + 1u);
}

// 64 x 4 NV scores of a row as a wave holds them: score (i, j) of a lane is that of token first + 256 i + j, if that is below `end`, else -inf.
struct Chunk {
    const float* row;
    uint32_t first, end;
    __device__ __forceinline__ uint32_t token(int i, int j) const { return first + 256u * i + j; }
    __device__ __forceinline__ bool valid(int i, int j) const { return token(i, j) < end; }      // (tokens before the row: far above it)
};

// A score with its token, as it goes into a list: becoming a key is left to the one lane that sorts it in.
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t token) { return (uint64_t)f2u(x) << 32 | token; }
__device__ __forceinline__ uint64_t key_of(uint64_t entry) { return place_key(u2f((uint32_t)(entry >> 32)), (uint32_t)entry); }

// The list of a wave's candidates in shared memory.
struct Candidates {
    uint64_t* entries;                           // LIST of them
    uint32_t count, top;
    float bar;                                   // at least `top` scores have been no smaller: later ones count where they are larger

    // cuts the list to the `top` largest, in order
    __device__ __forceinline__ void cut() {
        wave_fence();
        const uint32_t lane = __lane_id();
        const uint64_t own_a = lane < count ? entries[lane] : 0ull, own_b = lane + 64u < count ? entries[lane + 64u] : 0ull;
        const uint64_t a = lane < count ? key_of(own_a) : 0ull, b = lane + 64u < count ? key_of(own_b) : 0ull;
        uint32_t place_a, place_b = 0u;
        wave_fence();
        if (count <= 64u) {
            uint64_t keys[1];
            uint32_t places[1];
            keys[0] = a;
            places_of<1>(keys, count, count, reinterpret_cast<uint32_t*>(entries), places);
            place_a = places[0];
        } else {
            uint64_t keys[2];
            uint32_t places[2];
            keys[0] = a; keys[1] = b;
            places_of<2>(keys, count, count, reinterpret_cast<uint32_t*>(entries), places);
            place_a = places[0]; place_b = places[1];
        }
        if (lane < count && place_a < top) entries[place_a] = own_a;
        if (lane + 64u < count && place_b < top) entries[place_b] = own_b;
        wave_fence();
        count = min(count, top);
        bar = u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(entries[count - 1u] >> 32)));
    }
    // Takes from a chunk, whose tokens are behind those of the chunks before, what may be among the largest. `best`: the largest number of each of the lane's
    // vectors, `most` of all; `broken`: the lane has met a NaN, which does not show among the maxima but passes the comparisons that are made here.
    __device__ __forceinline__ void take(const float (&v)[NV][4], const float (&best)[NV], float most, bool broken, const Chunk& chunk) {
        const bool fresh = count == 0u;
        if (fresh) {
            bar = bar_of(most, top);
            if (bar == -INFINITY) bar = kth_largest(most, top);           // (much of it masked)
        } else if (__builtin_amdgcn_ballot_w64(!(most <= bar) || broken) == 0ull) return;
        // of the first scores those that reach the bar
        float from = fresh && bar != -INFINITY ? below(bar) : bar;
        uint32_t n;
#pragma nounroll
        for (bool again = false;; again = true) {
            n = count;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (__builtin_amdgcn_ballot_w64(!(best[i] <= from) || broken) == 0ull) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t mask = __builtin_amdgcn_ballot_w64(!(v[i][j] <= from));
                    if (mask != 0ull) {
                        const uint32_t more = (uint32_t)__popcll(mask);
                        if (n + more <= LIST && !(v[i][j] <= from)) entries[n + lanes_below(mask)] = entry_of(v[i][j], chunk.token(i, j));
                        n += more;
                    }
                }
            }
            if (n <= LIST) break;
            if (again) { one_by_one(chunk); return; }
            // more than there is room for: once more from a higher bar, that of the list cut to its largest or one that as many of these scores reach as do not
            // fill the list, which a bisection of their keys finds
            if (count > top) { cut(); from = bar; }
            uint32_t low = score_key(from), high = score_key(wave_max(most));
            for (int step = 0; step < 32 && high - low > 1u; ++step) {
                const uint32_t between = low + ((high - low) >> 1);
                const float x = key_score(between);
                uint32_t passing = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) passing += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(!(v[i][j] <= x)));
                if (passing < top) { high = between; continue; }
                low = between; from = x;
                if (count + passing <= LIST) break;
            }
        }
        count = n;
        if (fresh && count < top) {                                       // masked scores: as many as are missing, the first of them
            uint32_t need = top - count;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                uint32_t before = 0, all = 0;
                bool is[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    is[j] = v[i][j] == -INFINITY && chunk.valid(i, j);
                    const uint64_t mask = __builtin_amdgcn_ballot_w64(is[j]);
                    before += lanes_below(mask); all += (uint32_t)__popcll(mask);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (is[j] && before < need) entries[count + before] = entry_of(-INFINITY, chunk.token(i, j));
                    before += is[j];
                }
                const uint32_t taken = min(all, need);
                count += taken; need -= taken;
            }
        }
        if (count > top + 24u) cut();                                     // (a bar that stays low lets ever more pass)
    }
    // The `top` largest of the list and a chunk, one after the other, where more of the chunk pass than the list holds: many equal scores, or many large ones in few
    // lanes. The scores are read again (they are in the caches), so that this takes no registers from the loop over the row.
    __device__ __forceinline__ void one_by_one(const Chunk& chunk) {
        const uint32_t lane = __lane_id();
        wave_fence();
        const uint64_t a = lane < count ? key_of(entries[lane]) : 0ull, b = lane + 64u < count ? key_of(entries[lane + 64u]) : 0ull;
        uint64_t below = ~0ull;
        uint32_t n = 0;
#pragma nounroll
        for (; n < top; ++n) {
            uint64_t best = a < below ? a : 0ull;
            best = b < below && b > best ? b : best;
#pragma unroll 4
            for (int e = 0; e < 4 * NV; ++e) {
                const uint32_t token = chunk.first + 256u * (e >> 2) + (e & 3);
                const uint64_t key = token < chunk.end ? place_key(chunk.row[token], token) : 0ull;
                if (key < below && key > best) best = key;
            }
            best = lanes_allreduce(best, 64u, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
            if (best == 0ull) break;
            below = best;
            wave_fence();
            if (lane == 0u) entries[n] = entry_of(key_score((uint32_t)(best >> 32)), place_token(best));
        }
        wave_fence();
        count = n;
        bar = n == top ? key_score((uint32_t)(below >> 32)) : -INFINITY;
    }
};

struct Results { float *log_prob, *entropy, *log_sum, *top_log_prob; int32_t* top_token; float* log_sum_rest; };

__device__ __forceinline__ void write_padding(const Results& to, uint64_t row, uint32_t lane, uint32_t lanes, uint32_t top) {
    if (lane == 0u) {
        if (to.log_prob) to.log_prob[row] = 0.f;
        if (to.entropy) to.entropy[row] = 0.f;
        if (to.log_sum) to.log_sum[row] = 0.f;
        if (to.log_sum_rest) to.log_sum_rest[row] = 0.f;
    }
    for (uint32_t k = lane; k < top; k += lanes) {
        if (to.top_log_prob) to.top_log_prob[row * top + k] = 0.f;
        if (to.top_token) to.top_token[row * top + k] = -1;
    }
}
__device__ __forceinline__ void write_sums(const Results& to, uint64_t row, const Distribution& p, float score) {
    if (to.log_prob) to.log_prob[row] = p.log_prob(score);
    if (to.entropy) to.entropy[row] = p.entropy;
    if (to.log_sum) to.log_sum[row] = p.log_sum();
    if (to.log_sum_rest) to.log_sum_rest[row] = p.log_sum_rest();
}
__device__ __forceinline__ void write_alternative(const Results& to, uint64_t row, uint32_t top, uint32_t place, uint64_t key, const Distribution& p) {
    if (to.top_log_prob) to.top_log_prob[row * top + place] = p.log_prob(key_score((uint32_t)(key >> 32)));
    if (to.top_token) to.top_token[row * top + place] = (int32_t)place_token(key);
}

// A row in vectors of 16 aligned bytes.
struct Row {
    const float* x;
    uint32_t lead, V;                            // scores of other rows in the first vector; its own
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ Row(const float* logits, uint64_t row, uint32_t V) : x(logits + row * V), lead((uint32_t)(row * V) & 3u), V(V) { rsrc = make_rsrc(x - lead, (lead + V) * 4u); }
    __device__ __forceinline__ uint32_t vectors() const { return (lead + V + 3u) >> 2; }
    // vectors q + 64 i + lane, those below q1
    __device__ __forceinline__ void fetch(f32x4 (&to)[NV], uint32_t q, uint32_t q1) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t at = q + i * 64u + __lane_id();
            to[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at < q1 ? at * 16u : NOWHERE, 0, 0));
        }
    }
};

// A wave's part of a row: vectors [q0, q1) of it, the first of which are in `next`. SINGLE: no more than the wave takes at a time.
template <bool SINGLE, class Take>
__device__ __forceinline__ void read_row(const Row& row, uint32_t q0, uint32_t q1, f32x4 (&next)[NV], Sums& sums, Take take) {
    for (uint32_t q = q0; q < q1; q += NV * 64u) {
        float v[NV][4];
#pragma unroll
        for (int i = 0; i < NV; ++i) { v[i][0] = next[i].x; v[i][1] = next[i].y; v[i][2] = next[i].z; v[i][3] = next[i].w; }
        if (!SINGLE && q + NV * 64u < q1) row.fetch(next, q + NV * 64u, q1);
        const Chunk chunk{row.x, (q + __lane_id()) * 4u - row.lead, min(q1 * 4u - row.lead, row.V)};
        if (SINGLE || q == 0u || q + NV * 64u >= q1)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = chunk.valid(i, j) ? v[i][j] : -INFINITY;
        float best[NV], most = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            best[i] = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
            most = fmaxf(most, best[i]);
        }
        sums.move(fmaxf(sums.m, most));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums.add(v[i][j]);
        take(v, best, most, sums.s != sums.s, chunk);
        if (SINGLE) return;
    }
}

// put(place, key) for the `top` largest of `count` keys (up to 64 N, no two the same; zeros are none), by a wave; `room` holds 64 in shared memory. The alternatives'
// bar, for keys, raised until no more than 64 pass.
template <int N, class Put>
__device__ __forceinline__ void best_keys(const uint64_t* keys, uint32_t count, uint64_t* room, uint32_t top, Put put) {
    const uint32_t lane = __lane_id(), group = 64u >> (32u - (uint32_t)__clz((int)top - 1));
    uint64_t mine[N], bar = 0ull;
#pragma unroll
    for (int i = 0; i < N; ++i) mine[i] = i * 64u + lane < count ? keys[i * 64u + lane] : 0ull;
#pragma unroll
    for (int i = 0; i < N; ++i) bar = mine[i] > bar ? mine[i] : bar;
    wave_butterfly([&](auto step) {
        constexpr int S = decltype(step)::value;
        const uint64_t other = lane_xor<S>(bar);
        bar = ((uint32_t)S >= 64u / group) == (other > bar) ? other : bar;
    });
    auto passing = [&](auto passes) {
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(mine[i] != 0ull && passes(mine[i])));
        return n;
    };
    bar = of_lane(bar, 0u);
    if (passing([&](uint64_t key) { return key >= bar; }) > 64u) {
        // by the scores alone, and, where too many are equal, by the tokens among them (of neighbouring bars one lets at most one key more through)
        uint32_t low = (uint32_t)(bar >> 32), high = 0u, n = count;
#pragma unroll
        for (int i = 0; i < N; ++i) high = max(high, (uint32_t)(mine[i] >> 32));
        high = lanes_allreduce(high, 64u, [](uint32_t a, uint32_t b) { return max(a, b); }) + 1u;
#pragma nounroll
        while (n > 64u && high - low > 1u) {
            const uint32_t between = low + ((high - low) >> 1), here = passing([&](uint64_t key) { return (uint32_t)(key >> 32) >= between; });
            if (here >= top) { low = between; n = here; } else high = between;
        }
        bar = (uint64_t)low << 32;
        uint64_t most = (uint64_t)high << 32;
#pragma nounroll
        for (int i = 0; i < 33 && n > 64u; ++i) {
            const uint64_t between = bar + ((most - bar) >> 1);
            const uint32_t here = passing([&](uint64_t key) { return key >= between; });
            if (here >= top) { bar = between; n = here; } else most = between;
        }
    }
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool in = mine[i] >= bar && mine[i] != 0ull;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
        if (in && n + lanes_below(mask) < 64u) room[n + lanes_below(mask)] = mine[i];
        n += (uint32_t)__popcll(mask);
    }
    wave_fence();
    const uint64_t found[1] = {lane < n ? room[lane] : 0ull};
    uint32_t place[1];
    wave_fence();
    places_of<1>(found, n, n, reinterpret_cast<uint32_t*>(room), place);
    if (lane < n && place[0] < top) put(place[0], found[0]);
}

// A row to a wave.
template <bool SINGLE>
__device__ __forceinline__ void wave_body(const Results& to, const float* logits, const uint32_t* tokens, const LogProbsParams& P) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[4][LIST];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t row = (uint64_t)blockIdx.x * 4u + wave;
    // (asked for before it is known whether there is such a row, so that all arguments come with one wait: 65536 rows of 1000 67.0 us a pass, so 64.5)
    const uint32_t token = __builtin_amdgcn_readfirstlane(tokens[min(row, (uint64_t)P.rows - 1u)]);
    if (row >= P.rows) return;
    if (token >= P.V) { write_padding(to, row, lane, 64u, P.top); return; }
    const Row from(logits, row, P.V);
    const float score = from.x[token];
    Sums sums; sums.start();
    Candidates found{lists[wave], 0u, P.top, 0.f};
    f32x4 next[NV];
    from.fetch(next, 0u, from.vectors());
    read_row<SINGLE>(from, 0u, from.vectors(), next, sums, [&](const float (&v)[NV][4], const float (&best)[NV], float most, bool broken, const Chunk& chunk) {
        if (P.top != 0u) found.take(v, best, most, broken, chunk);
    });
    sums.join_lanes(64u);
    const Distribution p(sums);
    if (lane == 0u) write_sums(to, row, p, score);
    if (P.top == 0u) return;
    if (found.count > 64u) found.cut();
    wave_fence();
    const uint64_t key[1] = {lane < found.count ? key_of(found.entries[lane]) : 0ull};
    uint32_t place[1];
    wave_fence();
    places_of<1>(key, found.count, found.count, reinterpret_cast<uint32_t*>(found.entries), place);
    if (lane < found.count && place[0] < P.top) write_alternative(to, row, P.top, place[0], key[0], p);
}
#define LOG_PROBS_WAVE(name, SINGLE)                                                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void name(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token,    \
                                                           float* log_sum_rest, const float* logits, const uint32_t* tokens, LogProbsParams P) {        \
        wave_body<SINGLE>(Results{log_prob, entropy, log_sum, top_log_prob, top_token, log_sum_rest}, logits, tokens, P);                               \
    }
LOG_PROBS_WAVE(log_probs_wave, true)
LOG_PROBS_WAVE(log_probs_wave_long, false)

// A row, or a slice of one, to a block of four waves. With slices: sums and candidates go to `parts` ([rows, slices, 4] floats: m, s, w) and
// `keys` ([rows, top, slices]) for log_probs_join.
extern "C" __global__ __launch_bounds__(256, 4) void log_probs_block(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token, float* log_sum_rest,
                                                                     float* parts, uint64_t* keys, const float* logits, const uint32_t* tokens, LogProbsParams P) {
    constexpr uint32_t WAVES = 4;
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token, log_sum_rest};
    __shared__ __attribute__((aligned(16))) uint64_t lists[WAVES * LIST];
    __shared__ uint64_t all[WAVES * 32];
    __shared__ Sums of_wave[WAVES];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, slice = blockIdx.x % P.slices;
    const uint64_t row = blockIdx.x / P.slices;
    const Row from(logits, row, P.V);
    const uint32_t q0 = min((slice * WAVES + wave) * P.slice, from.vectors()), q1 = min(q0 + P.slice, from.vectors());
    f32x4 next[NV];
    if (P.slices != 1u) from.fetch(next, q0, q1);                         // (few rows: one round trip to memory less to wait for, and little read in vain for padding)
    const uint32_t token = __builtin_amdgcn_readfirstlane(tokens[row]);
    if (token >= P.V) {
        if (P.slices == 1u && wave == 0u) write_padding(to, row, lane, 64u, P.top);
        return;                                                           // (the whole block)
    }
    const float score = from.x[token];
    if (P.slices == 1u) from.fetch(next, q0, q1);
    Sums sums; sums.start();
    Candidates found{lists + wave * LIST, 0u, P.top, 0.f};
    if (q0 < q1) read_row<false>(from, q0, q1, next, sums, [&](const float (&v)[NV][4], const float (&best)[NV], float most, bool broken, const Chunk& chunk) {
        if (P.top != 0u) found.take(v, best, most, broken, chunk);
    });
    sums.join_lanes(64u);
    if (lane == 0u) of_wave[wave] = sums;
    const uint32_t share = P.top <= 12u ? 16u : 32u;                      // keys that a wave may leave, in any order
    if (P.top != 0u) {
        if (found.count > share) found.cut();
        wave_fence();
        if (lane < share) all[wave * share + lane] = lane < found.count ? key_of(found.entries[lane]) : 0ull;
    }
    __syncthreads();
    if (wave != 0u) return;
    sums = of_wave[lane & (WAVES - 1)];
    sums.join_lanes(WAVES);
    const Distribution p(sums);
    if (P.slices == 1u) {
        if (lane == 0u) write_sums(to, row, p, score);
    } else if (lane < 3u) parts[(row * P.slices + slice) * 4u + lane] = lane == 0u ? sums.m : lane == 1u ? sums.s : sums.w;
    if (P.top == 0u) return;
    uint64_t* const out = keys + row * P.slices * P.top + slice;
    uint32_t* const scores = reinterpret_cast<uint32_t*>(lists);
    auto keep = [&](uint32_t place, uint64_t key) {
        if (key == 0ull || place >= P.top) return;
        if (P.slices == 1u) write_alternative(to, row, P.top, place, key, p);
        else out[place * P.slices] = key;
    };
    uint32_t count;
    if (share == 16u) {
        const uint64_t mine[1] = {all[lane]};
        uint32_t places[1];
        count = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(mine[0] != 0ull));
        places_of<1>(mine, 64u, count, scores, places);
        keep(places[0], mine[0]);
    } else {
        const uint64_t mine[2] = {all[lane], all[lane + 64u]};
        uint32_t places[2];
        count = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(mine[0] != 0ull)) + (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(mine[1] != 0ull));
        places_of<2>(mine, 128u, count, scores, places);
        keep(places[0], mine[0]); keep(places[1], mine[1]);
    }
    if (P.slices != 1u && lane >= count && lane < P.top) out[lane * P.slices] = 0ull;      // (a slice may have fewer scores)
}

// Joins the slices of a row: a wave to a row.
extern "C" __global__ __launch_bounds__(64) void log_probs_join(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token, float* log_sum_rest,
                                                                const float* parts, const uint64_t* keys, const float* logits, const uint32_t* tokens, LogProbsParams P) {
    __shared__ __attribute__((aligned(16))) uint64_t room[64];
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token, log_sum_rest};
    const uint32_t lane = threadIdx.x;
    const uint64_t row = blockIdx.x;
    const uint32_t token = __builtin_amdgcn_readfirstlane(tokens[row]);
    Sums sums; sums.start();
    for (uint32_t k = lane; k < P.slices; k += 64u) {                     // (of padding: whatever is there)
        const float* const part = parts + (row * P.slices + k) * 4u;
        sums.join(Sums{part[0], part[1], part[2]});
    }
    if (token >= P.V) { write_padding(to, row, lane, 64u, P.top); return; }
    const float score = logits[row * P.V + token];
    sums.join_lanes(64u);
    const Distribution p(sums);
    if (lane == 0u) write_sums(to, row, p, score);
    if (P.top == 0u) return;
    const uint32_t count = P.slices * P.top;
    auto put = [&](uint32_t place, uint64_t key) { write_alternative(to, row, P.top, place, key, p); };
    if (count <= 256u) best_keys<4>(keys + row * count, count, room, P.top, put);
    else best_keys<16>(keys + row * count, count, room, P.top, put);
}

// Short rows: 2^log2_lanes lanes to a row, four vectors to a lane, and several rows to a wave. The alternatives one by one.
extern "C" __global__ __launch_bounds__(256) void log_probs_short(float* log_prob, float* entropy, float* log_sum, float* top_log_prob, int32_t* top_token,
                                                                  float* log_sum_rest, const float* logits, const uint32_t* tokens, LogProbsParams P) {
    const Results to{log_prob, entropy, log_sum, top_log_prob, top_token, log_sum_rest};
    const uint32_t lanes = 1u << P.log2_lanes, lane = threadIdx.x & (lanes - 1u);
    const uint64_t row = ((uint64_t)blockIdx.x * 256u + threadIdx.x) >> P.log2_lanes;
    const bool there = row < P.rows;
    const uint32_t token = there ? tokens[row] : 0xFFFFFFFFu;
    const bool given = token < P.V;
    const uint64_t start = row * P.V;
    const uint32_t lead = (uint32_t)start & 3u;
    const float* const x = logits + start;
    const float score = given ? x[token] : 0.f;
    float v[NV][4], best = -INFINITY;
    auto at = [&](int i, int j) { return (i * lanes + lane) * 4u + j - lead; };      // (before the row: far above V)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = -INFINITY;
        const uint32_t first = (i * lanes + lane) * 4u;
        if (given && first >= lead && first + 4u <= lead + P.V) {
            const f32x4 t = *reinterpret_cast<const f32x4*>(logits + (start - lead) + first);
            v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
        } else if (given)
#pragma unroll
            for (int j = 0; j < 4; ++j) if (at(i, j) < P.V) v[i][j] = x[at(i, j)];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) best = fmaxf(best, v[i][j]);
    Sums sums; sums.start();
    sums.move(fmaxf(sums.m, best));
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums.add(v[i][j]);
    sums.join_lanes(lanes);
    if (there && !given) write_padding(to, row, lane, lanes, P.top);
    const Distribution p(sums);
    if (given && lane == 0u) write_sums(to, row, p, score);
    if (P.top == 0u) return;
    // A place's key is the score's; which of the equal ones it is, the number of the first one behind the last place tells.
    uint32_t keys[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) keys[i][j] = at(i, j) < P.V ? score_key(v[i][j]) : 0u;
    for (uint32_t k = 0; k < P.top; ++k) {
        uint32_t key = 0u, number = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) key = max(key, keys[i][j]);
        key = lanes_allreduce(key, lanes, [](uint32_t a, uint32_t b) { return max(a, b); });
#pragma unroll
        for (int i = NV - 1; i >= 0; --i)
#pragma unroll
            for (int j = 3; j >= 0; --j) number = keys[i][j] == key && key != 0u ? at(i, j) : number;
        number = lanes_allreduce(number, lanes, [](uint32_t a, uint32_t b) { return min(a, b); });
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) keys[i][j] = at(i, j) == number ? 0u : keys[i][j];
        if (given && lane == (k & (lanes - 1u))) write_alternative(to, row, P.top, k, (uint64_t)key << 32 | (0xFFFFFFFFu - number), p);
    }
}

// ---------------------------------------------------------------------------------------------- gradient

// One read and one write per score. 2^log2_lanes lanes to a row (or to a slice of a long one), NV vectors of each in flight per lane; several rows to a block where
// they are short. Cotangents that are null are zeros. The tokens whose own log probabilities have cotangents are done once more behind the
// block's other stores: a score's value anew, and all its cotangents in one fixed order.
// What bounds it: memory, 4096 rows of 32000 (1.02 GB) 170 us, 6.0 TB/s; rows from the last one on, since the forward pass has left those in the
// 256 MB behind the L2s (198 us from the first one on).
template <bool ENTROPY>
__device__ __forceinline__ float grad_of(float x, float lse, float rest, float total, float gh, float H) {
    const float lp = (x - lse) - rest;
    // exp(lp): base 2, with the part of the exponent that its rounding loses
    const float t = lp * LOG2E, lost = __builtin_fmaf(lp, LOG2E, -t);
    float p = __builtin_amdgcn_exp2f(t);
    p = lp > -3e38f ? __builtin_fmaf(p, lost * 0.6931471805599453f, p) : p;
    const float d = ENTROPY ? __builtin_fmaf(gh, fmaxf(lp, -1e30f) + H, total) : total;
    return p == 0.f ? 0.f : -p * d;
}

extern "C" __global__ __launch_bounds__(256) void log_probs_grad(float* dx, const float* logits, const uint32_t* tokens, const float* log_sum, const float* log_sum_rest,
                                                                 const float* entropy, const float* g_log_prob, const float* g_entropy, const float* g_top, const int32_t* top_token, LogProbsParams P) {
    const uint32_t lanes = 1u << P.log2_lanes, lane = threadIdx.x & (lanes - 1u), side = 256u >> P.log2_lanes;
    const uint32_t rows = without_stream_bit(P.first), block = gridDim.x - 1u - blockIdx.x, slice = block % P.slices;
    const bool stream = streams_result(P.first);
    const uint64_t row0 = (uint64_t)(block / P.slices) * side, row = row0 + (threadIdx.x >> P.log2_lanes), start0 = row0 * P.V;
    const bool there = row < rows;
    const uint32_t at0 = ((uint32_t)start0 & 3u) + (uint32_t)(row - row0) * P.V, lead = at0 & 3u;      // where the row starts in the block's scores
    const uint32_t vectors = lead + P.V + 3u >> 2, q0 = slice * P.slice, q1 = there ? min(q0 + P.slice, vectors) : 0u;
    const uint32_t bytes = (((uint32_t)start0 & 3u) + (uint32_t)min((uint64_t)side, rows - row0) * P.V) * 4u;
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(logits + (start0 - (start0 & 3u)), bytes), d_rsrc = make_rsrc(dx + (start0 - (start0 & 3u)), bytes);
    const uint32_t token = there ? tokens[row] : 0xFFFFFFFFu;
    const float lse = there ? log_sum[row] : 0.f, rest = there && log_sum_rest ? log_sum_rest[row] : 0.f, H = there ? entropy[row] : 0.f;
    const bool nothing = token >= P.V || lse == -INFINITY;
    const float own = g_log_prob && there ? g_log_prob[row] : 0.f, gh = g_entropy && there ? g_entropy[row] : 0.f;
    float total = own;
    if (there)
#pragma unroll 8
        for (uint32_t k = 0; k < P.top; ++k) total += g_top[row * P.top + k];
    // rows of few lanes: every score looks for itself among the alternatives. (2319 rows of 12, all of them alternatives: 7 us, a lane to an alternative some 27)
    const bool few = P.log2_lanes <= 4u;
    const uint32_t from = at0 - lead;
    for (uint32_t q = q0 + lane; q < q1; q += lanes * NV) {
        f32x4 v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, q + i * lanes < q1 && !nothing ? (from + (q + i * lanes) * 4u) * 4u : NOWHERE, 0, 0));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t at = q + i * lanes;
            f32x4 d;
            if (g_entropy == nullptr)
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = nothing ? 0.f : grad_of<false>(v[i][j], lse, rest, total, gh, H);
            else
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = nothing ? 0.f : grad_of<true>(v[i][j], lse, rest, total, gh, H);
            if (few && !nothing) {
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] += at * 4u + j - lead == token ? own : 0.f;
#pragma unroll 4
                for (uint32_t k = 0; k < P.top; ++k) {
                    const uint32_t which = (uint32_t)top_token[row * P.top + k] + lead - at * 4u;
                    const float g = g_top[row * P.top + k];
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] += which == (uint32_t)j ? g : 0.f;
                }
            }
            if (at >= q1) continue;
            if (at * 4u >= lead && at * 4u + 4u <= lead + P.V) {
                const u32x4 t = u32x4{f2u(d[0]), f2u(d[1]), f2u(d[2]), f2u(d[3])};
                if (stream) __builtin_amdgcn_raw_buffer_store_b128(t, d_rsrc, (from + at * 4u) * 4u, 0, 2);
                else __builtin_amdgcn_raw_buffer_store_b128(t, d_rsrc, (from + at * 4u) * 4u, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (at * 4u + j - lead < P.V) dx[row * P.V + (at * 4u + j - lead)] = d[j];
            }
        }
    }
    if (few) return;
    __syncthreads();
    if (nothing || !there) return;
    // number k < top: alternative k, number `top`: the given token; in the slice that has its score
    for (uint32_t k = lane; k <= P.top; k += lanes) {
        const uint32_t mine = k < P.top ? (uint32_t)top_token[row * P.top + k] : token, vector = mine + lead >> 2;
        if (mine >= P.V || vector < q0 || vector >= q1) continue;
        const float x = logits[row * P.V + mine];
        float d = g_entropy == nullptr ? grad_of<false>(x, lse, rest, total, gh, H) : grad_of<true>(x, lse, rest, total, gh, H);
        if (mine == token) d += own;
#pragma unroll 8
        for (uint32_t i = 0; i < P.top; ++i) d += (uint32_t)top_token[row * P.top + i] == mine ? g_top[row * P.top + i] : 0.f;
        dx[row * P.V + mine] = d;
    }
}
