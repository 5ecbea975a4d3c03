// beam.hip -- beam search: the best continuations of a request's beams over the
// vocabulary (doe_beam_select), and dense states in the order of their parents
// (doe_beam_reorder_rows; page tables: kv_pages.hip).
//
// A candidate (beam, token) scores s_b + x_t - log sum_t' exp x_t', x the logits times
// the inverse temperature.  Within a row the order is that of the logits, so the first
// kernel reads them once and leaves, for every wave's part of a row, its `select` best
// logits and its share of the sum; the second one forms the rows' logarithms in 64 bits
// and picks among the parts.  Sixteen requests of eight beams, 248321 tokens, the best
// sixteen (127 MB): 27.9 us, 23.5 of them in the first kernel (5.4 TB/s; 18.6 without its
// lists), 6 in the second; four beams of 256000: 8.5, 4.0 and 4.4, chains of cold reads and
// barriers.  Powers and a part's sum of up to 2048 of them are f32 (their rounding is within
// 2^-18 of the logarithm, half a step of an f32 score from 2^6 on); from there on 64 bits.
#include "common.h"
#include "wave.h"

#include <float.h>
#include <math.h>
#include <algorithm>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));  // (rows of an odd vocabulary)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxBeams = 64, kMaxSelect = 64;
constexpr int kWaves = 4;
constexpr int kList = 256;   // a wave's shortlist
constexpr int kPick = 1024;  // threads of the second kernel
constexpr int kPool = 4096;  // its shortlist
constexpr int kMost = 128;   // groups of candidates
constexpr int kAhead = 4;    // entries of a thread's first list that are read at once

struct BeamArgs {
    const float *logits, *scores;
    const int32_t *finished;
    int64_t row_stride;
    int beams, vocab, select, parts, end_token;  // parts of a row: a wave each
    float inv_temperature, factor, factor_low;  // factor + factor_low = inv_temperature log2(e), factor_low above 0
    float per_part;   // 1 / parts
    uint64_t *cand;   // [row][select][part]: logit order, ~token; 0: none
    float2 *stats;    // [row][part]: the largest logit and the sum of their powers over it; 0: none above -infinity
    int32_t *parents, *tokens, *ended;
    float *best;
};

// Order of floats as unsigned numbers (no NaN).
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v);
    return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __uint_as_float(o ^ ((int)o < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float v, int token) {
    return (uint64_t)ordered(v + 0.0f) << 32 | (uint32_t)~token;  // (-0 is 0)
}

// A beam that offers its tokens: it has a score and has not ended.
__device__ __forceinline__ bool offers(const BeamArgs &a, int row) {
    const float s = a.scores[row];
    return s > -INFINITY && s < INFINITY && !(a.finished && a.finished[row]);
}

// exp(inv_temperature d), d at most 0.
__device__ __forceinline__ float power(const BeamArgs &a, float d) {
    return __builtin_amdgcn_exp2f(fmaf(d, a.factor, d * a.factor_low));
}

// What lanes of a wave write to LDS before it, its other lanes read behind it: the
// wave's LDS operations are in order, as long as the compiler leaves them so.
__device__ __forceinline__ void in_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return std::max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0x118, 0xf>(dpp_max<0x114, 0xf>(dpp_max<0x112, 0xf>(dpp_max<0x111, 0xf>(v))));
    return (uint32_t)__builtin_amdgcn_readlane((int)dpp_max<0x143, 0xc>(dpp_max<0x142, 0xa>(v)), 63);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    const uint32_t hi = wave_max((uint32_t)(v >> 32));
    return (uint64_t)hi << 32 | wave_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}
template <int CTRL>
__device__ __forceinline__ int dpp_take(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
// A bound that at least `select` of some values reach and few others, bit by bit: the largest
// key that enough of them reach, until no more than a quarter too many do.  count(key): how
// many; all reach `key`, which is 0 from `bit` on.
template <typename F>
__device__ __forceinline__ float bound_of_many(int select, const F &count, uint32_t key = 0, int bit = 31) {
    for (; bit >= 0; --bit) {
        const uint32_t next = key | 1u << bit;
        const int n = count(next);
        if (n < select) continue;
        key = next;
        if (n <= select + select / 4) break;
    }
    return key > ordered(-INFINITY) ? unordered(key) : -INFINITY;
}
// The same of the lanes' values, for up to kOne of them.  Up to kFew one lane after the other
// is taken, the largest but for six bits of its value, and the least of them is the bound:
// four of a wave 0.5 us less in a call than bit by bit, sixteen 1 us more.
constexpr int kFew = 8, kOne = 16;
__device__ __forceinline__ float bound_of_one(float v, int select) {
    if (select > kFew) {
        const uint32_t key = ordered(fmaxf(v, -INFINITY));
        // (from the first bit on in which they differ)
        const uint32_t most = wave_max(key), differ = most ^ ~wave_max(~key);
        const int bit = 31 - __builtin_clz(differ | 1);
        return bound_of_many(select, [&](uint32_t at) __attribute__((always_inline)) { return (int)__popcll(__ballot(key >= at)); },
                             most & ~((2u << bit) - 1), bit);
    }
    uint32_t key = (ordered(v) & ~63u) | (threadIdx.x & 63);
    bool taken = false;
    for (int c = 0; c < select; ++c) {
        const bool most = key == wave_max(key);
        taken = taken || most;
        key = most ? 0 : key;
    }
    return unordered(~wave_max(taken ? ~ordered(v) : 0u));
}

// Value e of a lane's, found by halves (they are registers).
template <int NV>
__device__ __forceinline__ float value_of(const f4 (&v)[NV], int e) {
    float s[2 * NV];
#pragma unroll
    for (int k = 0; k < 2 * NV; ++k) s[k] = e & 1 ? v[k / 2][k % 2 * 2 + 1] : v[k / 2][k % 2 * 2];
#pragma unroll
    for (int n = NV, bit = 2; n > 0; n /= 2, bit *= 2)
#pragma unroll
        for (int k = 0; k < n; ++k) s[k] = e & bit ? s[2 * k + 1] : s[2 * k];
    return s[0];
}

// A wave's part of a row: NV x 256 logits, four side by side a lane, kept in
// registers.  Those that reach the bound of the lanes' own largest ones go to a list in
// LDS, and their places in the order are counted.
template <int NV>
__global__ __launch_bounds__(64 * kWaves, NV == 8 ? 4 : 8) void beam_parts_kernel(BeamArgs a, int wgs) {
    __shared__ uint64_t lists[kWaves][kList];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int row = blockIdx.x / wgs, part = (blockIdx.x - row * wgs) * kWaves + wave;
    if (part >= a.parts) return;
    // (a beam that offers nothing: its parts are not looked at.  Short parts are a small call's,
    // which reads them all the same rather than wait for the answer)
    const bool wanted = offers(a, row);
    if (NV == 8 && !wanted) return;
    const float *x = a.logits + (int64_t)row * a.row_stride;
    // (parts by place, not by address: equal rows give equal bits)
    const int first = part * (256 * NV), e0 = first + 4 * lane;
    f4 v[NV];
    if (first + 256 * NV <= a.vocab) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            // (many logits past the caches: 30.8 to 30.2 us for 127 MB; few: 9.0 to 9.3)
            const f4_any *at = reinterpret_cast<const f4_any *>(x + e0 + 256 * j);
            if constexpr (NV == 8) v[j] = __builtin_nontemporal_load(at);
            else v[j] = *at;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = e0 + 256 * j;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][i] = e + i < a.vocab ? x[e + i] : -INFINITY;
        }
    }
    if (!wanted) return;
    float most4[NV], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        most4[j] = fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3]));
        most = fmaxf(most, most4[j]);
    }
    const int64_t slot = (int64_t)row * a.parts + part;
    uint64_t *cand = a.cand + (int64_t)row * a.select * a.parts + part;  // (then every parts-th)
    const float top = unordered(wave_max(ordered(most)));
    // an infinity or a NaN leaves a sum that is no number; -infinity adds 0 (factor_low > 0)
    f4 sums = {0.0f, 0.0f, 0.0f, 0.0f};
    if (top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i] += power(a, v[j][i] - top);
    } else {
        // (nothing above -infinity: a NaN all the same?)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i] += v[j][i] == v[j][i] ? 0.0f : v[j][i];
    }
    const float sum = doe::wave_sum((sums[0] + sums[1]) + (sums[2] + sums[3]));
    if (lane == 0) a.stats[slot] = make_float2(top, sum);
    if (!(sum > 0.0f)) {
        if (lane < a.select) cand[(int64_t)lane * a.parts] = 0;
        return;
    }
    float low;
    if (a.select <= kOne) {
        low = bound_of_one(most, a.select);
    } else {
        // (four values a lane: of one, nearly all would have to be taken)
        uint32_t key[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float m = most4[i * NV / 4];
#pragma unroll
            for (int j = i * NV / 4 + 1; j < (i + 1) * NV / 4; ++j) m = fmaxf(m, most4[j]);
            key[i] = ordered(fmaxf(m, -INFINITY));
        }
        low = bound_of_many(a.select, [&](uint32_t at) __attribute__((always_inline)) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) n += __popcll(__ballot(key[i] >= at));
            return n;
        });
    }
    // those that reach it: a bit each, and their places by a sum over the lanes (a ballot for every
    // value: 30.2 to 27.9 us for 127 MB)
    uint64_t *list = lists[wave];
    const float least = fmaxf(low, -FLT_MAX);
    uint32_t hits = 0;
#pragma unroll
    for (int e = 4 * NV - 1; e >= 0; --e) hits = 2 * hits + (v[e / 4][e % 4] >= least ? 1 : 0);
    const int upto = doe::wave_scan(__popc(hits)), count = __builtin_amdgcn_readlane(upto, 63);
    if (count <= kList) {
        int to = upto - __popc(hits);
        while (__any(hits)) {
            if (hits) {
                const int e = __builtin_ctz(hits);
                list[to++] = key_of(value_of(v, e), e0 + 256 * (e >> 2) + (e & 3));
                hits &= hits - 1;
            }
        }
        in_order();
        for (int t = lane; t < count; t += 64) {
            const uint64_t key = list[t];
            int before = 0;
#pragma unroll 4
            for (int j = 0; j < count; ++j) before += list[j] > key ? 1 : 0;
            if (before < a.select) cand[(int64_t)before * a.parts] = key;
        }
        if (lane >= count && lane < a.select) cand[(int64_t)lane * a.parts] = 0;
        return;
    }
    // (rarely: the large ones in few lanes, or as many equal ones) one after the other
    uint64_t last = ~0ull;
    for (int c = 0; c < a.select; ++c) {
        uint64_t next = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t key = v[j][i] > -INFINITY ? key_of(v[j][i], e0 + 256 * j + i) : 0;
                if (key < last && key > next) next = key;
            }
        last = wave_max(next);
        if (lane == 0) cand[(int64_t)c * a.parts] = last;
    }
}

// ln x of a positive number, to 1e-14: x = 2^e m, ln m = 2 (u + u^3 / 3 + ..), u = (m - 1) /
// (m + 1) within 0.172.
__device__ __forceinline__ double logarithm(double x) {
    int e = __builtin_amdgcn_frexp_exp(x);
    double m = __builtin_amdgcn_frexp_mant(x);  // [0.5, 1)
    if (m < 0.70710678118654752) {
        m *= 2.0;
        --e;
    }
    const double u = (m - 1.0) / (m + 1.0), w = u * u;
    double p = 1.0 / 15.0;
    p = fma(p, w, 1.0 / 13.0);
    p = fma(p, w, 1.0 / 11.0);
    p = fma(p, w, 1.0 / 9.0);
    p = fma(p, w, 1.0 / 7.0);
    p = fma(p, w, 1.0 / 5.0);
    p = fma(p, w, 1.0 / 3.0);
    return fma((double)e, 0.69314718055994531, 2.0 * fma(u * w, p, u));
}

// A request's pick: the rows' logarithms, a bound of the lists' best, the candidates that
// reach it, and their places in the order.  Entries of a place lie side by side for a beam's
// parts and are read before it is known which are wanted: sixteen requests of eight 6 us, 10
// with a list's entries side by side, read in turn, and a bound from the waves' own.  A list
// that goes on is read by a wave: eight requests of 32 beams of 32000, the best 64, of which
// few lists hold most, 10.7 us, 42 by the thread that found it.
__global__ __launch_bounds__(kPick) void beam_pick_kernel(BeamArgs a) {
    __shared__ double base[kMaxBeams], ended_at[kMaxBeams], pool[kPool];
    __shared__ uint64_t pool_at[kPool];  // a candidate's place, see `place`
    __shared__ uint64_t ahead[kAhead][kPick];
    __shared__ float bound_;
    __shared__ __align__(16) uint32_t most[kMost];  // of a group, as a number in their order; 0: none
    __shared__ int deep[kPick];  // lists that go on
    __shared__ int count_, deep_, sums[2][kPick / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int request = blockIdx.x, row0 = request * a.beams, C = a.select, lists = a.beams * a.parts;
    const uint64_t *cand = a.cand + (int64_t)row0 * a.parts * C;
    const double factor = a.inv_temperature;
    // (l + 1/2 is 2^-15 of an integer's place off it, the product within 2^-16)
    auto beam_of = [&](int l) __attribute__((always_inline)) { return (int)(((float)l + 0.5f) * a.per_part); };
    auto entry = [&](int l, int c) __attribute__((always_inline)) {
        const int b = beam_of(l);
        return cand[(uint32_t)((b * C + c) * a.parts + (l - b * a.parts))];
    };
    // this thread's first list, as far as it is likely to go (a beam without an offer leaves
    // its lists as they were: not used below)
    uint64_t own_list[kAhead];
#pragma unroll
    for (int c = 0; c < kAhead; ++c) own_list[c] = entry(std::min(tid, lists - 1), std::min(c, C - 1));
    if (tid == 0) count_ = deep_ = 0;
    if (tid < kMost) most[tid] = 0;
    for (int b = wave; b < a.beams; b += kPick / 64) {
        const float2 *stats = a.stats + (int64_t)(row0 + b) * a.parts;
        const float score = a.scores[row0 + b];
        const int ended = (a.finished ? a.finished : reinterpret_cast<const int32_t *>(a.scores))[row0 + b];
        float2 first[kAhead];  // (read whether they are used or not, so that one does not wait for another)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) first[i] = stats[std::min(lane + 64 * i, a.parts - 1)];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (lane + 64 * i >= a.parts) first[i] = make_float2(-INFINITY, 0.0f);
        const bool ok = score > -INFINITY && score < INFINITY, done = a.finished && ended;
        double start = -INFINITY;
        if (ok && !done) {
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) most = fmaxf(most, first[i].x);
            for (int p = lane + 64 * kAhead; p < a.parts; p += 64) most = fmaxf(most, stats[p].x);
            const float top = unordered(wave_max(ordered(most)));
            // (of none above -infinity a NaN, and a NaN stays one)
            double all = 0.0;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) all = fma((double)first[i].y, (double)power(a, first[i].x - top), all);
            for (int p = lane + 64 * kAhead; p < a.parts; p += 64) {
                const float2 s = stats[p];
                all = fma((double)s.y, (double)power(a, s.x - top), all);
            }
            all = doe::wave_sum(all);
            if (all > 0.0 && all < INFINITY) start = (double)score - ((double)top * factor + logarithm(all));
        }
        if (lane == 0) {
            base[b] = start;
            ended_at[b] = ok && done ? (double)score : -INFINITY;
        }
    }
#pragma unroll
    for (int c = 0; c < kAhead; ++c) ahead[c][tid] = own_list[c];
    __syncthreads();
    auto score_of = [&](uint64_t key, int b) {
        return key && base[b] > -INFINITY ? base[b] + factor * (double)unordered((uint32_t)(key >> 32)) : -INFINITY;
    };
    // of equal scores the lower place comes first: beam, then logit from the largest
    // (scores of a beam may be too near each other for 64 bits), then token
    auto place = [](int b, uint64_t key) { return (uint64_t)b << 56 | (uint64_t)~(uint32_t)(key >> 32) << 24 | ~(uint32_t)key; };
    auto end_place = [&](int b) { return (uint64_t)b << 56 | (uint32_t)a.end_token; };
    constexpr uint64_t kNone = ~0ull;
    auto head_of = [&](int l) { return l == tid ? ahead[0][tid] : entry(l, 0); };
    // the float at or below a score: a bound of these is below `select` of the scores
    auto below = [](double score) {
        const float f = (float)score;
        return (double)f > score ? unordered(ordered(f) - 1) : f;
    };
    int turn = 0;
    auto block_sum = [&](int n) __attribute__((always_inline)) {  // of the waves' numbers
        turn ^= 1;
        if (lane == 0) sums[turn][wave] = n;
        __syncthreads();
        n = sums[turn][lane & (kPick / 64 - 1)];
#pragma unroll
        for (int d = 1; d < kPick / 64; d <<= 1) n += __shfl_xor(n, d, 64);
        return __builtin_amdgcn_readfirstlane(n);
    };
    auto push = [&](double score, uint64_t at) {
        const int to = atomicAdd(&count_, 1);
        if (to < kPool) {
            pool[to] = score;
            pool_at[to] = at;
        }
    };
    const bool few = lists <= kPick / 4;
    // the candidates that reach a bound into the pool; how many
    auto gather = [&](double bound) {
        auto offer = [&](uint64_t key, int b) {
            const double s = score_of(key, b);
            const bool in = s > -INFINITY && s >= bound;
            if (in) push(s, place(b, key));
            return in;
        };
        if (few) {  // a thread an entry, not a list
            for (int i = tid; i < lists * C; i += kPick) offer(cand[i], i / (C * a.parts));
        }
        for (int l = few ? lists : tid; l < lists; l += kPick) {
            const int b = beam_of(l), known = l == tid ? std::min(C, kAhead) : 0;
            const double head = known ? 0.0 : score_of(entry(l, 0), b);
            bool more = known || (head > -INFINITY && head >= bound);
#pragma unroll 1
            for (int c = 0; more && c < known; ++c) more = offer(ahead[c][tid], b);
            if (!more || known == C) continue;
            const int to = atomicAdd(&deep_, 1);
            if (to < kPick) deep[to] = l;
            else for (int c = known; more && c < C; ++c) more = offer(entry(l, c), b);
        }
        if (!few && (C > kAhead || lists > kPick)) {
            // the rest of such a list at once, by a wave
            __syncthreads();
            for (int q = wave; q < std::min(deep_, kPick); q += kPick / 64) {
                const int l = deep[q], c = lane + (l < kPick ? kAhead : 0);
                if (c < C) offer(entry(l, c), beam_of(l));
            }
        }
        if (tid < a.beams && ended_at[tid] > -INFINITY && ended_at[tid] >= bound) push(ended_at[tid], end_place(tid));
        __syncthreads();
        return count_;
    };
    auto emptied = [&] {
        __syncthreads();
        if (tid == 0) count_ = deep_ = 0;
        if (tid < kMost) most[tid] = 0;
        __syncthreads();
    };
    constexpr int kEnough = 4 * kMaxSelect;  // whose order is counted
    // A bound: of 64 groups of candidates (128 if nearly all of 64 were to be taken) the
    // `select`-th best by themselves, equal ones in the groups' order.  `most` has been
    // cleared; give(offer): the candidates, by a number that finds their group.
    const int bits = C > 48 ? 7 : 6, sharers = kPick >> bits;
    auto group_bound = [&](const auto &give) __attribute__((always_inline)) {
        give([&](int i, double score) __attribute__((always_inline)) {
            if (score > -INFINITY) atomicMax(&most[(uint32_t)i * 0x9e3779b1u >> (32 - bits)], ordered(below(score)));
        });
        __syncthreads();
        // (sixteen or eight threads a group)
        const int group = tid / sharers, mine = tid & (sharers - 1);
        const uint32_t m = most[group];
        int before = 0;
        for (int i = 4 * mine; i < 1 << bits; i += 4 * sharers) {
            const u32x4 other = *reinterpret_cast<const u32x4 *>(most + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) before += other[e] > m || (other[e] == m && i + e < group) ? 1 : 0;
        }
        before += dpp_take<0xB1>(before);  // the neighbour, the other pair, the other four, the other eight
        before += dpp_take<0x4E>(before);
        before += dpp_take<0x141>(before);
        if (sharers == 16) before += dpp_take<0x140>(before);
        if (mine == 0 && before == C - 1) bound_ = m ? unordered(m) : -INFINITY;
        __syncthreads();
        return bound_;
    };
    const float bound = group_bound([&](const auto &offer) __attribute__((always_inline)) {
        if (few) {
            for (int i = tid; i < lists * C; i += kPick) offer(i, score_of(cand[i], i / (C * a.parts)));
            return;
        }
        for (int l = tid; l < lists; l += kPick) offer(l, score_of(head_of(l), beam_of(l)));
        // (few lists may hold most of many)
        if (C > kOne && tid < lists) {
#pragma unroll 1
            for (int c = 1; c < kAhead; ++c) offer(c * kPick + tid, score_of(ahead[c][tid], beam_of(tid)));
        }
    });
    int count = gather(bound);
    if (count > kPool) {
        // the lists' best by themselves: no more than `select` lists reach their bound, but for ties
        constexpr int kHeads = 8;
        uint32_t key[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int l = tid + i * kPick;
            key[i] = l < lists ? ordered(below(score_of(head_of(l), beam_of(l)))) : 0;
        }
        const float own = lists < C ? -INFINITY : bound_of_many(C, [&](uint32_t at) __attribute__((always_inline)) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < kHeads; ++i) n += __popcll(__ballot(key[i] >= at));
            for (int l = wave * 64 + lane + kHeads * kPick; l - lane < lists; l += kPick)
                n += __popcll(__ballot(l < lists && ordered(below(score_of(head_of(l), beam_of(l)))) >= at));
            return block_sum(n);
        });
        emptied();
        count = gather(own);
    }
    if (count > kEnough && count <= kPool) {
        constexpr int kEach = kPool / kPick;
        double s[kEach];
        uint64_t at[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const bool in = tid + i * kPick < count;
            s[i] = in ? pool[tid + i * kPick] : -INFINITY;
            at[i] = in ? pool_at[tid + i * kPick] : kNone;
        }
        emptied();
        const float own = group_bound([&](const auto &offer) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) offer(tid + i * kPick, s[i]);
        });
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (s[i] > -INFINITY && s[i] >= own) push(s[i], at[i]);
        __syncthreads();
        count = count_;
    }
    auto put = [&](int c, double score, uint64_t at) {
        const int64_t to = (int64_t)request * C + c;
        const bool none = at == kNone;
        const int b = none ? 0 : (int)(at >> 56), token = none ? -1 : (int)(at & 0xffffff);
        a.parents[to] = none ? -1 : row0 + b;
        a.tokens[to] = token;
        a.best[to] = none ? -INFINITY : (float)std::max<double>(score, -FLT_MAX);  // (masked by the lowest logit, at 1 / T above 1)
        if (a.ended) a.ended[to] = !none && (ended_at[b] > -INFINITY || token == a.end_token) ? 1 : 0;  // (it may be a.finished)
    };
    if (count <= kPool) {
        // sixteen threads a candidate
        for (int t = tid >> 4; t < count; t += kPick / 16) {
            const double s = pool[t];
            const uint64_t at = pool_at[t];
            int before = 0;
            for (int j = tid & 15; j < count; j += 16) before += pool[j] > s || (pool[j] == s && pool_at[j] < at) ? 1 : 0;
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) before += __shfl_xor(before, d, 64);
            if ((tid & 15) == 0 && before < C) put(before, s, at);
        }
        if (tid >= count && tid < C) put(tid, -INFINITY, kNone);
        return;
    }
    // (rarely: few full lists among many) one after the other
    double last = INFINITY;
    uint64_t last_at = 0;
    for (int c = 0; c < C; ++c) {
        double s = -INFINITY;
        uint64_t at = kNone;
        auto take = [&](double score, uint64_t where) {
            const bool behind = score < last || (score == last && where > last_at);
            if (score > -INFINITY && behind && (score > s || (score == s && where < at))) {
                s = score;
                at = where;
            }
        };
        for (int l = tid; l < lists; l += kPick)
            for (int e = 0; e < C; ++e) {
                const uint64_t key = entry(l, e);
                const double score = score_of(key, beam_of(l));
                if (score == -INFINITY) break;
                take(score, place(beam_of(l), key));
            }
        if (tid < a.beams) take(ended_at[tid], end_place(tid));
        __syncthreads();  // the last round's places have been read
        pool[tid] = s;
        pool_at[tid] = at;
        __syncthreads();
        for (int d = kPick / 2; d > 0; d >>= 1) {
            if (tid < d) {
                const double o = pool[tid + d];
                const uint64_t o_at = pool_at[tid + d];
                if (o > pool[tid] || (o == pool[tid] && o_at < pool_at[tid])) {
                    pool[tid] = o;
                    pool_at[tid] = o_at;
                }
            }
            __syncthreads();
        }
        last = pool[0];
        last_at = pool_at[0];
        if (tid == 0) put(c, last, last_at);
    }
}

// Row i of dst = row parents[i] of src in every layer, in pieces of 16 KB.
template <typename T>
__global__ __launch_bounds__(256) void beam_rows_kernel(const uint8_t *src, uint8_t *dst, const int32_t *parents, int64_t src_rows,
                                                        int64_t rows, int64_t row_bytes, int64_t layers, int64_t src_layer,
                                                        int64_t dst_layer) {
    constexpr int PIECE = 256 * 4 * (int)sizeof(T);
    const int64_t pieces = (row_bytes + PIECE - 1) / PIECE, all = rows * layers * pieces;
    for (int64_t w = blockIdx.x; w < all; w += gridDim.x) {
        const int64_t piece = w % pieces, rest = w / pieces, layer = rest / rows, i = rest - layer * rows;
        const int64_t parent = parents[i];
        if (parent < 0 || parent >= src_rows) continue;
        const int64_t at = piece * PIECE + threadIdx.x * (int)sizeof(T);
        const uint8_t *s = src + layer * src_layer + parent * row_bytes + at;
        uint8_t *d = dst + layer * dst_layer + i * row_bytes + at;
        T v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j * (PIECE / 4) < row_bytes) v[j] = *reinterpret_cast<const T *>(s + j * (PIECE / 4));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j * (PIECE / 4) < row_bytes) *reinterpret_cast<T *>(d + j * (PIECE / 4)) = v[j];
    }
}

// Vectors a lane: longer parts where there are rows enough to fill the device (128 rows of
// 248321: 45 us in parts of 1024, 37.5 of 2048, 37.6 of 4096, which spill registers), and
// sooner where a part's list is what costs (256 rows of 32000, the best 64: 35.4 and 25.9 us;
// 80 of 60000, 40: 19.2 and 18.4; 84 of 17880, 21: 13.4 and 15.5).
int vectors_of(int64_t rows, int64_t vocab, int64_t select) {
    return rows * vocab >= (int64_t)(select > kOne ? 2 : 8) << 20 ? 8 : 4;
}

struct BeamSizes {
    int vectors;
    int64_t parts, cand, bytes;
};
int beam_sizes(int64_t batch, int64_t beams, int64_t vocab, int64_t select, BeamSizes &z) {
    DOE_REQUIRE(beams > 0 && beams <= kMaxBeams, DOE_E_UNSUPPORTED, "beams %lld outside 1..%d", (long long)beams, kMaxBeams);
    DOE_REQUIRE(select > 0 && select <= kMaxSelect, DOE_E_UNSUPPORTED, "select %lld outside 1..%d", (long long)select, kMaxSelect);
    DOE_REQUIRE(vocab > 0 && vocab <= ((int64_t)1 << 24), DOE_E_UNSUPPORTED, "vocab %lld outside 1..2^24", (long long)vocab);
    DOE_REQUIRE(batch >= 0 && batch <= 65535, DOE_E_INVALID, "batch %lld outside 0..65535", (long long)batch);
    const int64_t rows = batch * beams;
    z.vectors = vectors_of(rows, vocab, select);
    z.parts = (vocab + 256 * z.vectors - 1) / (256 * z.vectors);
    z.cand = rows * z.parts * select * 8;
    z.bytes = std::max<int64_t>(16, z.cand + rows * z.parts * 8);
    return DOE_OK;
}

}  // namespace

extern "C" {

int doe_beam_select_workspace(int64_t batch, int64_t beams, int64_t vocab, int64_t select, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    BeamSizes z;
    const int rc = beam_sizes(batch, beams, vocab, select, z);
    if (rc) return rc;
    *bytes = z.bytes;
    return DOE_OK;
}

int doe_beam_select(const float *logits, int64_t row_stride, const float *scores, const int32_t *finished, int64_t batch,
                    int64_t beams, int64_t vocab, int64_t select, float inv_temperature, int64_t end_token, int32_t *parents,
                    int32_t *tokens, float *out_scores, int32_t *out_finished, void *workspace, int64_t workspace_bytes,
                    doe_stream_t stream) {
    BeamSizes z;
    int rc = beam_sizes(batch, beams, vocab, select, z);
    if (rc) return rc;
    DOE_REQUIRE(row_stride >= vocab, DOE_E_INVALID, "row stride %lld below vocab %lld", (long long)row_stride, (long long)vocab);
    // (factor_low, 2^-53 of it at the least, is above 0)
    DOE_REQUIRE(inv_temperature >= 0x1p-64f && isfinite(inv_temperature * 1.4426950408889634f), DOE_E_INVALID, "inv_temperature %g",
                (double)inv_temperature);
    DOE_REQUIRE(end_token < vocab && (end_token >= 0 || !finished), DOE_E_INVALID, "end_token %lld of %lld tokens%s", (long long)end_token,
                (long long)vocab, finished ? ", with finished beams" : "");
    DOE_REQUIRE(batch == 0 || (logits && scores && parents && tokens && out_scores), DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)logits & 3) == 0, DOE_E_INVALID, "logits must be 4-byte aligned");
    const int64_t in_bytes = 4 * batch * beams, out_bytes = 4 * batch * select;
    auto apart = [](const void *p, int64_t p_bytes, const void *q, int64_t q_bytes) {
        return !p || !q || (uintptr_t)p + (uintptr_t)p_bytes <= (uintptr_t)q || (uintptr_t)q + (uintptr_t)q_bytes <= (uintptr_t)p;
    };
    // in place only request by request, scores over scores and flags over flags
    const void *const outs[4] = {parents, tokens, out_scores, out_finished};
    for (int o = 0; o < 4; ++o)
        DOE_REQUIRE((apart(scores, in_bytes, outs[o], out_bytes) || (o == 2 && out_scores == scores && select == beams)) &&
                        (apart(finished, in_bytes, outs[o], out_bytes) || (o == 3 && out_finished == finished && select == beams)),
                    DOE_E_INVALID, "the outputs overlap scores or finished");
    DOE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= z.bytes, DOE_E_INVALID,
                "a 16-byte aligned workspace of %lld bytes is needed (got %lld)", (long long)z.bytes, (long long)workspace_bytes);
    for (int o = 1; o < 4; ++o)
        for (int p = 0; p < o; ++p)
            DOE_REQUIRE(apart(outs[p], out_bytes, outs[o], out_bytes), DOE_E_INVALID, "the outputs overlap each other");
    const int64_t rows = batch * beams, wgs = (z.parts + kWaves - 1) / kWaves;
    DOE_REQUIRE(rows * wgs < ((int64_t)1 << 24), DOE_E_UNSUPPORTED, "%lld rows of %lld logits", (long long)rows, (long long)vocab);
    if ((rc = doe::require_init())) return rc;
    if (batch == 0) return DOE_OK;
    BeamArgs a{};
    a.logits = logits;
    a.scores = scores;
    a.finished = finished;
    a.row_stride = row_stride;
    a.beams = (int)beams;
    a.vocab = (int)vocab;
    a.select = (int)select;
    a.parts = (int)z.parts;
    a.end_token = end_token < 0 ? -2 : (int)end_token;  // (-2: no token is)
    a.inv_temperature = inv_temperature;
    const double factor = inv_temperature * 1.4426950408889634074;
    a.factor = (float)factor;
    if ((double)a.factor >= factor) a.factor = nextafterf(a.factor, 0.0f);
    a.factor_low = (float)(factor - (double)a.factor);
    a.per_part = 1.0f / (float)z.parts;
    a.cand = static_cast<uint64_t *>(workspace);
    a.stats = reinterpret_cast<float2 *>(static_cast<uint8_t *>(workspace) + z.cand);
    a.parents = parents;
    a.tokens = tokens;
    a.best = out_scores;
    a.ended = out_finished;
    const hipStream_t st = (hipStream_t)stream;
    if (z.vectors == 8) hipLaunchKernelGGL(beam_parts_kernel<8>, dim3((unsigned)(rows * wgs)), dim3(64 * kWaves), 0, st, a, (int)wgs);
    else hipLaunchKernelGGL(beam_parts_kernel<4>, dim3((unsigned)(rows * wgs)), dim3(64 * kWaves), 0, st, a, (int)wgs);
    DOE_LAUNCH_CHECK("beam_parts_kernel");
    hipLaunchKernelGGL(beam_pick_kernel, dim3((unsigned)batch), dim3(kPick), 0, st, a);
    DOE_LAUNCH_CHECK("beam_pick_kernel");
    return DOE_OK;
}

int doe_beam_reorder_rows(const void *src, void *dst, const int32_t *parents, int64_t src_rows, int64_t rows, int64_t row_bytes,
                          int64_t layers, int64_t src_layer_stride, int64_t dst_layer_stride, doe_stream_t stream) {
    DOE_REQUIRE(src_rows >= 0 && src_rows < ((int64_t)1 << 31) && rows >= 0 && rows < ((int64_t)1 << 31) && layers >= 0 && layers <= 65535,
                DOE_E_INVALID, "%lld rows of %lld in %lld layers", (long long)rows, (long long)src_rows, (long long)layers);
    DOE_REQUIRE(row_bytes > 0 && row_bytes % 4 == 0 && row_bytes < ((int64_t)1 << 40), DOE_E_INVALID,
                "row_bytes %lld is not a positive multiple of 4", (long long)row_bytes);
    DOE_REQUIRE(std::max(src_rows, rows) <= ((int64_t)1 << 46) / row_bytes, DOE_E_INVALID, "%lld rows of %lld bytes",
                (long long)std::max(src_rows, rows), (long long)row_bytes);
    DOE_REQUIRE(layers <= 1 || (src_layer_stride >= src_rows * row_bytes && dst_layer_stride >= rows * row_bytes), DOE_E_INVALID,
                "layer strides %lld and %lld below the rows' bytes", (long long)src_layer_stride, (long long)dst_layer_stride);
    DOE_REQUIRE(layers <= 1 || (src_layer_stride % 4 == 0 && dst_layer_stride % 4 == 0 && src_layer_stride < ((int64_t)1 << 46) &&
                                dst_layer_stride < ((int64_t)1 << 46)),
                DOE_E_INVALID, "layer strides %lld and %lld", (long long)src_layer_stride, (long long)dst_layer_stride);
    const bool none = rows == 0 || layers == 0 || src_rows == 0;
    DOE_REQUIRE(none || (src && dst && parents), DOE_E_INVALID, "null pointer");
    DOE_REQUIRE((((uintptr_t)src | (uintptr_t)dst) & 3) == 0, DOE_E_INVALID, "src and dst must be 4-byte aligned");
    const int64_t src_bytes = (layers - 1) * src_layer_stride + src_rows * row_bytes, dst_bytes = (layers - 1) * dst_layer_stride + rows * row_bytes;
    DOE_REQUIRE(none || (uintptr_t)src + (uintptr_t)src_bytes <= (uintptr_t)dst || (uintptr_t)dst + (uintptr_t)dst_bytes <= (uintptr_t)src,
                DOE_E_INVALID, "src and dst overlap");
    const int rc = doe::require_init();
    if (rc) return rc;
    if (none) return DOE_OK;
    const bool wide = row_bytes % 16 == 0 && (((uintptr_t)src | (uintptr_t)dst) & 15) == 0 &&
                      (layers == 1 || (src_layer_stride % 16 == 0 && dst_layer_stride % 16 == 0));
    const int64_t piece = 256 * 4 * (wide ? 16 : 4), pieces = (row_bytes + piece - 1) / piece;
    const int64_t most = (int64_t)1 << 14;
    const unsigned wgs = (unsigned)(rows > most / layers / pieces ? most : rows * layers * pieces);
    if (wide)
        hipLaunchKernelGGL(beam_rows_kernel<u32x4>, dim3(wgs), dim3(256), 0, (hipStream_t)stream, static_cast<const uint8_t *>(src),
                           static_cast<uint8_t *>(dst), parents, src_rows, rows, row_bytes, layers, src_layer_stride, dst_layer_stride);
    else
        hipLaunchKernelGGL(beam_rows_kernel<uint32_t>, dim3(wgs), dim3(256), 0, (hipStream_t)stream, static_cast<const uint8_t *>(src),
                           static_cast<uint8_t *>(dst), parents, src_rows, rows, row_bytes, layers, src_layer_stride, dst_layer_stride);
    DOE_LAUNCH_CHECK("beam_rows_kernel");
    return DOE_OK;
}

}  // extern "C"
