// attn_mx4_prompt.hip -- causal GQA attention of prompt rows over the paged KV
// cache held in 4 bits (doe_attn_mx4_prompt).
//
// o = softmax(cap(q . k_p scale)) v over the positions p that a row sees: p <=
// pos, with a window p > pos - window; row i of a sequence's n is at position
// kv_len - n + i.  The query heads of a KV head share its K and V: a tile is 32 or
// 128 (row, head) pairs of one KV head, a wave 32 of them, a lane column one.
//   * S^T = K Q^T on v_mfma_f32_32x32x16_f16: K's codes go to f16 with their scales in
//     four conversions an operand, exactly.  f16 queries are operands as they stand,
//     f32 ones in hi and lo parts of one power of two for the row: 22 bits of each
//     dim, whatever the others are (down to 2^-38 of the largest).  The matrix cores'
//     own 4-bit operands against digits of Q in 6 bits (25 bits of the largest of 32
//     dims) took up to 12 % less, but lost dims far below the largest where the keys are
//     zero at the large ones: 1e-3 of the output at 2^15.
//   * S^T's sums are P^T's operand order of O^T = V^T P^T, on the same instruction:
//     P as f16 hi + lo whatever the output's type (one f16 of P would cost an f16
//     output as much again as its own rounding, 2e-4).
//   * V goes to f16 with its scales (v_cvt_scalef32_pk_f16_fp4) once for the waves
//     that share it, into LDS in operand order: the page layout holds the eight
//     positions of a lane half together, so a lane writes and reads 16-byte pieces.
//   * The running max is raised only when a score exceeds it by 2^8; P lies 2^7
//     above it, so that f16's small values lose no more than 2^-32 of the largest.
// A block's steps overlap with its neighbours': its weights stand beside the next
// one's scores, its P V beside the next V's way into LDS, so that the matrix and
// vector units of a SIMD work at once with one or two waves on it.  2048 rows after
// 8192 positions, 32 / 8 heads of 128 dims, f16: 440 us, 704 TFLOP/s of the 4 D
// operations a pair and position, where a large f16 matrix product reaches 1139; P's two
// parts make three products of two.  Its matrix units are busy 47 % of the cycles and
// vector instructions issue in 50: the two waves of a SIMD seldom do both at once.  32 /
// 16 heads of 160 (1500 rows after 2000 of 8 sequences, f32): 31 and 34 % with the one wave
// a SIMD that its registers allow, 796 us, 360 TFLOP/s; 8 / 1 of 512, whose waves add up
// their parts of every score through LDS: 28 and 39 %, 667 us, 344.  1000 rows at 8 / 4
// heads of 256 dims, f32: 28 us, of which 8 are a prologue (row, page table and query read
// one after the other) and most of the rest the last tiles' eight blocks a wave, where the
// mean is 4.3.
#include "mx4_cache.h"

#include <math.h>
#include <algorithm>
#include <type_traits>

namespace {

using doe::Mx4Factor;
using doe::Mx4Slab;
using doe::Mx4View;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kBias = 7.0f, kLazy = 8.0f;  // log2: P of the running max, and how far that may lag
constexpr int kWaves = 4;
// Workgroups that a CU holds, by their registers (at 512 by LDS as well).  64: three
// cost eight spilled registers at most and win (12 ragged prompts of up to 777 rows, a window,
// capped scores: 49.6 to 41.3 us); 512: 1500 rows after 2000 of 8 sequences at 8 / 1 heads
// 648 us for 1050 with one.
constexpr int per_cu(int head_dim) { return head_dim == 64 ? 3 : (head_dim == 128 || head_dim == 512 ? 2 : 1); }

struct PromptArgs {
    Mx4View c;
    const void *q;
    void *out;
    const int32_t *row_starts;
    int64_t q_stride, out_stride;
    int q_f16, out_f16, rows, num_heads, group, window, splits, tiles;
    float scale, softcap;
    float *part;  // [split][row][head][D], then [split][row][head][2]
};

// TEAM waves share a block's V (4: a tile of 128 pairs, 1: of 32, the waves taking
// every fourth block); head_dim 512: each wave holds a quarter of the dims of one
// tile of 32, and the waves add up their parts of a score.
template <int D, int TEAM>
struct Shape {
    static constexpr int kSlices = D == 512 ? 4 : 1, kDims = D / kSlices;  // of a wave
    static constexpr int kRows = D == 512 ? 32 : 32 * TEAM;                // pairs of a tile
    static constexpr int kBlocks = TEAM;                                   // blocks of a step
    static constexpr int kSteps = (kDims + 63) / 64, kTiles = kDims / 32, kOps = kDims / 16;
    static constexpr int kV = 32 * kDims * 2;                              // bytes of a block's V
    static constexpr int kBuffers = 8;                                     // two steps of four, or two blocks a wave
    static constexpr int kMerge = TEAM == 4 || D == 512 ? 0 : kWaves * 32 * D * 4;  // the waves' O at the end
    static constexpr int kScores = D == 512 ? kWaves * 32 * 32 * 4 : 0;
    static constexpr int kData = kBuffers * kV > kMerge ? kBuffers * kV : kMerge;
    static constexpr int kLds = kData + kScores + (D == 512 ? 0 : 1024);  // (512: half a CU's, to the byte)
};

// A lane's dims of a row, of K and of the queries alike: operand o has eight, of the
// 32 of group 2 (o / 4) + half (half: lane / 32); of a last group without a second
// (head_dim 160) each half has 16.
template <int D, int TEAM>
__device__ __forceinline__ constexpr int dims_of(int o, int half) {
    constexpr int PAIRED = Shape<D, TEAM>::kDims / 64 * 4;
    return o < PAIRED ? 64 * (o / 4) + 32 * half + 8 * (o % 4) : 16 * PAIRED + 16 * half + 8 * (o - PAIRED);
}

// A lane's K of a block: position lane % 32, the codes of an operand a word, and the
// scale bytes (operands 4 s .. 4 s + 3 in byte 2 (s % 2) of word s / 2).
template <int D, int TEAM>
struct KBlock {
    uint32_t k[Shape<D, TEAM>::kOps], s[(Shape<D, TEAM>::kSteps + 1) / 2];
};
template <int D, int TEAM>
__device__ __forceinline__ void load_k(KBlock<D, TEAM> &b, const uint8_t *slab, int shift, int x, int lane, int slice) {
    using S = Mx4Slab<D>;
    using P = Shape<D, TEAM>;
    const int m = lane & 31, lh = lane >> 5;
    const uint8_t *k = slab + (uint32_t)(S::k_code(x) + slice * (P::kDims / 2));
    const uint32_t at_k = m * (D / 2) + lh * 16, at_s = m * (D / 32);
    const uint8_t *s = slab + (uint32_t)(S::k_scale(shift, x) + slice * (P::kDims / 32));
#pragma unroll
    for (int o = 0; o + 4 <= P::kOps; o += 4) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(k + (uint32_t)(at_k + 8 * o));
        b.k[o] = w[0], b.k[o + 1] = w[1], b.k[o + 2] = w[2], b.k[o + 3] = w[3];
    }
    if constexpr (P::kOps % 4 != 0) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(k + (uint32_t)(at_k - lh * 8 + 8 * (P::kOps - 2)));
        b.k[P::kOps - 2] = w[0], b.k[P::kOps - 1] = w[1];
    }
    if constexpr (D == 64) {
        b.s[0] = *reinterpret_cast<const uint16_t *>(s + at_s) >> (8 * lh);
    } else if constexpr (D == 160) {
        b.s[0] = s[at_s + lh] | (uint32_t)s[at_s + 2 + lh] << 16;
        b.s[1] = s[at_s + 4];
    } else {
#pragma unroll
        for (int i = 0; i < P::kSteps / 2; ++i) b.s[i] = *reinterpret_cast<const uint32_t *>(s + (uint32_t)(at_s + 4 * i)) >> (8 * lh);
    }
}

// A lane's V of a block: quarter lane / 16 of the positions (eight), column
// lane % 16, with the scales of the one or two groups that its dims lie in.
template <int D, int TEAM>
struct VBlock {
    static constexpr int kBytes = Shape<D, TEAM>::kDims / 32;  // of a position
    uint32_t v[2 * kBytes], s[D == 160 ? 4 : 2];
};
template <int D, int TEAM>
__device__ __forceinline__ void load_v(VBlock<D, TEAM> &b, const uint8_t *slab, int shift, int x, int lane, int slice) {
    using S = Mx4Slab<D>;
    constexpr int N = VBlock<D, TEAM>::kBytes;
    const int c = lane & 15, g = lane >> 4;
    const uint8_t *v = slab + S::v_code(shift, x, 0) + lane * (D / 4) + slice * N;
    if constexpr (D == 512) {
#pragma unroll
        for (int j = 0; j < 8; ++j) b.v[j] = *reinterpret_cast<const uint32_t *>(v + j * (D / 32));
    } else {
#pragma unroll
        for (int i = 0; i < 2 * N; i += 2) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(v + 4 * i);
            b.v[i] = w[0], b.v[i + 1] = w[1];
        }
    }
    const int group = c * (D / 16) / 32;
    const uint8_t *s = slab + S::v_scale(shift, x, 0) + (g * (D / 32) + group) * 8;
    const u32x2 w = *reinterpret_cast<const u32x2 *>(s);
    b.s[0] = w[0], b.s[1] = w[1];
    if constexpr (D == 160) {
        const u32x2 u = *reinterpret_cast<const u32x2 *>(s + (group < 4 ? 8 : 0));
        b.s[2] = u[0], b.s[3] = u[1];
    }
}

// Whether one of the word's bytes is 255.
__device__ __forceinline__ bool any_nan_scale(uint32_t w) { return ((~w - 0x01010101u) & w & 0x80808080u) != 0; }

// V as f16 to LDS: piece (g, t, c) holds the eight positions of quarter g of dim c
// D / 16 + t.  Positions outside [lo, hi) and NaN blocks are zeros.
template <int D, int TEAM>
struct VScale {
    float s[8], s2[D == 160 ? 8 : 1];
    bool nan;  // one of the latter (in this lane)
};
template <int D, int TEAM>
__device__ __forceinline__ void v_scales(VScale<D, TEAM> &f, const VBlock<D, TEAM> &b, int p0, int lo, int hi, int lane) {
    const int g = lane >> 4;
    f.nan = false;
#pragma unroll
    for (int w = 0; w < (D == 160 ? 4 : 2); ++w) f.nan |= any_nan_scale(b.s[w]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        f.s[j] = doe::mx4_byte_scale(b.s[j >> 2], j & 3);
        if constexpr (D == 160) f.s2[j] = doe::mx4_byte_scale(b.s[2 + (j >> 2)], j & 3);
    }
    if (p0 < lo || p0 + 32 > hi || __any(f.nan)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int p = p0 + 16 * (j >> 2) + 4 * g + (j & 3);
            const bool in = p >= lo && p < hi;
            f.s[j] = in && (b.s[j >> 2] >> 8 * (j & 3) & 255) != doe::kMx4NanScale ? f.s[j] : 0.0f;
            if constexpr (D == 160)
                f.s2[j] = in && (b.s[2 + (j >> 2)] >> 8 * (j & 3) & 255) != doe::kMx4NanScale ? f.s2[j] : 0.0f;
        }
    }
}
// Dims 2 i and 2 i + 1 of a lane's.
template <int D, int TEAM>
__device__ __forceinline__ void stage_v(uint8_t *dst, const VBlock<D, TEAM> &b, const VScale<D, TEAM> &f, int i, int lane) {
    constexpr int N = VBlock<D, TEAM>::kBytes;
    const int c = lane & 15, g = lane >> 4;
    h8 *to = reinterpret_cast<h8 *>(dst) + g * Shape<D, TEAM>::kDims + c;
    h2 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int at = j * N + i;
        float s = f.s[j];
        if constexpr (D == 160) s = 5 * c % 16 + i >= 16 ? f.s2[j] : s;
        v[j] = doe::mx4_pair_at(b.v[at >> 2], s, at);
    }
    to[(2 * i) * 16] = h8{v[0][0], v[1][0], v[2][0], v[3][0], v[4][0], v[5][0], v[6][0], v[7][0]};
    to[(2 * i + 1) * 16] = h8{v[0][1], v[1][1], v[2][1], v[3][1], v[4][1], v[5][1], v[6][1], v[7][1]};
}

// A lane's queries as operands, pair lane % 32: f16 as they are (HALF), f32 as f16 hi
// and lo parts of q 2^e.
template <int D, int TEAM, bool HALF>
struct Query {
    static constexpr int kOps = Shape<D, TEAM>::kOps, kLo = HALF ? 1 : kOps;
    h8 hi[kOps], lo[kLo];
};
// N operands of f32 queries from `first` on.
template <int D, int TEAM, int N>
struct RawQuery {
    float f[8 * N];
};
template <int D, int TEAM, int N>
__device__ __forceinline__ uint32_t read_query(RawQuery<D, TEAM, N> &r, const float *q, int first, int half) {
    uint32_t top = 0;  // (as bits: a NaN is above all)
#pragma unroll
    for (int o = 0; o < N; ++o) {
        const int from = dims_of<D, TEAM>(first + o, half);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(q + from + i);
            r.f[8 * o + i] = v.x, r.f[8 * o + i + 1] = v.y, r.f[8 * o + i + 2] = v.z, r.f[8 * o + i + 3] = v.w;
        }
    }
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) top = max(top, __float_as_uint(r.f[i]) & 0x7fffffffu);
    return max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
}
__device__ __forceinline__ void split_query(h8 &hi, h8 &lo, const float *f, int e) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = __builtin_amdgcn_ldexpf(f[i], e);
        hi[i] = (_Float16)v;
        lo[i] = (_Float16)(v - (float)hi[i]);
    }
}

// The products [FROM, TO) of a block's scores, operand by operand.
template <int D, int TEAM, bool HALF, int FROM, int TO>
__device__ __forceinline__ void scores(const Query<D, TEAM, HALF> &q, const KBlock<D, TEAM> &k, f32x16 &acc) {
    if constexpr (FROM < TO) {
        const float f = doe::mx4_byte_scale(k.s[FROM / 8], FROM / 4 % 2 * 2);
        const uint32_t w = k.k[FROM];
        const h2 k0 = doe::mx4_pair<0>(w, f), k1 = doe::mx4_pair<1>(w, f), k2 = doe::mx4_pair<2>(w, f), k3 = doe::mx4_pair<3>(w, f);
        const h8 kf = {k0[0], k0[1], k1[0], k1[1], k2[0], k2[1], k3[0], k3[1]};
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q.hi[FROM], acc, 0, 0, 0);
        if constexpr (!HALF) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q.lo[FROM], acc, 0, 0, 0);
        scores<D, TEAM, HALF, FROM + 1, TO>(q, k, acc);
    }
}

// What lanes of a wave write to LDS before it, its other lanes read behind it: the
// wave's LDS operations are in order, as long as the compiler leaves them so.
__device__ __forceinline__ void in_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A value is wanted here: otherwise the compiler computes it where it is used.
template <typename T>
__device__ __forceinline__ void here(T &v) {
    __asm__ volatile("" : "+v"(v));
}

// The instruction scheduler's order for what stands before it in a block of code:
// one matrix instruction, then so many vector ones, N times.
template <int N, int VALU>
__device__ __forceinline__ void interleave() {
    if constexpr (N > 0) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
        interleave<N - 1, VALU>();
    }
}

// HALF: f16 queries.
template <int D, int TEAM, bool HALF>
__global__ __launch_bounds__(64 * kWaves, per_cu(D)) void attn_mx4_prompt_kernel(PromptArgs a) {
    using P = Shape<D, TEAM>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr bool kShare = TEAM == 4;                 // the waves share V
    constexpr bool kSliced = P::kSlices > 1;
    constexpr int kParts = HALF ? 1 : 2;               // matrix instructions of an operand
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n32 = lane & 31, lh = lane >> 5, shift = a.c.page_shift, G = a.group;
    const int slice = kSliced ? wave : 0;
    const int kvh = blockIdx.x % a.c.kv_heads;
    // the last tiles first: they see the most positions
    int tile = a.tiles - 1 - blockIdx.x / a.c.kv_heads, b = 0, start = 0, count = 1, all = 1;
    if (a.row_starts) {
        for (int b0 = 0;; b0 += 64) {
            if (b0 >= a.c.batch) return;
            const int i = b0 + lane;
            const int lo_ = i < a.c.batch ? a.row_starts[i] : 0, hi_ = i < a.c.batch ? a.row_starts[i + 1] : 0;
            const int rows = lo_ < 0 ? 0 : std::max(0, std::min(hi_, a.rows) - lo_);
            const int upto = doe::wave_scan((int)(((int64_t)rows * G + P::kRows - 1) / P::kRows));
            const uint64_t behind = __ballot(upto > tile);
            if (behind) {
                const int at = __builtin_ctzll(behind);
                b = b0 + at;
                start = __builtin_amdgcn_readlane(lo_, at);
                count = __builtin_amdgcn_readlane(rows, at);
                all = __builtin_amdgcn_readlane(hi_, at) - start;
                tile -= at ? __builtin_amdgcn_readlane(upto, at - 1) : 0;
                break;
            }
            tile -= __builtin_amdgcn_readlane(upto, 63);
        }
    } else {
        const int each = (G + P::kRows - 1) / P::kRows;
        b = tile / each;
        tile -= b * each;
        start = b;
    }
    const int L = doe::mx4_len(a.c, b), pairs = count * G, pair0 = tile * P::kRows;
    // positions [seen_from, seen_to) of a pair; pairs behind the last repeat it
    auto to_of = [&](int pr) { return std::max(0, L - all + pr / G + 1); };
    auto from_of = [&](int pr) { return a.window > 0 ? std::max(0, to_of(pr) - a.window) : 0; };
    const int wave0 = pair0 + (kShare ? 32 * wave : 0);          // this wave's first pair
    const int tile1 = std::min(pair0 + P::kRows, pairs) - 1, wave1 = std::min(wave0 + 32, pairs) - 1;
    const bool idle = wave1 < wave0;
    const int klo = from_of(pair0), khi = to_of(tile1);          // the tile's
    const int flo = idle ? 0 : from_of(wave1), fhi = to_of(std::min(wave0, pairs - 1));  // seen by all of its pairs
    const int mine = std::min(wave0 + n32, pairs - 1);
    const int lo = from_of(mine), hi = to_of(mine);
    const int row = start + mine / G, head = kvh * G + mine % G;

    // this split's blocks [b0, b1)
    int b0 = klo / 32, b1 = khi > klo ? (khi + 31) / 32 : b0;
    if (a.splits > 1) {
        int per = (b1 - b0 + a.splits - 1) / a.splits;
        per = (per + P::kBlocks - 1) / P::kBlocks * P::kBlocks;
        b0 += (int)blockIdx.y * per;
        b1 = std::min(b1, b0 + per);
    }
    // this wave's blocks: first, first + stride, .. (all of the tile's, or every fourth);
    // slabs of 64 of them at a time, a lane each: -1 where there is nothing to see
    constexpr int kStride = kShare || kSliced ? 1 : kWaves;
    const int first = kShare || kSliced ? b0 : b0 + wave, blocks = std::max(0, (b1 - first + kStride - 1) / kStride);
    const int32_t *table = a.c.table + (int64_t)b * a.c.table_stride;
    auto slabs = [&](int i0) __attribute__((always_inline)) {
        const int blk = first + (i0 + lane) * kStride;
        int page = -1;
        if (blk < b1) page = table[blk >> (shift - 5)];
        return page >= 0 && page < a.c.num_pages ? page * a.c.kv_heads + kvh : -1;
    };
    int list0 = slabs(0), list1 = slabs(64), base = 0;  // blocks base .. base + 127
    auto slab_index = [&](int i) __attribute__((always_inline)) {
        const int k = i - base;
        return __builtin_amdgcn_readlane(k < 64 ? list0 : list1, k & 63);
    };
    auto slab_at = [&](int index) __attribute__((always_inline)) {
        return a.c.pool + (uint64_t)(uint32_t)std::max(index, 0) * (uint32_t)Mx4Slab<D>::bytes(shift);
    };
    auto place = [&](int i) __attribute__((always_inline)) { return ((first + i * kStride) * 32) & ((1 << shift) - 1); };

    float *sx = reinterpret_cast<float *>(lds + P::kData);                 // scores of the slices
    int *flags = reinterpret_cast<int *>(lds + P::kData + P::kScores);     // [buffer]: a NaN among the block's V
    const int ahead = kShare ? wave : 0;       // the block of a step that this wave stages
    const int buffers = kShare ? 0 : 2 * wave;  // this wave's first buffer

    Query<D, TEAM, HALF> q;
    f32x16 o[P::kTiles], s;
#pragma unroll
    for (int t = 0; t < P::kTiles; ++t) o[t] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    Mx4Factor rowf;  // of a score

    KBlock<D, TEAM> kb;
    VBlock<D, TEAM> vb;
    VScale<D, TEAM> vs;
    int ahead_slab = slab_index(ahead);  // of the block in vb
    auto fetch_v = [&](int i) __attribute__((always_inline)) {
        ahead_slab = slab_index(i);
        load_v<D, TEAM>(vb, slab_at(ahead_slab), shift, place(i), lane, slice);
    };
    int nans = 0, nans_ahead = 0;  // NaN blocks among the V of the step at hand, of the one being staged
    auto scale_v = [&](int i, int buffer) __attribute__((always_inline)) {
        v_scales<D, TEAM>(vs, vb, (first + i * kStride) * 32, klo, ahead_slab < 0 ? 0 : khi, lane);
        nans_ahead = __any(vs.nan);
        if (kShare && lane == 0) flags[buffer] = nans_ahead;
    };
    fetch_v(ahead);
    int slab0 = slab_index(0), slab1 = slab_index(1);  // of the block at hand and the next
    load_k<D, TEAM>(kb, slab_at(slab0), shift, place(0), lane, slice);
    {
        const int64_t at = (int64_t)row * a.q_stride + (int64_t)head * D + slice * P::kDims;
        const float f = a.softcap > 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
        if constexpr (HALF) {
            typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
            u16x8 top = {};
#pragma unroll
            for (int o = 0; o < P::kOps; ++o) {
                q.hi[o] = *reinterpret_cast<const h8 *>(static_cast<const _Float16 *>(a.q) + at + dims_of<D, TEAM>(o, lh));
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x8, q.hi[o]) & (unsigned short)0x7fff);
            }
            int bad = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) bad |= top[i] >= 0x7c00;
            bad |= __shfl_xor(bad, 32, 64);
            if constexpr (kSliced) {  // (a slice that is no number: the pair's scores are none)
                if (bad) q.hi[0][0] = (_Float16)NAN;
                bad = 0;
            }
            rowf = doe::mx4_factor(f, bad ? 0x7f800000u : 0u, 0);
        } else if constexpr (kShare) {
            RawQuery<D, TEAM, P::kOps> raw;
            const uint32_t top = read_query(raw, static_cast<const float *>(a.q) + at, 0, lh);
            const int e = doe::mx4_query_exp(top);
#pragma unroll
            for (int o = 0; o < P::kOps; ++o) split_query(q.hi[o], q.lo[o], raw.f + 8 * o, e);
            rowf = doe::mx4_factor(f, top, e);
        } else {
            // the waves have the same pairs: a step or none each (or, sliced, a part of the
            // dims), one scale for them all, passed on in V's place
            uint32_t *tops = reinterpret_cast<uint32_t *>(lds);
            h8 *x = reinterpret_cast<h8 *>(lds);
            constexpr int N = kSliced ? P::kOps : 4;
            RawQuery<D, TEAM, N> raw;
            uint32_t top = 0;
            const bool have = kSliced || wave < P::kSteps;
            // (the last step of head_dim 160 has two operands: its others are read again)
            const int op0 = kSliced ? 0 : std::min(4 * wave, P::kOps - N);
            if (have) top = read_query(raw, static_cast<const float *>(a.q) + at, op0, lh);
            if (lh == 0) tops[wave * 32 + n32] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = max(top, tops[w * 32 + n32]);
            __syncthreads();
            const int e = doe::mx4_query_exp(top);
            rowf = doe::mx4_factor(f, top, e);
            if constexpr (kSliced) {
#pragma unroll
                for (int o = 0; o < P::kOps; ++o) split_query(q.hi[o], q.lo[o], raw.f + 8 * o, e);
            } else {
                if (have) {
#pragma unroll
                    for (int o = 0; o < N; ++o) {
                        h8 hi, lo;
                        split_query(hi, lo, raw.f + 8 * o, e);
                        x[(op0 + o) * 128 + lane] = hi, x[(op0 + o) * 128 + 64 + lane] = lo;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int o = 0; o < P::kOps; ++o) q.hi[o] = x[o * 128 + lane], q.lo[o] = x[o * 128 + 64 + lane];
                __syncthreads();
            }
        }
    }
    const float yf = a.softcap > 0.0f ? a.softcap * 1.4426950408889634f : rowf.post;
    const bool large = __any(rowf.pre != 1.0f);
    scale_v(ahead, buffers + ahead);
#pragma unroll
    for (int t = 0; t < P::kTiles; ++t) stage_v<D, TEAM>(lds + (buffers + ahead) * P::kV, vb, vs, t, lane);
    fetch_v(ahead + P::kBlocks);
    constexpr int kEarly = P::kOps / 4;  // operands of a block's scores that go beside the logs
    s = f32x16{};
    scores<D, TEAM, HALF, 0, P::kOps>(q, kb, s);
    load_k<D, TEAM>(kb, slab_at(slab1), shift, place(1), lane, slice);
    if (kShare) __syncthreads();
    else in_order();

    // O stays in the accumulation registers between the matrix instructions where it
    // takes many (the compiler would move it out at every block for the rare rescaling)
    auto keep = [&](f32x16 &v) __attribute__((always_inline)) {
        if constexpr (P::kTiles > 4) __asm__ volatile("" : "+a"(v));
    };

    // Block i: its weights beside the next one's scores, its P V beside the next V's
    // way into LDS (of a step's next V a quarter at each of its four blocks).
    auto block = [&](int i, auto u_) __attribute__((always_inline)) {
        constexpr int u = decltype(u_)::value;
        const int p0 = (first + i * kStride) * 32;
        const int buffer = kShare ? (i & 4) + u : buffers + (i & 1);
        const int into = kShare ? ((i & 4) ^ 4) + wave : buffers + (~i & 1);
        f32x16 next = f32x16{};
        if constexpr (u == 0) {
            if constexpr (kShare) {
                const int4 f = *reinterpret_cast<const int4 *>(flags + (i & 4));
                nans = f.x | f.y | f.z | f.w;
            } else {
                nans = nans_ahead;
            }
        }
        if constexpr (kSliced) {
            // [slice][r / 4][lane] float4
            float4 *to = reinterpret_cast<float4 *>(sx) + wave * 256 + lane;
            __syncthreads();  // the last block's scores have been read
#pragma unroll
            for (int r = 0; r < 4; ++r) to[64 * r] = make_float4(s[4 * r], s[4 * r + 1], s[4 * r + 2], s[4 * r + 3]);
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float4 e = reinterpret_cast<const float4 *>(sx)[w * 256 + 64 * r + lane];
                    v.x += e.x, v.y += e.y, v.z += e.z, v.w += e.w;
                }
                s[4 * r] = v.x, s[4 * r + 1] = v.y, s[4 * r + 2] = v.z, s[4 * r + 3] = v.w;
            }
        }
        // lane: pair n32, positions p0 + 8 (r / 4) + 4 lh + r % 4
        if (large) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= rowf.pre;
        }
        if (a.softcap > 0.0f) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = doe::mx4_tanh(s[r] * rowf.post);
        }
        float y[16];
        const int top_ = slab0 < 0 ? 0 : hi;
        const bool whole = slab0 >= 0 && p0 >= flo && p0 + 32 <= fhi;
        auto logs = [&](float ref) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) y[r] = fmaf(s[r], yf, -ref);
        };
        auto mask = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int p = p0 + 8 * (r >> 2) + 4 * lh + (r & 3);
                y[r] = p >= lo && p < top_ ? y[r] : -INFINITY;
            }
        };
        auto most = [&]() __attribute__((always_inline)) {
            float top = y[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, y[r]);
            return top;
        };
        logs(m);
        if (!whole) mask();
        const float over = most();
        scores<D, TEAM, HALF, 0, kEarly>(q, kb, next);
        interleave<kEarly * kParts, 6>();
        here(next);
        if (__any(over > kBias + kLazy)) {  // (m = -inf: any score)
            logs(0.0f);
            if (!whole) mask();
            float top = most();
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            float ref = top - kBias > m + kLazy ? top - kBias : m;
            ref = ref == INFINITY ? NAN : ref;  // (a score beyond f32: no numbers from here on)
            const float corr = ref == m ? 1.0f : __builtin_amdgcn_exp2f(m - ref);
            m = ref;
            l *= corr;
            if (i > 0) {  // (O is 0 before)
#pragma unroll
                for (int t = 0; t < P::kTiles; ++t) {
                    keep(o[t]);
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[t][r] *= corr;
                    keep(o[t]);
                }
            }
            logs(ref);
            if (!whole) mask();
        }
        // P^T operands: step h of two takes the positions of quarter lh + 2 h
        h8 ph[2], pl[2];
        float minus = -1.0f;  // (a value, so that e - hi is one instruction that takes hi as f16)
        here(minus);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int r = 4 * (h + 2 * (j >> 2)) + (j & 3);
                const float e0 = __builtin_amdgcn_exp2f(y[r]), e1 = __builtin_amdgcn_exp2f(y[r + 1]);
                l += e0 + e1;
                h2 hi_part = {(_Float16)e0, (_Float16)e1};
                here(hi_part);  // (rounded as a pair once, not each again for the lo part)
                ph[h][j] = hi_part[0], ph[h][j + 1] = hi_part[1];
                pl[h][j] = (_Float16)fmaf((float)hi_part[0], minus, e0);
                pl[h][j + 1] = (_Float16)fmaf((float)hi_part[1], minus, e1);
            }
        scores<D, TEAM, HALF, kEarly, P::kOps>(q, kb, next);
        interleave<(P::kOps - kEarly) * kParts, 6>();
        here(next);
        here(l);
        __builtin_amdgcn_sched_barrier(0);
        // the block after next follows the next one's K into its registers
        const int slab2 = slab_index(i + 2);
        load_k<D, TEAM>(kb, slab_at(slab2), shift, place(i + 2), lane, slice);
        if constexpr (u == 0) scale_v(i + P::kBlocks + ahead, into);
        __builtin_amdgcn_sched_barrier(0);
        const h8 *v = reinterpret_cast<const h8 *>(lds + buffer * P::kV) + lh * P::kDims + n32;
        uint8_t *to = lds + into * P::kV;
        constexpr int each = (P::kTiles + P::kBlocks - 1) / P::kBlocks;  // pieces staged at a block of a step
#pragma unroll
        for (int t = 0; t < P::kTiles; ++t) {
            const h8 v0 = v[32 * t], v1 = v[2 * P::kDims + 32 * t];
            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, ph[0], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, ph[1], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, pl[0], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, pl[1], o[t], 0, 0, 0);
            if (t < each && u * each + t < P::kTiles) stage_v<D, TEAM>(to, vb, vs, u * each + t, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (u == P::kBlocks - 1) fetch_v(i + 1 + P::kBlocks + ahead);
        if (__builtin_amdgcn_readfirstlane(nans)) {
            // NaN blocks were left out of V: they reach the pairs that see them
            const uint8_t *slab = slab_at(slab0);
            for (int x = 0; x < 32; ++x)
                for (int g = 0; g < D / 32; ++g) {
                    if (slab[Mx4Slab<D>::v_scale(shift, place(i) + x, g)] != doe::kMx4NanScale) continue;
                    const float bad = p0 + x >= lo && p0 + x < top_ ? NAN : 0.0f;
#pragma unroll
                    for (int t = 0; t < P::kTiles; ++t) {
                        keep(o[t]);
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int w = 8 * (r >> 2) + 4 * lh + (r & 3);
                            const int dim = (w & 15) * (D / 16) + slice * (P::kDims / 16) + 2 * t + (w >> 4);
                            o[t][r] += dim / 32 == g ? bad : 0.0f;
                        }
                        keep(o[t]);
                    }
                }
        }
        if constexpr (!kShare) in_order();
        s = next;
        slab0 = slab1;
        slab1 = slab2;
    };
    for (int i = 0; i < blocks; i += P::kBlocks) {
        if (i - base >= 64) {  // (after the last use of a block below base + 64: those ahead are at most eleven on)
            base += 64;
            list0 = list1;
            list1 = slabs(base + 64);
        }
        block(i, std::integral_constant<int, 0>());
        if constexpr (kShare) {
            block(i + 1, std::integral_constant<int, 1>());
            block(i + 2, std::integral_constant<int, 2>());
            block(i + 3, std::integral_constant<int, 3>());
            __syncthreads();
        }
    }

    l += __shfl_xor(l, 32, 64);
    const int64_t parts = (int64_t)a.splits * a.rows * a.num_heads;
    // dims d .. d + N - 1 of the pair (row, head), or its part of a split
    auto put = [&](int row, int head, int d, const float *v, auto n, float M, float sum, bool first) __attribute__((always_inline)) {
        constexpr int N = decltype(n)::value;
        if (a.splits > 1) {
            const int64_t at = ((int64_t)blockIdx.y * a.rows + row) * a.num_heads + head;
            float *to = a.part + at * D + d;
#pragma unroll
            for (int i = 0; i < N; ++i) to[i] = v[i];
            if (first) reinterpret_cast<float2 *>(a.part + parts * D)[at] = make_float2(M, sum);
            return;
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        const int64_t at = (int64_t)row * a.out_stride + (int64_t)head * D + d;
        if (a.out_f16) {
            _Float16 *to = static_cast<_Float16 *>(a.out) + at;
#pragma unroll
            for (int i = 0; i < N; i += 2) *reinterpret_cast<h2 *>(to + i) = h2{(_Float16)(v[i] * inv), (_Float16)(v[i + 1] * inv)};
        } else {
            float *to = static_cast<float *>(a.out) + at;
#pragma unroll
            for (int i = 0; i < N; i += 2) *reinterpret_cast<float2 *>(to + i) = make_float2(v[i] * inv, v[i + 1] * inv);
        }
    };
    if constexpr (kShare || kSliced) {
        if (idle || wave0 + n32 >= pairs) return;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int c = 8 * (r >> 2) + 4 * lh + (r & 3);
            float v[2 * P::kTiles];
#pragma unroll
            for (int t = 0; t < P::kTiles; ++t) v[2 * t] = o[t][r], v[2 * t + 1] = o[t][r + 8];
            put(row, head, c * (D / 16) + slice * (P::kDims / 16), v, std::integral_constant<int, 2 * P::kTiles>(), m, l,
                r == 0 && lh == 0 && slice == 0);
        }
    } else {
        // the waves' parts of the tile together: each wave's O as [4 t + position / 4][pair] float4
        __syncthreads();
        float4 *om = reinterpret_cast<float4 *>(lds) + wave * (32 * D / 4);
        float2 *ml = reinterpret_cast<float2 *>(lds + P::kData);  // [wave][pair]
        if (lh == 0) ml[wave * 32 + n32] = make_float2(m, l);
#pragma unroll
        for (int t = 0; t < P::kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                om[(t * 8 + 2 * r + lh) * 32 + n32] = make_float4(o[t][4 * r], o[t][4 * r + 1], o[t][4 * r + 2], o[t][4 * r + 3]);
        __syncthreads();
        // a thread two columns (D / 16 dims) of a pair: position c + 16 h of tile t is dim c D / 16 + 2 t + h
        for (int id = threadIdx.x; id < 512; id += 64 * kWaves) {
            const int pr = (id >> 2) & 31, c = (id >> 7) * 4 + (id & 3);
            if (pair0 + pr >= pairs) continue;
            float M = -INFINITY, lt = 0.0f, v[D / 16], f[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w * 32 + pr].x);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float2 e = ml[w * 32 + pr];
                f[w] = e.x == -INFINITY ? (e.y != e.y ? e.y : 0.0f) : __builtin_amdgcn_exp2f(e.x - M);  // (a NaN stays one)
                lt += e.y * f[w];
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                v[i] = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    v[i] += f[w] * reinterpret_cast<const float *>(lds)[((w * (D / 4) + (i >> 1) * 8 + (i & 1) * 4 + (c >> 2)) * 32 + pr) * 4 + (c & 3)];
            }
            const int pr_ = pair0 + pr;
            put(start + pr_ / G, kvh * G + pr_ % G, c * (D / 16), v, std::integral_constant<int, D / 16>(), M, lt, c == 0);
        }
    }
}

// The splits of a (row, head) joined; pairs of rows of no sequence have none and are left alone.
template <int D>
__global__ __launch_bounds__(256) void attn_mx4_prompt_join_kernel(PromptArgs a) {
    const int64_t pairs = (int64_t)a.rows * a.num_heads;
    const int64_t at = (int64_t)blockIdx.x * (1024 / D) + threadIdx.x / (D / 4);
    const int d = (int)(threadIdx.x % (D / 4)) * 4;
    if (threadIdx.x / (D / 4) >= 1024 / D || at >= pairs) return;
    const int64_t row = at / a.num_heads;
    if (a.row_starts && (row < a.row_starts[0] || row >= a.row_starts[a.c.batch])) return;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + a.splits * pairs * D);
    float M = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z = 0; z < a.splits; ++z) M = fmaxf(M, ml[z * pairs + at].x);
    for (int z = 0; z < a.splits; ++z) {
        const float2 e = ml[z * pairs + at];
        const float f = e.x == -INFINITY ? (e.y != e.y ? e.y : 0.0f) : __builtin_amdgcn_exp2f(e.x - M);
        const float4 o = *reinterpret_cast<const float4 *>(a.part + (z * pairs + at) * D + d);
        l += e.y * f;
        v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const int64_t to = row * a.out_stride + (at - row * a.num_heads) * D + d;
    if (a.out_f16) {
        _Float16 *o = static_cast<_Float16 *>(a.out) + to;
        o[0] = (_Float16)(v.x * inv), o[1] = (_Float16)(v.y * inv), o[2] = (_Float16)(v.z * inv), o[3] = (_Float16)(v.w * inv);
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

constexpr int kCus = 256, kMaxSplits = 16;

// Tiles of `rows` pairs that a call may have, by what the host knows.
int64_t tiles_of(bool starts, int64_t batch, int64_t rows, int64_t group, int tile_rows) {
    return starts ? rows * group / tile_rows + std::min(batch, rows) : batch * ((group + tile_rows - 1) / tile_rows);
}
int g_tile = 0;  // 0 automatic, 32 or 128 (up to head_dim 256) pairs

// Whether a call takes tiles of 128 pairs, whose waves share V's way into LDS, or of
// 32, whose waves take every fourth block.  The large ones need as many tiles as the
// device holds workgroups.  1500 rows after 2000 of 8 sequences, 32 against 128, f32
// and f16: 16 / 4 heads of 64 165 / 166 and 147 / 146 us, 16 / 4 of 128 274 / 266 and 235 /
// 220, 32 / 16 of 160 1049 / 798 and 852 / 650, 8 / 4 of 256 331 / 324 and 290 / 264; one
// prompt of 1000 rows (fewer tiles), f32: 16 / 28, 20 / 36 and 29 / 43 at 64, 128 and 256,
// but 67 / 60 at 160, where 16 KV heads make 256 tiles.
bool shared(int64_t head_dim, bool starts, int64_t batch, int64_t rows, int64_t num_heads, int64_t kv_heads) {
    if (head_dim == 512) return false;
    if (g_tile) return g_tile == 128;
    return tiles_of(starts, batch, rows, num_heads / kv_heads, 128) * kv_heads >= per_cu((int)head_dim) * kCus;
}
int64_t splits_of(bool share, bool starts, int64_t batch, int64_t rows, int64_t num_heads, int64_t kv_heads) {
    const int64_t wgs =
        std::max<int64_t>(1, tiles_of(starts, batch, rows, num_heads / kv_heads, share ? 128 : 32) * kv_heads);
    return std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, kCus / wgs));
}
int64_t workspace_of(int64_t head_dim, int64_t batch, int64_t rows, int64_t num_heads, int64_t kv_heads) {
    auto splits = [&](bool starts) {
        return splits_of(shared(head_dim, starts, batch, rows, num_heads, kv_heads), starts, batch, rows, num_heads, kv_heads);
    };
    const int64_t most = rows == batch ? std::max(splits(true), splits(false)) : splits(true);
    return most == 1 ? 16 : most * rows * num_heads * (head_dim + 2) * 4;
}

template <int D, int TEAM, bool HALF>
int launch(const PromptArgs &a, hipStream_t st) {
    constexpr int lds = Shape<D, TEAM>::kLds;
    static const hipError_t attr_rc = hipFuncSetAttribute((const void *)attn_mx4_prompt_kernel<D, TEAM, HALF>,
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    DOE_HIP_CHECK(attr_rc);
    const dim3 grid((unsigned)(a.tiles * a.c.kv_heads), (unsigned)a.splits);
    hipLaunchKernelGGL((attn_mx4_prompt_kernel<D, TEAM, HALF>), grid, dim3(64 * kWaves), lds, st, a);
    DOE_LAUNCH_CHECK("attn_mx4_prompt_kernel");
    if (a.splits == 1) return DOE_OK;
    const int64_t pairs = (int64_t)a.rows * a.num_heads, each = 1024 / D;
    hipLaunchKernelGGL(attn_mx4_prompt_join_kernel<D>, dim3((unsigned)((pairs + each - 1) / each)), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("attn_mx4_prompt_join_kernel");
    return DOE_OK;
}

template <int D>
int launch_d(PromptArgs &a, bool share, hipStream_t st) {
    if constexpr (D < 512) {
        if (share) return a.q_f16 ? launch<D, 4, true>(a, st) : launch<D, 4, false>(a, st);
    }
    return a.q_f16 ? launch<D, 1, true>(a, st) : launch<D, 1, false>(a, st);
}

}  // namespace

namespace doe {

int mx4_set_tile(int value) {
    DOE_REQUIRE(value == 0 || value == 32 || value == 128, DOE_E_INVALID, "attn_mx4.tile is 0, 32 or 128");
    g_tile = value;
    return DOE_OK;
}

}  // namespace doe

extern "C" {

int doe_attn_mx4_prompt_workspace(int64_t batch, int64_t rows, int64_t num_heads, int64_t num_kv_heads,
                                  int64_t head_dim, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    int64_t page = 0;
    const int rc = doe_mx4_page_bytes(32, num_kv_heads, head_dim, &page);
    if (rc) return rc;
    DOE_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 0 && num_heads > 0 && num_heads <= 65535 &&
                    num_heads % num_kv_heads == 0 && rows < ((int64_t)1 << 31) && rows * num_heads < ((int64_t)1 << 31),
                DOE_E_INVALID, "batch %lld, %lld rows, %lld heads over %lld", (long long)batch, (long long)rows,
                (long long)num_heads, (long long)num_kv_heads);
    *bytes = workspace_of(head_dim, batch, rows, num_heads, num_kv_heads);
    return DOE_OK;
}

int doe_attn_mx4_prompt(const doe_mx4_cache *cache, const void *q, int q_f16, int64_t q_row_stride, void *out,
                        int out_f16, int64_t out_row_stride, const int32_t *row_starts, int64_t rows, int64_t num_heads,
                        float scale, float softcap, int64_t sliding_window, void *workspace, int64_t workspace_bytes,
                        doe_stream_t stream) {
    PromptArgs a{};
    int rc = doe::mx4_view(cache, &a.c);
    if (rc) return rc;
    if ((rc = doe::mx4_attention_checks(a.c, num_heads, scale, softcap, sliding_window, q, out))) return rc;
    const int64_t d = cache->head_dim;
    DOE_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && rows * num_heads < ((int64_t)1 << 31), DOE_E_INVALID,
                "%lld rows of %lld heads", (long long)rows, (long long)num_heads);
    DOE_REQUIRE(row_starts || rows == a.c.batch, DOE_E_INVALID,
                "without row_starts a call takes one row a sequence (%lld rows, batch %d)", (long long)rows, a.c.batch);
    DOE_REQUIRE(q_row_stride >= num_heads * d && out_row_stride >= num_heads * d && q_row_stride * (q_f16 ? 2 : 4) % 16 == 0 &&
                    out_row_stride * (out_f16 ? 2 : 4) % 16 == 0,
                DOE_E_INVALID, "row strides below a row, or not multiples of 16 bytes");
    const int64_t need = workspace_of(d, a.c.batch, rows, num_heads, a.c.kv_heads);
    DOE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need, DOE_E_INVALID,
                "a 16-byte aligned workspace of %lld bytes is needed (got %lld)", (long long)need, (long long)workspace_bytes);
    const bool starts = row_starts != nullptr, share = shared(d, starts, a.c.batch, rows, num_heads, a.c.kv_heads);
    const int64_t tiles = tiles_of(starts, a.c.batch, rows, num_heads / a.c.kv_heads, share ? 128 : 32);
    DOE_REQUIRE(tiles * a.c.kv_heads < ((int64_t)1 << 24), DOE_E_UNSUPPORTED, "%lld rows of %lld heads in one call",
                (long long)rows, (long long)num_heads);  // (a launch has fewer than 2^32 threads)
    if ((rc = doe::require_init())) return rc;
    if (rows == 0 || a.c.batch == 0) return DOE_OK;
    a.q = q;
    a.out = out;
    a.row_starts = row_starts;
    a.rows = (int)rows;
    a.q_stride = q_row_stride;
    a.out_stride = out_row_stride;
    a.q_f16 = q_f16 != 0;
    a.out_f16 = out_f16 != 0;
    a.num_heads = (int)num_heads;
    a.group = (int)(num_heads / a.c.kv_heads);
    a.window = (int)sliding_window;
    a.scale = scale;
    a.softcap = softcap;
    a.tiles = (int)tiles;
    // no more splits than there are steps of eight blocks to share out
    int64_t blocks = ((int64_t)a.c.table_stride << a.c.page_shift) / 32;
    if (a.window > 0) blocks = std::min<int64_t>(blocks, (a.window + rows) / 32 + 2);
    a.splits = (int)std::max<int64_t>(1, std::min(splits_of(share, starts, a.c.batch, rows, num_heads, a.c.kv_heads), blocks / 8));
    a.part = static_cast<float *>(workspace);
    const hipStream_t st = (hipStream_t)stream;
    switch (d) {
        case 64: return launch_d<64>(a, share, st);
        case 128: return launch_d<128>(a, share, st);
        case 160: return launch_d<160>(a, share, st);
        case 256: return launch_d<256>(a, share, st);
        default: return launch_d<512>(a, share, st);
    }
}

}  // extern "C"
