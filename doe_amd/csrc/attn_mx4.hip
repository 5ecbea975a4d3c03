// attn_mx4.hip -- GQA attention of single tokens over the paged KV cache held in 4
// bits (doe_attn_mx4_decode): o = softmax(cap(q . k scale)) v for one query a
// sequence, whose length the kernel reads.
//
// A row is a sequence and up to eight query heads of one KV head, and is cut in
// blocks of 32 positions.  Rows with more blocks than an even share of the
// device's are split into equal pieces; a workgroup takes one piece (or row), its
// waves every fourth block.  Pieces leave their parts (o, m, l) in the caller's
// workspace and a second kernel joins them.
//   * S^T = K Q^T on v_mfma_f32_16x16x32_f16: 16 positions x 16 query rows, of
//     which 0..7 are the heads' f16 hi parts and 8..15 their lo parts (one
//     exchange of lane halves adds them: f32 quality for no more matrix work).
//     A lane reads D / 4 dims of a position in one piece and turns each dword of
//     codes into an operand with four v_cvt_scalef32_pk_f16_fp4, the block's
//     power of two applied by the same instruction.
//   * S^T's sums are P^T's operand order as they stand.  P goes to f16 as hi (rows
//     0..7) + lo (8..15), so it too is carried with 22 bits for nothing.
//   * O^T = V^T P^T: the page layout gives a lane its eight positions x D / 16 dims
//     in one piece; pairs of positions are brought together by v_perm.
//   * The running max is raised only when a score exceeds it by 2^8, P lies
//     2^7 above it, so that f16's small values lose no more than 2^-32 of the largest.
// No wave waits for another until a row's end.  Bound by the cache's bytes where
// there are many: 8 sequences of 32768, 64 / 8 heads of 128 dims (285 MB): 55 us with
// the join, the rate of a large copy (5.2 TB/s).  Bound by two dependent launches and
// a chain of cold reads (length, page table, K, then parts) where there are few: one
// of 4096, 8 / 4 heads of 256: 10.5 us, 7.6 + 3.1-3.7 of them in the kernels, which
// overlap a little.  A wave has a block's K and V under way while it works on the one
// before, which asks for enough waves more than for more blocks a wave: per_cu() is as
// many as the registers allow.
#include "mx4_cache.h"

#include <limits.h>
#include <math.h>
#include <algorithm>

namespace {

using doe::Mx4Factor;
using doe::Mx4Slab;
using doe::Mx4View;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kHeads = 8;
constexpr float kBias = 7.0f, kLazy = 8.0f;  // log2: P of the running max, and how far that may lag

struct TokenArgs {
    Mx4View c;
    const void *q;
    void *out;
    int q_f16, out_f16, num_heads, group, heads, groups;  // query heads of a KV head, of a row, rows of a KV head
    int window, per_row, by_row;
    float scale, softcap;
    float *part;    // split items' [gridDim.x][kHeads][D], then [gridDim.x][kHeads][2]
    int2 *joined;   // by_row: a row's first part (-1: not split) and their number; else at a row's first part the row and that number (others: -1)
};

// Workgroups of four waves that a CU holds at once, by the registers that a wave
// takes, and those that fill the device's 256 CUs in one round (head_dim 128: four
// leave a wave fewer registers, 56.6 us for 55.2 over 8 sequences of 32768).
template <int D>
constexpr int per_cu() { return D <= 160 ? 3 : (D <= 256 ? 2 : 1); }
template <int D>
constexpr int workgroups() { return 256 * per_cu<D>(); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return std::max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
// The same query row's value in the other half (hi / lo) of its sixteen.
__device__ __forceinline__ float other_half(float v) { return dpp<0x128>(v); }

// Blocks of the rows of a sequence of hi positions, the first seen one at lo; at
// least one (of an empty sequence it gives the zeros).
__device__ __forceinline__ int first_seen(const TokenArgs &a, int hi) { return a.window > 0 && hi > a.window ? hi - a.window : 0; }
__device__ __forceinline__ int blocks_of(const TokenArgs &a, int hi) {
    const int n = ((hi + 31) >> 5) - (first_seen(a, hi) >> 5);
    return n < 1 ? 1 : n;
}

// A lane's bytes of a block: its dims of K at two positions, with their scale
// bytes, and its dims of V at eight with theirs (head_dim 160: of both groups
// that its dims may lie in).
template <int D>
struct KBlock {
    uint32_t k[2][D / 32], ks[2];
};
template <int D>
struct VBlock {
    uint32_t v[D / 16], vs[D == 160 ? 4 : 2];
};

// n dwords at p (aligned to 4 bytes, 8 or 16 where n is a multiple of 2 or 4 and so
// the layout).  NT: past the caches.
template <bool NT, typename T>
__device__ __forceinline__ T load(const uint8_t *p) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
    else return *reinterpret_cast<const T *>(p);
}
template <bool NT, int N>
__device__ __forceinline__ void load_words(uint32_t *dst, const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 v = load<NT, u32x4>(p + 4 * i);
            dst[i] = v[0], dst[i + 1] = v[1], dst[i + 2] = v[2], dst[i + 3] = v[3];
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const u32x2 v = load<NT, u32x2>(p + 4 * i);
            dst[i] = v[0], dst[i + 1] = v[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = load<NT, uint32_t>(p + 4 * i);
    }
}

// A lane's (c16, g4) place within a block's sections: fixed, so that a load is a
// wave's address and this offset.
template <int D>
struct Place {
    uint32_t k, ks, v, vs;
    __device__ __forceinline__ Place(int c16, int g4)
        : k(c16 * (D / 2) + g4 * (D / 8)),
          ks(c16 * (D / 32) + (D == 64 ? g4 >> 1 : (D <= 160 ? g4 : g4 * (D / 128)))),
          v((g4 * 16 + c16) * (D / 4)),
          vs((g4 * (D / 32) + c16 * (D / 16) / 32) * 8) {}
};

// The block at position x of a page.
template <int D, bool NT>
__device__ __forceinline__ void load_k(KBlock<D> &b, const uint8_t *slab, int shift, int x, const Place<D> &at) {
    using S = Mx4Slab<D>;
    const uint8_t *k = slab + S::k_code(x), *ks = slab + S::k_scale(shift, x);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        load_words<NT, D / 32>(b.k[t], k + at.k + 16 * t * (D / 2));
        const uint8_t *s = ks + at.ks + 16 * t * (D / 32);
        if constexpr (D <= 128) b.ks[t] = s[0];
        else if constexpr (D == 160) b.ks[t] = s[0] | (uint32_t)s[1] << 8;
        else if constexpr (D == 256) b.ks[t] = *reinterpret_cast<const uint16_t *>(s);
        else b.ks[t] = *reinterpret_cast<const uint32_t *>(s);
    }
}
template <int D, bool NT>
__device__ __forceinline__ void load_v(VBlock<D> &b, const uint8_t *slab, int shift, int x, const Place<D> &at) {
    using S = Mx4Slab<D>;
    load_words<NT, D / 16>(b.v, slab + S::v_code(shift, x, 0) + at.v);
    const uint8_t *vs = slab + S::v_scale(shift, x, 0) + at.vs;
    load_words<NT, 2>(b.vs, vs);
    // (the second group of columns 13 .. 15 is the same one: their dims lie in it whole)
    if constexpr (D == 160) load_words<NT, 2>(b.vs + 2, vs + (at.vs / 8 % 5 < 4 ? 8 : 0));
}

// A row's running state in a wave: O^T tile T, dims (4 g4 + i) D / 16 + T of
// query row c16; P is 2^(score - m), l its sum.
template <int D>
struct State {
    f32x4 o[D / 16];
    float m, l;
};

// S^T of a block: query row c16, positions 16 t + 4 g4 + i at s[t][i], hi and lo
// parts of the query in their own rows.
template <int D>
__device__ __forceinline__ void scores(f32x4 *s, const h8 (*q)[64], const KBlock<D> &b, int lane, int g4) {
    s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const h8 qf = q[i][lane];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float f;
            if constexpr (D == 160) f = doe::mx4_byte_scale(g4 + i >= 4 ? b.ks[t] >> 8 : b.ks[t], 0);
            else f = doe::mx4_byte_scale(b.ks[t], D >= 128 ? i / 4 : 0);
            const uint32_t w = b.k[t][i];
            const h2 k0 = doe::mx4_pair<0>(w, f), k1 = doe::mx4_pair<1>(w, f), k2 = doe::mx4_pair<2>(w, f), k3 = doe::mx4_pair<3>(w, f);
            const h8 kf = {k0[0], k0[1], k1[0], k1[1], k2[0], k2[1], k3[0], k3[1]};
            s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf, s[t], 0, 0, 0);
        }
    }
}

// P^T of a block at positions p0 .. (those in [lo, hi) are seen), the state's
// reference raised and its sum carried on.  `lo_part`: 1 in the lanes of P's lo
// part, 0 in those of its hi part.
template <int D>
__device__ __forceinline__ h8 weights(const TokenArgs &a, State<D> &st, const f32x4 *s, const Mx4Factor &factor, bool large,
                                      float lo_part, int p0, int lo, int hi, int g4) {
    float v[8], y[8], rowf = factor.post;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s[j >> 2][j & 3] + other_half(s[j >> 2][j & 3]);
    if (large) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= factor.pre;
    }
    if (a.softcap > 0.0f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = doe::mx4_tanh(v[j] * rowf);
        rowf = a.softcap * 1.4426950408889634f;
    }
    const bool whole = p0 >= lo && p0 + 32 <= hi;
    // log2 of P: the score less the reference (first -inf: any seen score gives +inf)
    auto logs = [&](float ref) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = fmaf(v[j], rowf, -ref);
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int p = p0 + 16 * (j >> 2) + 4 * g4 + (j & 3);
                y[j] = p >= lo && p < hi ? y[j] : -INFINITY;
            }
        }
        return fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
    };
    if (__any(logs(st.m) > kBias + kLazy)) {
        float top = logs(0.0f);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        float ref = top - kBias > st.m + kLazy ? top - kBias : st.m;
        ref = ref == INFINITY ? NAN : ref;  // (a score beyond f32: no numbers from here on)
        const float corr = ref == st.m ? 1.0f : __builtin_amdgcn_exp2f(st.m - ref);
        st.m = ref;
        st.l *= corr;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) st.o[t][i] *= corr;
        logs(ref);
    }
    h8 pf;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float p0_ = __builtin_amdgcn_exp2f(y[j]), p1_ = __builtin_amdgcn_exp2f(y[j + 1]);
        st.l += p0_ + p1_;
        const h2 hi_part = {(_Float16)p0_, (_Float16)p1_};
        pf[j] = (_Float16)fmaf(-lo_part, (float)hi_part[0], p0_);
        pf[j + 1] = (_Float16)fmaf(-lo_part, (float)hi_part[1], p1_);
    }
    return pf;
}

// O^T += V^T P^T.  Position j of the lane's eight is at bytes j D / 32 ..; scale
// 0 where it is not seen (0 times a NaN is one).
template <int D>
__device__ __forceinline__ void values(State<D> &st, const h8 pf, const VBlock<D> &b, int p0, int lo, int hi, int c16, int g4) {
    float vs[8], vs2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        vs[j] = doe::mx4_byte_scale(b.vs[j >> 2], j & 3);
        if constexpr (D == 160) vs2[j] = doe::mx4_byte_scale(b.vs[2 + (j >> 2)], j & 3);
    }
    if (p0 < lo || p0 + 32 > hi) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int p = p0 + 16 * (j >> 2) + 4 * g4 + (j & 3);
            const bool in = p >= lo && p < hi;
            vs[j] = in ? vs[j] : 0.0f;
            if constexpr (D == 160) vs2[j] = in ? vs2[j] : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {  // dims 2 i and 2 i + 1 of the lane's
        h2 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = j * (D / 32) + i;
            float f = vs[j];
            if constexpr (D == 160) f = 5 * c16 % 16 + i >= 16 ? vs2[j] : f;
            v[j] = doe::mx4_pair_at(b.v[at >> 2], f, at);
        }
        const h8 v0 = {v[0][0], v[1][0], v[2][0], v[3][0], v[4][0], v[5][0], v[6][0], v[7][0]};
        const h8 v1 = {v[0][1], v[1][1], v[2][1], v[3][1], v[4][1], v[5][1], v[6][1], v[7][1]};
        st.o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf, st.o[2 * i], 0, 0, 0);
        st.o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf, st.o[2 * i + 1], 0, 0, 0);
    }
}

template <int D>
struct TokenLds {
    static constexpr int kRow = D + 4;
    h8 q[D / 32][64];  // a row's query operands
    Mx4Factor rowf[kHeads];
    float o[kWaves][kHeads][kRow];
    float2 ml[kWaves][kHeads];
};

// A row's queries, two heads a wave and D / 32 dims a lane, into operand order:
// lane (c16, g4) of step i takes dims g4 D / 4 + 8 i .. of head c16 % 8, scaled
// by a power of two, the f16 hi part (c16 < 8) or the lo part; rowf takes the
// scale out of a score again.  Heads that the row lacks are 0.
template <int D>
struct RawQuery {
    static constexpr int N = D / 32;
    float f[N];
};
template <int D>
__device__ __forceinline__ void read_query(RawQuery<D> &r, const TokenArgs &a, int64_t row, int heads, int wave, int lane) {
    constexpr int N = RawQuery<D>::N;
    const int head = 2 * wave + (lane >> 5);
    const int64_t at = row + (head < heads ? head : 0) * D + (lane & 31) * N;
    if (a.q_f16) {
        const _Float16 *p = static_cast<const _Float16 *>(a.q) + at;
#pragma unroll
        for (int i = 0; i < N; ++i) r.f[i] = (float)p[i];
    } else {
        const float *p = static_cast<const float *>(a.q) + at;
#pragma unroll
        for (int i = 0; i < N; ++i) r.f[i] = p[i];
    }
}
template <int D>
__device__ __forceinline__ void stage_query(const TokenArgs &a, const RawQuery<D> &r, TokenLds<D> &sm, int heads, int wave, int lane) {
    constexpr int N = RawQuery<D>::N;
    const int head = 2 * wave + (lane >> 5);
    uint32_t top = 0;  // (as bits: a NaN is above all)
#pragma unroll
    for (int i = 0; i < N; ++i) top = std::max(top, __float_as_uint(r.f[i]) & 0x7fffffffu);
    top = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(top))));
    top = std::max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    const int e = doe::mx4_query_exp(top);
    _Float16 *q = reinterpret_cast<_Float16 *>(sm.q);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int d = (lane & 31) * N + i, in = d % (D / 4);
        const float v = head < heads ? __builtin_amdgcn_ldexpf(r.f[i], e) : 0.0f;
        const _Float16 h = (_Float16)v;
        _Float16 *to = q + ((in / 8) * 64 + d / (D / 4) * 16 + head) * 8 + in % 8;
        to[0] = h;
        to[64] = (_Float16)(v - (float)h);
    }
    if ((lane & 31) == 0) {
        const float f = a.softcap > 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
        sm.rowf[head] = doe::mx4_factor(f, top, e);
    }
}

template <int D, bool NT>
__global__ __launch_bounds__(64 * kWaves, per_cu<D>()) void attn_mx4_token_kernel(TokenArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    TokenLds<D> &sm = *reinterpret_cast<TokenLds<D> *>(lds_raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g4 = lane >> 4, shift = a.c.page_shift;
    const int rows_of = a.c.kv_heads * a.groups;  // rows of a sequence
    // the sequences b0 .. b0 + 63, a lane each: their lengths and the pieces of their rows
    int b0 = 0, lens = 0, pieces_ = 0;
    uint32_t share = 0;
    auto read_lens = [&](int from) __attribute__((always_inline)) {
        b0 = from;
        lens = b0 + lane < a.c.batch ? doe::mx4_len(a.c, b0 + lane) : 0;
    };
    auto cut = [&] { pieces_ = b0 + lane < a.c.batch ? (int)(((uint32_t)blocks_of(a, lens) + share - 1) / share) : 0; };
    auto sum_of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(doe::wave_scan(v), 63) * rows_of; };
    int item = blockIdx.x, items0 = 0, slots0 = 0;  // items and split ones before sequence b0
    bool dense = true;                              // as many slots as items
    const bool one = a.c.batch == 1 && a.by_row;
    if (a.per_row) {
        read_lens(item / rows_of);
    } else if (one) {
        // one sequence: as many pieces a row as workgroups, of a round of the waves at least
        read_lens(0);
        const uint32_t n = blocks_of(a, __builtin_amdgcn_readfirstlane(lens));
        pieces_ = std::min(gridDim.x / rows_of, (n + kWaves - 1) / kWaves);
        share = (n + pieces_ - 1) / (uint32_t)pieces_;
        pieces_ = (n + share - 1) / share;
    } else {
        // the share of an item: the least that leaves no more items than workgroups, of
        // an even share, a half more at most, and what does in any case (with few rows
        // there are at most blocks / share + rows items, else those of split rows are at
        // most twice blocks / share)
        int sum = 0, items = INT_MAX;
        for (int from = (a.c.batch - 1) & ~63; from >= 0; from -= 64) {
            read_lens(from);
            sum += b0 + lane < a.c.batch ? blocks_of(a, lens) : 0;
        }
        const uint32_t total = (uint32_t)sum_of(sum), rows = a.c.batch * rows_of;
        const uint32_t even = (total + gridDim.x - 1) / gridDim.x, room = rows <= gridDim.x / 2 ? gridDim.x - rows : gridDim.x / 2;
        auto rounded = [](uint32_t n) { return n <= 4 * kWaves ? (n + kWaves - 1) & -kWaves : n; };  // whole rounds of the waves
        for (int more = 0; more < 5 && a.c.batch <= 64 && items > (int)gridDim.x; ++more) {
            share = rounded(even + even * more / 8);
            cut();
            items = sum_of(pieces_);
        }
        if (items > (int)gridDim.x) {
            share = rounded((total + room - 1) / room);
            int split = 0;
            items = 0;
            for (int from = (a.c.batch - 1) & ~63; from >= 0; from -= 64) {
                read_lens(from);
                cut();
                items += pieces_;
                split += pieces_ > 1 ? pieces_ : 0;
            }
            items = sum_of(items);
            split = sum_of(split);
            dense = items <= (int)gridDim.x;
            if (!dense) items = split;
        }
        if (!a.by_row && tid == 0 && (int)blockIdx.x >= items) a.joined[blockIdx.x] = make_int2(-1, 0);  // of no row
    }
    for (bool again = false;; again = true) {
        if (again) {  // (rarely: read once more rather than held over a row)
            item += gridDim.x;
            read_lens(b0);
            if (!a.per_row) cut();
            if (one) return;
        }
        int b, pieces = 1, first_item, first_slot = 0;
        if (a.per_row) {
            if (item != (int)blockIdx.x) return;
            b = b0;
            first_item = b * rows_of;
        } else if (one) {
            b = first_item = 0;
            pieces = __builtin_amdgcn_readfirstlane(pieces_);
            if (item >= pieces * rows_of) return;
        } else {
            for (;;) {
                if (b0 >= a.c.batch) return;
                const int upto = doe::wave_scan(pieces_);
                const uint64_t behind = __ballot(items0 + upto * rows_of > item);
                const int split = dense ? 0 : doe::wave_scan(pieces_ > 1 ? pieces_ : 0);
                if (behind) {
                    const int i = __builtin_ctzll(behind);
                    pieces = __builtin_amdgcn_readlane(pieces_, i);
                    b = b0 + i;
                    first_item = items0 + (__builtin_amdgcn_readlane(upto, i) - pieces) * rows_of;
                    first_slot = dense ? first_item : slots0 + (__builtin_amdgcn_readlane(split, i) - (pieces > 1 ? pieces : 0)) * rows_of;
                    break;
                }
                items0 += __builtin_amdgcn_readlane(upto, 63) * rows_of;
                slots0 += __builtin_amdgcn_readlane(split, 63) * rows_of;
                read_lens(b0 + 64);
                cut();
            }
        }
        const int hi = __builtin_amdgcn_readlane(lens, b - b0), lo = first_seen(a, hi), n = blocks_of(a, hi);
        const int r = (uint32_t)(item - first_item) / (uint32_t)pieces, piece = item - first_item - r * pieces;
        const int per = ((uint32_t)n + pieces - 1) / (uint32_t)pieces, first = piece * per, last = std::min(n, first + per);
        const int kvh = r / a.groups, head0 = kvh * a.group + (r - kvh * a.groups) * a.heads;
        const int heads = std::min(a.heads, (kvh + 1) * a.group - head0);
        const int blk0 = lo / 32 + first + wave, count = (last - first - wave + kWaves - 1) / kWaves;
        // the pages of up to 64 of this wave's blocks, a lane each; -1: none to see
        const int32_t *table = a.c.table + (int64_t)b * a.c.table_stride;
        auto pages = [&](int i0) __attribute__((always_inline)) {
            const int blk = blk0 + kWaves * (i0 + lane);
            int page = -1;
            if (i0 + lane < count && blk * 32 < hi) page = table[blk >> (shift - 5)];
            return page < a.c.num_pages ? page : -1;
        };
        int list = pages(0);
        RawQuery<D> raw;
        read_query<D>(raw, a, ((int64_t)b * a.num_heads + head0) * D, heads, wave, lane);
        auto slab_of = [&](int page) __attribute__((always_inline)) {
            return a.c.pool + ((int64_t)std::max(page, 0) * a.c.kv_heads + kvh) * Mx4Slab<D>::bytes(shift);
        };
        auto place = [&](int i) __attribute__((always_inline)) { return ((blk0 + kWaves * i) * 32) & ((1 << shift) - 1); };
        int in_wave = lane;
        __asm__ volatile("" : "+v"(in_wave));
        const Place<D> at_lane(in_wave & 15, in_wave >> 4);
        KBlock<D> kb;
        VBlock<D> vb;
        int page = __builtin_amdgcn_readfirstlane(list);
        load_k<D, NT>(kb, slab_of(page), shift, place(0), at_lane);
        load_v<D, NT>(vb, slab_of(page), shift, place(0), at_lane);
        stage_query<D>(a, raw, sm, heads, wave, lane);  // (while the first block is under way)
        __syncthreads();
        const Mx4Factor rowf = sm.rowf[c16 & 7];
        const float lo_part = c16 < 8 ? 0.0f : 1.0f;
        const bool large = __any(rowf.pre != 1.0f);
        State<D> st;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) st.o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        st.m = -INFINITY;
        st.l = 0.0f;
        for (int i = 0; i < count; ++i) {
            // the next block's K follows this one's into its registers, and V likewise
            // (the last block again at the end: not used)
            const int in = std::min(i + 1, count - 1);
            if ((in & 63) == 0 && in) list = pages(in);
            const int next = __builtin_amdgcn_readlane(list, in & 63);
            const uint8_t *slab = slab_of(next);
            const int p0 = (blk0 + kWaves * i) * 32, top = page < 0 ? 0 : hi;
            f32x4 s[2];
            scores<D>(s, sm.q, kb, lane, g4);
            __builtin_amdgcn_sched_barrier(0);
            load_k<D, NT>(kb, slab, shift, place(in), at_lane);
            __builtin_amdgcn_sched_barrier(0);
            const h8 pf = weights<D>(a, st, s, rowf, large, lo_part, p0, lo, top, g4);
            values<D>(st, pf, vb, p0, lo, top, c16, g4);
            __builtin_amdgcn_sched_barrier(0);
            load_v<D, NT>(vb, slab, shift, place(in), at_lane);
            __builtin_amdgcn_sched_barrier(0);
            page = next;
        }
        // the row's four waves together (the lane's places formed anew: held over the
        // blocks they would take the registers that O needs)
        int tid = threadIdx.x;
        __asm__ volatile("" : "+v"(tid));
        const int lane = tid & 63, c16 = lane & 15, g4 = lane >> 4;
        float l = st.l + __shfl_xor(st.l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (lane < kHeads) sm.ml[wave][lane] = make_float2(st.m, l);
        __syncthreads();
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sm.ml[w][c16 & 7].x);
        const float corr = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - M);
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = st.o[t][i] * corr;
                st.o[t][i] = v + other_half(v);
            }
        if (c16 < kHeads) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float *to = &sm.o[wave][c16][(4 * g4 + i) * (D / 16)];
#pragma unroll
                for (int t = 0; t + 1 < D / 16; t += 2) *reinterpret_cast<float2 *>(to + t) = make_float2(st.o[t][i], st.o[t + 1][i]);
            }
        }
        __syncthreads();
        const int slot = first_slot + r * pieces + piece;
        for (int e = tid; e < heads * (D / 4); e += 64 * kWaves) {
            const int h = e / (D / 4), d = (e - h * (D / 4)) * 4;
            float M2 = -INFINITY, lt = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) M2 = fmaxf(M2, sm.ml[w][h].x);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float2 ml = sm.ml[w][h];
                const float4 o = *reinterpret_cast<const float4 *>(&sm.o[w][h][d]);
                lt += ml.x == -INFINITY ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - M2);
                v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
            }
            if (pieces > 1) {
                const int64_t p = (int64_t)slot * kHeads + h;
                *reinterpret_cast<float4 *>(a.part + p * D + d) = v;
                if (d == 0) reinterpret_cast<float2 *>(a.part + (int64_t)gridDim.x * kHeads * D)[p] = make_float2(M2, lt);
            } else {
                const float inv = lt != 0.0f ? 1.0f / lt : 0.0f;
                const int64_t to = ((int64_t)b * a.num_heads + head0 + h) * D + d;
                if (a.out_f16) {
                    _Float16 *o = static_cast<_Float16 *>(a.out) + to;
                    o[0] = (_Float16)(v.x * inv), o[1] = (_Float16)(v.y * inv), o[2] = (_Float16)(v.z * inv), o[3] = (_Float16)(v.w * inv);
                } else {
                    *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to) =
                        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                }
            }
        }
        if (!a.per_row && tid == 0) {
            const int row = b * rows_of + r;
            if (!a.by_row && (dense || pieces > 1)) a.joined[slot] = piece || pieces == 1 ? make_int2(-1, 0) : make_int2(row, pieces);
            if (a.by_row && piece == 0) a.joined[row] = make_int2(pieces > 1 ? slot : -1, pieces);
        }
    }
}

// A split row's head: its parts, in the order of a fixed tree.  D / 4 lanes hold the
// dims, kJoin / (D / 4) groups take every so manieth part and meet in LDS.  2.7 - 4.7
// us: a dependent launch and two reads after one another, whatever the parts.
constexpr int kJoin = 512;
template <int D>
__global__ __launch_bounds__(kJoin) void attn_mx4_join_kernel(TokenArgs a, int wgs) {
    constexpr int L = D / 4, GROUPS = kJoin / L;
    __shared__ float4 so[GROUPS][L];
    __shared__ float2 sml[GROUPS];
    const int2 j = a.joined[blockIdx.x];
    if (j.x < 0) return;
    const int row = a.by_row ? (int)blockIdx.x : j.x, slot = a.by_row ? j.x : (int)blockIdx.x, pieces = j.y;
    const int rows_of = a.c.kv_heads * a.groups, b = row / rows_of, r = row - b * rows_of, kvh = r / a.groups;
    const int head0 = kvh * a.group + (r - kvh * a.groups) * a.heads, h = blockIdx.y;
    if (h >= std::min(a.heads, (kvh + 1) * a.group - head0)) return;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (int64_t)wgs * kHeads * D);
    const int grp = threadIdx.x / L, d = (threadIdx.x - grp * L) * 4;
    float M = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < GROUPS) {
#pragma unroll 4
        for (int s = grp; s < pieces; s += GROUPS) {
            const int64_t p = (int64_t)(slot + s) * kHeads + h;
            const float2 e = ml[p];
            const float4 o = *reinterpret_cast<const float4 *>(a.part + p * D + d);
            const float mn = fmaxf(M, e.x), f0 = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mn);
            const float f1 = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - mn);
            M = mn;
            l = l * f0 + e.y * f1;
            v.x = v.x * f0 + o.x * f1, v.y = v.y * f0 + o.y * f1, v.z = v.z * f0 + o.z * f1, v.w = v.w * f0 + o.w * f1;
        }
        so[grp][d / 4] = v;
        if (d == 0) sml[grp] = make_float2(M, l);
    }
    __syncthreads();
    if (grp > 0) return;
    for (int g = 0; g < GROUPS; ++g) M = fmaxf(M, sml[g].x);
    l = 0.0f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < GROUPS; ++g) {
        const float2 e = sml[g];
        const float4 o = so[g][d / 4];
        const float f = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - M);
        l += e.y * f;
        v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const int64_t to = ((int64_t)b * a.num_heads + head0 + h) * D + d;
    if (a.out_f16) {
        _Float16 *o = static_cast<_Float16 *>(a.out) + to;
        o[0] = (_Float16)(v.x * inv), o[1] = (_Float16)(v.y * inv), o[2] = (_Float16)(v.z * inv), o[3] = (_Float16)(v.w * inv);
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

template <int D>
int64_t workspace() {
    return (int64_t)workgroups<D>() * (kHeads * (D + 2) * 4 + 8);
}

int64_t workspace_of(int64_t head_dim) {
    switch (head_dim) {
        case 64: return workspace<64>();
        case 128: return workspace<128>();
        case 160: return workspace<160>();
        case 256: return workspace<256>();
        default: return workspace<512>();
    }
}

template <int D, bool NT>
int launch_token(const TokenArgs &a, unsigned wgs, hipStream_t st) {
    static const hipError_t attr_rc = hipFuncSetAttribute((const void *)attn_mx4_token_kernel<D, NT>,
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(TokenLds<D>));
    DOE_HIP_CHECK(attr_rc);
    hipLaunchKernelGGL((attn_mx4_token_kernel<D, NT>), dim3(wgs), dim3(64 * kWaves), sizeof(TokenLds<D>), st, a);
    DOE_LAUNCH_CHECK("attn_mx4_token_kernel");
    return DOE_OK;
}

// Whether a call reads its pages past the 256 MB last-level cache: when it may read
// more than half of that, up to head_dim 128 and with one row a KV head.  Up to there a
// lane has its piece of K in one load; wider ones take several, and further rows the
// same pages again, each a read of memory.  Past the cache and through it, pools of
// layers in turn (one pool again and again in brackets), 16 sequences: 4 KV heads of 128
// with 8 heads each 70 MB 23.7 and 24.2 us (22.7, 22.0), 140 MB 34.5 and 36.2 (33.6,
// 31.6), 290 MB 58.0 and 62.8 (58.2, 56.7); with 16 heads each 290 MB 107 and 96; of
// 256 290 MB 80 and 62, of 512 123 and 67; 16 of 160 74 and 64.
template <int D>
bool past_caches(const TokenArgs &a) {
    if (D > 128 || a.groups > 1) return false;
    int64_t pages = a.c.table_stride;  // of a sequence
    if (a.window > 0) pages = std::min<int64_t>(pages, (a.window >> a.c.page_shift) + 2);
    pages = std::min<int64_t>(a.c.num_pages, pages * a.c.batch);
    return (pages * a.c.kv_heads * (D + D / 16) << a.c.page_shift) > ((int64_t)128 << 20);
}

template <int D>
int launch(TokenArgs &a, void *ws, hipStream_t st) {
    const int64_t rows = (int64_t)a.c.batch * a.c.kv_heads * a.groups;
    int64_t most = ((int64_t)a.c.table_stride << a.c.page_shift) / 32;  // blocks of a row, as far as the host knows
    if (a.window > 0) most = std::min<int64_t>(most, a.window / 32 + 2);
    a.per_row = most <= 2 * kWaves || rows * most >= ((int64_t)1 << 31);
    int64_t wgs = rows;
    if (!a.per_row) {
        wgs = std::min<int64_t>(workgroups<D>(), rows * ((most + kWaves - 1) / kWaves));
        a.by_row = rows <= wgs;
        a.part = static_cast<float *>(ws);
        a.joined = reinterpret_cast<int2 *>(a.part + wgs * kHeads * (D + 2));
    }
    const int rc = past_caches<D>(a) ? launch_token<D, D <= 128>(a, (unsigned)wgs, st) : launch_token<D, false>(a, (unsigned)wgs, st);
    if (rc) return rc;
    if (a.per_row) return DOE_OK;
    hipLaunchKernelGGL(attn_mx4_join_kernel<D>, dim3((unsigned)(a.by_row ? rows : wgs), (unsigned)a.heads), dim3(kJoin), 0, st, a,
                       (int)wgs);
    DOE_LAUNCH_CHECK("attn_mx4_join_kernel");
    return DOE_OK;
}

}  // namespace

extern "C" {

int doe_attn_mx4_decode_workspace(int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                  int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    int64_t page = 0;
    const int rc = doe_mx4_page_bytes(32, num_kv_heads, head_dim, &page);
    if (rc) return rc;
    DOE_REQUIRE(batch >= 0 && batch <= 65535 && num_heads > 0 && num_heads <= 65535 && num_heads % num_kv_heads == 0,
                DOE_E_INVALID, "batch %lld, %lld heads over %lld", (long long)batch, (long long)num_heads, (long long)num_kv_heads);
    *bytes = workspace_of(head_dim);
    return DOE_OK;
}

int doe_attn_mx4_decode(const doe_mx4_cache *cache, const void *q, int q_f16, void *out, int out_f16, int64_t num_heads,
                        float scale, float softcap, int64_t sliding_window, void *workspace, int64_t workspace_bytes,
                        doe_stream_t stream) {
    TokenArgs a{};
    int rc = doe::mx4_view(cache, &a.c);
    if (rc) return rc;
    if ((rc = doe::mx4_attention_checks(a.c, num_heads, scale, softcap, sliding_window, q, out))) return rc;
    const int64_t need = workspace_of(cache->head_dim);
    DOE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need, DOE_E_INVALID,
                "a 16-byte aligned workspace of %lld bytes is needed (got %lld)", (long long)need, (long long)workspace_bytes);
    a.q = q;
    a.out = out;
    a.q_f16 = q_f16 != 0;
    a.out_f16 = out_f16 != 0;
    a.num_heads = (int)num_heads;
    a.group = (int)(num_heads / a.c.kv_heads);
    a.groups = (a.group + kHeads - 1) / kHeads;
    a.heads = (a.group + a.groups - 1) / a.groups;
    a.groups = (a.group + a.heads - 1) / a.heads;
    a.window = (int)sliding_window;
    a.scale = scale;
    a.softcap = softcap;
    DOE_REQUIRE((int64_t)a.c.batch * a.c.kv_heads * a.groups < ((int64_t)1 << 24), DOE_E_UNSUPPORTED, "batch %d of %d KV heads",
                a.c.batch, a.c.kv_heads);  // (a workgroup each: a launch has fewer than 2^32 threads)
    if ((rc = doe::require_init())) return rc;
    if (a.c.batch == 0) return DOE_OK;
    switch (cache->head_dim) {
        case 64: return launch<64>(a, workspace, (hipStream_t)stream);
        case 128: return launch<128>(a, workspace, (hipStream_t)stream);
        case 160: return launch<160>(a, workspace, (hipStream_t)stream);
        case 256: return launch<256>(a, workspace, (hipStream_t)stream);
        default: return launch<512>(a, workspace, (hipStream_t)stream);
    }
}

}  // extern "C"
