// mx4_cache.hip -- K / V rows into the paged cache held in 4 bits, and back.
//
// Quantisation of a block of 32 values x: a = max |x|, e = floor(log2 a) - 2,
// one more where a / 2^floor(log2 a) >= 1.75 (a then rounds to the next power of
// two among the codes), held within [-23, 13] so that every value is exact in
// f16; codes are the nearest E2M1 value of x 2^-e (exact in f32), ties to the
// even code, at most 6.  v_cvt_scalef32_pk_fp4_f32 rounds so: checked against
// comparisons over all codes' borders and their neighbours.  A block with an
// infinity or a NaN keeps scale byte 255 (codes 0) and reads as NaN throughout.
#include "mx4_cache.h"
#include "rope_rows.h"

#include <math.h>
#include <algorithm>

namespace {

using doe::Mx4Slab;
using doe::Mx4View;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

struct RowArgs {
    Mx4View c;
    const void *k, *v;
    float *k_out, *v_out;
    const int32_t *row_starts;
    int64_t rows, row_stride;
    // a rotating call: the workgroups from kv_wgs on take the queries
    doe::RopeRows r;
    int kv_wgs, q_rows, q_ways;
};

// The queries' part of a rotating call; false: this workgroup is one of the cache's.  They
// are read and written past the caches, which the codes alone then fill: 1900 rows of 32 /
// 16 heads of 256 appended and read back (364 MB) 75 to 64 us, attention behind it as fast.
__device__ __forceinline__ bool queries(const RowArgs &a, int head_dim, int *s_pos) {
    const int wg = (int)blockIdx.x - a.kv_wgs;
    if (wg < 0) return false;
    const int64_t row0 = (int64_t)(wg / a.q_ways) * a.q_rows;
    const int count = a.rows - row0 < a.q_rows ? (int)(a.rows - row0) : a.q_rows;
    doe::rotate_queries<true>(a.r, a.c.lens, doe::mx4_room(a.c), a.c.batch, a.row_starts, row0, count, head_dim,
                        wg % a.q_ways, s_pos);
    return true;
}
// The angles that dims d .. d + 3 of a head turn by at a position (of a rotated head whole,
// else its first two); where they do not turn, whatever lies at K's first row.
struct Angles {
    doe::f4 first, second;
};
__device__ __forceinline__ Angles angles_of(const RowArgs &a, int d, int pos) {
    const doe::RopeRows &r = a.r;
    const int half = r.rotary_dim / 2;
    const float *at = d < r.rotary_dim && pos < r.max_positions
                          ? r.freq + (int64_t)pos * r.rotary_dim + (r.interleaved ? d : 2 * (d < half ? d : d - half))
                          : static_cast<const float *>(a.k);
    return {*reinterpret_cast<const doe::f4 *>(at), *reinterpret_cast<const doe::f4 *>(at + (d < r.rotary_dim && !r.interleaved ? 4 : 0))};
}
// Dims d .. d + 3 of a head at `head`, of which `own` has been read, rotated.  The other
// dims of its pairs are another lane's of the head (D / 4 lanes, four dims each): in this
// wave up to 256 dims, read again from 512.
template <int D>
__device__ __forceinline__ float4 rotated(const RowArgs &a, const float4 own_, const float *head, int d, const Angles &t) {
    const doe::RopeRows &r = a.r;
    const doe::f4 own = {own_.x, own_.y, own_.z, own_.w};
    doe::f4 out = own;
    const int half = r.rotary_dim / 2;
    if (r.interleaved) {
        if (d < r.rotary_dim) out = doe::rotate_pairs(own, t.first);
    } else {
        const int other_d = d < half ? d + half : d - half;
        doe::f4 other;
        if constexpr (D <= 256 && D != 160) {
            const int lane = (threadIdx.x & 63) + (other_d - d) / 4;  // (past the rotated dims: not used)
#pragma unroll
            for (int i = 0; i < 4; ++i) other[i] = __shfl(own[i], lane, 64);
        } else {
            other = *reinterpret_cast<const doe::f4 *>(head + (d < r.rotary_dim ? other_d : d));
        }
        if (d < r.rotary_dim) {
            doe::f4 lo = d < half ? own : other, hi = d < half ? other : own;
            doe::rotate_halves(lo, hi, t.first, t.second);
            out = d < half ? lo : hi;
        }
    }
    return make_float4(out[0], out[1], out[2], out[3]);
}

// Bits of the largest magnitude over each 8 lanes, an infinity's or NaN's above
// all others (as numbers a maximum would drop a NaN).
__device__ __forceinline__ uint32_t max8(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));   // lane ^ 1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));   // lane ^ 2
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // the other four of eight
}

// The 4-bit codes of four values of a block that eight lanes hold (16 bits),
// and the block's scale byte.
__device__ __forceinline__ uint32_t quantise(const float4 x, int &scale) {
    const uint32_t m = 0x7fffffffu;
    const uint32_t top = max8(max(max(__float_as_uint(x.x) & m, __float_as_uint(x.y) & m),
                                  max(__float_as_uint(x.z) & m, __float_as_uint(x.w) & m)));
    int e = (int)((top + 0x200000u) >> 23) - 129;
    e = e < doe::kMx4MinExp ? doe::kMx4MinExp : (e > doe::kMx4MaxExp ? doe::kMx4MaxExp : e);
    scale = top < 0x7f800000u ? e + 127 : doe::kMx4NanScale;
    const float s = __uint_as_float((uint32_t)(e + 127) << 23);
    // (values beyond 6 x 2^13 only where e was held at 13)
    const float lim = 6.0f * s;
    auto in = [&](float v) { return fminf(fmaxf(v, -lim), lim); };
    uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, in(x.x), in(x.y), s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, in(x.z), in(x.w), s, 1) & 0xffffu;
    return scale == doe::kMx4NanScale ? 0u : q;
}

constexpr int kRowsPerWg = 16;
static_assert(kRowsPerWg >= doe::kRopeRowsPerWg, "positions of a workgroup's rows");

// One row's place, found once for a workgroup's rows.
struct Place {
    int64_t page;  // page * kv_heads, -1: none
    int x;
};

// head_dim 160, whose columns of V are ten dims.  A workgroup takes kRowsPerWg rows; a
// thread four dims of K and V of a row's head.  10430 rows of 16 heads (f32: 214 MB and 28
// of codes) are written in 87 us and read in 62 (2.8 and 3.9 TB/s), f16 written in 74: two
// bytes of K and one of V a store.
// ROPE: K is rotated on the way, and the queries with it.
template <bool F16, bool ROPE = false>
__global__ __launch_bounds__(256) void mx4_write_kernel(RowArgs a) {
    constexpr int D = 160;
    __shared__ Place place[kRowsPerWg];
    __shared__ int positions[ROPE ? kRowsPerWg : 1];
    if constexpr (ROPE) {
        if (queries(a, D, positions)) return;
    }
    const int64_t row0 = (int64_t)blockIdx.x * kRowsPerWg;
    if (threadIdx.x < kRowsPerWg) {
        const int64_t row = row0 + threadIdx.x;
        Place p{-1, 0};
        int b, pos;
        if (row < a.rows && doe::row_position(a.c.lens, doe::mx4_room(a.c), a.c.batch, a.row_starts, row, b, pos) && pos >= 0) {
            const int page = doe::mx4_page(a.c, b, pos);
            if (page >= 0) p = Place{(int64_t)page * a.c.kv_heads, pos & ((1 << a.c.page_shift) - 1)};
            if constexpr (ROPE) {
                if (pos >= a.r.max_positions) p.page = -1;
                positions[threadIdx.x] = pos;
            }
        }
        place[threadIdx.x] = p;
    }
    __syncthreads();
    using S = Mx4Slab<D>;
    constexpr int QUADS = D / 4;
    const int shift = a.c.page_shift, per_row = a.c.kv_heads * QUADS;
    for (int i = threadIdx.x; i < kRowsPerWg * per_row; i += 256) {
        const int r = i / per_row, in_row = i - r * per_row, head = in_row / QUADS, d = (in_row - head * QUADS) * 4;
        const Place p = place[r];
        if (p.page < 0) continue;
        const int64_t at = (row0 + r) * a.row_stride + (int64_t)head * D + d;
        float4 k, v;
        if constexpr (F16) {
            const h4 kh = *reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(a.k) + at);
            const h4 vh = *reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(a.v) + at);
            k = make_float4((float)kh[0], (float)kh[1], (float)kh[2], (float)kh[3]);
            v = make_float4((float)vh[0], (float)vh[1], (float)vh[2], (float)vh[3]);
        } else {
            k = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.k) + at);
            v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.v) + at);
            if constexpr (ROPE) k = rotated<D>(a, k, static_cast<const float *>(a.k) + at - d, d, angles_of(a, d, positions[r]));
        }
        int ks, vs;
        const uint32_t kc = quantise(k, ks), vc = quantise(v, vs);
        uint8_t *slab = a.c.pool + (p.page + head) * S::bytes(shift);
        *reinterpret_cast<uint16_t *>(slab + S::k_code(p.x) + d / 2) = (uint16_t)kc;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            slab[S::v_code(shift, p.x, (d + 2 * e) / 10) + (d + 2 * e) % 10 / 2] = (uint8_t)(vc >> (8 * e));
        if ((d & 31) == 0) {
            slab[S::k_scale(shift, p.x) + d / 32] = (uint8_t)ks;
            slab[S::v_scale(shift, p.x, d / 32)] = (uint8_t)vs;
        }
    }
}

__device__ __forceinline__ float4 values(uint32_t codes, int scale) {
    const float s = __uint_as_float(scale == doe::kMx4NanScale ? 0x7fc00000u : (uint32_t)scale << 23);
    const h2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 1);
    return make_float4((float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]);
}

__global__ __launch_bounds__(256) void mx4_read_kernel(RowArgs a) {
    constexpr int D = 160;
    __shared__ Place place[kRowsPerWg];
    __shared__ bool mine[kRowsPerWg];
    const int64_t row0 = (int64_t)blockIdx.x * kRowsPerWg;
    if (threadIdx.x < kRowsPerWg) {
        const int64_t row = row0 + threadIdx.x;
        Place p{-1, 0};
        int b, pos;
        if (row < a.rows && doe::row_position(a.c.lens, doe::mx4_room(a.c), a.c.batch, a.row_starts, row, b, pos) && pos >= 0) {
            const int page = doe::mx4_page(a.c, b, pos);
            if (page >= 0) p = Place{(int64_t)page * a.c.kv_heads, pos & ((1 << a.c.page_shift) - 1)};
        }
        place[threadIdx.x] = p;
        // rows of no sequence stay as they were
        mine[threadIdx.x] = row < a.rows && (!a.row_starts || (row >= a.row_starts[0] && row < a.row_starts[a.c.batch]));
    }
    __syncthreads();
    using S = Mx4Slab<D>;
    constexpr int QUADS = D / 4;
    const int shift = a.c.page_shift, per_row = a.c.kv_heads * QUADS;
    for (int i = threadIdx.x; i < kRowsPerWg * per_row; i += 256) {
        const int r = i / per_row, in_row = i - r * per_row, head = in_row / QUADS, d = (in_row - head * QUADS) * 4;
        const Place p = place[r];
        if (!mine[r]) continue;
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
        if (p.page >= 0) {
            const uint8_t *slab = a.c.pool + (p.page + head) * S::bytes(shift);
            const uint32_t kc = *reinterpret_cast<const uint16_t *>(slab + S::k_code(p.x) + d / 2);
            const uint32_t vc = slab[S::v_code(shift, p.x, d / 10) + d % 10 / 2] |
                                (uint32_t)slab[S::v_code(shift, p.x, (d + 2) / 10) + (d + 2) % 10 / 2] << 8;
            k = values(kc, slab[S::k_scale(shift, p.x) + d / 32]);
            v = values(vc, slab[S::v_scale(shift, p.x, d / 32)]);
        }
        const int64_t at = (row0 + r) * a.row_stride + (int64_t)head * D + d;
        *reinterpret_cast<float4 *>(a.k_out + at) = k;
        *reinterpret_cast<float4 *>(a.v_out + at) = v;
    }
}

// ---------------------------------------------------------------------------
// The other head dims: a unit is four consecutive positions, from a multiple of
// four on, of one head, and D / 4 lanes take four dims of each.  V's codes of a
// column's four positions lie in a row (D / 8 bytes), so the lanes hand them round
// through LDS, each to its own wave's lanes only, and move eight bytes each.  The rows of a sequence get rows / 4 + 2 places for units (as
// many as they can touch from any position on), so that a place's sequence is
// found in row_starts.  Both directions are bound by their bytes.  20864 rows of 8
// heads of 128 dims (171 MB of f32, 23 MB of codes) are written in 43 us and read
// in 34 (4.5 and 5.7 TB/s); with a thread on four dims of one position, and V's
// codes two bytes at a time, it was 66 and 45.  Rows are loaded past the caches,
// which the quantised ones alone then fill: it was 58 us before.
// The rows read back are the next kernel's input and stay there.
struct Four {
    int pos0, from, last;  // positions pos0 .. pos0 + 3; those in [from, last] have rows, those below 0 hold nothing
    int64_t row0;          // row of position pos0
    int page;              // -1: none
};
template <int D>
__device__ __forceinline__ bool find_four(const RowArgs &a, Four &f, int &head) {
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / (D / 4), place = unit / a.c.kv_heads;
    head = (int)(unit - place * a.c.kv_heads);
    int b = 0, at = 0, len = 0;
    int64_t n = 0;
    if (a.row_starts) {
        // the last sequence whose places begin at or before this one: a lane a sequence of 64,
        // read once for a wave's units (forty prompts of twenty rows appended and read back: 11.8
        // to 8.7 us from a search by each; 4000 of up to two, 64 dims: 12.0 to 8.9 written and 9.1
        // to 7.4 read from a search by each unit in turn)
        constexpr int LANES = D / 4 < 64 ? D / 4 : 64;
        const int lane = threadIdx.x & 63;
        int from, to, held, lo = 0, left = a.c.batch;
        auto read = [&]() __attribute__((always_inline)) {
            const bool in = lane < left;
            from = in ? a.row_starts[lo + lane] : 0;
            to = in ? a.row_starts[lo + lane + 1] : 0;
            held = in ? doe::mx4_len(a.c, lo + lane) : 0;
        };
        auto begun = [&](int mine) __attribute__((always_inline)) { return __ballot(lane < left && (from >> 2) + 2 * (lo + lane) <= mine); };
        if (left <= 64) read();
        for (int u = 0; u < 64 / LANES; ++u) {
            const int mine = __builtin_amdgcn_readlane((int)place, u * LANES);
            uint64_t before = u || a.c.batch <= 64 ? begun(mine) : 0;
            // (of more sequences the 64 from the first unit's on, and further ones where all of
            // these begin before a unit)
            if (a.c.batch > 64 && (u == 0 || (before >> (left - 1) && lo + left < a.c.batch))) {
                lo = 0;
                for (int all = a.c.batch; all > 64;) {  // 64 ways at a time
                    const int step = (all + 63) >> 6, i = lo + lane * step;
                    const uint64_t at_or_before = __ballot(i < lo + all && (a.row_starts[i] >> 2) + 2 * i <= mine);
                    const int last = at_or_before ? 63 - __builtin_clzll(at_or_before) : 0;
                    lo += last * step;
                    all = std::min(step, all - last * step);
                }
                left = std::min(64, a.c.batch - lo);
                read();
                before = begun(mine);
            }
            if (before == 0) continue;  // (n stays 0)
            const int last = 63 - __builtin_clzll(before);
            if (lane / LANES == u) {
                b = lo + last;
                at = __builtin_amdgcn_readlane(from, last);
                n = (int64_t)__builtin_amdgcn_readlane(to, last) - at;
                len = __builtin_amdgcn_readlane(held, last);
            }
        }
    } else {
        if (place >= a.c.batch) return false;
        b = at = (int)place;
        n = 1;
        len = doe::mx4_len(a.c, b);
    }
    int64_t four = a.row_starts ? place - (at >> 2) - 2 * (int64_t)b : 0;
    if (at < 0 || n <= 0 || four < 0) return false;
    f.from = (int)(len - n);
    f.last = len - 1;
    four += f.from >> 2;
    if (four > (f.last >> 2)) return false;
    f.pos0 = (int)four * 4;
    f.row0 = at + (f.pos0 - f.from);
    f.page = f.pos0 < 0 ? -1 : doe::mx4_page(a.c, b, f.pos0);
    return true;
}

// Codes of V of a unit between the lanes' order (a lane's four dims of position
// i: 16 bits of the 64) and the page's.  LDS operations of a wave are in order.
template <int D>
struct Exchange {
    static constexpr int C = D / 16, PER = C / 4;  // lanes of a column
    uint8_t *mine, *column;
    int at;
    __device__ __forceinline__ explicit Exchange(uint8_t *lds)
        : mine(lds + threadIdx.x * 8), column(lds + (threadIdx.x / PER) * PER * 8), at(threadIdx.x % PER * 2) {}
    __device__ __forceinline__ uint64_t to_page(const uint32_t *codes) const {
        if constexpr (PER == 1) return codes[0] | codes[1] << 16 | (uint64_t)(codes[2] | codes[3] << 16) << 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint16_t *>(column + i * (C / 2) + at) = (uint16_t)codes[i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        return *reinterpret_cast<const uint64_t *>(mine);
    }
    __device__ __forceinline__ void from_page(uint64_t w, uint32_t *codes) const {
        if constexpr (PER == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) codes[i] = (uint32_t)(w >> (16 * i)) & 0xffff;
        } else {
            *reinterpret_cast<uint64_t *>(mine) = w;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int i = 0; i < 4; ++i) codes[i] = *reinterpret_cast<const uint16_t *>(column + i * (C / 2) + at);
        }
    }
};

template <int D, bool F16, bool ROPE = false>
__global__ __launch_bounds__(256) void mx4_write_fours_kernel(RowArgs a) {
    using S = Mx4Slab<D>;
    constexpr int C = D / 16;
    __shared__ __align__(16) uint8_t lds[256 * 8];
    if constexpr (ROPE) {
        if (queries(a, D, reinterpret_cast<int *>(lds))) return;
    }
    const Exchange<D> x(lds);
    Four f;
    int head;
    if (!find_four<D>(a, f, head) || f.page < 0) return;  // (all lanes of a unit)
    const int shift = a.c.page_shift, x0 = f.pos0 & ((1 << shift) - 1), d = threadIdx.x % (D / 4) * 4;
    uint8_t *slab = a.c.pool + ((int64_t)f.page * a.c.kv_heads + head) * S::bytes(shift);
    float4 k[4], v[4];
    Angles angles[ROPE ? 4 : 1] = {};
    // the row of position i; where the unit has none there, of the nearest that it has
    auto held = [&](int i) __attribute__((always_inline)) { return std::max(f.from - f.pos0, std::min(i, f.last - f.pos0)); };
    auto row_at = [&](int i) __attribute__((always_inline)) {
        return std::max<int64_t>(0, std::min<int64_t>(f.row0 + held(i), a.rows - 1)) * a.row_stride + (int64_t)head * D;
    };
    auto read = [&](int i) __attribute__((always_inline)) {
        const int64_t at = row_at(i) + d;
        if constexpr (F16) {
            const h4 kh = __builtin_nontemporal_load(reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(a.k) + at));
            const h4 vh = __builtin_nontemporal_load(reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(a.v) + at));
            k[i] = make_float4((float)kh[0], (float)kh[1], (float)kh[2], (float)kh[3]);
            v[i] = make_float4((float)vh[0], (float)vh[1], (float)vh[2], (float)vh[3]);
        } else {
            const f4 kf = __builtin_nontemporal_load(reinterpret_cast<const f4 *>(static_cast<const float *>(a.k) + at));
            const f4 vf = __builtin_nontemporal_load(reinterpret_cast<const f4 *>(static_cast<const float *>(a.v) + at));
            k[i] = make_float4(kf[0], kf[1], kf[2], kf[3]);
            v[i] = make_float4(vf[0], vf[1], vf[2], vf[3]);
            if constexpr (ROPE) angles[i] = angles_of(a, d, f.pos0 + held(i));
        }
    };
    auto turn = [&](int i) __attribute__((always_inline)) {
        if constexpr (ROPE) k[i] = rotated<D>(a, k[i], static_cast<const float *>(a.k) + row_at(i), d, angles[i]);
    };
    auto put_k = [&](int at, const float4 &row) __attribute__((always_inline)) {
        int ks;
        const uint32_t kc = quantise(row, ks);
        *reinterpret_cast<uint16_t *>(slab + S::k_code(at) + d / 2) = (uint16_t)kc;
        if ((d & 31) == 0) slab[S::k_scale(shift, at) + d / 32] = (uint8_t)ks;
    };
    auto put_v = [&](int at, uint32_t vc, int vs) __attribute__((always_inline)) {
        *reinterpret_cast<uint16_t *>(slab + S::v_code(shift, at, d / C) + d % C / 2) = (uint16_t)vc;
        if ((d & 31) == 0) slab[S::v_scale(shift, at, d / 32)] = (uint8_t)vs;
    };
    if (!a.row_starts) {
        // one row a unit (4096 of 8 heads of 512: 42 us, 72 as a unit of four that lacks three)
        const int i = held(0);
        if (ROPE && f.pos0 + i >= a.r.max_positions) return;
        read(0);
        turn(0);
        put_k(x0 + i, k[0]);
        int vs;
        const uint32_t vc = quantise(v[0], vs);
        put_v(x0 + i, vc, vs);
        return;
    }
    // (all of a unit's reads before the first of them is used, and for the positions that it lacks
    // a row that it has: a read that a condition guards is waited for by itself)
#pragma unroll
    for (int i = 0; i < 4; ++i) read(i);
#pragma unroll
    for (int i = 0; i < 4; ++i) turn(i);
    bool in[4], all = true;
    uint32_t vc[4] = {};
    int vs[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        in[i] = f.pos0 + i >= f.from && f.pos0 + i <= f.last && f.row0 + i < a.rows;
        if constexpr (ROPE) in[i] = in[i] && f.pos0 + i < a.r.max_positions;
        all = all && in[i];
        if (!in[i]) continue;
        put_k(x0 + i, k[i]);
        vc[i] = quantise(v[i], vs[i]);
    }
    if (all) {
        const uint64_t w = x.to_page(vc);
        *reinterpret_cast<uint64_t *>(slab + S::v_code(shift, x0, d / C) + d % C * 2) = w;
        if ((d & 31) == 0)
            *reinterpret_cast<uint32_t *>(slab + S::v_scale(shift, x0, d / 32)) = vs[0] | vs[1] << 8 | vs[2] << 16 | (uint32_t)vs[3] << 24;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in[i]) put_v(x0 + i, vc[i], vs[i]);
    }
}

template <int D>
__global__ __launch_bounds__(256) void mx4_read_fours_kernel(RowArgs a) {
    using S = Mx4Slab<D>;
    constexpr int C = D / 16;
    __shared__ __align__(16) uint8_t lds[256 * 8];
    const Exchange<D> x(lds);
    Four f;
    int head;
    if (!find_four<D>(a, f, head)) return;  // (all lanes of a unit)
    const int shift = a.c.page_shift, x0 = f.pos0 & ((1 << shift) - 1), d = threadIdx.x % (D / 4) * 4;
    uint32_t kc[4] = {}, vc[4] = {}, vs = 0;
    int ks[4] = {};
    if (f.page >= 0) {
        const uint8_t *slab = a.c.pool + ((int64_t)f.page * a.c.kv_heads + head) * S::bytes(shift);
        const uint64_t w = *reinterpret_cast<const uint64_t *>(slab + S::v_code(shift, x0, d / C) + d % C * 2);
        vs = *reinterpret_cast<const uint32_t *>(slab + S::v_scale(shift, x0, d / 32));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kc[i] = *reinterpret_cast<const uint16_t *>(slab + S::k_code(x0 + i) + d / 2);
            ks[i] = slab[S::k_scale(shift, x0 + i) + d / 32];
        }
        x.from_page(w, vc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = f.row0 + i;
        if (f.pos0 + i < f.from || f.pos0 + i > f.last || row >= a.rows) continue;
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;  // (positions below 0, pages outside the pool)
        if (f.page >= 0) {
            k = values(kc[i], ks[i]);
            v = values(vc[i], vs >> (8 * i) & 0xff);
        }
        const int64_t at = row * a.row_stride + (int64_t)head * D + d;
        *reinterpret_cast<float4 *>(a.k_out + at) = k;
        *reinterpret_cast<float4 *>(a.v_out + at) = v;
    }
}

int row_checks(const Mx4View &c, int64_t head_dim, int64_t rows, int64_t row_stride, const int32_t *row_starts,
               const void *k, const void *v, int size) {
    DOE_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31), DOE_E_INVALID, "rows %lld", (long long)rows);
    DOE_REQUIRE(row_starts || rows == c.batch, DOE_E_INVALID, "without row_starts a call takes one row a sequence (%lld rows, batch %d)",
                (long long)rows, c.batch);
    DOE_REQUIRE(row_stride >= c.kv_heads * head_dim && row_stride * size % 16 == 0, DOE_E_INVALID,
                "row stride %lld below a row of %lld, or not a multiple of 16 bytes", (long long)row_stride,
                (long long)(c.kv_heads * head_dim));
    // (a launch has fewer than 2^32 threads; without row_starts a unit a sequence)
    DOE_REQUIRE((row_starts ? rows / 4 + 2 * (int64_t)c.batch : rows) * c.kv_heads * (head_dim == 160 ? 64 : head_dim / 4) <
                    ((int64_t)1 << 32) - 256,
                DOE_E_UNSUPPORTED, "%lld rows and %d sequences of %d heads", (long long)rows, c.batch, c.kv_heads);
    DOE_REQUIRE(rows == 0 || (k && v), DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, DOE_E_INVALID, "k and v must be 16-byte aligned");
    return DOE_OK;
}

// Workgroups for the rows' units.
template <int D>
dim3 fours_grid(const RowArgs &a) {
    const int64_t places = a.row_starts ? a.rows / 4 + 2 * (int64_t)a.c.batch : a.c.batch;
    return dim3((unsigned)((places * a.c.kv_heads * (D / 4) + 255) / 256));
}
dim3 rows_grid(const RowArgs &a) { return dim3((unsigned)((a.rows + kRowsPerWg - 1) / kRowsPerWg)); }

template <int D>
void launch_write(bool f16, hipStream_t st, const RowArgs &a) {
    if constexpr (D == 160) {
        if (f16) hipLaunchKernelGGL((mx4_write_kernel<true>), rows_grid(a), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((mx4_write_kernel<false>), rows_grid(a), dim3(256), 0, st, a);
    } else {
        if (f16) hipLaunchKernelGGL((mx4_write_fours_kernel<D, true>), fours_grid<D>(a), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((mx4_write_fours_kernel<D, false>), fours_grid<D>(a), dim3(256), 0, st, a);
    }
}

// Rotating: the queries' workgroups behind the cache's.
template <int D>
int launch_append(hipStream_t st, RowArgs &a) {
    const dim3 kv = D == 160 ? rows_grid(a) : fours_grid<D>(a);
    const doe::RopeShare share = doe::rope_share(a.rows, std::max<int64_t>(1, (int64_t)a.r.num_heads * (D / 8)));
    a.q_rows = share.rows_per_wg;
    a.q_ways = share.ways;
    a.kv_wgs = (int)kv.x;
    const unsigned q_wgs = a.r.num_heads ? (unsigned)((a.rows + a.q_rows - 1) / a.q_rows * a.q_ways) : 0;
    DOE_REQUIRE((int64_t)kv.x + q_wgs < (1 << 24), DOE_E_UNSUPPORTED, "%lld rows of %d and %d heads in one call", (long long)a.rows,
                a.r.num_heads, a.c.kv_heads);  // (a launch has fewer than 2^32 threads)
    if constexpr (D == 160) hipLaunchKernelGGL((mx4_write_kernel<false, true>), dim3(kv.x + q_wgs), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mx4_write_fours_kernel<D, false, true>), dim3(kv.x + q_wgs), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("mx4_write_kernel");
    return DOE_OK;
}

template <int D>
void launch_read(hipStream_t st, const RowArgs &a) {
    if constexpr (D == 160) hipLaunchKernelGGL(mx4_read_kernel, rows_grid(a), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mx4_read_fours_kernel<D>), fours_grid<D>(a), dim3(256), 0, st, a);
}

}  // namespace

namespace doe {

int mx4_view(const doe_mx4_cache *cache, Mx4View *view) {
    DOE_REQUIRE(cache, DOE_E_INVALID, "null cache");
    const doe_mx4_cache &c = *cache;
    DOE_REQUIRE(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 160 || c.head_dim == 256 || c.head_dim == 512,
                DOE_E_UNSUPPORTED, "head_dim %lld unsupported (64, 128, 160, 256, 512)", (long long)c.head_dim);
    int shift = 0;
    while (shift < 9 && ((int64_t)1 << shift) != c.page_size) ++shift;
    DOE_REQUIRE(shift >= 5 && shift <= 8, DOE_E_UNSUPPORTED, "page_size %lld unsupported (32, 64, 128, 256)",
                (long long)c.page_size);
    DOE_REQUIRE(c.num_kv_heads > 0 && c.num_kv_heads <= 1024, DOE_E_INVALID, "num_kv_heads %lld outside 1..1024",
                (long long)c.num_kv_heads);
    DOE_REQUIRE(c.num_pages > 0 && c.num_pages < ((int64_t)1 << 31) && c.num_pages * c.num_kv_heads < ((int64_t)1 << 31),
                DOE_E_INVALID, "num_pages %lld of %lld heads", (long long)c.num_pages, (long long)c.num_kv_heads);
    DOE_REQUIRE(c.batch >= 0 && c.batch <= 65535, DOE_E_INVALID, "batch %lld outside 0..65535", (long long)c.batch);
    DOE_REQUIRE(c.table_stride > 0 && c.table_stride * c.page_size < ((int64_t)1 << 30), DOE_E_INVALID,
                "table_stride %lld: a sequence holds fewer than 2^30 positions", (long long)c.table_stride);
    DOE_REQUIRE(c.pool && c.page_table && c.kv_lens, DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)c.pool & 15) == 0, DOE_E_INVALID, "the pool must be 16-byte aligned");
    view->pool = static_cast<uint8_t *>(c.pool);
    view->table = c.page_table;
    view->lens = c.kv_lens;
    view->num_pages = (int)c.num_pages;
    view->page_shift = shift;
    view->kv_heads = (int)c.num_kv_heads;
    view->batch = (int)c.batch;
    view->table_stride = (int)c.table_stride;
    return DOE_OK;
}

int mx4_attention_checks(const Mx4View &c, int64_t num_heads, float scale, float softcap, int64_t sliding_window,
                         const void *q, const void *out) {
    DOE_REQUIRE(num_heads > 0 && num_heads <= 65535 && num_heads % c.kv_heads == 0, DOE_E_INVALID,
                "num_heads %lld is not a positive multiple of num_kv_heads %d", (long long)num_heads, c.kv_heads);
    DOE_REQUIRE(isfinite(scale) && isfinite(softcap) && softcap >= 0.0f, DOE_E_INVALID, "scale %g, softcap %g", (double)scale,
                (double)softcap);
    DOE_REQUIRE(softcap == 0.0f || isfinite(scale / softcap), DOE_E_INVALID, "softcap %g too small for scale %g",
                (double)softcap, (double)scale);
    // (scores and caps are held in powers of two)
    DOE_REQUIRE(isfinite(scale * 1.4426950408889634f) && isfinite(softcap * 1.4426950408889634f), DOE_E_INVALID,
                "scale %g or softcap %g above 2.35e38", (double)scale, (double)softcap);
    DOE_REQUIRE(sliding_window >= 0 && sliding_window < ((int64_t)1 << 30), DOE_E_INVALID, "sliding_window %lld",
                (long long)sliding_window);
    DOE_REQUIRE(c.batch == 0 || (q && out), DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0, DOE_E_INVALID, "q and out must be 16-byte aligned");
    return DOE_OK;
}

}  // namespace doe

extern "C" {

int doe_mx4_page_bytes(int64_t page_size, int64_t num_kv_heads, int64_t head_dim, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    int32_t some = 0;
    doe_mx4_cache c{};
    c.pool = reinterpret_cast<void *>(16);
    c.page_table = c.kv_lens = &some;
    c.num_pages = c.table_stride = 1;
    c.page_size = page_size;
    c.num_kv_heads = num_kv_heads;
    c.head_dim = head_dim;
    Mx4View v;
    const int rc = doe::mx4_view(&c, &v);
    if (rc) return rc;
    *bytes = page_size * num_kv_heads * (head_dim + head_dim / 16);
    return DOE_OK;
}

int doe_mx4_kv_write(const doe_mx4_cache *cache, const void *k, const void *v, int in_f16, int64_t row_stride,
                     const int32_t *row_starts, int64_t rows, doe_stream_t stream) {
    RowArgs a{};
    int rc = doe::mx4_view(cache, &a.c);
    if (rc) return rc;
    if ((rc = row_checks(a.c, cache->head_dim, rows, row_stride, row_starts, k, v, in_f16 ? 2 : 4))) return rc;
    if ((rc = doe::require_init())) return rc;
    if (rows == 0 || a.c.batch == 0) return DOE_OK;
    a.k = k;
    a.v = v;
    a.row_starts = row_starts;
    a.rows = rows;
    a.row_stride = row_stride;
    const hipStream_t st = (hipStream_t)stream;
    switch (cache->head_dim) {
        case 64: launch_write<64>(in_f16, st, a); break;
        case 128: launch_write<128>(in_f16, st, a); break;
        case 160: launch_write<160>(in_f16, st, a); break;
        case 256: launch_write<256>(in_f16, st, a); break;
        default: launch_write<512>(in_f16, st, a); break;
    }
    DOE_LAUNCH_CHECK("mx4_write_kernel");
    return DOE_OK;
}

int doe_mx4_qkv_rope_append(const doe_mx4_cache *cache, const float *qkv, int64_t row_stride, void *q_out, int q_f16,
                            int64_t q_row_stride, int64_t num_heads, const float *freq_cis, int64_t max_positions,
                            int64_t rotary_dim, int interleaved, const int32_t *row_starts, int64_t rows, doe_stream_t stream) {
    RowArgs a{};
    int rc = doe::mx4_view(cache, &a.c);
    if (rc) return rc;
    const int64_t d = cache->head_dim;
    if ((rc = doe::rope_rows_checks(a.r, qkv, row_stride, q_out, q_f16, q_row_stride, num_heads, a.c.kv_heads, d, freq_cis,
                                    max_positions, rotary_dim, interleaved, row_starts, rows, a.c.batch)))
        return rc;
    const float *k = qkv + num_heads * d, *v = k + a.c.kv_heads * d;
    if ((rc = row_checks(a.c, d, rows, row_stride, row_starts, qkv ? k : nullptr, qkv ? v : nullptr, 4))) return rc;
    if ((rc = doe::require_init())) return rc;
    if (rows == 0 || a.c.batch == 0) return DOE_OK;
    a.k = k;
    a.v = v;
    a.row_starts = row_starts;
    a.rows = rows;
    a.row_stride = row_stride;
    const hipStream_t st = (hipStream_t)stream;
    switch (d) {
        case 64: return launch_append<64>(st, a);
        case 128: return launch_append<128>(st, a);
        case 160: return launch_append<160>(st, a);
        case 256: return launch_append<256>(st, a);
        default: return launch_append<512>(st, a);
    }
}

int doe_mx4_kv_read(const doe_mx4_cache *cache, float *k, float *v, int64_t row_stride, const int32_t *row_starts,
                    int64_t rows, doe_stream_t stream) {
    RowArgs a{};
    int rc = doe::mx4_view(cache, &a.c);
    if (rc) return rc;
    if ((rc = row_checks(a.c, cache->head_dim, rows, row_stride, row_starts, k, v, 4))) return rc;
    if ((rc = doe::require_init())) return rc;
    if (rows == 0 || a.c.batch == 0) return DOE_OK;
    a.k_out = k;
    a.v_out = v;
    a.row_starts = row_starts;
    a.rows = rows;
    a.row_stride = row_stride;
    const hipStream_t st = (hipStream_t)stream;
    switch (cache->head_dim) {
        case 64: launch_read<64>(st, a); break;
        case 128: launch_read<128>(st, a); break;
        case 160: launch_read<160>(st, a); break;
        case 256: launch_read<256>(st, a); break;
        default: launch_read<512>(st, a); break;
    }
    DOE_LAUNCH_CHECK("mx4_read_kernel");
    return DOE_OK;
}

}  // extern "C"
