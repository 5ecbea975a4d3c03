// rope_rows.h -- rows [q heads | k heads | v heads] of a fused projection rotated at
// their positions, for the kernels that append them to a paged cache
// (kv_append.hip, mx4_cache.hip).
//
// The arithmetic is doe_rope's: x0 c - x1 s and x0 s + x1 c, each product and sum
// rounded to f32.
#pragma once

#include "common.h"

namespace doe {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// What a rotating call takes besides its cache.
struct RopeRows {
    const float *qkv, *freq;  // freq [max_positions][rotary_dim / 2][cos, sin]
    void *q_out;
    int64_t row_stride, q_stride;
    int num_heads, rotary_dim, max_positions;
    int q_f16, interleaved;
};

// Two pairs (x, y), (z, w) side by side, rotated by the angles (cos, sin, cos, sin).
__device__ __forceinline__ f4 rotate_pairs(f4 v, f4 cs) {
#pragma clang fp contract(off)
    return f4{v[0] * cs[0] - v[1] * cs[1], v[0] * cs[1] + v[1] * cs[0], v[2] * cs[2] - v[3] * cs[3], v[2] * cs[3] + v[3] * cs[2]};
}
// Four pairs (lo[i], hi[i]) rotated.
__device__ __forceinline__ void rotate_halves(f4 &lo, f4 &hi, f4 cs01, f4 cs23) {
#pragma clang fp contract(off)
    const f4 c = {cs01[0], cs01[2], cs23[0], cs23[2]}, s = {cs01[1], cs01[3], cs23[1], cs23[3]};
    f4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = lo[i] * c[i] - hi[i] * s[i];
        b[i] = lo[i] * s[i] + hi[i] * c[i];
    }
    lo = a;
    hi = b;
}

// A unit is eight values of a head: of `rotary_dim` halves four dims and their four
// partners, otherwise eight dims side by side.  at0 and at1 are the places of its two
// fours.
struct RopeUnit {
    int at0, at1;
    bool halves;
};
__device__ __forceinline__ RopeUnit rope_unit(const RopeRows &r, int u) {
    const bool halves = !r.interleaved && 8 * u < r.rotary_dim;
    const int at = halves ? 4 * u : 8 * u;
    return {at, halves ? at + r.rotary_dim / 2 : at + 4, halves};
}
// Rotates a unit; `pos` within the table.
__device__ __forceinline__ void rotate_unit(const RopeRows &r, const RopeUnit &u, int pos, f4 &v0, f4 &v1) {
    if (u.at0 >= r.rotary_dim) return;
    const f4 *cs = reinterpret_cast<const f4 *>(r.freq + (int64_t)pos * r.rotary_dim + (u.halves ? 2 * u.at0 : u.at0));
    if (u.halves) {
        rotate_halves(v0, v1, cs[0], cs[1]);
    } else {
        v0 = rotate_pairs(v0, cs[0]);
        v1 = rotate_pairs(v1, cs[1]);
    }
}
// A unit of a query to q_out.
__device__ __forceinline__ void store_query(const RopeRows &r, int64_t row, int head, int head_dim, const RopeUnit &u, f4 v0, f4 v1) {
    const int64_t at = row * r.q_stride + (int64_t)head * head_dim;
    if (r.q_f16) {
        _Float16 *q = static_cast<_Float16 *>(r.q_out) + at;
        *reinterpret_cast<h4 *>(q + u.at0) = __builtin_convertvector(v0, h4);
        *reinterpret_cast<h4 *>(q + u.at1) = __builtin_convertvector(v1, h4);
    } else {
        float *q = static_cast<float *>(r.q_out) + at;
        *reinterpret_cast<f4 *>(q + u.at0) = v0;
        *reinterpret_cast<f4 *>(q + u.at1) = v1;
    }
}

// Positions of sequence b that its row of the page table can hold and has in use.
__device__ __forceinline__ int held_positions(const int32_t *lens, int64_t room, int b) {
    const int n = lens[b];
    return n < 0 ? 0 : (n > room ? (int)room : n);
}
// The sequence and position of row `row` of a call (row_starts null: row b of sequence
// b); false where it is of none.  A position below 0 has no place.
__device__ __forceinline__ bool row_position(const int32_t *lens, int64_t room, int batch, const int32_t *row_starts, int64_t row,
                                             int &b, int &pos) {
    int lo = 0;
    int64_t behind = 0;  // rows of the sequence from this one on
    if (row_starts) {
        int hi = batch;  // the last b with row_starts[b] <= row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (row_starts[mid] <= row) lo = mid;
            else hi = mid;
        }
        behind = row_starts[lo + 1] - row;
        if (row < row_starts[lo] || behind <= 0) return false;
    } else {
        lo = (int)row;
        behind = 1;
    }
    b = lo;
    pos = (int)(held_positions(lens, room, lo) - behind);
    return true;
}

// Dims d .. d + 3 of a head at x, of which `own` has been read, rotated.
__device__ __forceinline__ f4 rotate_four(const RopeRows &r, const float *x, int d, f4 own, int pos) {
#pragma clang fp contract(off)
    if (d >= r.rotary_dim) return own;
    const float *freq = r.freq + (int64_t)pos * r.rotary_dim;
    if (r.interleaved) return rotate_pairs(own, *reinterpret_cast<const f4 *>(freq + d));
    const int half = r.rotary_dim / 2, i = d < half ? d : d - half;
    const f4 other = *reinterpret_cast<const f4 *>(x + (d < half ? d + half : i));
    f4 lo = d < half ? own : other, hi = d < half ? other : own;
    rotate_halves(lo, hi, *reinterpret_cast<const f4 *>(freq + 2 * i), *reinterpret_cast<const f4 *>(freq + 2 * i + 4));
    return d < half ? lo : hi;
}

constexpr int kRopeRowsPerWg = 32;

// The queries of rows [row0, row0 + count), count <= kRopeRowsPerWg, by this workgroup
// of 256 threads: every ways-th 256 of their units from the way-th on.
__device__ __forceinline__ void rotate_queries(const RopeRows &r, const int32_t *lens, int64_t room, int batch,
                                               const int32_t *row_starts, int64_t row0, int count, int head_dim, int way, int ways,
                                               int *s_pos) {
    constexpr int kNone = -0x7fffffff;  // a row of no sequence is left as it was
    if ((int)threadIdx.x < count) {
        int b, pos;
        if (!row_position(lens, room, batch, row_starts, row0 + threadIdx.x, b, pos)) pos = kNone;
        s_pos[threadIdx.x] = pos;
    }
    __syncthreads();
    const int per_head = head_dim / 8, per_row = r.num_heads * per_head;
    for (int i = way * 256 + threadIdx.x; i < count * per_row; i += ways * 256) {
        const int in_block = i / per_row, in_row = i - in_block * per_row, head = in_row / per_head, pos = s_pos[in_block];
        if (pos == kNone) continue;
        const int64_t row = row0 + in_block;
        const RopeUnit u = rope_unit(r, in_row - head * per_head);
        const float *x = r.qkv + row * r.row_stride + (int64_t)head * head_dim;
        f4 v0 = *reinterpret_cast<const f4 *>(x + u.at0), v1 = *reinterpret_cast<const f4 *>(x + u.at1);
        if (pos >= 0 && pos < r.max_positions) rotate_unit(r, u, pos, v0, v1);
        store_query(r, row, head, head_dim, u, v0, v1);
    }
}

// What every rotating call checks of these; fills `r`.
int rope_rows_checks(RopeRows &r, const float *qkv, int64_t row_stride, void *q_out, int q_f16, int64_t q_row_stride,
                     int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const float *freq_cis, int64_t max_positions,
                     int64_t rotary_dim, int interleaved, const int32_t *row_starts, int64_t rows, int64_t batch);

}  // namespace doe
