// rope_rows.h -- rows [q heads | k heads | v heads] of a fused projection rotated at
// their positions, for the kernels that append them to a paged cache
// (kv_append.hip, mx4_cache.hip).
//
// The arithmetic is doe_rope's: x0 c - x1 s and x0 s + x1 c, each product and sum
// rounded to f32.
#pragma once

#include "ragged.h"

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
// Rotates a unit of dims below rotary_dim at a position of the table.
__device__ __forceinline__ void rotate_unit(const RopeRows &r, const RopeUnit &u, int pos, f4 &v0, f4 &v1) {
    const f4 *cs = reinterpret_cast<const f4 *>(r.freq + (int64_t)pos * r.rotary_dim + (u.halves ? 2 * u.at0 : u.at0));
    const f4 cs0 = cs[0], cs1 = cs[1];
    if (u.halves) {
        rotate_halves(v0, v1, cs0, cs1);
    } else {
        v0 = rotate_pairs(v0, cs0);
        v1 = rotate_pairs(v1, cs1);
    }
}
// PAST: past the caches.
template <bool PAST, typename T>
__device__ __forceinline__ T load(const T *p) {
    if constexpr (PAST) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool PAST, typename T>
__device__ __forceinline__ void store(T *p, T v) {
    if constexpr (PAST) __builtin_nontemporal_store(v, p);
    else *p = v;
}
// A unit of a query to q_out.
template <bool PAST>
__device__ __forceinline__ void store_query(const RopeRows &r, int64_t row, int head, int head_dim, const RopeUnit &u, f4 v0, f4 v1) {
    const int64_t at = row * r.q_stride + (int64_t)head * head_dim;
    if (r.q_f16) {
        _Float16 *q = static_cast<_Float16 *>(r.q_out) + at;
        store<PAST>(reinterpret_cast<h4 *>(q + u.at0), __builtin_convertvector(v0, h4));
        store<PAST>(reinterpret_cast<h4 *>(q + u.at1), __builtin_convertvector(v1, h4));
    } else {
        float *q = static_cast<float *>(r.q_out) + at;
        store<PAST>(reinterpret_cast<f4 *>(q + u.at0), v0);
        store<PAST>(reinterpret_cast<f4 *>(q + u.at1), v1);
    }
}

// Sequence and position of rows [row0, row0 + count), count at most 64, a lane of the
// calling wave each (found: whether it has one).  The 64 sequences from the first row's on
// are looked through at once, a lane each; rows behind those search for theirs.
__device__ __forceinline__ bool rows_positions(const int32_t *lens, int64_t room, int batch, const int32_t *row_starts, int64_t row0,
                                               int count, int &b, int &pos) {
    const int lane = threadIdx.x & 63;
    if (!row_starts) return lane < count && row_position(lens, room, batch, row_starts, row0 + lane, b, pos);
    int first = 0;
    for (int left = batch; left > 64;) {  // 64 ways at a time
        const int step = (left + 63) >> 6, at = first + lane * step;
        const uint64_t before = __ballot(at < first + left && row_starts[at] <= row0);
        const int last = before ? 63 - __builtin_clzll(before) : 0;
        first += last * step;
        left = left - last * step < step ? left - last * step : step;
    }
    const int n = batch - first < 64 ? batch - first : 64;
    const int start = lane < n ? row_starts[first + lane] : 0, end = lane < n ? row_starts[first + lane + 1] : 0;
    const int held = lane < n ? held_positions(lens, room, first + lane) : 0;
    bool found = false;
    for (int i = 0; i < count; ++i) {
        const uint64_t in = __ballot(lane < n && start <= row0 + i && row0 + i < end);
        if (in == 0) continue;
        const int at = 63 - __builtin_clzll(in);
        const int64_t p = __builtin_amdgcn_readlane(held, at) - ((int64_t)__builtin_amdgcn_readlane(end, at) - (row0 + i));
        if (lane == i) {
            found = true;
            b = first + at;
            pos = (int)p;
        }
    }
    if (first + n < batch && lane < count && !found && row0 + lane >= __builtin_amdgcn_readlane(end, n - 1))
        found = row_position(lens, room, batch, row_starts, row0 + lane, b, pos);
    return found;
}

// The rows of a rotating call over workgroups of 256 threads.  A thread has one unit, of
// the `units` of a row, in all of its workgroup's rows, so that what it is is found once: a
// workgroup holds several rows at once, or `ways` of them share a row's units; twice as many
// rows, the second read while the first turns, where 2048 workgroups are left (77 prompts of up
// to 405 rows to f16 pages: 42 us with one row a workgroup, 35 with two, 34.8 with three; eight
// of up to 2000 in three ways 78, 75.4 and 76).
constexpr int kRopeRowsPerWg = 16;
struct RopeShare {
    int rows_per_wg, ways;
};
inline RopeShare rope_share(int64_t rows, int64_t units) {
    const int64_t ways = (units + 255) / 256, at_once = units < 256 ? 256 / units : 1;
    const int64_t per = rows * ways >= 2 * 2048 * at_once ? 2 * at_once : at_once;
    return {(int)(per < kRopeRowsPerWg ? per : kRopeRowsPerWg), (int)ways};
}
struct RopeThread {
    int unit, first, step;  // its unit, first row (past all rows: it has none), and rows from one to the next
};
__device__ __forceinline__ RopeThread rope_thread(int units, int way) {
    if (units >= 256) return {way * 256 + (int)threadIdx.x, way * 256 + (int)threadIdx.x < units ? 0 : kRopeRowsPerWg, 1};
    const int at_once = 256 / units, first = threadIdx.x / units;
    return {(int)threadIdx.x - first * units, first < at_once ? first : kRopeRowsPerWg, at_once};
}

// The queries of rows [row0, row0 + count) by a workgroup.
constexpr int kNoRow = -0x7fffffff;  // the position of a row of no sequence: it is left as it was
template <bool PAST>
__device__ __forceinline__ void rotate_queries(const RopeRows &r, const int32_t *lens, int64_t room, int batch,
                                               const int32_t *row_starts, int64_t row0, int count, int head_dim, int way, int *s_pos) {
    const int per_head = head_dim / 8;
    const RopeThread me = rope_thread(r.num_heads * per_head, way);
    const int head = me.unit / per_head;
    const RopeUnit u = rope_unit(r, me.unit - head * per_head);
    const float *x = r.qkv + row0 * r.row_stride + (int64_t)head * head_dim;
    // (a row's values are on their way before its position is known, the next one's while it turns)
    f4 v0 = {}, v1 = {};
    auto read = [&](int i) __attribute__((always_inline)) {
        v0 = load<PAST>(reinterpret_cast<const f4 *>(x + i * r.row_stride + u.at0));
        v1 = load<PAST>(reinterpret_cast<const f4 *>(x + i * r.row_stride + u.at1));
    };
    if (me.first < count) read(me.first);
    if (threadIdx.x < 64) {
        int b, pos = kNoRow;
        if (!rows_positions(lens, room, batch, row_starts, row0, count, b, pos)) pos = kNoRow;
        if ((int)threadIdx.x < count) s_pos[threadIdx.x] = pos;
    }
    __syncthreads();
    for (int i = me.first; i < count; i += me.step) {
        const int pos = s_pos[i];
        f4 w0 = v0, w1 = v1;
        if (i + me.step < count) read(i + me.step);
        if (pos == kNoRow) continue;
        if (u.at0 < r.rotary_dim && pos >= 0 && pos < r.max_positions) rotate_unit(r, u, pos, w0, w1);
        store_query<PAST>(r, row0 + i, head, head_dim, u, w0, w1);
    }
}

// What every rotating call checks of these; fills `r`.
int rope_rows_checks(RopeRows &r, const float *qkv, int64_t row_stride, void *q_out, int q_f16, int64_t q_row_stride,
                     int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const float *freq_cis, int64_t max_positions,
                     int64_t rotary_dim, int interleaved, const int32_t *row_starts, int64_t rows, int64_t batch);

}  // namespace doe
