// kv_append.hip -- rows [q | k | v] of ragged requests rotated and appended to the f16
// pages of a paged cache (doe_qkv_rope_append).  A page holds page_size positions
// [num_kv_heads][head_dim], the order that doe_attention_dispatch reads with
// kv_layout 2.
//
// Bound by its bytes: eight prompts of up to 2000 rows, 32 / 8 heads of 128 dims, f16
// queries (387 MB): 75 us, 5.1 TB/s.  A thread has the same eight values of every row that
// its workgroup takes; a row is read before its position is known, and the next one while it
// turns (without: 81; the next one's angles with it: no change).  One token of 8 / 4 heads of
// 256: 2.7 us in the kernel, three dependent reads (length, page, angles) before its stores.
#include "rope_rows.h"

#include <algorithm>

namespace {

using doe::f4;
using doe::h4;

struct AppendArgs {
    doe::RopeRows r;
    _Float16 *k_pool, *v_pool;
    const int32_t *table, *lens, *row_starts;
    int64_t rows, room;
    int num_pages, page_size, kv_heads, head_dim, batch, table_stride, rows_per_wg;
};

__global__ __launch_bounds__(256) void qkv_rope_append_kernel(AppendArgs a) {
    __shared__ int s_pos[doe::kRopeRowsPerWg];
    __shared__ int64_t s_at[doe::kRopeRowsPerWg];  // the position's place in the pools, -1: none
    const int64_t row0 = (int64_t)blockIdx.x * a.rows_per_wg;
    const int count = (int)std::min<int64_t>(a.rows_per_wg, a.rows - row0);
    const int D = a.head_dim, per_head = D / 8;
    const doe::RopeThread me = doe::rope_thread((a.r.num_heads + 2 * a.kv_heads) * per_head, blockIdx.y);
    const int head = me.unit / per_head, in_head = me.unit - head * per_head, kv = head - a.r.num_heads;
    const bool is_q = kv < 0, is_v = kv >= a.kv_heads;
    const doe::RopeUnit u = is_v ? doe::RopeUnit{8 * in_head, 8 * in_head + 4, false} : doe::rope_unit(a.r, in_head);
    const bool turns = !is_v && u.at0 < a.r.rotary_dim;
    _Float16 *pool = is_v ? a.v_pool + (int64_t)(kv - a.kv_heads) * D : a.k_pool + (int64_t)kv * D;
    const float *x = a.r.qkv + row0 * a.r.row_stride + (int64_t)head * D;
    // (a row's values are on their way before its position is known, the next one's while it turns)
    f4 next0 = {}, next1 = {};
    auto read = [&](int i) __attribute__((always_inline)) {
        next0 = *reinterpret_cast<const f4 *>(x + i * a.r.row_stride + u.at0);
        next1 = *reinterpret_cast<const f4 *>(x + i * a.r.row_stride + u.at1);
    };
    if (me.first < count) read(me.first);
    if (threadIdx.x < 64) {
        int b, pos = doe::kNoRow;
        int64_t at = -1;
        if (!doe::rows_positions(a.lens, a.room, a.batch, a.row_starts, row0, count, b, pos)) {
            pos = doe::kNoRow;
        } else if (pos >= 0 && pos < a.r.max_positions) {
            const int in_table = pos / a.page_size, page = a.table[(int64_t)b * a.table_stride + in_table];
            if (page >= 0 && page < a.num_pages)
                at = ((int64_t)page * a.page_size + (pos - in_table * a.page_size)) * a.kv_heads * a.head_dim;
        }
        if ((int)threadIdx.x < count) {
            s_pos[threadIdx.x] = pos;
            s_at[threadIdx.x] = at;
        }
    }
    __syncthreads();
    for (int i = me.first; i < count; i += me.step) {
        const int pos = s_pos[i];
        const int64_t at = s_at[i];
        f4 v0 = next0, v1 = next1;
        if (i + me.step < count) read(i + me.step);
        if (pos == doe::kNoRow || (!is_q && at < 0)) continue;
        if (turns && pos >= 0 && pos < a.r.max_positions) doe::rotate_unit(a.r, u, pos, v0, v1);
        if (is_q) {
            doe::store_query<false>(a.r, row0 + i, head, D, u, v0, v1);
        } else {
            *reinterpret_cast<h4 *>(pool + at + u.at0) = __builtin_convertvector(v0, h4);
            *reinterpret_cast<h4 *>(pool + at + u.at1) = __builtin_convertvector(v1, h4);
        }
    }
}

}  // namespace

namespace doe {

int rope_rows_checks(RopeRows &r, const float *qkv, int64_t row_stride, void *q_out, int q_f16, int64_t q_row_stride,
                     int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const float *freq_cis, int64_t max_positions,
                     int64_t rotary_dim, int interleaved, const int32_t *row_starts, int64_t rows, int64_t batch) {
    DOE_REQUIRE(num_heads >= 0 && num_heads <= 65535, DOE_E_INVALID, "num_heads %lld outside 0..65535", (long long)num_heads);
    DOE_REQUIRE(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 8 == 0, DOE_E_UNSUPPORTED,
                "rotary_dim %lld unsupported (a multiple of 8 up to head_dim %lld)", (long long)rotary_dim, (long long)head_dim);
    DOE_REQUIRE(max_positions >= 0 && max_positions < ((int64_t)1 << 31), DOE_E_INVALID, "max_positions %lld", (long long)max_positions);
    DOE_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 28), DOE_E_INVALID, "rows %lld", (long long)rows);  // (a launch has fewer than 2^32 threads)
    DOE_REQUIRE(row_starts || rows == batch, DOE_E_INVALID, "without row_starts a call takes one row a sequence (%lld rows, batch %lld)",
                (long long)rows, (long long)batch);
    DOE_REQUIRE(row_stride >= (num_heads + 2 * num_kv_heads) * head_dim && row_stride % 4 == 0, DOE_E_INVALID,
                "row stride %lld below a row of %lld, or not a multiple of 16 bytes", (long long)row_stride,
                (long long)((num_heads + 2 * num_kv_heads) * head_dim));
    DOE_REQUIRE(num_heads == 0 || (q_row_stride >= num_heads * head_dim && q_row_stride * (q_f16 ? 2 : 4) % 16 == 0), DOE_E_INVALID,
                "q row stride %lld below a row of %lld, or not a multiple of 16 bytes", (long long)q_row_stride,
                (long long)(num_heads * head_dim));
    DOE_REQUIRE(rows == 0 || (qkv && (q_out || num_heads == 0) && (freq_cis || rotary_dim == 0 || max_positions == 0)), DOE_E_INVALID,
                "null pointer");
    DOE_REQUIRE(((uintptr_t)qkv & 15) == 0 && ((uintptr_t)q_out & 15) == 0 && ((uintptr_t)freq_cis & 15) == 0, DOE_E_INVALID,
                "qkv, q_out and freq_cis must be 16-byte aligned");
    // in place only element by element: f32, the same rows
    const uintptr_t from = (uintptr_t)qkv, to = (uintptr_t)q_out;
    const int64_t in_bytes = rows ? ((rows - 1) * row_stride + (num_heads + 2 * num_kv_heads) * head_dim) * 4 : 0;
    const int64_t out_bytes = rows && num_heads ? ((rows - 1) * q_row_stride + num_heads * head_dim) * (q_f16 ? 2 : 4) : 0;
    const bool apart = to + (uintptr_t)out_bytes <= from || from + (uintptr_t)in_bytes <= to;
    DOE_REQUIRE(apart || num_heads == 0 || (from == to && !q_f16 && q_row_stride == row_stride), DOE_E_INVALID,
                "q_out is apart from qkv or its own f32 q rows");
    r.qkv = qkv;
    r.freq = freq_cis;
    r.q_out = q_out;
    r.row_stride = row_stride;
    r.q_stride = q_row_stride;
    r.num_heads = (int)num_heads;
    r.rotary_dim = (int)rotary_dim;
    r.max_positions = (int)max_positions;
    r.q_f16 = q_f16 != 0;
    r.interleaved = interleaved != 0;
    return DOE_OK;
}

}  // namespace doe

extern "C" {

int doe_qkv_rope_append(const doe_f16_cache *cache, const float *qkv, int64_t row_stride, void *q_out, int q_f16,
                        int64_t q_row_stride, int64_t num_heads, const float *freq_cis, int64_t max_positions,
                        int64_t rotary_dim, int interleaved, const int32_t *row_starts, int64_t rows, doe_stream_t stream) {
    DOE_REQUIRE(cache, DOE_E_INVALID, "null cache");
    const doe_f16_cache &c = *cache;
    DOE_REQUIRE(c.head_dim > 0 && c.head_dim <= 1024 && c.head_dim % 8 == 0, DOE_E_UNSUPPORTED,
                "head_dim %lld unsupported (a multiple of 8 up to 1024)", (long long)c.head_dim);
    DOE_REQUIRE(c.num_kv_heads > 0 && c.num_kv_heads <= 1024, DOE_E_INVALID, "num_kv_heads %lld outside 1..1024",
                (long long)c.num_kv_heads);
    DOE_REQUIRE(c.num_pages > 0 && c.num_pages < ((int64_t)1 << 31), DOE_E_INVALID, "num_pages %lld", (long long)c.num_pages);
    DOE_REQUIRE(c.batch >= 0 && c.batch <= 65535, DOE_E_INVALID, "batch %lld outside 0..65535", (long long)c.batch);
    DOE_REQUIRE(c.page_size > 0 && c.table_stride > 0 && c.page_size < ((int64_t)1 << 30) && c.table_stride < ((int64_t)1 << 30) &&
                    c.table_stride * c.page_size < ((int64_t)1 << 30),
                DOE_E_INVALID, "page_size %lld x table_stride %lld: a sequence holds fewer than 2^30 positions",
                (long long)c.page_size, (long long)c.table_stride);
    DOE_REQUIRE(c.k_pool && c.v_pool && c.page_table && c.kv_lens, DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)c.k_pool & 15) == 0 && ((uintptr_t)c.v_pool & 15) == 0, DOE_E_INVALID, "the pools must be 16-byte aligned");
    AppendArgs a{};
    int rc = doe::rope_rows_checks(a.r, qkv, row_stride, q_out, q_f16, q_row_stride, num_heads, c.num_kv_heads, c.head_dim,
                                   freq_cis, max_positions, rotary_dim, interleaved, row_starts, rows, c.batch);
    if (rc) return rc;
    if ((rc = doe::require_init())) return rc;
    if (rows == 0 || c.batch == 0) return DOE_OK;
    a.k_pool = reinterpret_cast<_Float16 *>(c.k_pool);
    a.v_pool = reinterpret_cast<_Float16 *>(c.v_pool);
    a.table = c.page_table;
    a.lens = c.kv_lens;
    a.row_starts = row_starts;
    a.rows = rows;
    a.room = c.table_stride * c.page_size;
    a.num_pages = (int)c.num_pages;
    a.page_size = (int)c.page_size;
    a.kv_heads = (int)c.num_kv_heads;
    a.head_dim = (int)c.head_dim;
    a.batch = (int)c.batch;
    a.table_stride = (int)c.table_stride;
    const doe::RopeShare share = doe::rope_share(rows, (num_heads + 2 * c.num_kv_heads) * (c.head_dim / 8));
    a.rows_per_wg = share.rows_per_wg;
    const int64_t wgs = (rows + share.rows_per_wg - 1) / share.rows_per_wg;
    DOE_REQUIRE(wgs * share.ways < (1 << 24), DOE_E_UNSUPPORTED, "%lld rows of %lld and %lld heads in one call", (long long)rows,
                (long long)num_heads, (long long)c.num_kv_heads);  // (a launch has fewer than 2^32 threads)
    hipLaunchKernelGGL(qkv_rope_append_kernel, dim3((unsigned)wgs, (unsigned)share.ways), dim3(256), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("qkv_rope_append_kernel");
    return DOE_OK;
}

}  // extern "C"
