// attn_mx4_prompt.hip -- causal GQA attention of prompt rows over the paged KV
// cache held in 4 bits (doe_attn_mx4_prompt).
//
// o = sum_p softmax_p(cap(q . k_p scale)) v_p over the positions p that a row
// sees: p <= pos, p < kv_len, with a window p > pos - window.
//
// One workgroup a row and head: 256 positions at a time, a thread one score;
// then the running maximum and sum, and a thread one or two dims of P V.
#include "mx4_cache.h"

#include <math.h>

namespace {

using doe::Mx4Slab;
using doe::Mx4View;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

struct Args {
    Mx4View c;
    const void *q;
    void *out;
    const int32_t *row_starts;
    int64_t rows, q_stride, out_stride;
    int q_f16, out_f16, num_heads, window;
    float scale, softcap;
};

__device__ __forceinline__ float scale_of(int s) {
    return __uint_as_float(s == doe::kMx4NanScale ? 0x7fc00000u : (uint32_t)s << 23);
}

template <int D>
__global__ __launch_bounds__(256) void attn_mx4_rows_kernel(Args a) {
    using S = Mx4Slab<D>;
    __shared__ float qs[D], p_[256], red[4];
    __shared__ int page_[256];
    const int tid = threadIdx.x, head = blockIdx.x % a.num_heads;
    const int64_t row = blockIdx.x / a.num_heads;
    int b, pos;
    const bool seen = doe::mx4_row(a.c, a.row_starts, row, b, pos);
    if (a.row_starts && (row < a.row_starts[0] || row >= a.row_starts[a.c.batch])) return;
    const int kvh = head / (a.num_heads / a.c.kv_heads), shift = a.c.page_shift;
    int hi = 0, lo = 0;
    if (seen) {
        hi = min(pos + 1, doe::mx4_len(a.c, b));
        if (a.window > 0) lo = max(0, pos - a.window + 1);
    }
    for (int d = tid; d < D; d += 256) {
        const int64_t at = row * a.q_stride + (int64_t)head * D + d;
        qs[d] = a.q_f16 ? (float)static_cast<const _Float16 *>(a.q)[at] : static_cast<const float *>(a.q)[at];
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[(D + 255) / 256] = {};
    for (int p0 = lo; p0 < hi; p0 += 256) {
        const int p = p0 + tid, page = p < hi ? doe::mx4_page(a.c, b, p) : -1, x = p & ((1 << shift) - 1);
        float s = -INFINITY;
        if (page >= 0) {
            const uint8_t *slab = a.c.pool + ((int64_t)page * a.c.kv_heads + kvh) * S::bytes(shift);
            s = 0.0f;
            for (int g = 0; g < D / 32; ++g) {
                const float f = scale_of(slab[S::k_scale(shift, x) + g]);
                for (int d = 32 * g; d < 32 * g + 32; d += 2) {
                    const h2 k = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(slab[S::k_code(x) + d / 2], f, 0);
                    s = fmaf(qs[d], (float)k[0], s);
                    s = fmaf(qs[d + 1], (float)k[1], s);
                }
            }
            s *= a.scale;
            if (a.softcap > 0.0f) s = tanhf(s / a.softcap) * a.softcap;
        }
        page_[tid] = page;
        float top = s;
        for (int w = 1; w < 64; w <<= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float mref = mn == -INFINITY ? 0.0f : mn, corr = expf(m - mref);
        p_[tid] = expf(s - mref);
        m = mn;
        __syncthreads();
        l *= corr;
        for (int i = 0; i < (D + 255) / 256; ++i) o[i] *= corr;
        for (int j = 0; j < 256; ++j) {
            if (page_[j] < 0) continue;
            const float pj = p_[j];
            l += pj;
            const int xj = (p0 + j) & ((1 << shift) - 1);
            const uint8_t *slab = a.c.pool + ((int64_t)page_[j] * a.c.kv_heads + kvh) * S::bytes(shift);
            for (int i = 0; i < (D + 255) / 256; ++i) {
                const int d = tid + 256 * i;
                if (d >= D) continue;
                const float f = scale_of(slab[S::v_scale(shift, xj, d / 32)]);
                const h2 v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(slab[S::v_code(shift, xj, d / (D / 16)) + d % (D / 16) / 2], f, 0);
                o[i] = fmaf(pj, (float)v[d & 1], o[i]);
            }
        }
        __syncthreads();
    }
    for (int i = 0; i < (D + 255) / 256; ++i) {
        const int d = tid + 256 * i;
        if (d >= D) continue;
        const int64_t at = row * a.out_stride + (int64_t)head * D + d;
        const float v = l != 0.0f ? o[i] / l : 0.0f;
        if (a.out_f16) static_cast<_Float16 *>(a.out)[at] = (_Float16)v;
        else static_cast<float *>(a.out)[at] = v;
    }
}

int attention(Args &a, const doe_mx4_cache *cache, int64_t num_heads, int64_t sliding_window, void *workspace,
              int64_t workspace_bytes, int64_t need, hipStream_t st) {
    const int64_t d = cache->head_dim;
    int rc = doe::mx4_attention_checks(a.c, num_heads, a.scale, a.softcap, sliding_window, a.q, a.out);
    if (rc) return rc;
    DOE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need, DOE_E_INVALID,
                "a 16-byte aligned workspace of %lld bytes is needed (got %lld)", (long long)need, (long long)workspace_bytes);
    DOE_REQUIRE(a.rows >= 0 && a.rows * num_heads < ((int64_t)1 << 31), DOE_E_INVALID, "%lld rows of %lld heads",
                (long long)a.rows, (long long)num_heads);
    DOE_REQUIRE(a.row_starts || a.rows == a.c.batch, DOE_E_INVALID,
                "without row_starts a call takes one row a sequence (%lld rows, batch %d)", (long long)a.rows, a.c.batch);
    DOE_REQUIRE(a.q_stride >= num_heads * d && a.out_stride >= num_heads * d && a.q_stride * (a.q_f16 ? 2 : 4) % 16 == 0 &&
                    a.out_stride * (a.out_f16 ? 2 : 4) % 16 == 0,
                DOE_E_INVALID, "row strides below a row, or not multiples of 16 bytes");
    if ((rc = doe::require_init())) return rc;
    if (a.rows == 0 || a.c.batch == 0) return DOE_OK;
    a.num_heads = (int)num_heads;
    a.window = (int)sliding_window;
    const dim3 grid((unsigned)(a.rows * num_heads));
    switch (d) {
        case 64: hipLaunchKernelGGL(attn_mx4_rows_kernel<64>, grid, dim3(256), 0, st, a); break;
        case 128: hipLaunchKernelGGL(attn_mx4_rows_kernel<128>, grid, dim3(256), 0, st, a); break;
        case 160: hipLaunchKernelGGL(attn_mx4_rows_kernel<160>, grid, dim3(256), 0, st, a); break;
        case 256: hipLaunchKernelGGL(attn_mx4_rows_kernel<256>, grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL(attn_mx4_rows_kernel<512>, grid, dim3(256), 0, st, a); break;
    }
    DOE_LAUNCH_CHECK("attn_mx4_rows_kernel");
    return DOE_OK;
}

int workspace_size(int64_t batch, int64_t rows, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    int64_t page = 0;
    const int rc = doe_mx4_page_bytes(32, num_kv_heads, head_dim, &page);
    if (rc) return rc;
    DOE_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 0 && num_heads > 0 && num_heads <= 65535 &&
                    num_heads % num_kv_heads == 0 && rows * num_heads < ((int64_t)1 << 31),
                DOE_E_INVALID, "batch %lld, %lld rows, %lld heads over %lld", (long long)batch, (long long)rows,
                (long long)num_heads, (long long)num_kv_heads);
    *bytes = 16;
    return DOE_OK;
}

}  // namespace

extern "C" {

int doe_attn_mx4_prompt_workspace(int64_t batch, int64_t rows, int64_t num_heads, int64_t num_kv_heads,
                                  int64_t head_dim, int64_t *bytes) {
    return workspace_size(batch, rows, num_heads, num_kv_heads, head_dim, bytes);
}

int doe_attn_mx4_prompt(const doe_mx4_cache *cache, const void *q, int q_f16, int64_t q_row_stride, void *out,
                        int out_f16, int64_t out_row_stride, const int32_t *row_starts, int64_t rows, int64_t num_heads,
                        float scale, float softcap, int64_t sliding_window, void *workspace, int64_t workspace_bytes,
                        doe_stream_t stream) {
    Args a{};
    const int rc = doe::mx4_view(cache, &a.c);
    if (rc) return rc;
    a.q = q;
    a.out = out;
    a.row_starts = row_starts;
    a.rows = rows;
    a.q_stride = q_row_stride;
    a.out_stride = out_row_stride;
    a.q_f16 = q_f16;
    a.out_f16 = out_f16;
    a.scale = scale;
    a.softcap = softcap;
    return attention(a, cache, num_heads, sliding_window, workspace, workspace_bytes, 16, (hipStream_t)stream);
}

}  // extern "C"
