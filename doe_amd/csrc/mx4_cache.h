// mx4_cache.h -- the pages of the KV cache held in 4 bits, for the kernels that
// write and read them (mx4_cache.hip, attn_mx4.hip, attn_mx4_prompt.hip).
//
// A value is an E2M1 code (sign, two exponent bits, one mantissa bit: 0, 0.5,
// 1, 1.5, 2, 3, 4, 6) times 2^(scale - 127), one scale byte for 32 dims of a
// row.  The page layout is given in doe_mi355x.h; V is held in the order in
// which a lane of the P V product takes it: columns of D / 16 dims, and of 32
// positions the eight that a lane group holds side by side, so a lane's bytes
// of a block are one run and no byte is shared between positions.
#pragma once

#include "common.h"

namespace doe {

constexpr int kMx4MinExp = -23;         // every value exact in f16: 0.5 x 2^-23 is its
constexpr int kMx4MaxExp = 13;          // least, 6 x 2^13 within its range
constexpr int kMx4NanScale = 255;

// A cache as the kernels take it.
struct Mx4View {
    uint8_t *pool;
    const int32_t *table, *lens;
    int num_pages, page_shift, kv_heads, batch, table_stride;
};

// Byte offsets within the slab of one head of a page of 1 << shift positions.
template <int D>
struct Mx4Slab {
    static __device__ __forceinline__ int64_t bytes(int shift) { return (int64_t)(D + D / 16) << shift; }
    static __device__ __forceinline__ int k_code(int x) { return x * (D / 2); }
    static __device__ __forceinline__ int k_scale(int shift, int x) { return (D << shift) + x * (D / 32); }
    // column c of position x: D / 32 bytes
    static __device__ __forceinline__ int v_code(int shift, int x, int c) {
        return ((D / 2) << shift) + ((((x >> 5) * 4 + ((x >> 2) & 3)) * 16 + c) * 8 + ((x >> 4) & 1) * 4 + (x & 3)) * (D / 32);
    }
    static __device__ __forceinline__ int v_scale(int shift, int x, int group) {
        return ((D + D / 32) << shift) + (((x >> 5) * 4 + ((x >> 2) & 3)) * (D / 32) + group) * 8 + ((x >> 4) & 1) * 4 + (x & 3);
    }
};

// Positions of sequence b that the cache can hold and has in use.
__device__ __forceinline__ int mx4_len(const Mx4View &c, int b) {
    const int64_t room = (int64_t)c.table_stride << c.page_shift;
    const int n = c.lens[b];
    return n < 0 ? 0 : (n > room ? (int)room : n);
}

// The sequence b and position of row `row` of a call (row_starts null: row b of
// sequence b); false where it has none: rows before and behind the
// sequences', positions before 0.
__device__ __forceinline__ bool mx4_row(const Mx4View &c, const int32_t *row_starts, int64_t row, int &b, int &pos) {
    int lo = 0;
    int64_t first = row, next = row + 1;
    if (row_starts) {
        int hi = c.batch;  // the last b with row_starts[b] <= row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (row_starts[mid] <= row) lo = mid;
            else hi = mid;
        }
        first = row_starts[lo];
        next = row_starts[lo + 1];
        if (row < first || row >= next) return false;
    } else {
        lo = (int)row;
    }
    b = lo;
    const int64_t p = (int64_t)mx4_len(c, b) - (next - first) + (row - first);
    pos = (int)p;
    return p >= 0;
}

// The page of position pos of sequence b; -1 where the table names none of the pool.
__device__ __forceinline__ int mx4_page(const Mx4View &c, int b, int pos) {
    const int page = c.table[(int64_t)b * c.table_stride + (pos >> c.page_shift)];
    return page >= 0 && page < c.num_pages ? page : -1;
}

// Inclusive sum over the wave's lanes, in registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xf>(v);  // one lane further within sixteen, two, four, eight
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);     // the last lane of a sixteen to the next (rows 1 and 3)
    return dpp_add<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
}

// A scale byte as the conversions take it: they look at the exponent field alone,
// so the other bits may hold the byte's neighbours.
__device__ __forceinline__ float mx4_byte_scale(uint32_t word, int byte) {
    return __uint_as_float(byte == 3 ? word >> 1 : word << (23 - 8 * byte));
}
// The two values of a byte of codes in f16, exactly.
typedef _Float16 Mx4Pair __attribute__((ext_vector_type(2)));
template <int BYTE>
__device__ __forceinline__ Mx4Pair mx4_pair(uint32_t word, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, s, BYTE);
}
__device__ __forceinline__ Mx4Pair mx4_pair_at(uint32_t word, float s, int byte) {
    switch (byte & 3) {
        case 0: return mx4_pair<0>(word, s);
        case 1: return mx4_pair<1>(word, s);
        case 2: return mx4_pair<2>(word, s);
        default: return mx4_pair<3>(word, s);
    }
}

// tanh x to 2e-7 of itself, without a branch: (1 - e) / (1 + e), e = exp(-2 |x|), the
// quotient with one Newton step; below 0.3, where 1 - e cancels, the series x -
// x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835 (the next term is 5e-8 of it).
__device__ __forceinline__ float mx4_tanh(float x) {
    const float u = fabsf(x), e = __builtin_amdgcn_exp2f(u * -2.8853900817779268f);
    const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
    const float q = (1.0f - e) * fmaf(fmaf(-d, r, 1.0f), r, r), x2 = x * x;
    const float p = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return u < 0.3f ? x * p : copysignf(q, x);
}

// A query's f32 values go to the matrix cores as f16 hi and lo parts of q 2^e, e such
// that the largest (its bits without the sign: `top`) lies in [2^13, 2^14): of a value
// at most 2^-22 is lost, or 2^-38 of the largest where that is more.
__device__ __forceinline__ int mx4_query_exp(uint32_t top) {
    if (top == 0 || top >= 0x7f800000u) return 0;
    return 14 - __builtin_amdgcn_frexp_expf(__uint_as_float(top));  // -114 .. 162
}
// Takes that 2^e out of a score again, with the call's own factor f: s = s * pre * post.
// pre is 1 unless f 2^-e overflows (then f > 1, so that s pre overflows with s only).
// A query that is no number has scores that are none.
struct Mx4Factor {
    float pre, post;
};
__device__ __forceinline__ Mx4Factor mx4_factor(float f, uint32_t top, int e) {
    if (top >= 0x7f800000u) return {1.0f, __uint_as_float(0x7fc00000u)};
    const float post = __builtin_amdgcn_ldexpf(f, -e);
    if (fabsf(post) < __uint_as_float(0x7f800000u)) return {1.0f, post};
    return {__builtin_amdgcn_ldexpf(1.0f, -e), f};
}

// Checks a cache and turns it into the kernels' form; returns a DOE status.
int mx4_view(const doe_mx4_cache *cache, Mx4View *view);
// What both attentions check of a call.
int mx4_attention_checks(const Mx4View &c, int64_t num_heads, float scale, float softcap, int64_t sliding_window,
                         const void *q, const void *out);

}  // namespace doe
