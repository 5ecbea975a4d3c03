// lora.hip -- low-rank adapters of many requests beside a shared projection
// (doe_lora_add): y[r] += s_a B_a (A_a x[r]) for the adapter a of row r's request.
//
// Rows of their own (decode steps): lora_token_kernel, in one launch where A is small.  A
// workgroup takes a row and 1024 of its columns, forms the t = A x that they need itself
// (again in every workgroup of the row: A comes from the caches) and adds B t; else t is
// formed by a launch before.  One token beside a projection of 2048 to 2304, rank 16: 4.3
// us in the kernel, a chain of cold reads (adapter, A and x) and two exchanges; 64 of 48
// adapters beside q/k/v (19.6 MB): 6.8 us, 2.9 TB/s.
// Runs of rows (prompts): two launches over tiles of 32 rows of a segment.
//   * lora_down_tiles_kernel: t^T = A x^T on v_mfma_f32_16x16x32: a lane's x row is the
//     column of its sums, so that a row's scale is the lane's own.  x is f32: for f16
//     adapters it is taken as f16 hi + lo of x 2^e, e from the largest of the row seen so
//     far (22 bits of each value, down to 2^-38 of the largest), the sums rescaled when
//     that grows; for bf16 ones as three bf16 parts, its 24 bits.
//   * lora_up_tiles_kernel: y += t B^T on v_mfma_f32_32x32x16, t in parts as above, a
//     lane a column: rows of y are read and written in runs of 128 bytes.
// Bound by y's bytes: 4096 rows of twelve segments beside gate and up (2304 to 18432, rank
// 32, f16: 656 MB) 102 us, 6.4 TB/s with what the last-level cache still holds; 15 of them
// in the first kernel, 85 to 94 in the second.  2048 rows of four, 5376 to 21504, rank 64, bf16
// (410 MB): 90 us, 13 and 79, where every tile reads the 2.7 MB of an adapter's B again.
#include "common.h"
#include "wave.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct LoraArgs {
    const uint16_t *a, *b;
    const float *scales;
    const int32_t *adapters, *row_starts;
    const float *x;
    float *y, *t;  // t [split][rows][slices * rank]
    int64_t x_stride, y_stride;
    int segments, rows, num_adapters, rank, k, n, slices;
    int splits, columns;  // columns of a workgroup
    int slice_end[4], group_end[4];  // columns and workgroups up to a slice's end
};

// The slice that a workgroup's columns lie in, and the first of them.
__device__ __forceinline__ void columns_of(const LoraArgs &a, int group, int &slice, int &col, int &end) {
    slice = 0;
    while (group >= a.group_end[slice]) ++slice;
    const int first = slice ? a.group_end[slice - 1] : 0, begin = slice ? a.slice_end[slice - 1] : 0;
    col = begin + (group - first) * a.columns;
    end = std::min(a.slice_end[slice], col + a.columns);
}

__device__ __forceinline__ int adapter_at(const LoraArgs &a, int segment) {
    const int id = a.adapters[segment];
    return id >= 0 && id < a.num_adapters ? id : -1;
}
// The adapter of a row; -1: none.
__device__ __forceinline__ int adapter_of(const LoraArgs &a, int row) {
    int s = row;
    if (a.row_starts) {
        int lo = 0, hi = a.segments;  // the last segment that begins at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.row_starts[mid] <= row) lo = mid;
            else hi = mid;
        }
        if (row < a.row_starts[lo] || row >= a.row_starts[lo + 1]) return -1;
        s = lo;
    }
    return adapter_at(a, s);
}
// Tiles of 32 rows.  Segment i has the places from row_starts[i] / 32 + i on, one more than
// its rows can take at most, so that a place's segment is found by a search in
// row_starts, 64 ways at a time.  Returns the place's adapter (-1: none, or no rows).
constexpr int kTile = 32, kShift = 5;
__device__ __forceinline__ int find_tile(const LoraArgs &a, int place, int &row, int &count) {
    const int lane = threadIdx.x & 63;
    row = count = 0;
    int lo = 0, n = a.segments, start = 0, end = 0;
    for (;;) {
        const int step = (n + 63) >> 6, i = lo + lane * step;
        const bool in = i < lo + n;
        const int from = in ? a.row_starts[i] : 0, to = in && step == 1 ? a.row_starts[i + 1] : 0;
        const uint64_t at_or_before = __ballot(in && (from >> kShift) + i <= place);
        if (at_or_before == 0) return -1;
        const int at = 63 - __builtin_clzll(at_or_before);
        if (step == 1) {
            lo += at;
            start = __builtin_amdgcn_readlane(from, at);
            end = __builtin_amdgcn_readlane(to, at);
            break;
        }
        lo += at * step;
        n = std::min(step, n - at * step);
    }
    if (start < 0) return -1;
    const int64_t first = (int64_t)start + (int64_t)(place - (start >> kShift) - lo) * kTile;
    const int64_t left = std::min(end, a.rows) - first;
    if (left <= 0) return -1;
    row = (int)first;
    count = (int)std::min<int64_t>(kTile, left);
    return adapter_at(a, lo);
}
template <bool BF16>
__device__ __forceinline__ void weights8(const u32x4 w, float *f) {
    if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const h8 h = __builtin_bit_cast(h8, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
    }
}
// t[j] = A_j . x for the `rank` rows of A at `w`, into LDS: a wave four of them and a part
// of k, parts added in their order.
constexpr int kTokenWaves = 16, kMaxRank = 256;
template <bool BF16>
__device__ __forceinline__ void token_down(const LoraArgs &a, const uint16_t *w, const float *x, float *t, float (*part)[kTokenWaves]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int fours = a.rank / 4, ways = std::max(1, kTokenWaves / fours);  // waves of a four
    const int way = wave % ways, units = (a.k + 511) / 512, per = (units + ways - 1) / ways;
    for (int j0 = 4 * (wave / ways); j0 < a.rank; j0 += 4 * (kTokenWaves / ways)) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const uint16_t *rows = w + (int64_t)j0 * a.k;
#pragma unroll 2
        for (int u = way * per; u < std::min(units, (way + 1) * per); ++u) {
            const int at = u * 512 + lane * 8;
            if (at >= a.k) continue;
            const f4 x0 = *reinterpret_cast<const f4 *>(x + at), x1 = *reinterpret_cast<const f4 *>(x + at + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[8];
                weights8<BF16>(*reinterpret_cast<const u32x4 *>(rows + (int64_t)j * a.k + at), f);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[j] = fmaf(x1[i], f[i + 4], fmaf(x0[i], f[i], sum[j]));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sum[j] = doe::wave_sum_last(sum[j]);
            if (lane == 63) part[j0 + j][way] = sum[j];
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < a.rank; j += 64 * kTokenWaves) {
        float sum = 0.0f;
        for (int i = 0; i < ways; ++i) sum += part[j][i];
        t[j] = sum;
    }
    __syncthreads();
}

// This wave's part of four rows of A, k apart, times x: every `ways`-th 512 of k.  Two of
// them are on their way at once, whole (lanes past k take the first values, times 0): a
// load that a lane's condition guards is waited for by itself (a token of rank 64, 5376 to
// 21504: 9.4 to 8.9 us).  token_down, whose waves have one or two and whose lanes past k
// load nothing, is a form of its own: by this one 64 tokens of 2304 take 6.36 for 6.28 us,
// four of 16000 6.57 for 6.41, 214 of 232 26.3 for 25.8.
template <bool BF16>
__device__ __forceinline__ void four_dots(const uint16_t *rows, const float *x, int k, int way, int ways, float *sum) {
    const int units = (k + 511) / 512, mine = (threadIdx.x & 63) * 8;
    struct Unit {
        f4 x0, x1;
        u32x4 w[4];
    };
    auto load = [&](Unit &v, int u) __attribute__((always_inline)) {
        const int at = u * 512 + mine, from = at < k ? at : 0;
        v.x0 = *reinterpret_cast<const f4 *>(x + from);
        v.x1 = *reinterpret_cast<const f4 *>(x + from + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v.w[j] = *reinterpret_cast<const u32x4 *>(rows + (int64_t)j * k + from);
    };
    auto add = [&](const Unit &v, int u) __attribute__((always_inline)) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = u * 512 + mine < k ? (i < 4 ? v.x0[i & 3] : v.x1[i & 3]) : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[8];
            weights8<BF16>(v.w[j], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[j] = fmaf(y[i], f[i], sum[j]);
        }
    };
    for (int u = way; u < units; u += 2 * ways) {
        Unit v0, v1;
        load(v0, u);
        if (u + ways < units) load(v1, u + ways);
        add(v0, u);
        if (u + ways < units) add(v1, u + ways);
    }
}

// t of a row, four rows of A a workgroup, its waves every fourth 512 of k.
template <bool BF16>
__global__ __launch_bounds__(256) void lora_down_rows_kernel(LoraArgs a) {
    __shared__ float part[4][4];
    const int per_row = a.slices * a.rank, fours = per_row / 4, row = blockIdx.x / fours, j0 = (blockIdx.x - row * fours) * 4;
    const int id = adapter_of(a, row);
    if (id < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    four_dots<BF16>(a.a + ((int64_t)id * per_row + j0) * a.k, a.x + (int64_t)row * a.x_stride, a.k, wave, 4, sum);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sum[j] = doe::wave_sum_last(sum[j]);
        if (lane == 63) part[j][wave] = sum[j];
    }
    __syncthreads();
    const int j = threadIdx.x;
    if (j < 4) a.t[(int64_t)row * per_row + j0 + j] = (part[j][0] + part[j][1]) + (part[j][2] + part[j][3]);
}

// A thread a column; its B and y are on their way while t is formed (FUSED), or read.
template <bool BF16, bool FUSED>
__global__ __launch_bounds__(64 * kTokenWaves) void lora_token_kernel(LoraArgs a) {
    __shared__ __align__(16) float t[kMaxRank];
    __shared__ float part[FUSED ? kMaxRank : 1][kTokenWaves];
    const int groups = a.group_end[3], row = blockIdx.x / groups, id = adapter_of(a, row);
    if (id < 0) return;
    int slice, col, end;
    columns_of(a, blockIdx.x - row * groups, slice, col, end);
    col += threadIdx.x;
    constexpr int kAhead = 4;  // eights of the rank
    const uint16_t *b = a.b + ((int64_t)id * a.n + std::min(col, end - 1)) * a.rank;
    float *y = a.y + (int64_t)row * a.y_stride + std::min(col, end - 1), was = *y;
    u32x4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = *reinterpret_cast<const u32x4 *>(b + (8 * i < a.rank ? 8 * i : 0));
    const float scale = a.scales ? a.scales[id] : 1.0f;
    if constexpr (FUSED) {
        token_down<BF16>(a, a.a + ((int64_t)id * a.slices + slice) * a.rank * a.k, a.x + (int64_t)row * a.x_stride, t, part);
    } else {
        if ((int)threadIdx.x < a.rank) t[threadIdx.x] = a.t[((int64_t)row * a.slices + slice) * a.rank + threadIdx.x];
        __syncthreads();
    }
    if (col >= end) return;
    float sum = 0.0f;
    auto add = [&](const u32x4 &w, int j) __attribute__((always_inline)) {
        float f[8];
        weights8<BF16>(w, f);
        const f4 t0 = *reinterpret_cast<const f4 *>(t + j), t1 = *reinterpret_cast<const f4 *>(t + j + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fmaf(t1[i], f[4 + i], fmaf(t0[i], f[i], sum));
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (8 * i < a.rank) add(ahead[i], 8 * i);
    for (int j = 8 * kAhead; j < a.rank; j += 8) add(*reinterpret_cast<const u32x4 *>(b + j), j);
    *y = fmaf(scale, sum, was);
}

// ---- tiles of 32 rows ----------------------------------------------------------------

template <bool BF16>
struct Parts {
    using V = std::conditional_t<BF16, b8, h8>;
    static constexpr int kCount = BF16 ? 3 : 2;
    V v[kCount];
};
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma16(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(h8 a, h8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(b8 a, b8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Eight values, times a power of two, in parts whose sum has 22 bits of them (f16: hi,
// cut off, and lo of what that leaves) or all 24 (bf16: eight bits a part; `scale`
// is 1).
template <bool BF16>
__device__ __forceinline__ Parts<BF16> split8(const float *f, float scale) {
    Parts<BF16> p;
    u32x4 u[Parts<BF16>::kCount];
    float minus = -1.0f;  // (a value, so that g - hi is one instruction that takes hi as f16)
    __asm__ volatile("" : "+v"(minus));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f0 = f[2 * i], f1 = f[2 * i + 1];
        if constexpr (BF16) {
            constexpr uint32_t kUpper = 0x07060302u;  // the upper halves of both
            const float g0 = f0 - __uint_as_float(__float_as_uint(f0) & 0xffff0000u), g1 = f1 - __uint_as_float(__float_as_uint(f1) & 0xffff0000u);
            const float h0 = g0 - __uint_as_float(__float_as_uint(g0) & 0xffff0000u), h1 = g1 - __uint_as_float(__float_as_uint(g1) & 0xffff0000u);
            u[0][i] = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), kUpper);
            u[1][i] = __builtin_amdgcn_perm(__float_as_uint(g1), __float_as_uint(g0), kUpper);
            u[2][i] = __builtin_amdgcn_perm(__float_as_uint(h1), __float_as_uint(h0), kUpper);
        } else {
            const float g0 = f0 * scale, g1 = f1 * scale;
            const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(g0, g1));
            const h2 lo = {(_Float16)fmaf((float)hi[0], minus, g0), (_Float16)fmaf((float)hi[1], minus, g1)};
            u[0][i] = __builtin_bit_cast(uint32_t, hi);
            u[1][i] = __builtin_bit_cast(uint32_t, lo);
        }
    }
#pragma unroll
    for (int k = 0; k < Parts<BF16>::kCount; ++k) p.v[k] = __builtin_bit_cast(typename Parts<BF16>::V, u[k]);
    return p;
}
// e such that the largest magnitude of a row lies in [2^13, 2^14) times 2^-e, held within
// what 2^-e can be; `none` where there is none, or an infinity.
__device__ __forceinline__ int exponent_of(float top, int none) {
    return top > 0.0f && top < __builtin_inff() ? std::max(-112, std::min(112, __builtin_amdgcn_frexp_expf(top) - 14)) : none;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ float largest8(const float *f) {
    float top = fmaxf(fabsf(f[0]), fabsf(f[1]));
#pragma unroll
    for (int i = 2; i < 8; i += 2) top = fmaxf(fmaxf(top, fabsf(f[i])), fabsf(f[i + 1]));
    return top;
}

constexpr int kDownCols = 64;  // rows of A of a workgroup

// At most N vector-memory operations outstanding.
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
    __asm__ volatile("" ::: "memory");
}

// t^T of a tile and 64 rows of A over this split's share of k: the waves take every eighth
// step of 32 and are added up through LDS.  A step's x (32 rows of 128 bytes) and A (64 of
// 64) go to the wave's own LDS by direct loads, lanes in the rows' order, two steps under
// way: read as operands (a lane a row) straight from memory the sixteen lanes that a load
// takes at once lie in as many lines, four times its time.  16-byte pieces of a row are
// exchanged by row so that the lanes' reads fall on different banks.
constexpr int kDownWaves = 8, kStepBytes = 8192;
constexpr int kDownLds = kDownWaves * 2 * kStepBytes;  // (the sums take half of it at the end)
template <bool BF16>
__global__ __launch_bounds__(64 * kDownWaves, 2) void lora_down_tiles_kernel(LoraArgs a) {
    using P = Parts<BF16>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4, per_row = a.slices * a.rank;
    const int col_groups = (per_row + kDownCols - 1) / kDownCols;
    const int rest = blockIdx.x / col_groups, cols0 = (blockIdx.x - rest * col_groups) * kDownCols;
    const int tile = rest / a.splits, split = rest - tile * a.splits;
    int row0, count;
    const int id = find_tile(a, tile, row0, count);
    if (id < 0) return;
    const int steps = (a.k + 31) / 32, parts = kDownWaves * a.splits, part = kDownWaves * split + wave;
    const uint8_t *x = reinterpret_cast<const uint8_t *>(a.x + (int64_t)row0 * a.x_stride);
    const uint8_t *w = reinterpret_cast<const uint8_t *>(a.a + (int64_t)id * per_row * a.k);
    const uint32_t k4 = 4 * a.k;
    // this lane's place in the loads: eight rows of x and sixteen of A each
    uint32_t x_at[4], w_at[4];
    const uint32_t x_piece = ((lane & 7) ^ (lane >> 4)) * 16, w_piece = ((lane & 3) ^ (lane >> 4)) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x_at[i] = (uint32_t)std::min(8 * i + (lane >> 3), count - 1) * (uint32_t)a.x_stride * 4;
        w_at[i] = (uint32_t)std::min(cols0 + 16 * i + (lane >> 2), per_row - 1) * (uint32_t)a.k * 2;
    }
    uint8_t *mine = lds + wave * 2 * kStepBytes;
    auto load = [&](int step, int buffer) __attribute__((always_inline)) {
        // (past the end: k's first values, and weights of zero below)
        uint8_t *to = mine + buffer * kStepBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (rows 8 i .. 8 i + 7: the exchange goes by row / 2)
            const uint32_t at = 128 * step + (x_piece ^ (64 * (i & 1)));
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(x + (x_at[i] + (at < k4 ? at : 0))),
                                             (__attribute__((address_space(3))) void *)(to + 1024 * i), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = 64 * step + w_piece;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(w + (w_at[i] + (2 * at < k4 ? at : 0))),
                                             (__attribute__((address_space(3))) void *)(to + 4096 + 1024 * i), 16, 0, 0);
        }
    };
    f4 acc[2][4];
    constexpr int kUnscaled = -120;
    int e[2] = {kUnscaled, kUnscaled};  // of the scale of a lane's row
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    load(part, 0);
    load(part + parts, 1);
    int buffer = 0;
#pragma unroll 1
    for (int step = part; step < steps; step += parts, buffer ^= 1) {
        wait_vm<8>();  // this step's have landed; the next one's are younger
        const uint8_t *from = mine + buffer * kStepBytes;
        f4 raw[2][2];
        u32x4 wt[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint8_t *row = from + (16 * r + c16) * 128;
            const int turn = c16 >> 1;  // (row / 2) % 8
            raw[r][0] = *reinterpret_cast<const f4 *>(row + ((2 * g4) ^ turn) * 16);
            raw[r][1] = *reinterpret_cast<const f4 *>(row + ((2 * g4 + 1) ^ turn) * 16);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) wt[c] = *reinterpret_cast<const u32x4 *>(from + 4096 + (16 * c + c16) * 64 + (g4 ^ (c16 >> 2)) * 16);
        // (in registers before the next loads overwrite them)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        load(step + 2 * parts, buffer);
        const bool in = 128 * step + 32 * g4 < (int)k4;
#pragma unroll
        for (int c = 0; c < 4; ++c) wt[c] = in ? wt[c] : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = raw[r][i >> 2][i & 3];
            if constexpr (!BF16) {
                int want = exponent_of(largest8(f), kUnscaled);
                if (__any(want > e[r] + 1)) {
                    want = std::max(want, __shfl_xor(want, 16, 64));
                    want = std::max(want, __shfl_xor(want, 32, 64));
                    const int next = want > e[r] + 1 ? want : e[r];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][c][i] = __builtin_amdgcn_ldexpf(acc[r][c][i], e[r] - next);
                    e[r] = next;
                }
            }
            const P p = split8<BF16>(f, BF16 ? 1.0f : power_of_two(-e[r]));
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < P::kCount; ++i) acc[r][c] = mfma16(__builtin_bit_cast(typename P::V, wt[c]), p.v[i], acc[r][c]);
        }
    }
    wait_vm<0>();
    __syncthreads();  // every wave is done with its buffers
    f4 *sums = reinterpret_cast<f4 *>(lds);  // [wave][r][c][lane]
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if constexpr (!BF16)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r][c][i] = __builtin_amdgcn_ldexpf(acc[r][c][i], e[r]);
            sums[((wave * 2 + r) * 4 + c) * 64 + lane] = acc[r][c];
        }
    __syncthreads();
    static_assert(kDownWaves == 8, "a thread four sums");
    const int c = wave & 3, r = wave >> 2, row = 16 * r + c16, col = cols0 + 16 * c + 4 * g4;
    if (row >= count || col >= per_row) return;
    f4 s = sums[(r * 4 + c) * 64 + lane];
#pragma unroll
    for (int v = 1; v < kDownWaves; ++v) s += sums[((v * 2 + r) * 4 + c) * 64 + lane];
    *reinterpret_cast<f4 *>(a.t + ((int64_t)split * a.rows + row0 + row) * per_row + col) = s;
}

// y += s t B^T of a tile of 32 rows and a workgroup's columns, 32 of them a wave at a
// time.  RS: steps of 16 of the rank.  y is read and written past the caches: B, read
// again for every tile, stays there (four prompts at rank 64: 94 to 80 us).  Tiles of 64
// rows, which read B half as often, take more registers than there are: 94 to 109 us beside
// gate and up, 80 to 155 at rank 64; as two halves one after the other 104 and 82.
template <bool BF16, int RS>
__global__ __launch_bounds__(256, 2) void lora_up_tiles_kernel(LoraArgs a) {
    using P = Parts<BF16>;
    __shared__ typename P::V ops[RS][P::kCount][64];
    __shared__ float row_scale[kTile];
    __shared__ uint32_t tops[kTile];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n32 = lane & 31, lh = lane >> 5, groups = a.group_end[3], tile = blockIdx.x / groups;
    int row0, count, slice, col0, end;
    const int id = find_tile(a, tile, row0, count);
    if (id < 0) return;
    columns_of(a, blockIdx.x - tile * groups, slice, col0, end);
    const float scale = a.scales ? a.scales[id] : 1.0f;
    if (tid < kTile) tops[tid] = 0;
    __syncthreads();
    {
        // t, its splits added in their order: a thread eight values of a row at a time
        constexpr int kThreads = 256 / kTile, N = (2 * RS + kThreads - 1) / kThreads;  // of a row; units of one
        const int row = tid % kTile, first = tid / kTile, per_row = a.slices * a.rank;
        float f[N][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = first + kThreads * i;
            f4 v0 = {0.0f, 0.0f, 0.0f, 0.0f}, v1 = v0;
            if (8 * u < a.rank && row < count) {
                const float *t = a.t + (int64_t)(row0 + row) * per_row + slice * a.rank + 8 * u;
                // (four splits' reads at once; from rank 33 on that costs registers and 2 us of 89)
#pragma unroll(RS <= 2 ? 4 : 1)
                for (int z = 0; z < a.splits; ++z, t += (int64_t)a.rows * per_row) {
                    v0 += *reinterpret_cast<const f4 *>(t);
                    v1 += *reinterpret_cast<const f4 *>(t + 4);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i][j] = v0[j], f[i][4 + j] = v1[j];
            top = fmaxf(top, largest8(f[i]));
        }
        int e = 0;
        if constexpr (!BF16) {
            atomicMax(&tops[row], __float_as_uint(top));
            __syncthreads();
            e = exponent_of(__uint_as_float(tops[row]), 0);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = first + kThreads * i;
            if (u >= 2 * RS) continue;
            const P p = split8<BF16>(f[i], power_of_two(-e));
#pragma unroll
            for (int k = 0; k < P::kCount; ++k) ops[u >> 1][k][(u & 1) * 32 + row] = p.v[k];
        }
        if (first == 0) row_scale[row] = scale * power_of_two(e);
    }
    __syncthreads();
    float rs[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) rs[r] = row_scale[8 * (r >> 2) + 4 * lh + (r & 3)];

    float *y = a.y + (int64_t)row0 * a.y_stride;
    const uint16_t *b = a.b + (int64_t)id * a.n * a.rank;
    struct Block {
        float y[16];
        u32x4 b[RS];
    };
    auto work = [&](auto whole_) __attribute__((always_inline)) {
        constexpr bool whole = decltype(whole_)::value;
        // a lane's place in y: its column and the first of its rows (of four in every eight)
        auto at = [&](int r, int col) __attribute__((always_inline)) {
            return y + (8 * (r >> 2) + (r & 3)) * a.y_stride + (uint32_t)(4 * lh * (uint32_t)a.y_stride + (uint32_t)col);
        };
        auto mine = [&](int r) __attribute__((always_inline)) { return whole || 8 * (r >> 2) + 4 * lh + (r & 3) < count; };
        auto load = [&](Block &v, int c0) __attribute__((always_inline)) {
            const int col = c0 + n32;
            if (col >= end) return;
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                v.b[s] = u32x4{0, 0, 0, 0};
                const int k = 16 * s + 8 * lh;
                if (k < a.rank) v.b[s] = *reinterpret_cast<const u32x4 *>(b + (int64_t)col * a.rank + k);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (mine(r)) v.y[r] = __builtin_nontemporal_load(at(r, col));
        };
        auto add = [&](Block &v, int c0) __attribute__((always_inline)) {
            const int col = c0 + n32;
            f32x16 acc = {};
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int k = 0; k < P::kCount; ++k) {
                    acc = mfma32(ops[s][k][lane], __builtin_bit_cast(typename P::V, v.b[s]), acc);
                    if (s % 4 == 3 && k == P::kCount - 1) __builtin_amdgcn_sched_barrier(0);  // (t's parts are not read all at once)
                }
            if (col >= end) return;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (mine(r)) __builtin_nontemporal_store(fmaf(acc[r], rs[r], v.y[r]), at(r, col));
        };
        int c = col0 + 32 * wave;
        Block v0 = {};
        if constexpr (RS <= 4) {
            Block v1 = {};
            if (c < end) load(v0, c);
            for (; c < end; c += 256) {
                if (c + 128 < end) load(v1, c + 128);
                add(v0, c);
                if (c + 256 < end) load(v0, c + 256);
                if (c + 128 < end) add(v1, c + 128);
            }
        } else {
            for (; c < end; c += 128) {
                load(v0, c);
                add(v0, c);
            }
        }
    };
    if (count == kTile) work(std::integral_constant<bool, true>());
    else work(std::integral_constant<bool, false>());
}

// ---- the host's side -------------------------------------------------------------------

int lora_checks(const doe_lora *l, int64_t rows, LoraArgs &a) {
    DOE_REQUIRE(l && l->a && l->b, DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(l->rank > 0 && l->rank <= 256 && l->rank % 8 == 0, DOE_E_UNSUPPORTED,
                "rank %lld unsupported (a multiple of 8 up to 256)", (long long)l->rank);
    DOE_REQUIRE(l->k > 0 && l->k <= ((int64_t)1 << 20) && l->k % 8 == 0, DOE_E_UNSUPPORTED,
                "k %lld unsupported (a multiple of 8 up to 2^20)", (long long)l->k);
    DOE_REQUIRE(l->slices >= 1 && l->slices <= 4, DOE_E_INVALID, "slices %lld outside 1..4", (long long)l->slices);
    DOE_REQUIRE(l->num_adapters > 0 && l->num_adapters < ((int64_t)1 << 24), DOE_E_INVALID, "num_adapters %lld",
                (long long)l->num_adapters);
    int64_t n = 0;
    for (int s = 0; s < 4; ++s) {
        if (s < l->slices) {
            DOE_REQUIRE(l->slice_n[s] > 0 && l->slice_n[s] <= ((int64_t)1 << 22), DOE_E_INVALID, "slice_n[%d] %lld", s,
                        (long long)l->slice_n[s]);
            n += l->slice_n[s];
        }
        a.slice_end[s] = (int)n;
    }
    DOE_REQUIRE(((uintptr_t)l->a & 15) == 0 && ((uintptr_t)l->b & 15) == 0, DOE_E_INVALID, "a and b must be 16-byte aligned");
    DOE_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 24), DOE_E_INVALID, "rows %lld", (long long)rows);
    a.a = static_cast<const uint16_t *>(l->a);
    a.b = static_cast<const uint16_t *>(l->b);
    a.scales = l->scales;
    a.num_adapters = (int)l->num_adapters;
    a.rank = (int)l->rank;
    a.k = (int)l->k;
    a.n = (int)n;
    a.slices = (int)l->slices;
    a.rows = (int)rows;
    return DOE_OK;
}

constexpr int kMaxSplits = 8, kCus = 256;

// Workgroups a slice of `columns` each.
void set_columns(LoraArgs &a, int columns) {
    a.columns = columns;
    int groups = 0;
    for (int s = 0; s < 4; ++s) {
        const int begin = s ? a.slice_end[s - 1] : 0;
        groups += (a.slice_end[s] - begin + columns - 1) / columns;
        a.group_end[s] = groups;
    }
}
// Whether a call takes tiles: where segments have rows to share weights, and what the rows
// would read of them by themselves, or their workgroups, cost more than the tiles'
// launches.  Rows by themselves against tiles, rank 16 of 2304 to 4096 columns in three
// slices: 64 rows (22 MB) of 32 segments 7.3 and 13.3 us, 128 (45 MB) 12.9 and 13.6, 256 (90
// MB) 19.8 and 14.6, 512 31.9 and 16.7; rank 64 of 5376 to 21504, 16 rows of 8 (55 MB) 19.5
// and 17.7, 64 41.6 and 19.5; rank 8 of 1024 to 300, 600 rows (600 workgroups) 10.0 and 10.6;
// rank 32 of 256 to 62 in three slices, 638 rows (1914) 26.9 and 10.2.
bool by_tiles(const LoraArgs &a, bool starts, int64_t segments) {
    const int64_t bytes = 2 * (int64_t)a.rows * a.rank * ((int64_t)a.slices * a.k + a.n);
    return starts && a.rows >= 2 * segments && (bytes > (48 << 20) || (int64_t)a.rows * a.group_end[3] > 640);
}
int64_t tiles_of(const LoraArgs &a, int64_t segments) { return a.rows / kTile + segments; }
// Splits of k: workgroups for the device, two steps of 32 a wave at least.
int64_t most_splits(const LoraArgs &a) {
    return std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, (a.k + 31) / 32 / (2 * kDownWaves)));
}
int splits_of(const LoraArgs &a, int64_t tiles) {
    const int64_t wgs = tiles * ((a.slices * a.rank + kDownCols - 1) / kDownCols);
    return (int)std::max<int64_t>(1, std::min(most_splits(a), kCus / wgs));
}
// Copies of t for any count of segments, and for any fewer rows: rows times splits_of, of
// which a call has more than one only where tiles x column groups (of rows / 32 at the
// least) leave CUs over.
int64_t workspace_of(const LoraArgs &a) {
    const int64_t per_row = (int64_t)a.slices * a.rank, groups = (per_row + kDownCols - 1) / kDownCols;
    const int64_t split_rows = std::min<int64_t>(a.rows * most_splits(a), kCus * kTile / groups);
    return std::max<int64_t>(16, 4 * per_row * std::max<int64_t>(a.rows, split_rows));
}

// Whether a call of rows forms t again in every workgroup that uses it: one launch instead
// of two, for what a workgroup then reads of A by itself and all of them together.  One
// launch against two: a token of rank 16, 2048 to 2304 5.0 and 7.0 us, of 5376 to 21504 (172
// KB a workgroup) 6.4 and 7.0, of rank 64 (688 KB) 14.5 and 9.8; 64 tokens of rank 16, 2304 to
// 4096 (19 MB) 7.2 and 10.7, 128 (38 MB) 11.6 and 11.2, 200 to 9216 (147 MB) 38.5 and 17.3.
bool in_one(const LoraArgs &a, int64_t wgs) {
    const int64_t bytes = 2 * (int64_t)a.rank * a.k;
    return bytes <= (256 << 10) && wgs * bytes <= (36 << 20);
}

// A launch has fewer than 2^32 threads.
int fits(const LoraArgs &a, int64_t threads) {
    DOE_REQUIRE(threads < ((int64_t)1 << 32), DOE_E_UNSUPPORTED, "%d rows of %d columns in one call", a.rows, a.n);
    return DOE_OK;
}

template <bool BF16, int RS>
int launch_up(const LoraArgs &a, int64_t segments, hipStream_t st) {
    const int64_t wgs = tiles_of(a, segments) * a.group_end[3];
    hipLaunchKernelGGL((lora_up_tiles_kernel<BF16, RS>), dim3((unsigned)wgs), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("lora_up_tiles_kernel");
    return DOE_OK;
}

template <bool BF16>
int launch(LoraArgs &a, bool starts, int64_t segments, hipStream_t st) {
    int rc;
    set_columns(a, 64 * kTokenWaves);
    if (!by_tiles(a, starts, segments)) {
        const int64_t wgs = (int64_t)a.rows * a.group_end[3], down = (int64_t)a.rows * a.slices * a.rank / 4;
        if ((rc = fits(a, wgs * 64 * kTokenWaves)) || (rc = fits(a, down * 256))) return rc;
        if (in_one(a, wgs)) {
            hipLaunchKernelGGL((lora_token_kernel<BF16, true>), dim3((unsigned)wgs), dim3(64 * kTokenWaves), 0, st, a);
        } else {
            hipLaunchKernelGGL(lora_down_rows_kernel<BF16>, dim3((unsigned)down), dim3(256), 0, st, a);
            DOE_LAUNCH_CHECK("lora_down_rows_kernel");
            hipLaunchKernelGGL((lora_token_kernel<BF16, false>), dim3((unsigned)wgs), dim3(64 * kTokenWaves), 0, st, a);
        }
        DOE_LAUNCH_CHECK("lora_token_kernel");
        return DOE_OK;
    }
    const int64_t tiles = tiles_of(a, segments), col_groups = (a.slices * a.rank + kDownCols - 1) / kDownCols;
    a.splits = splits_of(a, tiles);
    // 512 columns a workgroup, fewer where that leaves the device short of them (150 rows of four,
    // 512 columns: 13.8 to 10.7 us; 27 of five, 8577: 19.8 to 16.4)
    for (int columns = 512; columns >= 128; columns /= 2) {
        set_columns(a, columns);
        if (tiles * a.group_end[3] >= 2 * kCus) break;
    }
    const int64_t wgs = tiles * a.splits * col_groups;
    // (both before either runs)
    if ((rc = fits(a, wgs * 64 * kDownWaves)) || (rc = fits(a, tiles * a.group_end[3] * 256))) return rc;
    static const hipError_t attr_rc = hipFuncSetAttribute((const void *)lora_down_tiles_kernel<BF16>,
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, kDownLds);
    DOE_HIP_CHECK(attr_rc);
    hipLaunchKernelGGL(lora_down_tiles_kernel<BF16>, dim3((unsigned)wgs), dim3(64 * kDownWaves), kDownLds, st, a);
    DOE_LAUNCH_CHECK("lora_down_tiles_kernel");
    if (a.rank <= 16) return launch_up<BF16, 1>(a, segments, st);
    if (a.rank <= 32) return launch_up<BF16, 2>(a, segments, st);
    if (a.rank <= 64) return launch_up<BF16, 4>(a, segments, st);
    if (a.rank <= 128) return launch_up<BF16, 8>(a, segments, st);
    return launch_up<BF16, 16>(a, segments, st);
}

}  // namespace

extern "C" {

int doe_lora_workspace(const doe_lora *lora, int64_t rows, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    LoraArgs a{};
    const int rc = lora_checks(lora, rows, a);
    if (rc) return rc;
    *bytes = workspace_of(a);
    return DOE_OK;
}

int doe_lora_add(const doe_lora *lora, const int32_t *adapters, const int32_t *row_starts, int64_t segments,
                 const float *x, int64_t x_row_stride, float *y, int64_t y_row_stride, int64_t rows, void *workspace,
                 int64_t workspace_bytes, doe_stream_t stream) {
    LoraArgs a{};
    int rc = lora_checks(lora, rows, a);
    if (rc) return rc;
    DOE_REQUIRE(segments >= 0 && segments < ((int64_t)1 << 24), DOE_E_INVALID, "segments %lld", (long long)segments);
    DOE_REQUIRE(row_starts || segments == rows, DOE_E_INVALID, "without row_starts a segment is a row (%lld segments, %lld rows)",
                (long long)segments, (long long)rows);
    DOE_REQUIRE(x_row_stride >= a.k && x_row_stride % 4 == 0 && x_row_stride < ((int64_t)1 << 24), DOE_E_INVALID,
                "x_row_stride %lld outside k %d .. 2^24, or not a multiple of 4", (long long)x_row_stride, a.k);
    DOE_REQUIRE(y_row_stride >= a.n && y_row_stride < ((int64_t)1 << 26), DOE_E_INVALID,
                "y_row_stride %lld outside the %d columns .. 2^26", (long long)y_row_stride, a.n);
    DOE_REQUIRE(rows == 0 || segments == 0 || (adapters && x && y), DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 3) == 0, DOE_E_INVALID, "x must be 16-byte, y 4-byte aligned");
    // whole, or column by column within rows of the same stride
    const uintptr_t from = (uintptr_t)x, to = (uintptr_t)y, row = 4 * (uintptr_t)x_row_stride;
    const uintptr_t behind = to >= from ? (to - from) % row : (row - (from - to) % row) % row;  // of x's row to y's
    const bool columns = x_row_stride == y_row_stride && behind >= 4 * (uintptr_t)a.k && behind + 4 * (uintptr_t)a.n <= row;
    DOE_REQUIRE(rows == 0 || columns || from + (uintptr_t)(((rows - 1) * x_row_stride + a.k) * 4) <= to ||
                    to + (uintptr_t)(((rows - 1) * y_row_stride + a.n) * 4) <= from,
                DOE_E_INVALID, "x and y are apart from each other");
    const int64_t need = workspace_of(a);
    DOE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need, DOE_E_INVALID,
                "a 16-byte aligned workspace of %lld bytes is needed (got %lld)", (long long)need, (long long)workspace_bytes);
    if ((rc = doe::require_init())) return rc;
    if (rows == 0 || segments == 0) return DOE_OK;
    a.adapters = adapters;
    a.row_starts = row_starts;
    a.segments = (int)segments;
    a.x = x;
    a.y = y;
    a.t = static_cast<float *>(workspace);
    a.x_stride = x_row_stride;
    a.y_stride = y_row_stride;
    const hipStream_t st = (hipStream_t)stream;
    return lora->bf16 ? launch<true>(a, row_starts, segments, st) : launch<false>(a, row_starts, segments, st);
}

}  // extern "C"
