// lora.hip -- low-rank adapters of many requests beside a shared projection
// (doe_lora_add): y[r] += s_a B_a (A_a x[r]) for the adapter a of row r's request.
//
// Rows of their own (decode steps): lora_token_kernel, one launch.  A workgroup takes a
// row and some of its columns, forms the t = A x that they need itself (again in every
// workgroup of the row: A comes from the caches) and adds B t.
// Runs of rows (prompts): two launches over tiles of 32 rows of a segment.
//   * lora_down_tiles_kernel: t^T = A x^T on v_mfma_f32_16x16x32: a lane's x row is the
//     column of its sums, so that a row's scale is the lane's own.  x is f32: for f16
//     adapters it is taken as f16 hi + lo of x 2^e, e from the largest of the row seen so
//     far (22 bits of each value, down to 2^-38 of the largest), the sums rescaled when
//     that grows; for bf16 ones as three bf16 parts, its 24 bits.
//   * lora_up_tiles_kernel: y += t B^T on v_mfma_f32_32x32x16, t in parts as above, a
//     lane a column: rows of y are read and written in runs of 128 bytes.
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
    int splits, tiles, columns;  // columns of a workgroup
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
// Tile `tile` of 32 rows: its adapter (-1: none, or no such tile), first row and rows.
constexpr int kTile = 32;
__device__ __forceinline__ int find_tile(const LoraArgs &a, int tile, int &row, int &count) {
    const int lane = threadIdx.x & 63;
    row = count = 0;
    if (!a.row_starts) {
        row = tile;
        count = 1;
        return tile < a.rows ? adapter_at(a, tile) : -1;
    }
    for (int s0 = 0; s0 < a.segments; s0 += 64) {
        const int s = s0 + lane;
        const int lo = s < a.segments ? a.row_starts[s] : 0, hi = s < a.segments ? a.row_starts[s + 1] : 0;
        const int rows = lo < 0 ? 0 : std::max(0, std::min(hi, a.rows) - lo);
        const int upto = doe::wave_scan((rows + kTile - 1) / kTile);
        const uint64_t behind = __ballot(upto > tile);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            const int in = tile - (at ? __builtin_amdgcn_readlane(upto, at - 1) : 0);
            row = __builtin_amdgcn_readlane(lo, at) + in * kTile;
            count = std::min(kTile, __builtin_amdgcn_readlane(rows, at) - in * kTile);
            return adapter_at(a, s0 + at);
        }
        tile -= __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
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
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
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
            sum[j] = wave_sum(sum[j]);
            if (lane == 0) part[j0 + j][way] = sum[j];
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

// A row's columns from `col` to `end`, a thread each.
template <bool BF16>
__device__ __forceinline__ void token_up(const LoraArgs &a, int row, int id, const float *t, int col, int end) {
    const float scale = a.scales ? a.scales[id] : 1.0f;
    for (int c = col + threadIdx.x; c < end; c += 64 * kTokenWaves) {
        const uint16_t *b = a.b + ((int64_t)id * a.n + c) * a.rank;
        float sum = 0.0f;
        for (int j = 0; j < a.rank; j += 8) {
            float f[8];
            weights8<BF16>(*reinterpret_cast<const u32x4 *>(b + j), f);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(t[j + i], f[i], sum);
        }
        float *y = a.y + (int64_t)row * a.y_stride + c;
        *y = fmaf(scale, sum, *y);
    }
}

template <bool BF16>
__global__ __launch_bounds__(64 * kTokenWaves) void lora_token_kernel(LoraArgs a) {
    __shared__ __align__(16) float t[kMaxRank];
    __shared__ float part[kMaxRank][kTokenWaves];
    const int groups = a.group_end[3], row = blockIdx.x / groups, id = adapter_of(a, row);
    if (id < 0) return;
    int slice, col, end;
    columns_of(a, blockIdx.x - row * groups, slice, col, end);
    token_down<BF16>(a, a.a + ((int64_t)id * a.slices + slice) * a.rank * a.k, a.x + (int64_t)row * a.x_stride, t, part);
    token_up<BF16>(a, row, id, t, col, end);
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

// Eight values in parts whose sum has 22 bits of them (f16) or all (bf16).
template <bool BF16>
__device__ __forceinline__ Parts<BF16> split8(const float *f) {
    Parts<BF16> p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (BF16) {
            const __bf16 b0 = (__bf16)f[i];
            const float r0 = f[i] - (float)b0;
            const __bf16 b1 = (__bf16)r0;
            p.v[0][i] = b0;
            p.v[1][i] = b1;
            p.v[2][i] = (__bf16)(r0 - (float)b1);
        } else {
            const _Float16 h = (_Float16)f[i];
            p.v[0][i] = h;
            p.v[1][i] = (_Float16)(f[i] - (float)h);
        }
    }
    return p;
}
// e such that the largest of a row (its bits without the sign) lies in [2^13, 2^14) times
// 2^-e; 0 for none, infinities and NaN.
__device__ __forceinline__ int exponent_of(uint32_t top) {
    return top == 0 || top >= 0x7f800000u ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(top)) - 14;
}

constexpr int kDownCols = 64;  // rows of A of a workgroup

// Two steps of 32 of k: a lane's eight values of two x rows and of four rows of A each.
struct DownRaw {
    f4 x[2][2][2];  // [step][row tile][half]
    u32x4 w[2][4];  // [step][column tile]
};

// t^T of a tile and 64 rows of A over this split's share of k: the waves a quarter of it
// each, added up through LDS.
template <bool BF16>
__global__ __launch_bounds__(256, 2) void lora_down_tiles_kernel(LoraArgs a) {
    using P = Parts<BF16>;
    __shared__ f4 sums[4][2][4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4, per_row = a.slices * a.rank;
    const int col_groups = (per_row + kDownCols - 1) / kDownCols;
    int rest = blockIdx.x / col_groups, row0, count;
    const int cols0 = (blockIdx.x - rest * col_groups) * kDownCols, tile = rest / a.splits, split = rest - tile * a.splits;
    const int id = find_tile(a, tile, row0, count);
    if (id < 0) return;
    const int steps = (a.k + 31) / 32, parts = 4 * a.splits, part = 4 * split + wave;
    const int from = (int)((int64_t)steps * part / parts), to = (int)((int64_t)steps * (part + 1) / parts);
    const float *x[2];
    const uint16_t *w[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) x[r] = a.x + (int64_t)(row0 + std::min(16 * r + c16, count - 1)) * a.x_stride;
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = a.a + ((int64_t)id * per_row + std::min(cols0 + 16 * c + c16, per_row - 1)) * a.k;
    auto load = [&](DownRaw &v, int step) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            // (past the end: k's first values against weights of zero)
            const bool in = step + s < to && 32 * (step + s) + 8 * g4 < a.k;
            const int at = in ? 32 * (step + s) + 8 * g4 : 0;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                v.x[s][r][0] = *reinterpret_cast<const f4 *>(x[r] + at);
                v.x[s][r][1] = *reinterpret_cast<const f4 *>(x[r] + at + 4);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const u32x4 u = *reinterpret_cast<const u32x4 *>(w[c] + at);
                v.w[s][c] = in ? u : u32x4{0, 0, 0, 0};
            }
        }
    };
    f4 acc[2][4];
    int e[2] = {-1000, -1000};  // of the scale of a lane's row
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](const DownRaw &v) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if constexpr (!BF16) {
                uint32_t top = 0;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = std::max(top, __float_as_uint(v.x[s][r][h][i]) & 0x7fffffffu);
                int want = top == 0 || top >= 0x7f800000u ? -1000 : exponent_of(top);
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
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = BF16 ? v.x[s][r][i >> 2][i & 3] : __builtin_amdgcn_ldexpf(v.x[s][r][i >> 2][i & 3], -e[r]);
                const P p = split8<BF16>(f);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < P::kCount; ++i) acc[r][c] = mfma16(__builtin_bit_cast(typename P::V, v.w[s][c]), p.v[i], acc[r][c]);
            }
        }
    };
    DownRaw v0, v1;
    if (from < to) load(v0, from);
    for (int s = from; s < to; s += 4) {
        load(v1, s + 2);
        add(v0);
        load(v0, s + 4);
        if (s + 2 < to) add(v1);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if constexpr (!BF16)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r][c][i] = __builtin_amdgcn_ldexpf(acc[r][c][i], e[r]);
            sums[wave][r][c][lane] = acc[r][c];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int l = i & 63, c = i >> 6 & 3, r = i >> 8, row = 16 * r + (l & 15), col = cols0 + 16 * c + 4 * (l >> 4);
        if (row >= count || col >= per_row) continue;
        const f4 s = (sums[0][r][c][l] + sums[1][r][c][l]) + (sums[2][r][c][l] + sums[3][r][c][l]);
        *reinterpret_cast<f4 *>(a.t + ((int64_t)split * a.rows + row0 + row) * per_row + col) = s;
    }
}

// y += s t B^T of a tile and a workgroup's columns, 32 of them a wave at a time.  RS: steps
// of 16 of the rank.
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
        constexpr int N = (2 * RS + 7) / 8;
        const int row = tid & 31, per_row = a.slices * a.rank;
        float f[N][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = (tid >> 5) + 8 * i;
            f4 v0 = {0.0f, 0.0f, 0.0f, 0.0f}, v1 = v0;
            if (8 * u < a.rank && row < count) {
                const float *t = a.t + (int64_t)(row0 + row) * per_row + slice * a.rank + 8 * u;
                for (int z = 0; z < a.splits; ++z, t += (int64_t)a.rows * per_row) {
                    v0 += *reinterpret_cast<const f4 *>(t);
                    v1 += *reinterpret_cast<const f4 *>(t + 4);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i][j] = v0[j], f[i][4 + j] = v1[j];
#pragma unroll
            for (int j = 0; j < 8; ++j) top = std::max(top, __float_as_uint(f[i][j]) & 0x7fffffffu);
        }
        int e = 0;
        if constexpr (!BF16) {
            atomicMax(&tops[row], top);
            __syncthreads();
            e = exponent_of(tops[row]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = (tid >> 5) + 8 * i;
            if (u >= 2 * RS) continue;
            if constexpr (!BF16)
#pragma unroll
                for (int j = 0; j < 8; ++j) f[i][j] = __builtin_amdgcn_ldexpf(f[i][j], -e);
            const P p = split8<BF16>(f[i]);
#pragma unroll
            for (int k = 0; k < P::kCount; ++k) ops[u >> 1][k][(u & 1) * 32 + row] = p.v[k];
        }
        if (tid < kTile) row_scale[row] = __builtin_amdgcn_ldexpf(scale, e);
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
                if (mine(r)) v.y[r] = *at(r, col);
        };
        auto add = [&](Block &v, int c0) __attribute__((always_inline)) {
            const int col = c0 + n32;
            f32x16 acc = {};
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int k = 0; k < P::kCount; ++k) acc = mfma32(ops[s][k][lane], __builtin_bit_cast(typename P::V, v.b[s]), acc);
            if (col >= end) return;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (mine(r)) *at(r, col) = fmaf(acc[r], rs[r], v.y[r]);
        };
        Block v0 = {}, v1 = {};
        int c = col0 + 32 * wave;
        if (c < end) load(v0, c);
        for (; c < end; c += 256) {
            if (c + 128 < end) load(v1, c + 128);
            add(v0, c);
            if (c + 256 < end) load(v0, c + 256);
            if (c + 128 < end) add(v1, c + 128);
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

// Whether a call takes tiles: runs of rows long enough to share a tile's weights.
bool by_tiles(const LoraArgs &a, bool starts, int64_t segments) { return starts && a.rows >= 8 * segments; }
int64_t tiles_of(const LoraArgs &a, int64_t segments) { return a.rows / kTile + std::min<int64_t>(segments, a.rows); }
// Splits of k: enough workgroups for the device, two steps of 32 a wave at least.
int splits_of(const LoraArgs &a, int64_t tiles) {
    const int64_t wgs = tiles * ((a.slices * a.rank + kDownCols - 1) / kDownCols), steps = (a.k + 31) / 32;
    return (int)std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, 2 * kCus / std::max<int64_t>(1, wgs), steps / 8}));
}
int64_t workspace_of(const LoraArgs &a) {
    return std::max<int64_t>(16, 4 * (int64_t)a.rows * a.slices * a.rank * kMaxSplits);
}

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
// A launch has fewer than 2^32 threads.
int fits(const LoraArgs &a, int64_t threads) {
    DOE_REQUIRE(threads < ((int64_t)1 << 32), DOE_E_UNSUPPORTED, "%d rows of %d columns in one call", a.rows, a.n);
    return DOE_OK;
}

template <bool BF16, int RS>
int launch_up(const LoraArgs &a, hipStream_t st) {
    const int64_t wgs = (int64_t)a.tiles * a.group_end[3];
    const int rc = fits(a, wgs * 256);
    if (rc) return rc;
    hipLaunchKernelGGL((lora_up_tiles_kernel<BF16, RS>), dim3((unsigned)wgs), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("lora_up_tiles_kernel");
    return DOE_OK;
}

template <bool BF16>
int launch(LoraArgs &a, bool starts, int64_t segments, hipStream_t st) {
    int rc;
    if (!by_tiles(a, starts, segments)) {
        set_columns(a, 1024);
        const int64_t wgs = (int64_t)a.rows * a.group_end[3];
        if ((rc = fits(a, wgs * 64 * kTokenWaves))) return rc;
        hipLaunchKernelGGL(lora_token_kernel<BF16>, dim3((unsigned)wgs), dim3(64 * kTokenWaves), 0, st, a);
        DOE_LAUNCH_CHECK("lora_token_kernel");
        return DOE_OK;
    }
    const int64_t tiles = tiles_of(a, segments), col_groups = (a.slices * a.rank + kDownCols - 1) / kDownCols;
    a.splits = splits_of(a, tiles);
    a.tiles = (int)tiles;
    set_columns(a, 512);
    if ((rc = fits(a, tiles * a.splits * col_groups * 256)) || (rc = fits(a, tiles * a.group_end[3] * 256))) return rc;
    hipLaunchKernelGGL(lora_down_tiles_kernel<BF16>, dim3((unsigned)(tiles * a.splits * col_groups)), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("lora_down_tiles_kernel");
    if (a.rank <= 16) return launch_up<BF16, 1>(a, st);
    if (a.rank <= 32) return launch_up<BF16, 2>(a, st);
    if (a.rank <= 64) return launch_up<BF16, 4>(a, st);
    if (a.rank <= 128) return launch_up<BF16, 8>(a, st);
    return launch_up<BF16, 16>(a, st);
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
    DOE_REQUIRE(x_row_stride >= a.k && x_row_stride % 4 == 0 && x_row_stride < ((int64_t)1 << 32), DOE_E_INVALID,
                "x_row_stride %lld below k %d, or not a multiple of 4", (long long)x_row_stride, a.k);
    DOE_REQUIRE(y_row_stride >= a.n && y_row_stride < ((int64_t)1 << 26), DOE_E_INVALID, "y_row_stride %lld below the %d columns", (long long)y_row_stride, a.n);
    DOE_REQUIRE(rows == 0 || segments == 0 || (adapters && x && y), DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 3) == 0, DOE_E_INVALID, "x must be 16-byte, y 4-byte aligned");
    const uintptr_t from = (uintptr_t)x, to = (uintptr_t)y;
    DOE_REQUIRE(rows == 0 || from + (uintptr_t)(((rows - 1) * x_row_stride + a.k) * 4) <= to ||
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
