// lora.hip -- low-rank adapters of many requests beside a shared projection
// (doe_lora_add): y[r] += s_a B_a (A_a x[r]) for the adapter a of row r's request.
#include "common.h"

#include <algorithm>

namespace {

struct LoraArgs {
    const uint16_t *a, *b;
    const float *scales;
    const int32_t *adapters, *row_starts;
    const float *x;
    float *y, *t;  // t [rows][slices * rank]
    int64_t x_stride, y_stride;
    int segments, rows, num_adapters, rank, k, n, slices;
    int slice_end[4];
};

template <bool BF16>
__device__ __forceinline__ float weight(uint16_t w) {
    if constexpr (BF16) return __uint_as_float((uint32_t)w << 16);
    else return (float)__builtin_bit_cast(_Float16, w);
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
    const int id = a.adapters[s];
    return id >= 0 && id < a.num_adapters ? id : -1;
}

// A wave a value of t.
template <bool BF16>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    const int lane = threadIdx.x & 63, per_row = a.slices * a.rank;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = (int)(unit / per_row), j = (int)(unit - (int64_t)row * per_row);
    if (row >= a.rows) return;
    const int id = adapter_of(a, row);
    if (id < 0) return;
    const uint16_t *w = a.a + ((int64_t)id * per_row + j) * a.k;
    const float *x = a.x + (int64_t)row * a.x_stride;
    float sum = 0.0f;
    for (int i = lane; i < a.k; i += 64) sum = fmaf(x[i], weight<BF16>(w[i]), sum);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) a.t[(int64_t)row * per_row + j] = sum;
}

// A thread a value of y.
template <bool BF16>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    const int tiles = (a.n + 255) / 256, row = blockIdx.x / tiles, col = (blockIdx.x - row * tiles) * 256 + threadIdx.x;
    const int id = adapter_of(a, row);
    if (id < 0 || col >= a.n) return;
    int s = 0;
    while (col >= a.slice_end[s]) ++s;
    const float *t = a.t + ((int64_t)row * a.slices + s) * a.rank;
    const uint16_t *w = a.b + ((int64_t)id * a.n + col) * a.rank;
    float sum = 0.0f;
    for (int j = 0; j < a.rank; ++j) sum = fmaf(t[j], weight<BF16>(w[j]), sum);
    const float scale = a.scales ? a.scales[id] : 1.0f;
    float *y = a.y + (int64_t)row * a.y_stride + col;
    *y = fmaf(scale, sum, *y);
}

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

int64_t workspace_of(const LoraArgs &a) { return std::max<int64_t>(16, 4 * (int64_t)a.rows * a.slices * a.rank); }

template <bool BF16>
int launch(const LoraArgs &a, hipStream_t st) {
    const int64_t units = (int64_t)a.rows * a.slices * a.rank;
    DOE_REQUIRE((units + 3) / 4 < (1 << 24) && (int64_t)a.rows * ((a.n + 255) / 256) < (1 << 24), DOE_E_UNSUPPORTED,
                "%d rows of %d columns in one call", a.rows, a.n);  // (a launch has fewer than 2^32 threads)
    hipLaunchKernelGGL(lora_down_kernel<BF16>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("lora_down_kernel");
    hipLaunchKernelGGL(lora_up_kernel<BF16>, dim3((a.n + 255) / 256 * a.rows), dim3(256), 0, st, a);
    DOE_LAUNCH_CHECK("lora_up_kernel");
    return DOE_OK;
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
    DOE_REQUIRE(y_row_stride >= a.n && y_row_stride < ((int64_t)1 << 32), DOE_E_INVALID, "y_row_stride %lld below the %d columns", (long long)y_row_stride, a.n);
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
    return lora->bf16 ? launch<true>(a, (hipStream_t)stream) : launch<false>(a, (hipStream_t)stream);
}

}  // extern "C"
