// kv_pages.hip -- the pages of a paged KV cache: extending, forking, freeing and
// compacting sequences, and copying pages, all on the device (a captured step
// replays them with the lengths of the moment).
//
// The state is page_table [max_seqs][table_stride], kv_lens [max_seqs] and
// page_refs [num_pages], the number of sequences that hold a page (0: free).
// What is copied is bound by its bytes: 96 last pages of 26 layers (290 MB read and
// written, part of it from the last-level cache) 39 us, half of a pool (746 MB) 147 us,
// the rate of a large copy.  A plan is one workgroup's chain of dependent reads and of
// its own code's lines, fetched as it runs: 5.1 us for 256 sequences of a pool of 40000
// pages (7.3 with sums through memory, unrolled scans and the compiler's divisions).
// Splitting it over workgroups would take launches of 3 - 4 us each between its steps.
// A plan kernel of one workgroup checks the call as a whole, takes the lowest
// free pages in the order of the call's entries and writes *status; the copies
// and the long tables are a second, wide kernel that reads the plan.  A call
// that cannot be done whole (status not 0) changes nothing.
#include "common.h"
#include "wave.h"

#include <algorithm>

namespace {

constexpr int kPlan = 1024;  // threads of a plan workgroup

struct PageArgs {
    uint8_t *pools;
    int64_t layers, layer_stride, page_bytes;
    int32_t *table, *lens, *refs, *status;
    const int32_t *first, *second;  // the call's two lists (sequences, amounts; parents, children; sources, destinations)
    int n, max_seqs, table_stride, num_pages, page_size;
    double page_inv;  // 1 / page_size
    // workspace: plan[0] pages to copy; by_seq [max_seqs] and by_page [num_pages]
    // hold the entry that names a sequence or page; need [n] running sums of pages;
    // taken [num_pages] free pages in order; pair [2 n or num_pages] copies
    int32_t *plan, *by_seq, *by_page, *need, *taken, *pair;
};

// Inclusive sum over the workgroup; `total` the last thread's.
__device__ __forceinline__ int scan(int v, int *wave_sums, int &total) {
    static_assert(kPlan == 1024, "sixteen waves");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    v = doe::wave_scan(v);
    __syncthreads();  // the last call's sums have been read
    if (lane == 63) wave_sums[wave] = v;
    __syncthreads();
    const int upto = doe::scan16(wave_sums[lane & 15]);
    total = __builtin_amdgcn_readlane(upto, 15);
    return v + (wave ? __builtin_amdgcn_readlane(upto, wave - 1) : 0);
}

// Which of a thread's four pages p .. are free, a bit each.
__device__ __forceinline__ uint32_t free_bits(const PageArgs &a, int p) {
    // (read whether they are there or not, so that one does not wait for another)
    int refs[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) refs[j] = a.refs[std::min(p + j, a.num_pages - 1)];
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) bits |= p + j < a.num_pages && refs[j] == 0 ? 1u << j : 0u;
    return bits;
}

// The lowest free pages into a.taken (and the first kPlan into `near`, in LDS), at
// least `want` of them where there are as many; returns how many were found (the
// same for every thread).  `bits`: those of the first pages, read before.
__device__ int take_free(const PageArgs &a, int want, uint32_t bits, int *wave_sums, int *near) {
    int found = 0;
    for (int p0 = 0; p0 < a.num_pages && found < want; p0 += 4 * kPlan) {
        const int p = p0 + 4 * (int)threadIdx.x;
        if (p0) bits = free_bits(a, p);
        const int mine = __popc(bits);
        int total;
        int at = found + scan(mine, wave_sums, total) - mine;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (bits >> j & 1) {
                if (at < kPlan) near[at] = p + j;
                else if (at < want) a.taken[at] = p + j;
                ++at;
            }
        found += total;
    }
    __syncthreads();
    return found;
}
__device__ __forceinline__ int taken(const PageArgs &a, const int *near, int t) { return t < kPlan ? near[t] : a.taken[t]; }

// Every entry's count of pages (count(i)) summed into a.need (the first kPlan into
// `near`, in LDS, instead); the total.
template <typename F>
__device__ int sum_needs(const PageArgs &a, int *wave_sums, int *near, const F &count) {
    int sum = 0;
    for (int i0 = 0; i0 < a.n; i0 += kPlan) {
        const int i = i0 + (int)threadIdx.x;
        int total;
        const int upto = scan(i < a.n ? count(i) : 0, wave_sums, total);
        if (i < kPlan) near[i] = sum + upto;
        else if (i < a.n) a.need[i] = sum + upto;
        sum += total;
    }
    __syncthreads();
    return sum;
}

// The full ones of len positions' pages (the reciprocal's error is far below the half
// by which len + 1/2 clears the quotients' borders), and all of them.
__device__ __forceinline__ int full_pages(const PageArgs &a, int len) { return (int)(((double)len + 0.5) * a.page_inv); }
__device__ __forceinline__ int pages_of(const PageArgs &a, int len) { return full_pages(a, len + a.page_size - 1); }

// Each of `list` marks its place; afterwards mark[list[i]] == i for every i where no value comes twice.
__device__ void mark_all(const int32_t *list, int n, int limit, int32_t *mark) {
    for (int i = threadIdx.x; i < n; i += kPlan)
        if (list[i] >= 0 && list[i] < limit) mark[list[i]] = i;
    __syncthreads();
}

// The chain of dependent reads is all this kernel's time: a thread's first entry
// and the first pages' counts are read once, all at the start; places, sums and pages of
// the first kPlan entries go through LDS, and so do the marks of sequences as far as
// they fit there.
__global__ __launch_bounds__(kPlan) void pages_extend_kernel(PageArgs a) {
    constexpr int kMarks = 1 << 16;
    __shared__ int wave_sums[kPlan / 64], sums[kPlan], pages[kPlan];
    __shared__ int2 place[kPlan];
    __shared__ uint32_t marks[kMarks / 32];
    const int tid = threadIdx.x;
    struct Entry {
        int s, add, len;
    };
    auto read = [&](int i) {
        Entry e{-1, 0, 0};
        if (i < a.n) {
            e.s = a.first[i];
            e.add = a.second[i];
            if (e.s >= 0 && e.s < a.max_seqs) e.len = a.lens[e.s];
        }
        return e;
    };
    const uint32_t bits = free_bits(a, 4 * tid);
    const Entry mine = read(tid);
    auto entry = [&](int i) { return i == tid ? mine : read(i); };
    const bool few = a.max_seqs <= kMarks;
    if (few) {
        for (int w = tid; w < (a.max_seqs + 31) / 32; w += kPlan) marks[w] = 0;
        __syncthreads();
    } else {
        mark_all(a.first, a.n, a.max_seqs, a.by_seq);
    }
    auto twice = [&](int s, int i) { return few ? (atomicOr(&marks[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) != 0 : a.by_seq[s] != i; };
    bool bad = false;
    for (int i = tid; i < a.n; i += kPlan) {
        const Entry e = entry(i);
        if (e.s < 0 || e.s >= a.max_seqs || twice(e.s, i) || e.add < 0) {
            bad = true;
            continue;
        }
        bad = bad || e.len < 0 || (int64_t)e.len + e.add > (int64_t)a.table_stride * a.page_size;
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) *a.status = -1;
        return;
    }
    const int want = sum_needs(a, wave_sums, sums, [&](int i) {
        const Entry e = entry(i);
        const int held = pages_of(a, e.len);
        if (i < kPlan) place[i] = make_int2(e.s, held);
        return pages_of(a, e.len + e.add) - held;
    });
    const int found = take_free(a, want, bits, wave_sums, pages);
    if (found < want) {
        if (tid == 0) *a.status = want - found;
        return;
    }
    auto sum = [&](int i) { return i < kPlan ? sums[i] : a.need[i]; };
    for (int t = tid; t < want; t += kPlan) {
        int lo = 0, hi = a.n - 1;  // the first entry whose running sum is above t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sum(mid) > t) hi = mid;
            else lo = mid + 1;
        }
        const int2 at = lo < kPlan ? place[lo] : make_int2(a.first[lo], pages_of(a, a.lens[a.first[lo]]));
        const int page = taken(a, pages, t);
        a.table[(int64_t)at.x * a.table_stride + at.y + t - (lo ? sum(lo - 1) : 0)] = page;
        a.refs[page] = 1;
    }
    if (a.n > kPlan) __syncthreads();
    for (int i = tid; i < a.n; i += kPlan) {
        const Entry e = entry(i);
        a.lens[e.s] = e.len + e.add;
    }
    if (tid == 0) *a.status = 0;
}

__global__ __launch_bounds__(kPlan) void pages_fork_plan_kernel(PageArgs a) {
    __shared__ int wave_sums[kPlan / 64], sums[kPlan], pages[kPlan];
    const uint32_t bits = free_bits(a, 4 * (int)threadIdx.x);
    mark_all(a.second, a.n, a.max_seqs, a.by_seq);
    bool bad = false;
    for (int i = threadIdx.x; i < a.n; i += kPlan) {
        const int p = a.first[i], c = a.second[i];
        if (p < 0 || p >= a.max_seqs || c < 0 || c >= a.max_seqs || a.by_seq[c] != i || a.lens[c] != 0) {
            bad = true;
            continue;
        }
        // a parent that the call forks into (the mark may be an older call's)
        const int j = a.by_seq[p];
        bad = bad || (j >= 0 && j < a.n && a.second[j] == p);
        bad = bad || a.lens[p] < 0 || a.lens[p] > (int64_t)a.table_stride * a.page_size;
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) {
            *a.status = -1;
            a.plan[0] = 0;
        }
        return;
    }
    const int want = sum_needs(a, wave_sums, sums, [&](int i) {
        const int len = a.lens[a.first[i]];
        return pages_of(a, len) - full_pages(a, len);
    });
    const int found = take_free(a, want, bits, wave_sums, pages);
    if (found < want) {
        if (threadIdx.x == 0) {
            *a.status = want - found;
            a.plan[0] = 0;
        }
        return;
    }
    for (int i = threadIdx.x; i < a.n; i += kPlan) {
        const int len = a.lens[a.first[i]];
        const int full = full_pages(a, len);
        if (len == full * a.page_size) continue;
        const int t = (i < kPlan ? sums[i] : a.need[i]) - 1, page = taken(a, pages, t);
        if (i < kPlan) a.need[i] = t + 1;  // (the copying kernel reads it)
        a.pair[2 * t] = a.table[(int64_t)a.first[i] * a.table_stride + full];
        a.pair[2 * t + 1] = page;
        a.refs[page] = 1;
    }
    if (threadIdx.x == 0) {
        *a.status = 0;
        a.plan[0] = want;
    }
}

__device__ __forceinline__ int64_t quotient(int64_t v, int64_t by) {
    return (v | by) >> 32 ? v / by : (int64_t)((uint32_t)v / (uint32_t)by);
}
// The pages pair[2 i] -> pair[2 i + 1], i < count, of every layer in pieces of 16 KB, layer by
// layer: the copies of one page follow each other and read it from the caches (twelve
// prompts forked eight times: 43.4 us, 50.1 with a page's layers side by side).
__device__ void copy_pages(const PageArgs &a, int count, int64_t first, int64_t step) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int PIECE = 256 * 16 * 4;
    const int64_t pieces = (a.page_bytes + PIECE - 1) / PIECE, all = (int64_t)count * a.layers * pieces;
    for (int64_t w = first; w < all; w += step) {
        const int64_t rest = quotient(w, pieces), piece = w - rest * pieces, layer = quotient(rest, count), i = rest - layer * count;
        const int src = a.pair[2 * i], dst = a.pair[2 * i + 1];
        if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages) continue;
        const int64_t at = piece * PIECE + threadIdx.x * 16;
        const uint8_t *s = a.pools + layer * a.layer_stride + (int64_t)src * a.page_bytes + at;
        uint8_t *d = a.pools + layer * a.layer_stride + (int64_t)dst * a.page_bytes + at;
        u32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j * 4096 < a.page_bytes) v[j] = *reinterpret_cast<const u32x4 *>(s + j * 4096);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j * 4096 < a.page_bytes) *reinterpret_cast<u32x4 *>(d + j * 4096) = v[j];
    }
}

// Children's rows (the parent's whole pages shared, the last one their own) and the copies.
__global__ __launch_bounds__(256) void pages_fork_kernel(PageArgs a) {
    if (*a.status != 0) return;
    const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    const int64_t entries = (int64_t)a.n * a.table_stride;
    for (int64_t t = tid; t < entries; t += step) {
        const int i = (int)(t / a.table_stride), col = (int)(t - (int64_t)i * a.table_stride);
        const int p = a.first[i], c = a.second[i], len = a.lens[p], full = full_pages(a, len);
        int page = -1;
        if (col < full) {
            page = a.table[(int64_t)p * a.table_stride + col];
            if (page >= 0 && page < a.num_pages) atomicAdd(&a.refs[page], 1);
        } else if (col == full && len != full * a.page_size) {
            page = a.pair[2 * (a.need[i] - 1) + 1];
        }
        a.table[(int64_t)c * a.table_stride + col] = page;
        if (col == 0) a.lens[c] = len;
    }
    copy_pages(a, a.plan[0], blockIdx.x, gridDim.x);
}

// One workgroup a listed sequence.  The exchange of its length makes one of
// several that name the same sequence the one that gives its pages back; the
// first also reports whether every entry names a sequence.
__global__ __launch_bounds__(256) void pages_free_kernel(PageArgs a) {
    __shared__ int len_;
    const int s = a.first[blockIdx.x];
    const bool ok = s >= 0 && s < a.max_seqs;
    if (threadIdx.x == 0) len_ = ok ? atomicExch(&a.lens[s], 0) : 0;
    if (blockIdx.x == 0) {
        bool bad = false;
        for (int i = threadIdx.x; i < a.n; i += 256) bad = bad || a.first[i] < 0 || a.first[i] >= a.max_seqs;
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0) *a.status = bad ? -1 : 0;
    }
    __syncthreads();
    if (len_ <= 0) return;
    const int held = pages_of(a, (int)min((int64_t)len_, (int64_t)a.table_stride * a.page_size));
    for (int col = threadIdx.x; col < a.table_stride; col += 256) {
        int32_t *e = &a.table[(int64_t)s * a.table_stride + col];
        if (col < held && *e >= 0 && *e < a.num_pages) atomicSub(&a.refs[*e], 1);
        *e = -1;
    }
}

__global__ __launch_bounds__(kPlan) void pages_compact_plan_kernel(PageArgs a) {
    __shared__ int wave_sums[kPlan / 64], pages[kPlan];
    int mine = 0, total;
    for (int p = threadIdx.x; p < a.num_pages; p += kPlan) mine += a.refs[p] != 0;
    scan(mine, wave_sums, total);
    const int live = total;
    take_free(a, live, free_bits(a, 4 * (int)threadIdx.x), wave_sums, pages);  // in order: those below `live` take the pages above it, as many
    int moved = 0;
    for (int p0 = 0; p0 < a.num_pages; p0 += kPlan) {
        const int p = p0 + (int)threadIdx.x;
        const bool high = p < a.num_pages && p >= live && a.refs[p] != 0;
        const int at = moved + scan(high, wave_sums, total) - 1;
        const int to = high ? taken(a, pages, at) : p;
        if (p < a.num_pages) a.by_page[p] = to;
        if (high) {
            a.pair[2 * at] = p;
            a.pair[2 * at + 1] = to;
        }
        moved += total;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moved; i += kPlan) {
        a.refs[a.pair[2 * i + 1]] = a.refs[a.pair[2 * i]];
        a.refs[a.pair[2 * i]] = 0;
    }
    if (threadIdx.x == 0) {
        a.plan[0] = moved;
        *a.status = 0;
    }
}

__global__ __launch_bounds__(256) void pages_compact_kernel(PageArgs a) {
    const int count = a.plan[0];
    if (count == 0) return;
    const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    const int64_t entries = (int64_t)a.max_seqs * a.table_stride;
    for (int64_t t = tid; t < entries; t += step) {
        const int s = (int)(t / a.table_stride), col = (int)(t - (int64_t)s * a.table_stride);
        if ((int64_t)col * a.page_size >= a.lens[s]) continue;
        const int page = a.table[t];
        if (page >= 0 && page < a.num_pages && a.by_page[page] != page) a.table[t] = a.by_page[page];
    }
    copy_pages(a, count, blockIdx.x, gridDim.x);
}

__global__ __launch_bounds__(kPlan) void pages_copy_plan_kernel(PageArgs a) {
    mark_all(a.second, a.n, a.num_pages, a.by_page);
    bool bad = false;
    for (int i = threadIdx.x; i < a.n; i += kPlan) {
        const int s = a.first[i], d = a.second[i];
        if (s < 0 || s >= a.num_pages || d < 0 || d >= a.num_pages || a.by_page[d] != i) {
            bad = true;
            continue;
        }
        // a source that some entry writes (the mark may be an older call's)
        const int j = a.by_page[s];
        bad = bad || (j >= 0 && j < a.n && a.second[j] == s);
        a.pair[2 * i] = s;
        a.pair[2 * i + 1] = d;
    }
    const int any = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        *a.status = any ? -1 : 0;
        a.plan[0] = any ? 0 : a.n;
    }
}

__global__ __launch_bounds__(256) void pages_copy_kernel(PageArgs a) { copy_pages(a, a.plan[0], blockIdx.x, gridDim.x); }

// ---------------------------------------------------------------------------
// Reordering: slot i becomes what the slot of parents[i] was, all at once.  The plan
// takes a fresh page for every heir of a partly filled last page but one (the parent's
// own slot, else the first heir); the wide kernel reads its columns of all rows before
// it writes any of them.  Twelve requests of eight beams, 26 last pages of 52 layers (177
// MB): 33 us, 5.3 TB/s, behind 4.8 of the plan; three of four 4.2 and 3.7.
constexpr int kReorder = 8192;  // sequences of a call: their marks and a column of their rows fit in LDS

struct ReorderArgs {
    PageArgs p;        // first: parents; second: the slots (null: 0 .. n - 1); by_seq, taken, pair, need as above
    int32_t *old_len;  // [n] of the slots before
    int32_t *heirs;    // [n]
    int32_t *fresh;    // [n] an heir's own last page, -1: none
    int columns;       // of a workgroup
};
__device__ __forceinline__ int slot_of(const ReorderArgs &a, int i) { return a.p.second ? a.p.second[i] : i; }

constexpr int kWhole = -0x7fffffff;  // in place of a last page: there is none but whole ones
__global__ __launch_bounds__(kPlan) void pages_reorder_plan_kernel(ReorderArgs r) {
    const PageArgs &a = r.p;
    extern __shared__ int marks[];  // of each slot: heirs, keeper, its last page before
    __shared__ int wave_sums[kPlan / 64], sums[kPlan], pages[kPlan];
    int *heirs = marks, *keeper = marks + a.n, *last = marks + 2 * a.n;
    const int tid = threadIdx.x;
    const uint32_t bits = free_bits(a, 4 * tid);
    for (int i = tid; i < a.n; i += kPlan) {
        heirs[i] = 0;
        keeper[i] = a.n;
    }
    if (a.second) mark_all(a.second, a.n, a.max_seqs, a.by_seq);
    __syncthreads();
    bool bad = false;
    for (int i = tid; i < a.n; i += kPlan) {
        const int s = slot_of(r, i), p = a.first[i], seq = std::max(0, std::min(s, a.max_seqs - 1)), len = a.lens[seq];
        const int full = full_pages(a, std::max(0, len));
        const int page = a.table[(int64_t)seq * a.table_stride + std::min(full, a.table_stride - 1)];
        if (s != seq || (a.second && a.by_seq[s] != i) || p >= a.n) {
            bad = true;
            continue;
        }
        bad = bad || len < 0 || len > (int64_t)a.table_stride * a.page_size;
        r.old_len[i] = len;
        last[i] = len > full * a.page_size ? page : kWhole;
        if (p >= 0) {
            atomicAdd(&heirs[p], 1);
            atomicMin(&keeper[p], p == i ? -1 : i);
        }
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) {
            *a.status = -1;
            a.plan[0] = 0;
        }
        return;
    }
    auto own_page = [&](int i) {
        const int p = a.first[i];
        return p >= 0 && keeper[p] != (p == i ? -1 : i) && last[p] != kWhole ? 1 : 0;
    };
    const int want = sum_needs(a, wave_sums, sums, own_page);
    const int found = take_free(a, want, bits, wave_sums, pages);
    if (found < want) {
        if (tid == 0) {
            *a.status = want - found;
            a.plan[0] = 0;
        }
        return;
    }
    for (int i = tid; i < a.n; i += kPlan) {
        r.heirs[i] = heirs[i];
        int page = -1;
        if (own_page(i)) {
            const int t = (i < kPlan ? sums[i] : a.need[i]) - 1, p = a.first[i];
            page = taken(a, pages, t);
            a.pair[2 * t] = last[p];
            a.pair[2 * t + 1] = page;
            a.refs[page] = 1;
        }
        r.fresh[i] = page;
    }
    if (tid == 0) {
        *a.status = 0;
        a.plan[0] = want;
    }
}

__global__ __launch_bounds__(256) void pages_reorder_kernel(ReorderArgs r) {
    const PageArgs &a = r.p;
    extern __shared__ int old[];  // [n][columns]
    if (*a.status != 0) return;
    const int C = r.columns, col0 = blockIdx.x * C, cells = a.n * C;
    if (col0 < a.table_stride) {
        for (int t = threadIdx.x; t < cells; t += 256) {
            const int i = t / C, col = col0 + t - i * C;
            old[t] = col < a.table_stride ? a.table[(int64_t)slot_of(r, i) * a.table_stride + col] : -1;
        }
        __syncthreads();
        for (int t = threadIdx.x; t < cells; t += 256) {
            const int i = t / C, c = t - i * C, col = col0 + c;
            if (col >= a.table_stride) continue;
            const int s = slot_of(r, i), p = a.first[i];
            int page = -1;
            if (p >= 0) {
                const int len = r.old_len[p], full = full_pages(a, len);
                if (col < full || (col == full && len > full * a.page_size)) page = old[p * C + c];
                if (col == full && r.fresh[i] >= 0) page = r.fresh[i];
                if (col == 0) a.lens[s] = len;
            } else if (col == 0) {
                a.lens[s] = 0;
            }
            a.table[(int64_t)s * a.table_stride + col] = page;
            // what slot i held is held by its heirs from here on
            const int len = r.old_len[i], full = full_pages(a, len), was = old[t], heirs = r.heirs[i];
            const int more = col < full ? heirs - 1 : (col == full && len > full * a.page_size && heirs == 0 ? -1 : 0);
            if (more != 0 && was >= 0 && was < a.num_pages) atomicAdd(&a.refs[was], more);
        }
    }
    copy_pages(a, a.plan[0], blockIdx.x, gridDim.x);
}

int reorder_workspace_ints(int64_t num_pages, int64_t max_seqs, int64_t n, int64_t *ints) {
    DOE_REQUIRE(num_pages > 0 && num_pages < ((int64_t)1 << 30), DOE_E_INVALID, "num_pages %lld", (long long)num_pages);
    DOE_REQUIRE(max_seqs > 0 && max_seqs <= ((int64_t)1 << 24), DOE_E_INVALID, "max_seqs %lld", (long long)max_seqs);
    DOE_REQUIRE(n >= 0 && n <= kReorder, DOE_E_UNSUPPORTED, "n %lld outside 0..%d", (long long)n, kReorder);
    *ints = 16 + num_pages + max_seqs + 6 * n;
    return DOE_OK;
}

int workspace_ints(int64_t num_pages, int64_t max_seqs, int64_t n, int64_t *ints) {
    DOE_REQUIRE(num_pages > 0 && num_pages < ((int64_t)1 << 30), DOE_E_INVALID, "num_pages %lld", (long long)num_pages);
    DOE_REQUIRE(max_seqs >= 0 && max_seqs <= ((int64_t)1 << 24), DOE_E_INVALID, "max_seqs %lld", (long long)max_seqs);
    DOE_REQUIRE(n >= 0 && n < ((int64_t)1 << 24), DOE_E_INVALID, "n %lld", (long long)n);
    *ints = 16 + 3 * num_pages + max_seqs + 3 * n;
    return DOE_OK;
}

int page_workspace(PageArgs &a, void *workspace, int64_t workspace_bytes) {
    int64_t ints = 0;
    const int rc = workspace_ints(a.num_pages, a.max_seqs, a.n, &ints);
    if (rc) return rc;
    DOE_REQUIRE(workspace && workspace_bytes >= 4 * ints, DOE_E_INVALID, "a workspace of %lld bytes is needed (got %lld)",
                (long long)(4 * ints), (long long)workspace_bytes);
    DOE_REQUIRE(((uintptr_t)workspace & 15) == 0, DOE_E_INVALID, "the workspace must be 16-byte aligned");
    a.plan = static_cast<int32_t *>(workspace);
    a.by_seq = a.plan + 16;
    a.need = a.by_seq + a.max_seqs;
    a.by_page = a.need + a.n;
    a.taken = a.by_page + a.num_pages;
    a.pair = a.taken + a.num_pages;  // 2 max(n, num_pages / 2)
    return DOE_OK;
}

int pool_checks(const PageArgs &a) {
    DOE_REQUIRE(a.layers >= 0 && a.layers <= 65535, DOE_E_INVALID, "layers %lld", (long long)a.layers);
    if (a.layers == 0) return DOE_OK;
    DOE_REQUIRE(a.pools, DOE_E_INVALID, "null pools");
    DOE_REQUIRE(a.page_bytes > 0 && a.page_bytes % 16 == 0 && a.layer_stride % 16 == 0 && ((uintptr_t)a.pools & 15) == 0,
                DOE_E_INVALID, "pools, page_bytes and layer_stride must be multiples of 16");
    DOE_REQUIRE(a.page_bytes < ((int64_t)1 << 32), DOE_E_INVALID, "page_bytes %lld", (long long)a.page_bytes);
    DOE_REQUIRE(a.layer_stride >= a.num_pages * a.page_bytes, DOE_E_INVALID, "layer_stride %lld below %d pages of %lld bytes",
                (long long)a.layer_stride, a.num_pages, (long long)a.page_bytes);
    return DOE_OK;
}

int page_args(PageArgs &a, const doe_kv_pages *p, const int32_t *first, const int32_t *second, int64_t n, bool lists,
              int32_t *status) {
    DOE_REQUIRE(p && p->page_table && p->kv_lens && p->page_refs && status, DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(n >= 0 && n < ((int64_t)1 << 24), DOE_E_INVALID, "n %lld", (long long)n);
    DOE_REQUIRE(n == 0 || !lists || first, DOE_E_INVALID, "null list");
    DOE_REQUIRE(p->max_seqs > 0 && p->max_seqs <= ((int64_t)1 << 24), DOE_E_INVALID, "max_seqs %lld", (long long)p->max_seqs);
    DOE_REQUIRE(p->num_pages > 0 && p->num_pages < ((int64_t)1 << 30), DOE_E_INVALID, "num_pages %lld", (long long)p->num_pages);
    DOE_REQUIRE(p->page_size > 0 && p->table_stride > 0 && p->page_size < ((int64_t)1 << 30) &&
                    p->table_stride < ((int64_t)1 << 30) && p->page_size * p->table_stride < ((int64_t)1 << 30),
                DOE_E_INVALID, "page_size %lld x table_stride %lld: a sequence holds fewer than 2^30 positions",
                (long long)p->page_size, (long long)p->table_stride);
    a = PageArgs{};
    a.pools = static_cast<uint8_t *>(p->pools);
    a.layers = p->layers;
    a.layer_stride = p->layer_stride;
    a.page_bytes = p->page_bytes;
    a.table = p->page_table;
    a.lens = p->kv_lens;
    a.refs = p->page_refs;
    a.status = status;
    a.first = first;
    a.second = second;
    a.n = (int)n;
    a.max_seqs = (int)p->max_seqs;
    a.table_stride = (int)p->table_stride;
    a.num_pages = (int)p->num_pages;
    a.page_size = (int)p->page_size;
    a.page_inv = 1.0 / a.page_size;
    return DOE_OK;
}

// Workgroups of a wide kernel: one for each 16 KB piece and 256 entries, at most eight a CU.
unsigned wide_grid(const PageArgs &a, int64_t copies, int64_t entries) {
    const int64_t pieces = a.layers > 0 ? std::min<int64_t>(copies * a.layers, 2048) * ((a.page_bytes + 16383) / 16384) : 0;
    const int64_t want = std::max(pieces, (entries + 255) / 256);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(want, 2048));
}

}  // namespace

extern "C" {

int doe_kv_pages_workspace(int64_t num_pages, int64_t max_seqs, int64_t n, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    int64_t ints = 0;
    const int rc = workspace_ints(num_pages, max_seqs, n, &ints);
    if (rc) return rc;
    *bytes = 4 * ints;
    return DOE_OK;
}

int doe_kv_pages_extend(const doe_kv_pages *pages, const int32_t *seqs, const int32_t *add, int64_t n, int32_t *status,
                        void *workspace, int64_t workspace_bytes, doe_stream_t stream) {
    PageArgs a;
    int rc = page_args(a, pages, seqs, add, n, true, status);
    if (rc) return rc;
    DOE_REQUIRE(n == 0 || add, DOE_E_INVALID, "null list");
    DOE_REQUIRE(n * pages->table_stride < ((int64_t)1 << 31), DOE_E_UNSUPPORTED, "%lld entries of up to %lld pages",
                (long long)n, (long long)pages->table_stride);
    if ((rc = page_workspace(a, workspace, workspace_bytes))) return rc;
    if ((rc = doe::require_init())) return rc;
    hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_extend_kernel");
    return DOE_OK;
}

int doe_kv_pages_fork(const doe_kv_pages *pages, const int32_t *parents, const int32_t *children, int64_t n, int32_t *status,
                      void *workspace, int64_t workspace_bytes, doe_stream_t stream) {
    PageArgs a;
    int rc = page_args(a, pages, parents, children, n, true, status);
    if (rc) return rc;
    DOE_REQUIRE(n == 0 || children, DOE_E_INVALID, "null list");
    if ((rc = pool_checks(a))) return rc;
    if ((rc = page_workspace(a, workspace, workspace_bytes))) return rc;
    if ((rc = doe::require_init())) return rc;
    hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_fork_plan_kernel");
    if (n == 0) return DOE_OK;
    hipLaunchKernelGGL(pages_fork_kernel, dim3(wide_grid(a, n, n * (int64_t)a.table_stride)), dim3(256), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_fork_kernel");
    return DOE_OK;
}

int doe_kv_pages_free(const doe_kv_pages *pages, const int32_t *seqs, int64_t n, int32_t *status, doe_stream_t stream) {
    PageArgs a;
    int rc = page_args(a, pages, seqs, nullptr, n, true, status);
    if (rc) return rc;
    if ((rc = doe::require_init())) return rc;
    if (n == 0) return doe::fill_bytes_async(status, 0, 4, (hipStream_t)stream);
    hipLaunchKernelGGL(pages_free_kernel, dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_free_kernel");
    return DOE_OK;
}

int doe_kv_pages_compact(const doe_kv_pages *pages, int32_t *status, void *workspace, int64_t workspace_bytes,
                         doe_stream_t stream) {
    PageArgs a;
    int rc = page_args(a, pages, nullptr, nullptr, 0, false, status);
    if (rc) return rc;
    if ((rc = pool_checks(a))) return rc;
    if ((rc = page_workspace(a, workspace, workspace_bytes))) return rc;
    if ((rc = doe::require_init())) return rc;
    hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_compact_plan_kernel");
    hipLaunchKernelGGL(pages_compact_kernel, dim3(wide_grid(a, a.num_pages / 2, (int64_t)a.max_seqs * a.table_stride)), dim3(256), 0,
                       (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_compact_kernel");
    return DOE_OK;
}

int doe_kv_pages_copy(void *pools, int64_t layers, int64_t layer_stride, int64_t page_bytes, int64_t num_pages,
                      const int32_t *sources, const int32_t *destinations, int64_t n, int32_t *status, void *workspace,
                      int64_t workspace_bytes, doe_stream_t stream) {
    DOE_REQUIRE(status, DOE_E_INVALID, "null pointer");
    DOE_REQUIRE(n >= 0 && n < ((int64_t)1 << 24), DOE_E_INVALID, "n %lld", (long long)n);
    DOE_REQUIRE(n == 0 || (sources && destinations), DOE_E_INVALID, "null list");
    DOE_REQUIRE(num_pages > 0 && num_pages < ((int64_t)1 << 30), DOE_E_INVALID, "num_pages %lld", (long long)num_pages);
    PageArgs a{};
    a.pools = static_cast<uint8_t *>(pools);
    a.layers = layers;
    a.layer_stride = layer_stride;
    a.page_bytes = page_bytes;
    a.status = status;
    a.first = sources;
    a.second = destinations;
    a.n = (int)n;
    a.num_pages = (int)num_pages;
    int rc = pool_checks(a);
    if (rc) return rc;
    if ((rc = page_workspace(a, workspace, workspace_bytes))) return rc;
    if ((rc = doe::require_init())) return rc;
    hipLaunchKernelGGL(pages_copy_plan_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_copy_plan_kernel");
    if (n == 0 || layers == 0) return DOE_OK;
    hipLaunchKernelGGL(pages_copy_kernel, dim3(wide_grid(a, n, 0)), dim3(256), 0, (hipStream_t)stream, a);
    DOE_LAUNCH_CHECK("pages_copy_kernel");
    return DOE_OK;
}

int doe_beam_reorder_pages_workspace(int64_t num_pages, int64_t max_seqs, int64_t n, int64_t *bytes) {
    DOE_REQUIRE(bytes, DOE_E_INVALID, "null argument");
    int64_t ints = 0;
    const int rc = reorder_workspace_ints(num_pages, max_seqs, n, &ints);
    if (rc) return rc;
    *bytes = 4 * ints;
    return DOE_OK;
}

int doe_beam_reorder_pages(const doe_kv_pages *pages, const int32_t *seqs, const int32_t *parents, int64_t n, int32_t *status,
                           void *workspace, int64_t workspace_bytes, doe_stream_t stream) {
    ReorderArgs r{};
    PageArgs &a = r.p;
    int rc = page_args(a, pages, parents, seqs, n, true, status);
    if (rc) return rc;
    DOE_REQUIRE(seqs || n <= a.max_seqs, DOE_E_INVALID, "%lld sequences of %d slots", (long long)n, a.max_seqs);
    if ((rc = pool_checks(a))) return rc;
    int64_t ints = 0;
    if ((rc = reorder_workspace_ints(a.num_pages, a.max_seqs, n, &ints))) return rc;
    DOE_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= 4 * ints, DOE_E_INVALID,
                "a 16-byte aligned workspace of %lld bytes is needed (got %lld)", (long long)(4 * ints), (long long)workspace_bytes);
    if ((rc = doe::require_init())) return rc;
    if (n == 0) return doe::fill_bytes_async(status, 0, 4, (hipStream_t)stream);
    a.plan = static_cast<int32_t *>(workspace);
    a.by_seq = a.plan + 16;
    a.taken = a.by_seq + a.max_seqs;
    a.need = a.taken + a.num_pages;
    a.pair = a.need + n;
    r.old_len = a.pair + 2 * n;
    r.heirs = r.old_len + n;
    r.fresh = r.heirs + n;
    // a workgroup's cells fit in 32 KB, and the columns spread over the device
    r.columns = (int)std::max<int64_t>(1, std::min<int64_t>({64, kReorder / n, (a.table_stride + 255) / 256 * 16}));
    const int64_t chunks = (a.table_stride + r.columns - 1) / r.columns;
    DOE_REQUIRE(chunks < (1 << 24), DOE_E_UNSUPPORTED, "%lld sequences of up to %d pages", (long long)n, a.table_stride);
    const int lds = (int)(12 * n);
    static const hipError_t attr_rc = hipFuncSetAttribute((const void *)pages_reorder_plan_kernel,
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, 12 * kReorder);
    DOE_HIP_CHECK(attr_rc);
    hipLaunchKernelGGL(pages_reorder_plan_kernel, dim3(1), dim3(kPlan), lds, (hipStream_t)stream, r);
    DOE_LAUNCH_CHECK("pages_reorder_plan_kernel");
    const unsigned wgs = (unsigned)std::max<int64_t>(chunks, wide_grid(a, n, 0));
    hipLaunchKernelGGL(pages_reorder_kernel, dim3(wgs), dim3(256), (size_t)n * r.columns * 4, (hipStream_t)stream, r);
    DOE_LAUNCH_CHECK("pages_reorder_kernel");
    return DOE_OK;
}

}  // extern "C"
