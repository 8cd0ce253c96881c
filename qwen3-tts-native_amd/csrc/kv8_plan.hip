// Block tables, row starts, row positions and slots of one step of many
// sequences, made on the device from the sequences' lengths, so that a step
// (plan, append, attention) needs no host round trip and can be a HIP graph.
//
// Sequence s holds L tokens in ceil(L / P) pages of P tokens and brings n:
//   n < 0   it ends: its pages go on the stack of free pages, in order;
//   n >= 0  it is let in if its table has room for L + n tokens, then if the
//           rows of all that were let in so far and its own fit the row
//           buffers, then if the stack still holds the pages it needs after
//           what those before it took (a sequence without rows, or that needs
//           no page, always passes).  Its pages come from the stack's top, its row i gets
//           position L + i and slot table[(L + i) / P] * P + (L + i) % P.
// Each "so far" is a prefix sum over the sequences that passed the test before
// it, not over the finally admitted ones: three scans instead of a serial walk,
// and the same answer whatever the order of execution.
//
// The sequences that get pages are therefore the first ones that ask for any,
// so that page i of the step is the stack's entry i below its top, whoever
// gets it.
//
// Bound by latency: dependent trips to memory and four block scans on a few
// kilobytes.  One workgroup does the scans (a grid-wide scan would need a
// second launch to hand sums over); pages and rows are then dealt to threads
// one by one, each finding its sequence by bisection of the scan in LDS (a
// wave a sequence: 1000 sequences with 23205 rows 22.7 us, now 13.6; eight with a
// row each 3.7).
#include "kv8.hpp"

#include <algorithm>
#include <climits>

namespace q3 {
namespace {

constexpr int kMaxThreads = 1024;
// Rows up to which the scanning workgroup writes the row map too.
constexpr int kRowsInOneLaunch = 2048;
constexpr int kRowThreads = 256;
constexpr int kRowStartsInLds = 4096;
// Sums end here, far above any capacity: they are only compared with one.
constexpr unsigned kMost = 1u << 30;

__device__ __forceinline__ unsigned add(unsigned a, unsigned b) { return min(a + b, kMost); }

template <int kControl, int kRowMask>
__device__ __forceinline__ unsigned moved(unsigned v) {
    return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, kRowMask, 0xf, false));
}

// Inclusive prefix sum over the block in thread order; total = the block's sum.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* lds, unsigned& total) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    v = add(v, moved<0x111, 0xf>(v));  // row_shr:1
    v = add(v, moved<0x112, 0xf>(v));
    v = add(v, moved<0x114, 0xf>(v));
    v = add(v, moved<0x118, 0xf>(v));
    v = add(v, moved<0x142, 0xa>(v));  // row_bcast:15 into rows 1, 3
    v = add(v, moved<0x143, 0xc>(v));  // row_bcast:31 into rows 2, 3
    const unsigned last = static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
    if (waves == 1) {
        total = last;
        return v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) lds[wave] = v;
    __syncthreads();
    unsigned before = 0, sum = 0;
    for (int w = 0; w < waves; ++w) {
        before = w == wave ? sum : before;
        sum = add(sum, lds[w]);
    }
    total = sum;
    return add(v, before);
}

// The thread of the block whose share of the items, given by inclusive prefix
// sums, holds item i.
__device__ __forceinline__ int owner_of(const unsigned* upto, unsigned i) {
    int at = 0;
    for (int step = blockDim.x >> 1; step > 0; step >>= 1) at += upto[at + step - 1] <= i ? step : 0;
    return at;
}

// page_tokens is a power of two
__device__ __forceinline__ int pages_of(long long tokens, int page_tokens) {
    return static_cast<int>((tokens + page_tokens - 1) >> __builtin_ctz(page_tokens));
}

// Position and slot of one row of a sequence.
__device__ __forceinline__ void write_row(const Kv8PlanArgs& a, int sequence, int row, int position) {
    const int shift = __builtin_ctz(a.page_tokens);
    const int page = a.tables[static_cast<size_t>(sequence) * a.table_stride + (position >> shift)];
    a.row_positions[row] = position;
    a.row_slots[row] = page >= 0 && page < a.pages ? (page << shift) + (position & (a.page_tokens - 1)) : -1;
}

template <bool kRows>
__global__ __launch_bounds__(kMaxThreads) void kv8_plan_kernel(Kv8PlanArgs a) {
    __shared__ unsigned lds[kMaxThreads / 64], upto_lds[kMaxThreads];
    __shared__ int from_lds[kMaxThreads], taken_lds, refused_lds;
    const long long room = static_cast<long long>(a.table_stride) * a.page_tokens;
    // what a sequence holds; a length its table cannot hold counts as a full table
    auto length_of = [&](int s) { return static_cast<int>(min(static_cast<long long>(max(a.lengths[s], 0)), room)); };
    auto table_of = [&](int s) { return a.tables + static_cast<size_t>(s) * a.table_stride; };
    unsigned stack = min(max(*a.free_count, 0), a.pages);
    if (threadIdx.x == 0) taken_lds = refused_lds = 0;

    // ---- pages of sequences that end ----
    for (int first = 0; first < a.sequences; first += blockDim.x) {
        const int s = first + threadIdx.x;
        const int held = s < a.sequences && a.new_tokens[s] < 0 ? pages_of(length_of(s), a.page_tokens) : 0;
        if (__syncthreads_count(held) == 0) continue;
        unsigned count = 0;
        const unsigned upto = block_scan(held, lds, count);
        upto_lds[threadIdx.x] = upto;
        __syncthreads();
        count = min(count, a.pages - stack);  // the stack has a place for every page once
        for (unsigned i = threadIdx.x; i < count; i += blockDim.x) {
            const int owner = owner_of(upto_lds, i);
            a.free_pages[stack + i] = table_of(first + owner)[i - (owner > 0 ? upto_lds[owner - 1] : 0)];
        }
        stack += count;
    }
    __syncthreads();

    // ---- who is let in, their pages and rows ----
    unsigned asked_rows = 0, asked_pages = 0, out = 0;
    for (int first = 0; first < a.sequences; first += blockDim.x) {
        const int s = first + threadIdx.x;
        const bool mine = s < a.sequences;
        const int length = mine ? length_of(s) : 0, asked = mine ? a.new_tokens[s] : 0;
        const bool ends = asked < 0;
        const int held = pages_of(length, a.page_tokens);
        unsigned rows = max(asked, 0), sum = 0;
        bool fits = mine && !ends && static_cast<long long>(length) + rows <= room;
        const unsigned upto_rows = add(asked_rows, block_scan(fits ? min(rows, kMost) : 0, lds, sum));
        asked_rows = add(asked_rows, sum);
        fits &= rows == 0 || upto_rows <= static_cast<unsigned>(a.rows_capacity);
        const unsigned need = fits ? pages_of(static_cast<long long>(length) + rows, a.page_tokens) - held : 0;
        const unsigned upto_pages = block_scan(need, lds, sum);
        fits &= need == 0 || add(asked_pages, upto_pages) <= stack;
        upto_lds[threadIdx.x] = upto_pages;
        from_lds[threadIdx.x] = held;
        if (fits && need > 0) atomicMax(&taken_lds, static_cast<int>(asked_pages + upto_pages));
        if (mine && !ends && !fits) atomicAdd(&refused_lds, 1);
        __syncthreads();
        const unsigned taken = taken_lds;
        for (unsigned i = threadIdx.x; asked_pages + i < taken; i += blockDim.x) {
            const int owner = owner_of(upto_lds, i);
            const unsigned j = i - (owner > 0 ? upto_lds[owner - 1] : 0);
            table_of(first + owner)[from_lds[owner] + j] = a.free_pages[stack - 1 - (asked_pages + i)];
        }
        asked_pages = add(asked_pages, sum);
        if (!fits) rows = 0;
        const unsigned upto = block_scan(rows, lds, sum);
        if (mine) {
            a.new_lengths[s] = ends ? 0 : length + static_cast<int>(rows);
            a.row_starts[s] = static_cast<int>(out + upto - rows);
        }
        if constexpr (kRows) {
            __syncthreads();
            upto_lds[threadIdx.x] = upto;
            from_lds[threadIdx.x] = length;
            __syncthreads();
            for (unsigned i = threadIdx.x; i < sum; i += blockDim.x) {
                const int owner = owner_of(upto_lds, i);
                const unsigned j = i - (owner > 0 ? upto_lds[owner - 1] : 0);
                write_row(a, first + owner, static_cast<int>(out + i), from_lds[owner] + static_cast<int>(j));
            }
        }
        __syncthreads();
        out += sum;
    }
    if (threadIdx.x == 0) {
        a.row_starts[a.sequences] = static_cast<int>(out);
        *a.new_free_count = static_cast<int>(stack) - taken_lds;
        *a.refused = refused_lds;
    }
    if constexpr (kRows) {
        for (int r = static_cast<int>(out + threadIdx.x); r < a.rows_capacity; r += blockDim.x) {
            a.row_positions[r] = 0;
            a.row_slots[r] = -1;
        }
    }
}

// The row map of a step with many rows: a thread a row, its sequence by
// bisection of the row starts, in LDS where they fit.
__global__ __launch_bounds__(kRowThreads) void kv8_plan_rows_kernel(Kv8PlanArgs a) {
    __shared__ int starts_lds[kRowStartsInLds];
    const int* starts = a.row_starts;
    const int row = blockIdx.x * kRowThreads + threadIdx.x;
    const int end = starts[a.sequences];
    if (a.sequences < kRowStartsInLds && static_cast<int>(blockIdx.x) * kRowThreads < end) {
        for (int s = threadIdx.x; s <= a.sequences; s += kRowThreads) starts_lds[s] = a.row_starts[s];
        __syncthreads();
        starts = starts_lds;
    }
    if (row >= a.rows_capacity) return;
    if (row >= end) {
        a.row_positions[row] = 0;
        a.row_slots[row] = -1;
        return;
    }
    int low = 0, high = a.sequences;  // row_starts[low] <= row < row_starts[high]
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (starts[middle] <= row) low = middle;
        else high = middle;
    }
    write_row(a, low, row, a.new_lengths[low] - starts[low + 1] + row);
}

}  // namespace

hipError_t launch_kv8_plan(const Kv8PlanArgs& a, hipStream_t stream) {
    const auto given = [](const void* p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 4 == 0; };
    if (a.sequences < 1 || a.table_stride < 1 || a.pages < 1 || a.rows_capacity < 0 ||
        a.rows_capacity >= static_cast<int>(kMost) ||
        (a.page_tokens != 16 && a.page_tokens != 32 && a.page_tokens != 64) || a.pages > INT_MAX / a.page_tokens ||
        a.table_stride > INT_MAX / a.page_tokens || !given(a.new_tokens) || !given(a.lengths) ||
        !given(a.new_lengths) || !given(a.tables) || !given(a.free_pages) || !given(a.free_count) ||
        !given(a.new_free_count) || !given(a.row_starts) || !given(a.refused) ||
        (a.rows_capacity > 0 && (!given(a.row_positions) || !given(a.row_slots)))) {
        return hipErrorInvalidValue;
    }
    const bool together = a.rows_capacity <= kRowsInOneLaunch;
    const int most = std::max(a.sequences, together ? a.rows_capacity : 0);
    const int threads = most <= 64 ? 64 : most <= 256 ? 256 : kMaxThreads;
    if (together) {
        kv8_plan_kernel<true><<<1, threads, 0, stream>>>(a);
        return hipGetLastError();
    }
    kv8_plan_kernel<false><<<1, threads, 0, stream>>>(a);
    const hipError_t st = hipGetLastError();
    if (st != hipSuccess) return st;
    kv8_plan_rows_kernel<<<(a.rows_capacity + kRowThreads - 1) / kRowThreads, kRowThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace q3
