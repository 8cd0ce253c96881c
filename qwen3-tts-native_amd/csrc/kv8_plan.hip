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
// Bound by latency: a few dependent trips to memory and four block scans on a
// few kilobytes.  One workgroup does the scans (a grid-wide scan would need a
// second launch to hand sums over).
#include "kv8.hpp"

#include <climits>

namespace q3 {
namespace {

constexpr int kMaxThreads = 1024;
// Rows up to which the scanning workgroup writes the row map too.
constexpr int kRowsInOneLaunch = 2048;
constexpr int kRowThreads = 256;

// Inclusive prefix sum over the block in thread order; total = the block's sum.
__device__ __forceinline__ long long block_scan(long long v, long long* lds, long long& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long other = __shfl_up(v, d, 64);
        if (lane >= d) v += other;
    }
    if (waves == 1) {
        total = __shfl(v, 63, 64);
        return v;
    }
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    long long before = 0, sum = 0;
    for (int w = 0; w < waves; ++w) {
        before += w < wave ? lds[w] : 0;
        sum += lds[w];
    }
    __syncthreads();
    total = sum;
    return v + before;
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
    __shared__ long long lds[kMaxThreads / 64];
    const int lane = threadIdx.x & 63;
    const long long room = static_cast<long long>(a.table_stride) * a.page_tokens;
    int stack = min(max(*a.free_count, 0), a.pages);
    // what a sequence holds; a length its table cannot hold counts as a full table
    auto length_of = [&](int s) { return static_cast<int>(min(static_cast<long long>(max(a.lengths[s], 0)), room)); };

    // ---- pages of sequences that end ----
    for (int first = 0; first < a.sequences; first += blockDim.x) {
        const int s = first + threadIdx.x;
        const int held = s < a.sequences && a.new_tokens[s] < 0 ? pages_of(length_of(s), a.page_tokens) : 0;
        long long sum = 0;
        const long long after = block_scan(held, lds, sum);
        const int place = static_cast<int>(min(stack + after - held, static_cast<long long>(a.pages)));
        for (unsigned long long todo = __ballot(held > 0); todo != 0; todo &= todo - 1) {
            const int from = __ffsll(todo) - 1;
            const int count = __shfl(held, from, 64), to = __shfl(place, from, 64);
            const int* table = a.tables + static_cast<size_t>(first + (threadIdx.x & ~63) + from) * a.table_stride;
            for (int j = lane; j < count; j += 64) {
                if (j < a.pages - to) a.free_pages[to + j] = table[j];
            }
        }
        stack = static_cast<int>(min(static_cast<long long>(stack) + sum, static_cast<long long>(a.pages)));
    }
    __syncthreads();

    // ---- who is let in, their pages and rows ----
    long long asked_rows = 0, asked_pages = 0, taken = 0, out = 0;
    long long refused = 0;
    for (int first = 0; first < a.sequences; first += blockDim.x) {
        const int s = first + threadIdx.x;
        const bool mine = s < a.sequences;
        const int length = mine ? length_of(s) : 0, asked = mine ? a.new_tokens[s] : 0;
        const bool ends = asked < 0;
        const int held = pages_of(length, a.page_tokens);
        int rows = max(asked, 0);
        bool fits = mine && !ends && static_cast<long long>(length) + rows <= room;
        long long sum = 0;
        const long long upto_rows = asked_rows + block_scan(fits ? rows : 0, lds, sum);
        fits &= rows == 0 || upto_rows <= a.rows_capacity;
        asked_rows += sum;
        int need = fits ? pages_of(static_cast<long long>(length) + rows, a.page_tokens) - held : 0;
        const long long upto = asked_pages + block_scan(need, lds, sum);
        asked_pages += sum;
        fits &= need == 0 || upto <= stack;
        if (!fits) need = rows = 0;
        const int start = static_cast<int>(out + block_scan(rows, lds, sum)) - rows;
        out += sum;
        block_scan(need, lds, sum);
        taken += sum;
        block_scan(mine && !ends && !fits ? 1 : 0, lds, sum);
        refused += sum;
        if (mine) {
            a.new_lengths[s] = ends ? 0 : length + rows;
            a.row_starts[s] = start;
        }
        // page j of a sequence: the stack's entry below those of the sequences before it
        const int top = stack - 1 - static_cast<int>(min(upto, static_cast<long long>(INT_MAX))) + need;
        for (unsigned long long todo = __ballot(need > 0); todo != 0; todo &= todo - 1) {
            const int from = __ffsll(todo) - 1;
            const int count = __shfl(need, from, 64), begin = __shfl(held, from, 64), at = __shfl(top, from, 64);
            int* table = a.tables + static_cast<size_t>(first + (threadIdx.x & ~63) + from) * a.table_stride;
            for (int j = lane; j < count; j += 64) table[begin + j] = a.free_pages[at - j];
        }
        if constexpr (kRows) {
            __syncthreads();
            for (unsigned long long todo = __ballot(rows > 0); todo != 0; todo &= todo - 1) {
                const int from = __ffsll(todo) - 1;
                const int count = __shfl(rows, from, 64), begin = __shfl(start, from, 64), at = __shfl(length, from, 64);
                for (int j = lane; j < count; j += 64) {
                    write_row(a, first + (threadIdx.x & ~63) + from, begin + j, at + j);
                }
            }
        }
    }
    if (threadIdx.x == 0) {
        a.row_starts[a.sequences] = static_cast<int>(out);
        *a.new_free_count = stack - static_cast<int>(taken);
        *a.refused = static_cast<int>(refused);
    }
    if constexpr (kRows) {
        for (int r = static_cast<int>(out) + threadIdx.x; r < a.rows_capacity; r += blockDim.x) {
            a.row_positions[r] = 0;
            a.row_slots[r] = -1;
        }
    }
}

// The row map of a step with many rows: a thread a row, its sequence by
// bisection of the row starts.
__global__ __launch_bounds__(kRowThreads) void kv8_plan_rows_kernel(Kv8PlanArgs a) {
    const int row = blockIdx.x * kRowThreads + threadIdx.x;
    if (row >= a.rows_capacity) return;
    if (row >= a.row_starts[a.sequences]) {
        a.row_positions[row] = 0;
        a.row_slots[row] = -1;
        return;
    }
    int low = 0, high = a.sequences;  // row_starts[low] <= row < row_starts[high]
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (a.row_starts[middle] <= row) low = middle;
        else high = middle;
    }
    write_row(a, low, row, a.new_lengths[low] - a.row_starts[low + 1] + row);
}

}  // namespace

hipError_t launch_kv8_plan(const Kv8PlanArgs& a, hipStream_t stream) {
    const auto given = [](const void* p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 4 == 0; };
    if (a.sequences < 1 || a.table_stride < 1 || a.pages < 1 || a.rows_capacity < 0 ||
        (a.page_tokens != 16 && a.page_tokens != 32 && a.page_tokens != 64) || a.pages > INT_MAX / a.page_tokens ||
        a.table_stride > INT_MAX / a.page_tokens || !given(a.new_tokens) || !given(a.lengths) ||
        !given(a.new_lengths) || !given(a.tables) || !given(a.free_pages) || !given(a.free_count) ||
        !given(a.new_free_count) || !given(a.row_starts) || !given(a.refused) ||
        (a.rows_capacity > 0 && (!given(a.row_positions) || !given(a.row_slots)))) {
        return hipErrorInvalidValue;
    }
    const int threads = a.sequences <= 64 ? 64 : a.sequences <= 256 ? 256 : kMaxThreads;
    if (a.rows_capacity <= kRowsInOneLaunch) {
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
