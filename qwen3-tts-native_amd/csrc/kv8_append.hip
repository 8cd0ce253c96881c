// Stores key and value rows in the paged 8-bit cache (kv8.hpp).
//
// A run is the rows of one call that go into one page: consecutive rows with
// consecutive slots.  Per page and head, for keys and values apart:
//   c = largest finite magnitude of the run / 127 in fp32          (int8)
//   c = the smallest power of two with 448 c >= that magnitude      (e4m3)
//   S = c where the run begins the page, else max(S_old, c)
//   new tokens      q = rne(x / S), to the format's range; infinities become
//                   its largest value, NaN becomes 0, so that a page never
//                   holds a NaN
//   earlier tokens  q = rne(q * S_old / S) where the scale grew
// x / S is the product with the reciprocal in 64 bits: the rounding to 8 bits
// is the only one.  e4m3 takes powers of two because its step is relative to
// the value: a finer scale would gain nothing, and growth would round every
// earlier value once more, where halving is exact (above its subnormals).
// An int8's step is absolute: a power of two would waste up to one bit of it.
// Tokens behind the run in its last granule become 0 where the granule begins
// with the run and keep their bytes where it does not: nothing reads them
// before a later run writes them.
//
// A wave owns a (run, head, keys or values): nobody else touches the page's
// bytes of that head, so granules that the run enters half-way are read,
// merged and written whole.  Lane (token, 16-dimension group) quantises in the
// keys' layout; values take their layout through 2 KB of LDS.  Bound by HBM for
// prompts, by the chain slot -> scale and page -> store for single tokens.
#include "kv8.hpp"

#include <climits>

namespace q3 {
namespace {

using namespace kv8;

// Bytes of four values from their quotients x / S.
template <int kFormat>
__device__ __forceinline__ unsigned hold4(double a, double b, double c, double d) {
    if constexpr (kFormat == kKv8Int8) {
        // NaN passes neither bound: fmax returns the bound, so it is caught by the callers
        const auto one = [](double v) { return static_cast<unsigned>(static_cast<int>(fmin(fmax(rint(v), -127.0), 127.0))) & 0xffu; };
        return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
    } else {
        const auto one = [](double v) { return fminf(fmaxf(static_cast<float>(v), -448.0f), 448.0f); };
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(one(a), one(b), 0, false);
        return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(one(c), one(d), w, true));
    }
}

// Held values in a page whose scale changed by `ratio` = S_old / S.
template <int kFormat>
__device__ __forceinline__ unsigned rescale4(unsigned w, double ratio) {
    if constexpr (kFormat == kKv8Int8) {
        const int v = static_cast<int>(w);
        return hold4<kFormat>(static_cast<signed char>(v) * ratio, static_cast<signed char>(v >> 8) * ratio,
                              static_cast<signed char>(v >> 16) * ratio, (v >> 24) * ratio);
    } else {
        const auto at = [&](float x) { return static_cast<double>(x) * ratio; };
        return hold4<kFormat>(at(__builtin_amdgcn_cvt_f32_fp8(w, 0)), at(__builtin_amdgcn_cvt_f32_fp8(w, 1)),
                              at(__builtin_amdgcn_cvt_f32_fp8(w, 2)), at(__builtin_amdgcn_cvt_f32_fp8(w, 3)));
    }
}

template <int kFormat>
__device__ __forceinline__ float scale_for(float largest) {
    if constexpr (kFormat == kKv8Int8) {
        return largest / 127.0f;
    } else {
        if (largest == 0.0f) return 0.0f;
        // largest = part * 2^exponent, part in [0.5, 1); 448 = 0.875 * 2^9
        int exponent;
        const float part = frexpf(largest, &exponent);
        return ldexpf(1.0f, part <= 0.875f ? exponent - 9 : exponent - 8);
    }
}

__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = max(v, __shfl_xor(v, d, 64));
    return v;
}

template <int kFormat, int kGranules>  // granules of a page
__device__ void append_run(const Kv8Cache& cache, const Kv8AppendArgs& a, int row, int count, int slot, int head,
                           bool is_value, unsigned char* lds) {
    constexpr int kPage = kGranules * kKv8Granule;
    const int lane = threadIdx.x & 63;
    const int page = slot / kPage, offset = slot % kPage, end = offset + count;
    const int first_granule = offset / kKv8Granule, granules_end = (end + kKv8Granule - 1) / kKv8Granule;
    const size_t of_page = static_cast<size_t>(page) * cache.key_value_heads + head;
    unsigned char* bytes = (is_value ? cache.value_pages : cache.key_pages) + of_page * (kGranules * kKv8GranuleBytes);
    float* scale_at = (is_value ? cache.value_scales : cache.key_scales) + of_page;
    const int stride = is_value ? a.value_stride : a.key_stride;
    const bf16_t* rows = (is_value ? a.value : a.key) + static_cast<size_t>(head) * kKv8HeadDimension;

    // the page's scale and the granule that the run enters half-way, beside the rows
    const bool keeps = offset > 0, enters = offset % kKv8Granule != 0;
    const float old_scale = keeps ? *scale_at : 0.0f;
    uint4 before[2];
    if (enters) {
        const uint4* from = reinterpret_cast<const uint4*>(bytes + first_granule * kKv8GranuleBytes) + lane;
        before[0] = from[0], before[1] = from[64];
    }
    // lane (token of the granule, group of 16 dimensions)
    const int token = lane >> 2, group = lane & 3;
    uint4 x[kGranules][2][2];
    int largest_bits = 0;
#pragma unroll
    for (int g = 0; g < kGranules; ++g) {
        const int t = g * kKv8Granule + token;
        const bool mine = t >= offset && t < end;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                x[g][c][u] = uint4{0, 0, 0, 0};
                if (mine) {
                    x[g][c][u] = *reinterpret_cast<const uint4*>(rows + static_cast<size_t>(row + t - offset) * stride +
                                                                 c * 64 + group * 16 + u * 8);
                }
            }
    }
#pragma unroll
    for (int g = 0; g < kGranules; ++g)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned w[4] = {x[g][c][u].x, x[g][c][u].y, x[g][c][u].z, x[g][c][u].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int lo = w[i] & 0x7fff, hi = (w[i] >> 16) & 0x7fff;
                    largest_bits = max(largest_bits, lo < 0x7f80 ? lo : 0);
                    largest_bits = max(largest_bits, hi < 0x7f80 ? hi : 0);
                }
            }
    largest_bits = wave_max(largest_bits);
    const float wanted = scale_for<kFormat>(__uint_as_float(static_cast<unsigned>(largest_bits) << 16));
    // a scale that is no number cannot be kept: its tokens are lost, the new ones are not
    const float scale = wanted >= old_scale ? wanted : old_scale == old_scale ? old_scale : wanted;
    const double inverse = scale > 0.0f ? 1.0 / static_cast<double>(scale) : 0.0;
    const bool grew = keeps && scale != old_scale;
    const double ratio = scale > 0.0f ? static_cast<double>(old_scale) / static_cast<double>(scale) : 1.0;

    // bytes of tokens before the run in the new scale
    auto moved = [&](uint4 w) {
        return uint4{rescale4<kFormat>(w.x, ratio), rescale4<kFormat>(w.y, ratio), rescale4<kFormat>(w.z, ratio),
                     rescale4<kFormat>(w.w, ratio)};
    };
    if (grew) {
        for (int g = 0; g < first_granule; ++g) {
            uint4* at = reinterpret_cast<uint4*>(bytes + g * kKv8GranuleBytes) + lane;
            const uint4 w0 = at[0], w1 = at[64];
            at[0] = moved(w0), at[64] = moved(w1);
        }
    }
#pragma unroll
    for (int g = 0; g < kGranules; ++g) {
        if (g < first_granule || g >= granules_end) continue;
        uint4 fresh[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4& half = x[g][c][i >> 1];
                const unsigned lo = i & 1 ? half.z : half.x, hi = i & 1 ? half.w : half.y;
                const auto at = [&](unsigned bits) {
                    const float v = __uint_as_float(bits);
                    return v == v ? static_cast<double>(v) * inverse : 0.0;
                };
                // an infinity times a zero reciprocal (a run without a finite magnitude) is held as 0
                const auto fine = [](double v) { return v == v ? v : 0.0; };
                w[i] = hold4<kFormat>(fine(at(lo << 16)), fine(at(lo & 0xffff0000u)), fine(at(hi << 16)),
                                      fine(at(hi & 0xffff0000u)));
            }
            fresh[c] = uint4{w[0], w[1], w[2], w[3]};
        }
        const int base = g * kKv8Granule;
        const bool merge = enters && g == first_granule;
        uint4 keep[2] = {uint4{0, 0, 0, 0}, uint4{0, 0, 0, 0}};
        if (merge) {
#pragma unroll
            for (int c = 0; c < 2; ++c) keep[c] = before[c];
        }
        uint4* to = reinterpret_cast<uint4*>(bytes + g * kKv8GranuleBytes) + lane;
        if (!is_value) {
            const int t = base + token;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (merge) {
                    if (t < offset) fresh[c] = grew ? moved(keep[c]) : keep[c];
                    else if (t >= end) fresh[c] = keep[c];
                }
                to[c * 64] = fresh[c];
            }
        } else {
            // token `token`, dimensions 64 c + 16 group + e: byte (token / 4) * 256 + e * 16 + group * 4 + token % 4
            __syncthreads();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const unsigned w[4] = {fresh[c].x, fresh[c].y, fresh[c].z, fresh[c].w};
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    lds[c * 1024 + (token >> 2) * 256 + e * 16 + group * 4 + (token & 3)] =
                        static_cast<unsigned char>(w[e >> 2] >> (8 * (e & 3)));
                }
            }
            __syncthreads();
            // lane (token / 4, d % 16)
            const int t = base + 4 * (lane >> 4);
            const unsigned earlier = byte_mask(t, 0, offset), later = byte_mask(t, end, INT_MAX);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint4 w = reinterpret_cast<const uint4*>(lds)[c * 64 + lane];
                if (merge) {
                    const uint4 scaled = grew ? moved(keep[c]) : keep[c];
                    const auto pick = [&](unsigned n, unsigned m, unsigned o) {
                        return (n & ~(earlier | later)) | (m & earlier) | (o & later);
                    };
                    w = uint4{pick(w.x, scaled.x, keep[c].x), pick(w.y, scaled.y, keep[c].y),
                              pick(w.z, scaled.z, keep[c].z), pick(w.w, scaled.w, keep[c].w)};
                }
                to[c * 64] = w;
            }
        }
    }
    if (lane == 0 && (!keeps || grew)) *scale_at = scale;
}

// A wave looks at kRows rows and takes the runs that begin there.
template <int kFormat, int kGranules, int kRows>
__global__ __launch_bounds__(64) void kv8_append_kernel(Kv8Cache cache, Kv8AppendArgs a) {
    __shared__ __align__(16) unsigned char lds[kKv8GranuleBytes];
    constexpr int kPage = kGranules * kKv8Granule;
    const int lane = threadIdx.x;
    const int first = blockIdx.x * kRows;
    const int head = blockIdx.y;
    const bool is_value = blockIdx.z != 0;
    const int slots = cache.pages * kPage;
    auto slot_of = [&](int row) {
        if (row < 0 || row >= a.rows) return -1;
        const int s = a.row_slots[row];
        return s >= 0 && s < slots ? s : -1;
    };
    bool begins = false;
    if (lane < kRows) {
        const int mine = slot_of(first + lane), last = slot_of(first + lane - 1);
        begins = mine >= 0 && !(last >= 0 && mine == last + 1 && mine % kPage != 0);
    }
    for (unsigned long long todo = __ballot(begins); todo != 0; todo &= todo - 1) {
        const int row = first + __ffsll(todo) - 1;
        const int slot = a.row_slots[row];
        // the run: rows that follow one another up to the page's end
        const bool follows = lane < kPage - slot % kPage && slot_of(row + lane) == slot + lane;
        const unsigned long long stops = ~__ballot(follows);
        const int count = stops == 0 ? 64 : __ffsll(stops) - 1;
        append_run<kFormat, kGranules>(cache, a, row, count, slot, head, is_value, lds);
    }
}

template <int kFormat, int kGranules>
hipError_t launch_pages(const Kv8Cache& cache, const Kv8AppendArgs& a, hipStream_t stream) {
    // One row a wave while that leaves the launch small: a row's wave starts
    // at once and single tokens of many sequences do not queue behind one
    // another.  Prompts: 15 of 16 rows begin no run.
    constexpr int kRows = 16;
    if (static_cast<long long>(a.rows) * cache.key_value_heads <= 4096) {
        kv8_append_kernel<kFormat, kGranules, 1>
            <<<dim3(a.rows, cache.key_value_heads, 2), 64, 0, stream>>>(cache, a);
    } else {
        kv8_append_kernel<kFormat, kGranules, kRows>
            <<<dim3((a.rows + kRows - 1) / kRows, cache.key_value_heads, 2), 64, 0, stream>>>(cache, a);
    }
    return hipGetLastError();
}

template <int kFormat>
hipError_t launch_format(const Kv8Cache& cache, const Kv8AppendArgs& a, hipStream_t stream) {
    switch (cache.page_tokens) {
        case 16: return launch_pages<kFormat, 1>(cache, a, stream);
        case 32: return launch_pages<kFormat, 2>(cache, a, stream);
        default: return launch_pages<kFormat, 4>(cache, a, stream);
    }
}

}  // namespace

bool kv8_cache_ok(const Kv8Cache& c, bool pointers) {
    const auto aligned = [](const void* p, size_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; };
    return (c.format == kKv8Int8 || c.format == kKv8E4m3) &&
           (c.page_tokens == 16 || c.page_tokens == 32 || c.page_tokens == 64) && c.pages >= 1 &&
           c.pages <= INT_MAX / c.page_tokens && c.key_value_heads >= 1 && c.key_value_heads <= 65535 &&
           (!pointers || (aligned(c.key_pages, 16) && aligned(c.value_pages, 16) && aligned(c.key_scales, 4) &&
                          aligned(c.value_scales, 4)));
}

hipError_t launch_kv8_append(const Kv8Cache& cache, const Kv8AppendArgs& a, hipStream_t stream) {
    if (!kv8_cache_ok(cache) || a.rows < 0) return hipErrorInvalidValue;
    if (a.rows == 0) return hipSuccess;
    const long long width = static_cast<long long>(cache.key_value_heads) * kKv8HeadDimension;
    if (a.key == nullptr || a.value == nullptr || a.row_slots == nullptr || a.key_stride < width ||
        a.value_stride < width || a.key_stride % 8 != 0 || a.value_stride % 8 != 0 ||
        reinterpret_cast<uintptr_t>(a.key) % 16 != 0 || reinterpret_cast<uintptr_t>(a.value) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(a.row_slots) % 4 != 0) {
        return hipErrorInvalidValue;
    }
    return cache.format == kKv8Int8 ? launch_format<kKv8Int8>(cache, a, stream)
                                    : launch_format<kKv8E4m3>(cache, a, stream);
}

}  // namespace q3
