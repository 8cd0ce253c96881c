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
// A workgroup owns a (run, head, keys or values), a wave each granule of the
// page: nobody else touches the page's bytes of that head, so granules that
// the run enters half-way are read, merged and written whole.  Lane (token,
// 16-dimension group) quantises in the keys' layout; values take theirs by two
// 4 x 4 transpositions in registers, of bytes over the lanes of four tokens
// and of words over the four lane groups.  Bound by HBM for prompts (16379 rows,
// 8 heads, int8: 4.2 TB/s), by the chain slot -> page and scale -> store for
// single tokens.
#include "kv8.hpp"

#include <algorithm>
#include <climits>

namespace q3 {
namespace {

using namespace kv8;

constexpr int kRows = 64;  // rows that a workgroup looks at for runs

// Bytes of four values from their quotients x / S.  Adding 1.5 * 2^52 rounds to
// the nearest whole number, ties to even, and leaves it in the low bits.
template <int kFormat>
__device__ __forceinline__ unsigned hold4(double a, double b, double c, double d) {
    if constexpr (kFormat == kKv8Int8) {
        const auto one = [](double v) {
            return static_cast<unsigned>(__builtin_bit_cast(unsigned long long, v + 6755399441055744.0));
        };
        const unsigned low = __builtin_amdgcn_perm(one(b), one(a), 0x0c0c0400u);
        return __builtin_amdgcn_perm(one(d), one(c), 0x04000c0cu) | low;
    } else {
        const auto one = [](double v) { return fminf(fmaxf(static_cast<float>(v), -448.0f), 448.0f); };
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(one(a), one(b), 0, false);
        return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(one(c), one(d), w, true));
    }
}

// Held values in a page whose scale changed by `ratio` = S_old / S, at most 1.
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
__device__ __forceinline__ uint4 rescale16(uint4 w, double ratio) {
    return uint4{rescale4<kFormat>(w.x, ratio), rescale4<kFormat>(w.y, ratio), rescale4<kFormat>(w.z, ratio),
                 rescale4<kFormat>(w.w, ratio)};
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

template <int kControl>
__device__ __forceinline__ unsigned max_moved(unsigned v) {
    return max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, 0xf, 0xf, true)));
}

// The largest value over the workgroup's waves.
template <int kWaves>
__device__ __forceinline__ unsigned block_max(unsigned v, unsigned* lds) {
    v = max(v, static_cast<unsigned>(__builtin_amdgcn_permlane32_swap(v, v, false, false)[1]));  // lanes 0-31 see 32-63
    v = max(v, static_cast<unsigned>(__builtin_amdgcn_permlane16_swap(v, v, false, false)[1]));  // lanes 0-15 see 16-31
    v = max_moved<0x108>(v);  // row_shl:8 and below
    v = max_moved<0x104>(v);
    v = max_moved<0x102>(v);
    v = max_moved<0x101>(v);
    v = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
    if constexpr (kWaves == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = max(v, lds[w]);
    return v;
}

// Of the four lanes 4 n .. 4 n + 3, lane k gets byte k of each one's word.
__device__ __forceinline__ unsigned transpose_bytes(unsigned w, int lane) {
    const unsigned next = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w), 0xb1, 0xf, 0xf, true));  // lane ^ 1
    w = __builtin_amdgcn_perm(next, w, lane & 1 ? 0x03070105u : 0x06020400u);
    const unsigned far = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w), 0x4e, 0xf, 0xf, true));  // lane ^ 2
    return __builtin_amdgcn_perm(far, w, lane & 2 ? 0x03020706u : 0x05040100u);
}

// Word j of the lane in group g of 16 becomes word g of the lane in group j.
__device__ __forceinline__ uint4 transpose_groups(uint4 w) {
    const auto a = __builtin_amdgcn_permlane32_swap(w.x, w.z, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w.y, w.w, false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return uint4{c[0], c[1], d[0], d[1]};
}

typedef unsigned short ushortx2_t __attribute__((ext_vector_type(2)));

template <int kFormat, int kGranules>  // granules of a page
__device__ __forceinline__ void append_run(const Kv8Cache& cache, const Kv8AppendArgs& a, int row, int count, int slot, int head,
                                           bool is_value, unsigned* lds) {
    constexpr int kPage = kGranules * kKv8Granule;
    const int lane = threadIdx.x & 63, granule = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int page = slot / kPage, offset = slot % kPage, end = offset + count;
    const int first = granule * kKv8Granule;  // the wave's granule's first token
    const size_t of_page = static_cast<size_t>(page) * cache.key_value_heads + head;
    unsigned char* bytes = (is_value ? cache.value_pages : cache.key_pages) + of_page * (kGranules * kKv8GranuleBytes);
    float* scale_at = (is_value ? cache.value_scales : cache.key_scales) + of_page;
    const int stride = is_value ? a.value_stride : a.key_stride;
    const bf16_t* rows = (is_value ? a.value : a.key) + static_cast<size_t>(head) * kKv8HeadDimension;

    // lane (token of the granule, group of 16 dimensions), and where its 16
    // bytes lie: keys token by token, values as (token / 4, d % 16) after the
    // transpositions, which bring lane (group, token / 4, token % 4) the words of
    // d % 16 = 4 group + token % 4
    const int token = lane & 15, group = lane >> 4;
    const int place = is_value ? (token >> 2) * 256 + (4 * group + (token & 3)) * 16 : token * 64 + group * 16;
    uint4* to = reinterpret_cast<uint4*>(bytes + granule * kKv8GranuleBytes + place);  // and 64 further for the upper dimensions

    // the rows, beside the page's scale and a granule that the run enters half-way
    const bool keeps = offset > 0;
    const bool touched = first < end && first + kKv8Granule > offset;  // by the run
    const bool merges = touched && first < offset;
    const bool mine = first + token >= offset && first + token < end;
    const float old_scale = keeps ? *scale_at : 0.0f;
    uint4 x[2][2], before[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            x[c][u] = uint4{0, 0, 0, 0};
            if (mine) {
                x[c][u] = *reinterpret_cast<const uint4*>(rows + static_cast<size_t>(row + first + token - offset) * stride +
                                                          c * 64 + group * 16 + u * 8);
            }
        }
    if (merges) before[0] = to[0], before[1] = to[64];

    ushortx2_t most{0, 0};
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned w[4] = {x[c][u].x, x[c][u].y, x[c][u].z, x[c][u].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(ushortx2_t, w[i] & 0x7fff7fffu));
        }
    unsigned largest = block_max<kGranules>(max(most[0], most[1]), lds);
    const bool odd = largest >= 0x7f80u;  // an infinity or a NaN is among them: looked for one by one
    if (odd) {
        unsigned finite = 0;
        for (int c = 0; c < 2; ++c)
            for (int u = 0; u < 2; ++u)
                for (int i = 0; i < 4; ++i) {
                    const unsigned w = i == 0 ? x[c][u].x : i == 1 ? x[c][u].y : i == 2 ? x[c][u].z : x[c][u].w;
                    const unsigned lo = w & 0x7fffu, hi = w >> 16 & 0x7fffu;
                    finite = max(finite, lo < 0x7f80u ? lo : 0u);
                    finite = max(finite, hi < 0x7f80u ? hi : 0u);
                }
        largest = block_max<kGranules>(finite, lds);
    }
    const float wanted = scale_for<kFormat>(__uint_as_float(largest << 16));
    // a scale that is no number cannot be kept: its tokens are lost, the new ones are not
    const float scale = wanted >= old_scale ? wanted : old_scale == old_scale ? old_scale : wanted;
    const double inverse = scale > 0.0f ? 1.0 / static_cast<double>(scale) : 0.0;
    const bool grew = keeps && scale != old_scale;
    double ratio = scale > 0.0f ? static_cast<double>(old_scale) / static_cast<double>(scale) : 1.0;
    if (!(ratio <= 1.0)) ratio = 0.0;

    if (touched) {
        uint4 fresh[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4& eight = x[c][i >> 1];
                const unsigned lo = i & 1 ? eight.z : eight.x, hi = i & 1 ? eight.w : eight.y;
                const auto quotient = [&](unsigned bits) { return static_cast<double>(__uint_as_float(bits)) * inverse; };
                double v[4] = {quotient(lo << 16), quotient(lo & 0xffff0000u), quotient(hi << 16), quotient(hi & 0xffff0000u)};
                if (odd) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // NaN, also of an infinity in a run without a finite magnitude, becomes 0
                        constexpr double kRange = kFormat == kKv8Int8 ? 127.0 : 448.0;
                        v[e] = v[e] == v[e] ? fmin(fmax(v[e], -kRange), kRange) : 0.0;
                    }
                }
                w[i] = hold4<kFormat>(v[0], v[1], v[2], v[3]);
            }
            fresh[c] = uint4{w[0], w[1], w[2], w[3]};
        }
        if (!is_value) {
            if (merges) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (first + token < offset) fresh[c] = grew ? rescale16<kFormat>(before[c], ratio) : before[c];
                    else if (first + token >= end) fresh[c] = before[c];
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                fresh[c] = transpose_groups(uint4{transpose_bytes(fresh[c].x, lane), transpose_bytes(fresh[c].y, lane),
                                                  transpose_bytes(fresh[c].z, lane), transpose_bytes(fresh[c].w, lane)});
            }
            if (merges) {
                const int four = first + (token & ~3);
                const unsigned earlier = byte_mask(four, 0, offset), later = byte_mask(four, end, INT_MAX);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint4 scaled = grew ? rescale16<kFormat>(before[c], ratio) : before[c];
                    const auto pick = [&](unsigned n, unsigned m, unsigned o) {
                        return (n & ~(earlier | later)) | (m & earlier) | (o & later);
                    };
                    fresh[c] = uint4{pick(fresh[c].x, scaled.x, before[c].x), pick(fresh[c].y, scaled.y, before[c].y),
                                     pick(fresh[c].z, scaled.z, before[c].z), pick(fresh[c].w, scaled.w, before[c].w)};
                }
            }
        }
        to[0] = fresh[0], to[64] = fresh[1];
    } else if (grew && first < offset) {
        const uint4 w0 = to[0], w1 = to[64];
        to[0] = rescale16<kFormat>(w0, ratio), to[64] = rescale16<kFormat>(w1, ratio);
    }
    if (threadIdx.x == 0 && (!keeps || grew)) *scale_at = scale;
}

// `slices` workgroups look at the same kRows rows and take the runs that begin
// there in turn.
template <int kFormat, int kGranules>
__global__ __launch_bounds__(64 * kGranules) void kv8_append_kernel(Kv8Cache cache, Kv8AppendArgs a, int slices) {
    __shared__ unsigned lds[kGranules];
    constexpr int kPage = kGranules * kKv8Granule;
    const int lane = threadIdx.x & 63;
    const int first = static_cast<int>(blockIdx.x / slices) * kRows, slice = blockIdx.x % slices;
    const int head = blockIdx.y;
    const bool is_value = blockIdx.z != 0;
    const int slots = cache.pages * kPage;
    auto slot_of = [&](int row) {
        if (row < 0 || row >= a.rows) return -1;
        const int s = a.row_slots[row];
        return s >= 0 && s < slots ? s : -1;
    };
    // the rows, the one before them, and those behind them that a run which begins here can have
    const int before = slot_of(first - 1), mine = slot_of(first + lane), later = slot_of(first + kRows + lane);
    int last = __builtin_amdgcn_update_dpp(0, mine, 0x138, 0xf, 0xf, false);  // wave_shr:1
    if (lane == 0) last = before;
    const bool begins = mine >= 0 && !(last >= 0 && mine == last + 1 && mine % kPage != 0);
    // this workgroup's turns among the runs
    const unsigned turn = __popcll(__ballot(begins) & ((1ull << lane) - 1));
    for (unsigned long long todo = __ballot(begins && turn % static_cast<unsigned>(slices) == static_cast<unsigned>(slice)); todo != 0; todo &= todo - 1) {
        const int from = __ffsll(todo) - 1;
        const int slot = __builtin_amdgcn_readlane(mine, from);
        // the run: rows that follow one another up to the page's end
        const int most = kPage - slot % kPage;
        const unsigned long long here = __ballot(lane >= from && lane - from < most && mine == slot + lane - from) >> from;
        const unsigned long long there = __ballot(kRows + lane - from < most && later == slot + kRows + lane - from);
        int count = ~here == 0 ? kRows : __ffsll(~here) - 1;
        if (count == kRows - from) count += ~there == 0 ? kRows : __ffsll(~there) - 1;
        append_run<kFormat, kGranules>(cache, a, first + from, count, slot, head, is_value, lds);
    }
}

template <int kFormat, int kGranules>
hipError_t launch_pages(const Kv8Cache& cache, const Kv8AppendArgs& a, hipStream_t stream) {
    // Single tokens of many sequences begin a run in every row, prompts in one
    // of a page's: several workgroups share 64 rows' runs, as many as a prompt
    // has there at least, and more while the launch stays small, since one that
    // finds none costs its start.  1024 / 2048 / 4096 workgroups, us: 256 single
    // tokens 9.2 / 7.4 / 6.9, four prompts of 512 rows 5.1 / 5.0 / 7.7, with pages
    // of 64 tokens (four waves) 7.4 / 11.7 / 18.4.
    constexpr int kLeast = kRows / (kGranules * kKv8Granule);
    constexpr int kWorkgroups = kGranules == 4 ? 1024 : 2048;
    const long long groups = (a.rows + kRows - 1) / kRows, units = groups * cache.key_value_heads * 2;
    const int slices = static_cast<int>(std::clamp<long long>(kWorkgroups / units, kLeast, kRows));
    kv8_append_kernel<kFormat, kGranules>
        <<<dim3(static_cast<unsigned>(groups * slices), cache.key_value_heads, 2), 64 * kGranules, 0, stream>>>(cache, a, slices);
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
