// The paged 8-bit key/value cache: layout, number formats and launch
// arguments shared by its three operators (kv8_plan.hip, kv8_append.hip,
// kv8_attention.hip).
//
// A page holds 16, 32 or 64 tokens of every key/value head; per head it is a
// run of granules of 16 tokens, 2048 bytes of keys in one array of pages and
// 2048 bytes of values in another.  Within a granule a byte lies where the
// attention's matrix instructions take it, so that a wave reads a granule in
// two contiguous 1 KB loads and needs no exchange between lanes:
//   key   (token t, dimension d): (d / 64) * 1024 + t * 64 + d % 64
//         lane (t, d / 16 % 4) holds 16 dimensions of one token: the key
//         operand of two 16x16x32 products (the query is read in that order)
//   value (token t, dimension d): (d / 64) * 1024 + (t / 4) * 256 +
//         (d % 16) * 16 + (d / 16 % 4) * 4 + t % 4
//         lane (t / 4, d % 16) holds four tokens of four dimensions 16 apart:
//         a lane's scores of a granule are those of its four tokens, which
//         makes both operands of the value product without a transposition
// Each page has one fp32 scale per head for its keys and one for its values.
#pragma once

#include "q3_common.hpp"

namespace q3 {

enum Kv8Format : int { kKv8Int8 = 0, kKv8E4m3 = 1 };

constexpr int kKv8HeadDimension = 128;
constexpr int kKv8Granule = 16;         // tokens
constexpr int kKv8GranuleBytes = 2048;  // of one head's keys or values

struct Kv8Cache {
    int format = kKv8Int8;
    int page_tokens = 16;
    int pages = 0;
    int key_value_heads = 0;
    uint8_t* key_pages = nullptr;  // [pages][key_value_heads][page_tokens / 16][2048]
    uint8_t* value_pages = nullptr;
    float* key_scales = nullptr;  // [pages][key_value_heads]
    float* value_scales = nullptr;
};

struct Kv8PlanArgs {
    int sequences = 0, page_tokens = 0, pages = 0, table_stride = 0, rows_capacity = 0;
    const int* new_tokens = nullptr;
    const int* lengths = nullptr;
    int* new_lengths = nullptr;
    int* tables = nullptr;
    int* free_pages = nullptr;
    const int* free_count = nullptr;
    int* new_free_count = nullptr;
    int* row_starts = nullptr;
    int* row_positions = nullptr;
    int* row_slots = nullptr;
    int* refused = nullptr;
};
hipError_t launch_kv8_plan(const Kv8PlanArgs& args, hipStream_t stream);

struct Kv8AppendArgs {
    int rows = 0, key_stride = 0, value_stride = 0;
    const bf16_t* key = nullptr;
    const bf16_t* value = nullptr;
    const int* row_slots = nullptr;
};
hipError_t launch_kv8_append(const Kv8Cache& cache, const Kv8AppendArgs& args, hipStream_t stream);

struct Kv8AttentionArgs {
    int query_heads = 0, rows = 0, query_stride = 0, out_stride = 0;
    int sequences = 0, table_stride = 0, max_rows = 0, max_length = 0, window = 0;
    float scale = 0.0f;
    const bf16_t* query = nullptr;
    bf16_t* out = nullptr;
    const int* tables = nullptr;
    const int* lengths = nullptr;
    const int* row_starts = nullptr;
    float* workspace = nullptr;
    size_t workspace_bytes = 0;
};
hipError_t launch_kv8_attention(const Kv8Cache& cache, const Kv8AttentionArgs& args, hipStream_t stream);
// What a call with these sizes uses where it is given that much (0: it needs
// none); pointers are not looked at.
hipError_t kv8_attention_workspace(const Kv8Cache& cache, const Kv8AttentionArgs& args, size_t& bytes);

// Format, page size, head count and (where `pointers`) the arrays.
bool kv8_cache_ok(const Kv8Cache& cache, bool pointers = true);

#if defined(__HIPCC__)
namespace kv8 {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx2_t __attribute__((ext_vector_type(2)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));

// Two floats to a pair of bf16, nearest even.
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(floatx2_t{lo, hi}, bf16x2_t));
}

// Four held values as bf16, in units of their scale: exact in both formats
// (at most 8 significant bits).
template <int kFormat>
__device__ __forceinline__ uint2 bf16_of(unsigned w) {
    if constexpr (kFormat == kKv8Int8) {
        const int v = static_cast<int>(w);
        return uint2{pack_bf16(static_cast<float>(static_cast<signed char>(v)),
                               static_cast<float>(static_cast<signed char>(v >> 8))),
                     pack_bf16(static_cast<float>(static_cast<signed char>(v >> 16)), static_cast<float>(v >> 24))};
    } else {
        return uint2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
    }
}

template <int kFormat>
__device__ __forceinline__ bf16x8_t bf16x8_of(unsigned lo, unsigned hi) {
    const uint2 a = bf16_of<kFormat>(lo), b = bf16_of<kFormat>(hi);
    return __builtin_bit_cast(bf16x8_t, uint4{a.x, a.y, b.x, b.y});
}

// 0xff in the bytes of tokens first .. first + 3 that lie in [begin, end).
__device__ __forceinline__ unsigned byte_mask(int first, int begin, int end) {
    const int lo = min(max(begin - first, 0), 4), hi = min(max(end - first, 0), 4);
    const unsigned below = hi == 4 ? 0xffffffffu : (1u << (8 * hi)) - 1u;
    const unsigned skip = lo == 4 ? 0xffffffffu : (1u << (8 * lo)) - 1u;
    return below & ~skip;
}

}  // namespace kv8
#endif

}  // namespace q3
