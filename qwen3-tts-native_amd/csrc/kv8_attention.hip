// Ragged causal attention over the paged 8-bit cache (kv8.hpp).
//
// Rows r of sequence s are the last ones of its length: position p = length -
// rows + i attends to tokens max(0, p - window + 1) .. p (window 0: all).  With
// q.k the product over 128 dimensions and k = held * key scale of its page:
//   o = sum_j exp(scale * q.k_j - m) v_j / sum_j exp(scale * q.k_j - m)
// A row whose tokens are none (an empty sequence, a table entry that is no
// page) becomes 0.  Held values are at most 8 bits wide, so they are exact as
// bf16 operands of the matrix instructions; scales are applied in fp32, the
// keys' to the scores, the values' to the weights; maxima, sums and
// accumulators are fp32.
#include "kv8.hpp"

#include <climits>
#include <cmath>

namespace q3 {

namespace {

using namespace kv8;

constexpr int kDim = kKv8HeadDimension;
constexpr int kMaxGroup = 16;  // query heads of a key/value head: the columns of the smallest product
constexpr float kLog2E = 1.44269504088896340736f;

struct Params {
    Kv8AttentionArgs a;
    Kv8Cache cache;
    int group = 1;     // query heads of a key/value head
    float scale2 = 0;  // scale * log2(e)
    int splits = 1;    // workgroups that share a context
    int columns = 16;  // of a partial result: (row, head of the group) pairs
    float* partial_out = nullptr;   // [sequence][kv head][column][split][128]
    float2* partial_sums = nullptr;  // [sequence][kv head][column][split] (maximum, sum)
};

// The rows of a sequence that exist, and where they lie in it.
struct Rows {
    int first, count, position;  // row 0's position
    int length;                  // tokens that the table can hold
};
__device__ __forceinline__ Rows rows_of(const Params& p, int sequence) {
    Rows r;
    const int begin = p.a.row_starts[sequence], end = p.a.row_starts[sequence + 1];
    const long long room = static_cast<long long>(p.a.table_stride) * p.cache.page_tokens;
    r.first = max(begin, 0);
    r.count = min(end, p.a.rows) - r.first;
    const int length = max(p.a.lengths[sequence], 0);
    r.position = length - (end - begin) + (r.first - begin);
    r.length = static_cast<int>(min(static_cast<long long>(length), room));
    return r;
}

// ---------------------------------------------------------------------------
// Few rows: up to 16 (row, head) pairs of one key/value head are the columns
// of 16x16x32 products, keys and values are read once for all of them.
// ---------------------------------------------------------------------------
constexpr int kWaves = 4;
constexpr int kStep = 64;  // tokens of a wave's step
constexpr int kStepGranules = kStep / kKv8Granule;

template <int kFormat, int kPageGranules>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_few_rows_kernel(Params p) {
    __shared__ __align__(16) float out_lds[kWaves][8 * 64 * 4];
    __shared__ float max_lds[kWaves][16], sum_lds[kWaves][16];
    constexpr int kPage = kPageGranules * kKv8Granule;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, quad = lane >> 4;
    const int split = blockIdx.x, kv_head = blockIdx.y, sequence = blockIdx.z;
    const Rows rows = rows_of(p, sequence);
    if (rows.count <= 0) return;
    const int rows_per_tile = 16 / p.group;
    const int head = kv_head * p.group + column % p.group;
    const int* table = p.a.tables + static_cast<size_t>(sequence) * p.a.table_stride;
    const size_t page_bytes = static_cast<size_t>(p.cache.key_value_heads) * (kPageGranules * kKv8GranuleBytes);
    const unsigned char* values = p.cache.value_pages + kv_head * (kPageGranules * kKv8GranuleBytes) + lane * 16;
    // lane (token, 16-dimension group) of the keys: byte token * 64 + group * 16
    const unsigned char* keys_of_lane = p.cache.key_pages + kv_head * (kPageGranules * kKv8GranuleBytes) +
                                        (lane & 15) * 64 + quad * 16;

    for (int tile = 0; tile < rows.count; tile += rows_per_tile) {
        const int row = tile + column / p.group;
        const bool mine = column < rows_per_tile * p.group && row < rows.count;
        const int position = mine ? rows.position + row : -1;
        // the query's dimensions 64 c + 16 quad + 8 u + 0 .. 7: those of the key bytes of this lane's group
        bf16x8_t q[2][2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint4 w{0, 0, 0, 0};
                if (mine) {
                    w = *reinterpret_cast<const uint4*>(p.a.query +
                                                        static_cast<size_t>(rows.first + row) * p.a.query_stride +
                                                        head * kDim + c * 64 + quad * 16 + u * 8);
                }
                q[c][u] = __builtin_bit_cast(bf16x8_t, w);
            }
        // tokens [begin, end) of this tile's rows, in steps dealt to the splits, then to the waves
        const int last = min(tile + rows_per_tile, rows.count) - 1;
        const int end = min(rows.position + last + 1, rows.length);
        const int begin = p.a.window > 0 ? max(rows.position + tile - p.a.window + 1, 0) & ~(kStep - 1) : 0;
        const int steps = end > begin ? (end - begin + kStep - 1) / kStep : 0;
        const int share = (steps + p.splits - 1) / p.splits;
        const int steps_begin = split * share, steps_end = min(steps_begin + share, steps);
        const int lowest = p.a.window > 0 ? position - p.a.window : -1;  // tokens above it count

        float maximum = -INFINITY, sum = 0.0f;
        floatx4_t acc[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        for (int step = steps_begin + wave; step < steps_end; step += kWaves) {
            const int token0 = begin + step * kStep;
            uint4 k[kStepGranules][2], v[kStepGranules][2];
            float key_scale[kStepGranules], value_scale[kStepGranules];
            int held[kStepGranules];  // tokens of the granule that hold something
#pragma unroll
            for (int g = 0; g < kStepGranules; ++g) {
                const int first = token0 + g * kKv8Granule;
                const int at = min(first, (end - 1) & ~(kKv8Granule - 1));  // past the end: the last one again
                int page = table[at / kPage];
                held[g] = min(max(end - first, 0), kKv8Granule);
                if (page < 0 || page >= p.cache.pages) page = 0, held[g] = 0;
                const size_t offset = page * page_bytes + at % kPage / kKv8Granule * kKv8GranuleBytes;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    k[g][c] = *reinterpret_cast<const uint4*>(keys_of_lane + offset + c * 1024);
                    v[g][c] = *reinterpret_cast<const uint4*>(values + offset + c * 1024);
                }
                const size_t scale_at = static_cast<size_t>(page) * p.cache.key_value_heads + kv_head;
                key_scale[g] = p.cache.key_scales[scale_at] * p.scale2;
                value_scale[g] = held[g] > 0 ? p.cache.value_scales[scale_at] : 0.0f;
            }
            float s[kStepGranules][4];
            float top = maximum;
#pragma unroll
            for (int g = 0; g < kStepGranules; ++g) {
                floatx4_t dot{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16x8_of<kFormat>(k[g][c].x, k[g][c].y), q[c][0], dot, 0, 0, 0);
                    dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16x8_of<kFormat>(k[g][c].z, k[g][c].w), q[c][1], dot, 0, 0, 0);
                }
                const int first = token0 + g * kKv8Granule + 4 * quad;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = first + i;
                    const bool counts = token <= position && token > lowest && 4 * quad + i < held[g];
                    s[g][i] = counts ? dot[i] * key_scale[g] : -INFINITY;
                    top = fmaxf(top, s[g][i]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float reference = top == -INFINITY ? 0.0f : top;  // nothing counted yet: weights become 0
            const float shrink = __builtin_amdgcn_exp2f(maximum - reference);
            maximum = top;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[d] *= shrink;
            // weights times the values' scale as two bf16, the second what the first leaves: 16 bits of them
            unsigned high[kStepGranules][2], low[kStepGranules][2];
#pragma unroll
            for (int g = 0; g < kStepGranules; ++g) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[g][i] - reference);
                    sum += e;
                    w[i] = e * value_scale[g];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    high[g][i] = pack_bf16(w[2 * i], w[2 * i + 1]);
                    low[g][i] = pack_bf16(w[2 * i] - __uint_as_float(high[g][i] << 16),
                                          w[2 * i + 1] - __uint_as_float(high[g][i] & 0xffff0000u));
                }
                if (held[g] < kKv8Granule) {
                    // bytes behind the length may hold anything, an e4m3 NaN too, which a zero weight would not silence
                    const unsigned mask = byte_mask(4 * quad, 0, held[g]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) v[g][c] = uint4{v[g][c].x & mask, v[g][c].y & mask, v[g][c].z & mask, v[g][c].w & mask};
                }
            }
#pragma unroll
            for (int g = 0; g < kStepGranules; g += 2) {
                const bf16x8_t ph = __builtin_bit_cast(bf16x8_t, uint4{high[g][0], high[g][1], high[g + 1][0], high[g + 1][1]});
                const bf16x8_t pl = __builtin_bit_cast(bf16x8_t, uint4{low[g][0], low[g][1], low[g + 1][0], low[g + 1][1]});
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const unsigned a[4] = {v[g][c].x, v[g][c].y, v[g][c].z, v[g][c].w};
                    const unsigned b[4] = {v[g + 1][c].x, v[g + 1][c].y, v[g + 1][c].z, v[g + 1][c].w};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const bf16x8_t value = bf16x8_of<kFormat>(a[t], b[t]);
                        acc[c * 4 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, ph, acc[c * 4 + t], 0, 0, 0);
                        acc[c * 4 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, pl, acc[c * 4 + t], 0, 0, 0);
                    }
                }
            }
        }
        // over the lanes of a column, then over the waves
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (quad == 0) max_lds[wave][column] = maximum, sum_lds[wave][column] = sum;
        __syncthreads();
        float top = max_lds[0][column];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, max_lds[w][column]);
        const float reference = top == -INFINITY ? 0.0f : top;
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total += sum_lds[w][column] * __builtin_amdgcn_exp2f(max_lds[w][column] - reference);
        const float mine_shrinks = __builtin_amdgcn_exp2f(maximum - reference);
#pragma unroll
        for (int d = 0; d < 8; ++d) *reinterpret_cast<floatx4_t*>(&out_lds[wave][(d * 64 + lane) * 4]) = acc[d] * mine_shrinks;
        __syncthreads();
        // wave w: dimensions 32 w .. 32 w + 31 (two tiles of 16) of every column
        if (mine) {
            const size_t slot = ((static_cast<size_t>(sequence) * p.cache.key_value_heads + kv_head) * p.columns + tile * p.group + column) * p.splits + split;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int d = 2 * wave + j;
                floatx4_t o = *reinterpret_cast<const floatx4_t*>(&out_lds[0][(d * 64 + lane) * 4]);
#pragma unroll
                for (int w = 1; w < kWaves; ++w) o += *reinterpret_cast<const floatx4_t*>(&out_lds[w][(d * 64 + lane) * 4]);
                if (p.splits == 1) {
                    const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
                    bf16_t* to = p.a.out + static_cast<size_t>(rows.first + row) * p.a.out_stride + head * kDim + 16 * d + 4 * quad;
                    *reinterpret_cast<uint2*>(to) = uint2{pack_bf16(o[0] * inverse, o[1] * inverse), pack_bf16(o[2] * inverse, o[3] * inverse)};
                } else {
                    *reinterpret_cast<floatx4_t*>(p.partial_out + slot * kDim + 16 * d + 4 * quad) = o;
                }
            }
            if (p.splits > 1 && wave == 0 && quad == 0) p.partial_sums[slot] = float2{top, total};
        }
        __syncthreads();
    }
}

template <int kFormat>
hipError_t launch_few_rows(const Params& p, hipStream_t stream) {
    const dim3 grid(p.splits, p.cache.key_value_heads, p.a.sequences);
    switch (p.cache.page_tokens) {
        case 16: kv8_few_rows_kernel<kFormat, 1><<<grid, 64 * kWaves, 0, stream>>>(p); break;
        case 32: kv8_few_rows_kernel<kFormat, 2><<<grid, 64 * kWaves, 0, stream>>>(p); break;
        default: kv8_few_rows_kernel<kFormat, 4><<<grid, 64 * kWaves, 0, stream>>>(p); break;
    }
    return hipGetLastError();
}

bool sizes_ok(const Kv8Cache& c, const Kv8AttentionArgs& a) {
    return kv8_cache_ok(c, false) && a.rows >= 0 && a.sequences >= 0 && a.sequences <= 65535 && a.query_heads >= 1 &&
           a.query_heads % c.key_value_heads == 0 && a.query_heads / c.key_value_heads <= kMaxGroup && a.window >= 0 &&
           std::isfinite(a.scale) && a.max_rows >= 1 && a.max_length >= 1;
}

bool args_ok(const Kv8Cache& c, const Kv8AttentionArgs& a) {
    const auto aligned = [](const void* p, size_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; };
    const long long width = static_cast<long long>(a.query_heads) * kDim;
    return kv8_cache_ok(c) && a.query_stride >= width && a.out_stride >= width && a.query_stride % 8 == 0 &&
           a.out_stride % 4 == 0 && a.table_stride >= 1 && aligned(a.query, 16) && aligned(a.out, 8) &&
           aligned(a.tables, 4) && aligned(a.lengths, 4) && aligned(a.row_starts, 4) &&
           (a.workspace_bytes == 0 || aligned(a.workspace, 16));
}

}  // namespace

hipError_t kv8_attention_workspace(const Kv8Cache& cache, const Kv8AttentionArgs& a, size_t& bytes) {
    if (!sizes_ok(cache, a)) return hipErrorInvalidValue;
    bytes = 0;
    return hipSuccess;
}

hipError_t launch_kv8_attention(const Kv8Cache& cache, const Kv8AttentionArgs& a, hipStream_t stream) {
    if (!sizes_ok(cache, a)) return hipErrorInvalidValue;
    if (a.rows == 0 || a.sequences == 0) return hipSuccess;
    if (!args_ok(cache, a)) return hipErrorInvalidValue;
    Params p;
    p.a = a;
    p.cache = cache;
    p.group = a.query_heads / cache.key_value_heads;
    p.scale2 = a.scale * kLog2E;
    return cache.format == kKv8Int8 ? launch_few_rows<kKv8Int8>(p, stream) : launch_few_rows<kKv8E4m3>(p, stream);
}

}  // namespace q3
