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

#include <algorithm>
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
    int splits = 1;    // workgroups that share a context of few rows
    int columns = 16;  // (row, head of the group) pairs that a shared context can have
    int few = INT_MAX;  // pairs up to which a sequence counts as one of few rows
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

// Workgroups that share the context of a sequence of few rows: 0 where it is
// not one, 1 where its results do not fit the partial ones' place (more rows
// than the caller said).
__device__ __forceinline__ int splits_of(const Params& p, const Rows& r) {
    if (r.count <= 0 || r.count > p.few / p.group) return 0;
    return r.count <= p.columns / p.group ? p.splits : 1;
}
__device__ __forceinline__ size_t partial_slot(const Params& p, int sequence, int kv_head, int column) {
    return ((static_cast<size_t>(sequence) * p.cache.key_value_heads + kv_head) * p.columns + column) * p.splits;
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
    const int kv_head = blockIdx.x, split = blockIdx.y, sequence = blockIdx.z;
    const Rows rows = rows_of(p, sequence);
    const int splits = splits_of(p, rows);
    if (split >= splits) return;
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
        const int share = (steps + splits - 1) / splits;
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
            const size_t slot = partial_slot(p, sequence, kv_head, column) + split;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int d = 2 * wave + j;
                floatx4_t o = *reinterpret_cast<const floatx4_t*>(&out_lds[0][(d * 64 + lane) * 4]);
#pragma unroll
                for (int w = 1; w < kWaves; ++w) o += *reinterpret_cast<const floatx4_t*>(&out_lds[w][(d * 64 + lane) * 4]);
                if (splits == 1) {
                    const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
                    bf16_t* to = p.a.out + static_cast<size_t>(rows.first + row) * p.a.out_stride + head * kDim + 16 * d + 4 * quad;
                    *reinterpret_cast<uint2*>(to) = uint2{pack_bf16(o[0] * inverse, o[1] * inverse), pack_bf16(o[2] * inverse, o[3] * inverse)};
                } else {
                    *reinterpret_cast<floatx4_t*>(p.partial_out + slot * kDim + 16 * d + 4 * quad) = o;
                }
            }
            if (splits > 1 && wave == 0 && quad == 0) p.partial_sums[slot] = float2{top, total};
        }
        __syncthreads();
    }
}

// Joins the results of workgroups that shared a context: a wave a (row, head).
__global__ __launch_bounds__(64 * kWaves) void kv8_join_kernel(Params p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv_head = blockIdx.x, sequence = blockIdx.y;
    const Rows rows = rows_of(p, sequence);
    const int splits = splits_of(p, rows);
    if (splits <= 1) return;
    for (int column = wave; column < rows.count * p.group; column += kWaves) {
        const size_t slot = partial_slot(p, sequence, kv_head, column);
        float top = -INFINITY;
        for (int i = lane; i < splits; i += 64) top = fmaxf(top, p.partial_sums[slot + i].x);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        const float reference = top == -INFINITY ? 0.0f : top;
        float total = 0.0f;
        floatx2_t o{0.f, 0.f};
        for (int i = 0; i < splits; ++i) {
            const float2 part = p.partial_sums[slot + i];
            const float share = __builtin_amdgcn_exp2f(part.x - reference);
            total += part.y * share;
            o += *reinterpret_cast<const floatx2_t*>(p.partial_out + (slot + i) * kDim + 2 * lane) * share;
        }
        const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
        const int row = rows.first + column / p.group, head = kv_head * p.group + column % p.group;
        *reinterpret_cast<unsigned*>(p.a.out + static_cast<size_t>(row) * p.a.out_stride + head * kDim + 2 * lane) =
            pack_bf16(o[0] * inverse, o[1] * inverse);
    }
}

// ---------------------------------------------------------------------------
// Many rows: a wave owns 32 (row, head) pairs of a key/value head as the
// columns of 32x32x16 products, the block's waves share its keys and values,
// which go through LDS as bf16: a byte is converted once for all columns.
// Scores are formed transposed, S^T = K Q^T, with key rows dealt so that a
// lane's scores are those of eight consecutive tokens, the operand of the value
// product O^T = V^T P^T: weights never leave their lane.
// ---------------------------------------------------------------------------
constexpr int kTile = 64;  // tokens in LDS at a time
constexpr int kTileGranules = kTile / kKv8Granule;
// a maximum may stay this far (log2) behind the scores before the sums are scaled anew
constexpr float kSlack = 8.0f;

template <int kFormat, int kPageGranules, int kManyWaves>
__global__ __launch_bounds__(64 * kManyWaves, 2) void kv8_many_rows_kernel(Params p) {
    static_assert(kManyWaves == kTileGranules, "a wave stages a granule");
    __shared__ __align__(16) unsigned char key_lds[2][kTile * kDim * 2];    // [token][16-byte groups of dimensions, swizzled]
    __shared__ __align__(16) unsigned char value_lds[2][kTile * kDim * 2];  // [dimension][16-byte groups of tokens, swizzled]
    __shared__ float key_scale_lds[2][kTileGranules], value_scale_lds[2][kTileGranules];
    __shared__ int held_lds[2][kTileGranules];
    constexpr int kPage = kPageGranules * kKv8Granule;
    constexpr int kColumns = 32 * kManyWaves;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 31, half = lane >> 5;
    const int kv_head = blockIdx.x, sequence = blockIdx.z;
    const Rows rows = rows_of(p, sequence);
    if (rows.count <= 0 || splits_of(p, rows) > 0) return;
    const int* table = p.a.tables + static_cast<size_t>(sequence) * p.a.table_stride;
    const size_t page_bytes = static_cast<size_t>(p.cache.key_value_heads) * (kPageGranules * kKv8GranuleBytes);
    const unsigned char* keys = p.cache.key_pages + kv_head * (kPageGranules * kKv8GranuleBytes) + lane * 16;
    const unsigned char* values = p.cache.value_pages + kv_head * (kPageGranules * kKv8GranuleBytes) + lane * 16;
    const int pairs = rows.count * p.group;
    const int tiles = (pairs + kColumns - 1) / kColumns;

    // the longest rows first: they are the launch's tail
    for (int tile = tiles - 1 - static_cast<int>(blockIdx.y); tile >= 0; tile -= gridDim.y) {
        const int pair = tile * kColumns + wave * 32 + column;
        const bool mine = pair < pairs;
        const int row = min(pair, pairs - 1) / p.group;
        const int head = kv_head * p.group + pair % p.group;
        const int position = rows.position + row;
        const int lowest = p.a.window > 0 ? position - p.a.window : -1;  // tokens above it count
        bf16x8_t q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            uint4 w{0, 0, 0, 0};
            if (mine) {
                w = *reinterpret_cast<const uint4*>(p.a.query + static_cast<size_t>(rows.first + row) * p.a.query_stride +
                                                    head * kDim + 16 * k + 8 * half);
            }
            q[k] = __builtin_bit_cast(bf16x8_t, w);
        }
        // the block's and the wave's positions
        const int first_row = tile * kColumns / p.group;
        const int last_row = min(tile * kColumns + kColumns - 1, pairs - 1) / p.group;
        const int end = min(rows.position + last_row + 1, rows.length);
        const int begin = p.a.window > 0 ? max(rows.position + first_row - p.a.window + 1, 0) & ~(kTile - 1) : 0;
        const int steps = end > begin ? (end - begin + kTile - 1) / kTile : 0;
        const int wave_pair = tile * kColumns + wave * 32;
        const bool wave_lives = wave_pair < pairs;
        const int wave_first = rows.position + min(wave_pair, pairs - 1) / p.group;
        const int wave_last = rows.position + min(wave_pair + 31, pairs - 1) / p.group;

        uint4 k_bytes[2], v_bytes[2];
        float key_scale = 0.f, value_scale = 0.f;
        int held = 0;
        auto load = [&](int step) {
            const int first = begin + step * kTile + wave * kKv8Granule;
            const int at = min(first, (end - 1) & ~(kKv8Granule - 1));
            int page = table[at / kPage];
            held = min(max(end - first, 0), kKv8Granule);
            if (page < 0 || page >= p.cache.pages) page = 0, held = 0;
            const size_t offset = page * page_bytes + at % kPage / kKv8Granule * kKv8GranuleBytes;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                k_bytes[c] = *reinterpret_cast<const uint4*>(keys + offset + c * 1024);
                v_bytes[c] = *reinterpret_cast<const uint4*>(values + offset + c * 1024);
            }
            const size_t scale_at = static_cast<size_t>(page) * p.cache.key_value_heads + kv_head;
            key_scale = p.cache.key_scales[scale_at] * p.scale2;
            value_scale = p.cache.value_scales[scale_at];
        };
        auto stage = [&](int buffer) {
            // keys: lane (token, 16-dimension group): two 16-byte groups of bf16 for each half of the dimensions
            const int token = wave * kKv8Granule + (lane >> 2);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint2 a = bf16_of<kFormat>(k_bytes[c].x), b = bf16_of<kFormat>(k_bytes[c].y);
                const uint2 d = bf16_of<kFormat>(k_bytes[c].z), e = bf16_of<kFormat>(k_bytes[c].w);
                const int group = 8 * c + 2 * (lane & 3);
                *reinterpret_cast<uint4*>(&key_lds[buffer][token * 256 + (group ^ (token & 15)) * 16]) = uint4{a.x, a.y, b.x, b.y};
                *reinterpret_cast<uint4*>(&key_lds[buffer][token * 256 + ((group + 1) ^ (token & 15)) * 16]) = uint4{d.x, d.y, e.x, e.y};
            }
            // values: lane (token / 4, d % 16): four tokens of dimensions 64 c + 16 t + d % 16
            const unsigned mask = byte_mask(4 * (lane >> 4), 0, held);
            const int place = 2 * wave + (lane >> 5);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const unsigned w[4] = {v_bytes[c].x, v_bytes[c].y, v_bytes[c].z, v_bytes[c].w};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int d = 64 * c + 16 * t + (lane & 15);
                    *reinterpret_cast<uint2*>(&value_lds[buffer][d * 128 + (place ^ (d >> 1 & 7)) * 16 + (lane >> 4 & 1) * 8]) =
                        bf16_of<kFormat>(w[t] & mask);
                }
            }
            if (lane == 0) {
                key_scale_lds[buffer][wave] = held > 0 ? key_scale : 0.0f;
                value_scale_lds[buffer][wave] = held > 0 ? value_scale : 0.0f;
                held_lds[buffer][wave] = held;
            }
        };

        float maximum = -INFINITY, sum = 0.0f;
        floatx16_t acc[4];
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
        if (steps > 0) load(0);
        for (int step = 0; step < steps; ++step) {
            const int buffer = step & 1;
            stage(buffer);
            if (step + 1 < steps) load(step + 1);
            __syncthreads();
            const int token0 = begin + step * kTile;
            if (!wave_lives || token0 > wave_last || (p.a.window > 0 && token0 + kTile - 1 <= wave_first - p.a.window)) continue;
            // row i of a 32-token tile is token i with bits 2 and 3 exchanged
            const int token = (column & 19) | (column & 4) << 1 | (column & 8) >> 1;
            floatx16_t s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
                const unsigned char* from = &key_lds[buffer][(32 * t + token) * 256];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const bf16x8_t a = *reinterpret_cast<const bf16x8_t*>(from + ((2 * k + half) ^ (token & 15)) * 16);
                    s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[k], s[t], 0, 0, 0);
                }
            }
            float factor[kTileGranules], value_factor[kTileGranules];
            bool whole = token0 + kTile - 1 <= wave_first && (p.a.window == 0 || token0 > wave_last - p.a.window);
#pragma unroll
            for (int g = 0; g < kTileGranules; ++g) {
                factor[g] = key_scale_lds[buffer][g];
                value_factor[g] = value_scale_lds[buffer][g];
                whole &= held_lds[buffer][g] == kKv8Granule;
            }
            // s[t][i]: token 32 t + 16 (i / 8) + 8 half + i % 8
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] *= factor[2 * t + (i >> 3)];
            if (!__builtin_amdgcn_readfirstlane(whole)) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int of_granule = 8 * half + (i & 7);
                        const int at = token0 + 32 * t + 16 * (i >> 3) + of_granule;
                        const bool counts = at <= position && at > lowest && of_granule < held_lds[buffer][2 * t + (i >> 3)];
                        s[t][i] = counts ? s[t][i] : -INFINITY;
                    }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > maximum + kSlack)) {
                const float next = fmaxf(maximum, top);
                const float shrink = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(maximum - next);
                maximum = next;
                sum *= shrink;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= shrink;
            }
            const float reference = maximum == -INFINITY ? 0.0f : maximum;
            bf16x8_t weights[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                unsigned w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = __builtin_amdgcn_exp2f(s[g >> 1][8 * (g & 1) + 2 * i] - reference);
                    const float b = __builtin_amdgcn_exp2f(s[g >> 1][8 * (g & 1) + 2 * i + 1] - reference);
                    sum += a + b;
                    w[i] = pack_bf16(a * value_factor[g], b * value_factor[g]);
                }
                weights[g] = __builtin_bit_cast(bf16x8_t, uint4{w[0], w[1], w[2], w[3]});
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int dimension = 32 * d + column;
                const unsigned char* from = &value_lds[buffer][dimension * 128];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const bf16x8_t a = *reinterpret_cast<const bf16x8_t*>(from + ((2 * g + half) ^ (dimension >> 1 & 7)) * 16);
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, weights[g], acc[d], 0, 0, 0);
                }
            }
        }
        __syncthreads();  // the next tile of rows stages into the buffers
        sum += __shfl_xor(sum, 32, 64);
        if (mine) {
            const float inverse = sum > 0.0f ? 1.0f / sum : 0.0f;
            bf16_t* to = p.a.out + static_cast<size_t>(rows.first + row) * p.a.out_stride + head * kDim + 4 * half;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    *reinterpret_cast<uint2*>(to + 32 * d + 8 * i) =
                        uint2{pack_bf16(acc[d][4 * i] * inverse, acc[d][4 * i + 1] * inverse),
                              pack_bf16(acc[d][4 * i + 2] * inverse, acc[d][4 * i + 3] * inverse)};
                }
        }
    }
}

template <int kFormat, int kPageGranules>
hipError_t launch_pages(const Params& p, hipStream_t stream) {
    const bool many = p.few != INT_MAX;
    if (!many || p.a.sequences > 1) {
        kv8_few_rows_kernel<kFormat, kPageGranules>
            <<<dim3(p.cache.key_value_heads, p.splits, p.a.sequences), 64 * kWaves, 0, stream>>>(p);
        if (p.splits > 1) {
            kv8_join_kernel<<<dim3(p.cache.key_value_heads, p.a.sequences), 64 * kWaves, 0, stream>>>(p);
        }
    }
    if (many) {
        const int pairs = std::min(p.a.max_rows, p.a.rows) * p.group;
        const int tiles = (pairs + 127) / 128;
        kv8_many_rows_kernel<kFormat, kPageGranules, 4>
            <<<dim3(p.cache.key_value_heads, std::min(tiles, 65535), p.a.sequences), 256, 0, stream>>>(p);
    }
    return hipGetLastError();
}

template <int kFormat>
hipError_t launch_format(const Params& p, hipStream_t stream) {
    switch (p.cache.page_tokens) {
        case 16: return launch_pages<kFormat, 1>(p, stream);
        case 32: return launch_pages<kFormat, 2>(p, stream);
        default: return launch_pages<kFormat, 4>(p, stream);
    }
}

// How a call's work is dealt out.
struct Dealt {
    bool many;    // sequences of many rows may be among them
    int columns;  // as in Params
    int splits;
};
constexpr int kBytesOfPartial = (kDim + 2) * 4;
Dealt dealt_of(const Kv8Cache& cache, const Kv8AttentionArgs& a, size_t workspace_bytes) {
    Dealt d;
    const int group = a.query_heads / cache.key_value_heads;
    const int rows = std::max(1, std::min(a.max_rows, a.rows));
    d.many = static_cast<long long>(rows) * group > 16;
    d.columns = std::min(16 / group, rows) * group;
    // Contexts are shared until two workgroups a CU are there, each with a step for every wave
    const long long blocks = static_cast<long long>(std::max(a.sequences, 1)) * cache.key_value_heads;
    const int reach = a.window > 0 ? std::min(a.window + rows, a.max_length) : a.max_length;
    const long long wanted = std::min<long long>((512 + blocks - 1) / blocks, (reach + kWaves * kStep - 1) / (kWaves * kStep));
    const long long fits = static_cast<long long>(workspace_bytes / (static_cast<size_t>(blocks) * d.columns * kBytesOfPartial));
    d.splits = static_cast<int>(std::max<long long>(1, std::min<long long>({wanted, fits, 64})));
    if (d.many && a.sequences == 1) d.splits = 1;  // one prompt: no sequence of few rows
    return d;
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
    const Dealt d = dealt_of(cache, a, SIZE_MAX);
    bytes = d.splits == 1 ? 0 : static_cast<size_t>(a.sequences) * cache.key_value_heads * d.columns * d.splits * kBytesOfPartial;
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
    const Dealt d = dealt_of(cache, a, a.workspace_bytes);
    p.columns = d.columns;
    p.splits = d.splits;
    p.few = !d.many ? INT_MAX : a.sequences > 1 ? 16 : 0;
    const size_t slots = static_cast<size_t>(a.sequences) * cache.key_value_heads * d.columns * d.splits;
    p.partial_out = a.workspace;
    p.partial_sums = reinterpret_cast<float2*>(a.workspace + slots * kDim);
    return cache.format == kKv8Int8 ? launch_format<kKv8Int8>(p, stream) : launch_format<kKv8E4m3>(p, stream);
}

}  // namespace q3
