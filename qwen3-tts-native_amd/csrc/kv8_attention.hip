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

constexpr int kFewWaves = 4;
constexpr int kStep = 64;  // tokens of a step of its waves
constexpr int kMostSplits = 64;
// Workgroups for sequences of many rows: column waves x key groups of 4 x 1, 4 x 2, 2 x 4.
enum Many : int { kNone = 0, kWide, kHalved, kQuartered };

struct Params {
    Kv8AttentionArgs a;
    Kv8Cache cache;
    int group = 1;     // query heads of a key/value head
    float scale2 = 0;  // |scale| * log2(e)
    unsigned flip = 0;  // sign bits of a pair of bf16: the query's are flipped for a negative scale
    int splits = 1;    // workgroups that share a context of few rows, where it has few_tiles tiles
    int columns = 16;  // (row, head of the group) pairs that a shared context can have
    int waves = kFewWaves;  // of a workgroup of few rows
    int many = kNone;
    int few = INT_MAX;  // pairs up to which a sequence counts as one of few rows
    int few_rows = 0, shared_rows = 0, tile_rows = 0;  // rows of `few`, `columns` and 16 pairs
    int few_tiles = 1;  // workgroups among which the tiles of its rows are dealt
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

// a / b for 0 <= a < 2^20, b > 0: the reciprocal's error times a / b is far below the
// 0.5 / b to the next whole number.  Integer divisions' chains cost 0.4 us a call.
__device__ __forceinline__ int quotient(int a, int b) {
    return static_cast<int>((static_cast<float>(a) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(b)));
}
// How a sequence of few rows is dealt to its workgroups: `tiles` of them take its
// tiles in turn, `splits` of those share their context.  No splits where it is none
// of few rows, one where its results do not fit the partial ones' place (more
// rows than the caller said).  A sequence of fewer tiles than the largest leaves
// workgroups over: they take shares, of a step of every wave at least (a token
// over 4000 where 256 rows may come 39 us without, 10.8 with; four sequences 59 / 22).
struct Shares {
    int tiles, splits;
};
__device__ __forceinline__ Shares shares_of(const Params& p, const Rows& r) {
    if (r.count <= 0 || r.count > p.few_rows) return Shares{1, 0};
    if (r.count > p.shared_rows) return Shares{p.few_tiles, 1};
    if (p.few_tiles == 1 || p.splits == 1) return Shares{p.few_tiles, p.splits};
    const int tiles = quotient(r.count + p.tile_rows - 1, p.tile_rows);
    const int reach = p.a.window > 0 ? static_cast<int>(min(static_cast<long long>(p.a.window) + r.count, static_cast<long long>(r.length))) : r.length;
    const int steps = (reach + kFewWaves * kStep - 1ll) / (kFewWaves * kStep);
    return Shares{tiles, max(1, min(min(quotient(p.splits * p.few_tiles, tiles), kMostSplits), steps))};
}
// A split's place among a column's is its number; columns are `splits` apart.
__device__ __forceinline__ size_t partial_slot(const Params& p, int sequence, int kv_head, int column, int splits) {
    return (static_cast<size_t>(sequence) * p.cache.key_value_heads + kv_head) * p.columns * p.splits + static_cast<size_t>(column) * splits;
}

// Pages and scales of a wave's next 64 granules, one a lane, so that no step
// waits for its table entry, then for its scales, before it can ask for bytes.
struct Lookup {
    int page;  // -1: none
    float key_scale, value_scale;
};
// `token` is the first of the lane's granule; tokens [low, end) are those that
// any of the rows attends to.  Nothing else of a sequence is looked at as a
// number: pages in front of a window may have been given to others.
template <int kPage>
__device__ __forceinline__ Lookup look_up(const Params& p, const int* table, int kv_head, int token, int low, int end) {
    const int at = min(token, (end - 1) & ~(kKv8Granule - 1));  // past the end: the last one again
    int page = table[at / kPage];
    if (page < 0 || page >= p.cache.pages) page = -1;
    const size_t scale_at = static_cast<size_t>(max(page, 0)) * p.cache.key_value_heads + kv_head;
    const bool counts = page >= 0 && token < end && token + kKv8Granule > low;
    return Lookup{page, counts ? p.cache.key_scales[scale_at] * p.scale2 : 0.0f, counts ? p.cache.value_scales[scale_at] : 0.0f};
}
__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float of_lane(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// ---------------------------------------------------------------------------
// Few rows: a tile of up to 16 (row, head) pairs of one key/value head is the columns
// of 16x16x32 products, keys and values are read once for all of them.  Nothing
// goes through LDS before the end: a lane's 16 bytes of keys are two operands'
// rows, its scores' four tokens are those of its four bytes of each dimension.
// A wave's weights are two bf16, the second what the first leaves, so that
// outputs carry no other rounding than their own; the products have room for it.
// Bound by HBM where the batch is large (256 sequences of 1111..8192 tokens,
// int8, 16 / 8 heads: 446 us, 5.5 TB/s; 64 of 33..4096, e4m3: 60 us, 4.5 TB/s, the
// longest ones' tail; one of 65521: 33 us, 4.1 TB/s), below by the chain
// table -> bytes -> products (eight of 97..1024 tokens: 9 us with the join).
// Rows of short prompts, and some rows over a long context, are tiles in
// workgroups of their own (one prompt of 801: 20 us; 32 over 16000 tokens: 28).
// ---------------------------------------------------------------------------
constexpr int kStepGranules = kStep / kKv8Granule;

template <int kWaves>
struct FewShared {
    __align__(16) float out[kWaves][8 * 64 * 4];
    float maximum[kWaves][16], sum[kWaves][16];
};

template <int kFormat, int kPageGranules, int kWaves>
__device__ __forceinline__ void few_rows(const Params& p, FewShared<kWaves>& lds, int share) {
    auto& out_lds = lds.out;
    auto& max_lds = lds.maximum;
    auto& sum_lds = lds.sum;
    constexpr int kPage = kPageGranules * kKv8Granule;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, quad = lane >> 4;
    const int kv_head = blockIdx.x, sequence = blockIdx.z;
    const Rows rows = rows_of(p, sequence);
    const auto [tiles, splits] = shares_of(p, rows);
    const int split = quotient(share, tiles);
    const int first_tile = tiles - 1 - (share - split * tiles);  // a prompt's longest first
    if (split >= splits) return;
    const int rows_per_tile = p.tile_rows;
    const int head = kv_head * p.group + column % p.group;
    const int* table = p.a.tables + static_cast<size_t>(sequence) * p.a.table_stride;
    const size_t page_bytes = static_cast<size_t>(p.cache.key_value_heads) * (kPageGranules * kKv8GranuleBytes);
    const unsigned char* values = p.cache.value_pages + kv_head * (kPageGranules * kKv8GranuleBytes) + lane * 16;
    // lane (token, 16-dimension group) of the keys: byte token * 64 + group * 16
    const unsigned char* keys_of_lane = p.cache.key_pages + kv_head * (kPageGranules * kKv8GranuleBytes) +
                                        (lane & 15) * 64 + quad * 16;

    for (int tile = first_tile * rows_per_tile; tile < rows.count; tile += tiles * rows_per_tile) {
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
                    w = uint4{w.x ^ p.flip, w.y ^ p.flip, w.z ^ p.flip, w.w ^ p.flip};
                }
                q[c][u] = __builtin_bit_cast(bf16x8_t, w);
            }
        // tokens [begin, end) of this tile's rows, in steps dealt to the splits, then to the waves
        const int last = min(tile + rows_per_tile, rows.count) - 1;
        const int end = min(rows.position + last + 1, rows.length);
        const int low = p.a.window > 0 ? max(rows.position + tile - p.a.window + 1, 0) : 0;
        const int begin = low & ~(kStep - 1);
        const int steps = end > begin ? (end - begin + kStep - 1) / kStep : 0;
        const int steps_each = (steps + splits - 1) / splits;
        const int steps_begin = split * steps_each, steps_end = min(steps_begin + steps_each, steps);
        const int lowest = p.a.window > 0 ? position - p.a.window : -1;  // tokens above it count

        float maximum = -INFINITY, sum = 0.0f;
        floatx4_t acc[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        // the wave's i-th step and its granules; their bytes are asked for as
        // soon as the registers of the step before are free
        const int mine_steps = steps_end > steps_begin + wave ? (steps_end - steps_begin - wave + kWaves - 1) / kWaves : 0;
        constexpr int kLooked = 64 / kStepGranules;  // steps of a look-up
        const auto token_of = [&](int i) { return begin + (steps_begin + wave + i * kWaves) * kStep; };
        uint4 k[kStepGranules][2], v[kStepGranules][2];
        Lookup looked{};
        const auto look = [&](int i) {
            looked = look_up<kPage>(p, table, kv_head, token_of(i + lane / kStepGranules) + lane % kStepGranules * kKv8Granule, low, end);
        };
        const auto offset_of = [&](int i, int g) {
            const int page = max(of_lane(looked.page, i % kLooked * kStepGranules + g), 0);
            const int at = min(token_of(i) + g * kKv8Granule, (end - 1) & ~(kKv8Granule - 1));
            return page * page_bytes + at % kPage / kKv8Granule * kKv8GranuleBytes;
        };
        const auto load = [&](uint4 (&to)[kStepGranules][2], const unsigned char* from, int i) {
#pragma unroll
            for (int g = 0; g < kStepGranules; ++g) {
                const unsigned char* at = from + offset_of(i, g);
#pragma unroll
                for (int c = 0; c < 2; ++c) to[g][c] = *reinterpret_cast<const uint4*>(at + c * 1024);
            }
        };
        if (mine_steps > 0) {
            look(0);
            load(k, keys_of_lane, 0);
            load(v, values, 0);
        }
        for (int i = 0; i < mine_steps; ++i) {
            const int token0 = token_of(i);
            float key_scale[kStepGranules], value_scale[kStepGranules];
            int held[kStepGranules];  // tokens of the granule that hold something
#pragma unroll
            for (int g = 0; g < kStepGranules; ++g) {
                const int from = i % kLooked * kStepGranules + g;
                key_scale[g] = of_lane(looked.key_scale, from);
                value_scale[g] = of_lane(looked.value_scale, from);
                held[g] = of_lane(looked.page, from) < 0 ? 0 : min(max(end - token0 - g * kKv8Granule, 0), kKv8Granule);
            }
            const bool more = i + 1 < mine_steps;
            if (more && (i + 1) % kLooked == 0) look(i + 1);
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
                for (int e = 0; e < 4; ++e) {
                    const int token = first + e;
                    const bool counts = token <= position && token > lowest && 4 * quad + e < held[g];
                    s[g][e] = counts ? dot[e] * key_scale[g] : -INFINITY;
                    top = fmaxf(top, s[g][e]);
                }
            }
            if (more) load(k, keys_of_lane, i + 1);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float reference = top == -INFINITY ? 0.0f : top;  // nothing counted yet: weights become 0
            const float shrink = __builtin_amdgcn_exp2f(maximum - reference);
            maximum = top;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[d] *= shrink;
            // weights times the values' scale as two bf16, the second what the first leaves: 16 bits of them
            unsigned high[kStepGranules][2], rest[kStepGranules][2];
#pragma unroll
            for (int g = 0; g < kStepGranules; ++g) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = __builtin_amdgcn_exp2f(s[g][e] - reference);
                    sum += weight;
                    w[e] = weight * value_scale[g];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    high[g][e] = pack_bf16(w[2 * e], w[2 * e + 1]);
                    rest[g][e] = pack_bf16(w[2 * e] - __uint_as_float(high[g][e] << 16),
                                           w[2 * e + 1] - __uint_as_float(high[g][e] & 0xffff0000u));
                }
                const int skipped = low - token0 - g * kKv8Granule;
                if (held[g] < kKv8Granule || skipped > 0) {
                    // bytes that do not count may hold anything, an e4m3 NaN too, which a zero weight would not silence
                    const unsigned mask = byte_mask(4 * quad, skipped, held[g]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) v[g][c] = uint4{v[g][c].x & mask, v[g][c].y & mask, v[g][c].z & mask, v[g][c].w & mask};
                }
            }
#pragma unroll
            for (int g = 0; g < kStepGranules; g += 2) {
                const bf16x8_t ph = __builtin_bit_cast(bf16x8_t, uint4{high[g][0], high[g][1], high[g + 1][0], high[g + 1][1]});
                const bf16x8_t pl = __builtin_bit_cast(bf16x8_t, uint4{rest[g][0], rest[g][1], rest[g + 1][0], rest[g + 1][1]});
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
            if (more) load(v, values, i + 1);
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
        // wave w: dimension tiles of 16, every column
        if (mine) {
            const size_t slot = partial_slot(p, sequence, kv_head, tile * p.group + column, splits) + split;
#pragma unroll
            for (int j = 0; j < 8 / kWaves; ++j) {
                const int d = 8 / kWaves * wave + j;
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

// Two waves a SIMD: with registers for three (168) the compiler spills, and
// 256 sequences up to 8192 tokens take 601 us instead of 445.
template <int kFormat, int kPageGranules, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_few_rows_kernel(Params p) {
    __shared__ FewShared<kWaves> lds;
    few_rows<kFormat, kPageGranules, kWaves>(p, lds, blockIdx.y);
}

// Joins the results of workgroups that shared a context: a workgroup a (row,
// head), its 8 groups of 32 lanes take every eighth of the partial results
// (one wave for all of them: 18 us for 64 of a row, now 4).
constexpr int kJoinGroups = 8;
__global__ __launch_bounds__(32 * kJoinGroups) void kv8_join_kernel(Params p) {
    __shared__ float max_lds[kJoinGroups], sum_lds[kJoinGroups];
    __shared__ __align__(16) float out_lds[kJoinGroups][kDim];
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const int column = blockIdx.x, kv_head = blockIdx.y, sequence = blockIdx.z;
    const Rows rows = rows_of(p, sequence);
    const int splits = shares_of(p, rows).splits;
    if (splits <= 1 || column >= rows.count * p.group) return;
    const size_t slot = partial_slot(p, sequence, kv_head, column, splits);
    float top = -INFINITY, total = 0.0f;
    floatx4_t o{0.f, 0.f, 0.f, 0.f};
    for (int i = group; i < splits; i += kJoinGroups) {
        const float2 part = p.partial_sums[slot + i];
        const floatx4_t values = *reinterpret_cast<const floatx4_t*>(p.partial_out + (slot + i) * kDim + 4 * lane);
        const float next = fmaxf(top, part.x), reference = next == -INFINITY ? 0.0f : next;
        const float shrink = __builtin_amdgcn_exp2f(top - reference), share = __builtin_amdgcn_exp2f(part.x - reference);
        total = total * shrink + part.y * share;
        o = o * shrink + values * share;
        top = next;
    }
    if (lane == 0) max_lds[group] = top, sum_lds[group] = total;
    *reinterpret_cast<floatx4_t*>(&out_lds[group][4 * lane]) = o;
    __syncthreads();
    if (threadIdx.x >= kDim / 2) return;
    top = max_lds[0];
#pragma unroll
    for (int g = 1; g < kJoinGroups; ++g) top = fmaxf(top, max_lds[g]);
    const float reference = top == -INFINITY ? 0.0f : top;
    floatx2_t sums{0.f, 0.f};
    total = 0.0f;
#pragma unroll
    for (int g = 0; g < kJoinGroups; ++g) {
        const float share = __builtin_amdgcn_exp2f(max_lds[g] - reference);
        total += sum_lds[g] * share;
        sums += *reinterpret_cast<const floatx2_t*>(&out_lds[g][2 * threadIdx.x]) * share;
    }
    const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
    const int row = rows.first + column / p.group, head = kv_head * p.group + column % p.group;
    *reinterpret_cast<unsigned*>(p.a.out + static_cast<size_t>(row) * p.a.out_stride + head * kDim + 2 * threadIdx.x) =
        pack_bf16(sums[0] * inverse, sums[1] * inverse);
}

// ---------------------------------------------------------------------------
// Many rows: a wave owns 32 (row, head) pairs of a key/value head as the
// columns of 32x32x16 products; the block's waves share its keys and values,
// which go through LDS as bf16: a byte is converted once for all columns.
// Scores are formed transposed, S^T = K Q^T, with key rows dealt so that a
// lane's scores are those of eight consecutive tokens, the operand of the value
// product O^T = V^T P^T: weights never leave their lane.
// Waves are kColumnWaves x kKeyWaves: those of a key group take the same 64 of
// every 64 * kKeyWaves tokens, and the groups' results are joined at the end.
// Prompts of 1777..4096 rows, 32 / 8 heads: 361 us, 850 TFLOP/s (the library's
// large product reaches 1213); one of 1024 rows, 16 / 8 heads: 24 us, latency.
// Two waves a SIMD share the matrix cores (40 % of a busy CU's time), the vector
// unit (52 %) and LDS (40 %), none of them full: leaving out the exponentials, the
// value products, the staging or the loads saves 6 to 12 % each.
// ---------------------------------------------------------------------------
constexpr int kTile = 64;  // tokens of a wave's step
constexpr int kTileGranules = kTile / kKv8Granule;
// Rows of a tile in LDS, as bf16: 16 bytes of padding put the rows that 16 lanes
// read at once in different banks, and leave one address for all of a lane's reads.
constexpr int kKeyRow = kDim * 2 + 16, kValueRow = kTile * 2 + 16;
// a maximum may stay this far (log2) behind the scores before the sums are scaled anew
constexpr float kSlack = 8.0f;
// Smallest value scale that goes into the weights as it is, see stage().
constexpr float kLeastScale = 0x1p-60f;

// Four held values times `factor` as bf16.
template <int kFormat>
__device__ __forceinline__ uint2 scaled_bf16_of(unsigned w, float factor) {
    const uint2 v = bf16_of<kFormat>(w);
    return uint2{pack_bf16(__uint_as_float(v.x << 16) * factor, __uint_as_float(v.x & 0xffff0000u) * factor),
                 pack_bf16(__uint_as_float(v.y << 16) * factor, __uint_as_float(v.y & 0xffff0000u) * factor)};
}

// What a step has to know of a granule: the keys' scale times the scores', log2
// of the values' scale and its reciprocal, tokens that hold something.
struct __align__(16) Granule {
    float key_scale, value_log, value_inverse;
    int held;
};

template <int kColumnWaves, int kKeyWaves>
struct ManyShared {
    static constexpr int kBuffers = kKeyWaves == 1 ? 2 : 1;
    unsigned char keys[kBuffers][kKeyWaves][kTile * kKeyRow];    // [token][dimension]
    unsigned char values[kBuffers][kKeyWaves][kDim * kValueRow];  // [dimension][token]
    Granule granules[kBuffers][kKeyWaves][kTileGranules];
    float maximum[kKeyWaves][kColumnWaves][32], sum[kKeyWaves][kColumnWaves][32];
};

template <int kFormat, int kPageGranules, int kColumnWaves, int kKeyWaves>
__device__ __forceinline__ void many_rows(const Params& p, unsigned char* dynamic_lds, int first_tile, int tiles_apart) {
    using Shared = ManyShared<kColumnWaves, kKeyWaves>;
    Shared& lds = *reinterpret_cast<Shared*>(dynamic_lds);
    constexpr int kBuffers = Shared::kBuffers;
    constexpr int kPage = kPageGranules * kKv8Granule;
    constexpr int kColumns = 32 * kColumnWaves;
    constexpr int kStepTokens = kTile * kKeyWaves;
    constexpr int kStaged = kTileGranules / kColumnWaves;  // granules that a wave stages
    static_assert(kStaged * kColumnWaves == kTileGranules, "column waves stage a tile's granules");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column_wave = wave % kColumnWaves, key_wave = wave / kColumnWaves;
    const int column = lane & 31, half = lane >> 5;
    const int kv_head = blockIdx.x, sequence = blockIdx.z;
    const Rows rows = rows_of(p, sequence);
    if (rows.count <= 0 || shares_of(p, rows).splits > 0) return;
    const int* table = p.a.tables + static_cast<size_t>(sequence) * p.a.table_stride;
    const size_t page_bytes = static_cast<size_t>(p.cache.key_value_heads) * (kPageGranules * kKv8GranuleBytes);
    const unsigned char* keys = p.cache.key_pages + kv_head * (kPageGranules * kKv8GranuleBytes) + lane * 16;
    const unsigned char* values = p.cache.value_pages + kv_head * (kPageGranules * kKv8GranuleBytes) + lane * 16;
    const int pairs = rows.count * p.group;
    const int tiles = (pairs + kColumns - 1) / kColumns;

    // the longest rows first: they are the launch's tail
    for (int tile = tiles - 1 - first_tile; tile >= 0; tile -= tiles_apart) {
        const int pair = tile * kColumns + column_wave * 32 + column;
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
                w = uint4{w.x ^ p.flip, w.y ^ p.flip, w.z ^ p.flip, w.w ^ p.flip};
            }
            q[k] = __builtin_bit_cast(bf16x8_t, w);
        }
        // the block's and the wave's positions
        const int first_row = tile * kColumns / p.group;
        const int last_row = min(tile * kColumns + kColumns - 1, pairs - 1) / p.group;
        const int end = min(rows.position + last_row + 1, rows.length);
        const int low = p.a.window > 0 ? max(rows.position + first_row - p.a.window + 1, 0) : 0;
        const int begin = low & ~(kTile - 1);
        const int steps = end > begin ? (end - begin + kStepTokens - 1) / kStepTokens : 0;
        const int wave_pair = tile * kColumns + column_wave * 32;
        const bool wave_lives = wave_pair < pairs;
        const int wave_first = rows.position + min(wave_pair, pairs - 1) / p.group;
        const int wave_last = rows.position + min(wave_pair + 31, pairs - 1) / p.group;

        uint4 k_bytes[kStaged][2], v_bytes[kStaged][2];
        Granule staged[kStaged];
        float value_scale[kStaged];
        int skipped[kStaged];  // tokens of the granule in front of every row's window
        constexpr int kLooked = 64 / kStaged;  // steps of a look-up
        const auto token_of = [&](int step, int j) {
            return begin + step * kStepTokens + key_wave * kTile + (column_wave * kStaged + j) * kKv8Granule;
        };
        Lookup looked{};
        float looked_log = 0.0f, looked_inverse = 1.0f;
        auto load = [&](int step) {
            if (step % kLooked == 0) {
                looked = look_up<kPage>(p, table, kv_head, token_of(step + lane / kStaged, lane % kStaged), low, end);
                // Values' scale goes into the weights as a power, 2^(score + log2 scale); below kLeastScale the values
                // take the rest of it, so that a page of tiny values does not push its weights, which the sum
                // needs, out of fp32.
                const float kept = fmaxf(looked.value_scale, kLeastScale);
                looked_log = __builtin_amdgcn_logf(kept);
                looked_inverse = 1.0f / kept;
            }
#pragma unroll
            for (int j = 0; j < kStaged; ++j) {
                const int from = step % kLooked * kStaged + j, first = token_of(step, j);
                const int page = of_lane(looked.page, from);
                const int at = min(first, (end - 1) & ~(kKv8Granule - 1));
                const size_t offset = max(page, 0) * page_bytes + at % kPage / kKv8Granule * kKv8GranuleBytes;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    k_bytes[j][c] = *reinterpret_cast<const uint4*>(keys + offset + c * 1024);
                    v_bytes[j][c] = *reinterpret_cast<const uint4*>(values + offset + c * 1024);
                }
                staged[j] = Granule{of_lane(looked.key_scale, from), of_lane(looked_log, from), of_lane(looked_inverse, from),
                                    page < 0 ? 0 : min(max(end - first, 0), kKv8Granule)};
                value_scale[j] = of_lane(looked.value_scale, from);
                skipped[j] = low - first;
            }
        };
        auto stage = [&](int buffer) {
#pragma unroll
            for (int j = 0; j < kStaged; ++j) {
                const int granule = column_wave * kStaged + j;
                // keys: lane (token, 16-dimension group): two 16-byte groups of bf16 for each half of the dimensions
                const int token = lane >> 2;
                unsigned char* to = &lds.keys[buffer][key_wave][(granule * kKv8Granule + token) * kKeyRow + (lane & 3) * 32];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint2 a = bf16_of<kFormat>(k_bytes[j][c].x), b = bf16_of<kFormat>(k_bytes[j][c].y);
                    const uint2 d = bf16_of<kFormat>(k_bytes[j][c].z), e = bf16_of<kFormat>(k_bytes[j][c].w);
                    *reinterpret_cast<uint4*>(to + c * 128) = uint4{a.x, a.y, b.x, b.y};
                    *reinterpret_cast<uint4*>(to + c * 128 + 16) = uint4{d.x, d.y, e.x, e.y};
                }
                // values: lane (token / 4, d % 16): four tokens of dimensions 64 c + 16 t + d % 16
                unsigned char* values_to = &lds.values[buffer][key_wave][(lane & 15) * kValueRow + granule * 32 + (lane >> 4) * 8];
                unsigned mask = 0xffffffffu;
                if (staged[j].held < kKv8Granule || skipped[j] > 0) mask = byte_mask(4 * (lane >> 4), skipped[j], staged[j].held);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const unsigned w[4] = {v_bytes[j][c].x, v_bytes[j][c].y, v_bytes[j][c].z, v_bytes[j][c].w};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        *reinterpret_cast<uint2*>(values_to + (64 * c + 16 * t) * kValueRow) = bf16_of<kFormat>(w[t] & mask);
                    }
                }
                if (value_scale[j] < kLeastScale) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const unsigned w[4] = {v_bytes[j][c].x, v_bytes[j][c].y, v_bytes[j][c].z, v_bytes[j][c].w};
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            *reinterpret_cast<uint2*>(values_to + (64 * c + 16 * t) * kValueRow) =
                                scaled_bf16_of<kFormat>(w[t] & mask, value_scale[j] * (1.0f / kLeastScale));
                        }
                    }
                }
                if (lane == 0) lds.granules[buffer][key_wave][granule] = staged[j];
            }
        };

        float maximum = -INFINITY, sum = 0.0f;
        floatx16_t acc[4];
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
        // row i of a 32-token tile is token i with bits 2 and 3 exchanged
        const int key_row = (column & 19) | (column & 4) << 1 | (column & 8) >> 1;
        auto compute = [&](int buffer, int token0) {
            const unsigned char* keys_from = &lds.keys[buffer][key_wave][key_row * kKeyRow + half * 16];
            const unsigned char* values_from = &lds.values[buffer][key_wave][column * kValueRow + half * 16];
            bf16x8_t fragment[16];
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int t = 0; t < 2; ++t) fragment[2 * k + t] = *reinterpret_cast<const bf16x8_t*>(keys_from + 32 * t * kKeyRow + 32 * k);
            floatx16_t s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fragment[2 * k + t], q[k], s[t], 0, 0, 0);
            bf16x8_t value[16];
#pragma unroll
            for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) value[4 * d + g] = *reinterpret_cast<const bf16x8_t*>(values_from + 32 * d * kValueRow + 32 * g);
            Granule of[kTileGranules];
            bool whole = token0 + kTile - 1 <= wave_first && (p.a.window == 0 || token0 > wave_last - p.a.window);
#pragma unroll
            for (int g = 0; g < kTileGranules; ++g) {
                of[g] = lds.granules[buffer][key_wave][g];
                whole &= of[g].held == kKv8Granule;
            }
            // s[t][i]: token 32 t + 16 (i / 8) + 8 half + i % 8, in units of its granule's scale
            if (!__builtin_amdgcn_readfirstlane(whole)) {
                // kept a branch: the compiler would fold its 160 operations into every step
                asm volatile("");
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int of_granule = 8 * half + (i & 7);
                        const int at = token0 + 32 * t + 16 * (i >> 3) + of_granule;
                        const bool counts = at <= position && at > lowest && of_granule < of[2 * t + (i >> 3)].held;
                        s[t][i] = counts ? s[t][i] : -INFINITY;
                    }
#pragma unroll
                for (int g = 0; g < kTileGranules; ++g) {
                    // -infinity stays what it is: 0 * -infinity would not
                    of[g].key_scale = fmaxf(of[g].key_scale, 0x1p-126f);
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int g = 0; g < kTileGranules; ++g) {
                float most = s[g >> 1][8 * (g & 1)];
#pragma unroll
                for (int i = 1; i < 8; ++i) most = fmaxf(most, s[g >> 1][8 * (g & 1) + i]);
                top = fmaxf(top, most * of[g].key_scale);
            }
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
            for (int g = 0; g < kTileGranules; ++g) {
                const float shift = of[g].value_log - reference;
                unsigned w[4];
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + 2 * i], of[g].key_scale, shift));
                    const float b = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + 2 * i + 1], of[g].key_scale, shift));
                    part += a;
                    part += b;
                    w[i] = pack_bf16(a, b);
                }
                sum = fmaf(part, of[g].value_inverse, sum);
                weights[g] = __builtin_bit_cast(bf16x8_t, uint4{w[0], w[1], w[2], w[3]});
            }
#pragma unroll
            for (int d = 2; d < 4; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) value[4 * d + g] = *reinterpret_cast<const bf16x8_t*>(values_from + 32 * d * kValueRow + 32 * g);
#pragma unroll
            for (int e = 0; e < 4; e += 2)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int d = e; d < e + 2; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value[4 * d + g], weights[g], acc[d], 0, 0, 0);
        };
        if (steps > 0) load(0);
        for (int step = 0; step < steps; ++step) {
            const int buffer = kBuffers == 2 ? step & 1 : 0;
            stage(buffer);
            if (step + 1 < steps) load(step + 1);
            __syncthreads();
            const int token0 = begin + step * kStepTokens + key_wave * kTile;
            // nothing of this wave's rows lies before their window or behind their last position
            if (wave_lives && token0 <= wave_last && (p.a.window == 0 || token0 + kTile - 1 > wave_first - p.a.window)) {
                compute(buffer, token0);
            }
            if constexpr (kBuffers == 1) __syncthreads();
        }
        __syncthreads();  // the buffers are free: for the key groups' results, for the next tile of rows
        sum += __shfl_xor(sum, 32, 64);
        if constexpr (kKeyWaves > 1) {
            if (half == 0) lds.maximum[key_wave][column_wave][column] = maximum, lds.sum[key_wave][column_wave][column] = sum;
            __syncthreads();
            float top = lds.maximum[0][column_wave][column];
#pragma unroll
            for (int g = 1; g < kKeyWaves; ++g) top = fmaxf(top, lds.maximum[g][column_wave][column]);
            const float reference = top == -INFINITY ? 0.0f : top;
            sum = 0.0f;
#pragma unroll
            for (int g = 0; g < kKeyWaves; ++g) {
                sum += lds.sum[g][column_wave][column] * __builtin_amdgcn_exp2f(lds.maximum[g][column_wave][column] - reference);
            }
            const float shrink = __builtin_amdgcn_exp2f(maximum - reference);
            // a column wave's 16 KB of each key group but the first, lane by lane
            float* place = reinterpret_cast<float*>(dynamic_lds) + lane * 4;
            static_assert(sizeof(lds.keys) + sizeof(lds.values) >= (kKeyWaves - 1) * kColumnWaves * 64 * 64 * 4, "results fit");
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= shrink;
            if (key_wave > 0) {
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        *reinterpret_cast<floatx4_t*>(place + (((key_wave - 1) * kColumnWaves + column_wave) * 16 + d * 4 + i) * 256) =
                            floatx4_t{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
                    }
            }
            __syncthreads();
            if (key_wave == 0) {
#pragma unroll
                for (int g = 0; g < kKeyWaves - 1; ++g)
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const floatx4_t o = *reinterpret_cast<const floatx4_t*>(place + ((g * kColumnWaves + column_wave) * 16 + d * 4 + i) * 256);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[d][4 * i + e] += o[e];
                        }
            }
            __syncthreads();
        }
        if (mine && key_wave == 0) {
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

// Sequences of few rows and of many in one launch, so that neither waits for
// the other's last workgroup: workgroups y < splits take the former's shares,
// the others the latter's tiles; a sequence has one of the two.  Sequence after
// sequence, and heads side by side: with eight key/value heads each XCD's L2
// holds one head of one sequence at a time (every sequence's longest tiles
// first instead, four prompts of 1777..4096 rows 363 -> 555 us).
template <int kFormat, int kPageGranules, int kColumnWaves, int kKeyWaves>
__global__ __launch_bounds__(64 * kColumnWaves * kKeyWaves, 2) void kv8_all_rows_kernel(Params p) {
    constexpr int kWaves = kColumnWaves * kKeyWaves;
    extern __shared__ __align__(16) unsigned char dynamic_lds[];
    const int shares = p.few > 0 ? p.splits * p.few_tiles : 0, y = blockIdx.y;
    if (y < shares) {
        few_rows<kFormat, kPageGranules, kWaves>(p, *reinterpret_cast<FewShared<kWaves>*>(dynamic_lds), y);
    } else {
        many_rows<kFormat, kPageGranules, kColumnWaves, kKeyWaves>(p, dynamic_lds, y - shares, gridDim.y - shares);
    }
}

template <int kFormat, int kPageGranules, int kColumnWaves, int kKeyWaves>
hipError_t launch_all_rows(const Params& p, hipStream_t stream) {
    const auto kernel = kv8_all_rows_kernel<kFormat, kPageGranules, kColumnWaves, kKeyWaves>;
    static std::atomic<unsigned long long> prepared{0};
    constexpr int kWaves = kColumnWaves * kKeyWaves;
    constexpr int kBytes = std::max(sizeof(ManyShared<kColumnWaves, kKeyWaves>), sizeof(FewShared<kWaves>));
    if (const hipError_t st = set_dynamic_lds_once(prepared, reinterpret_cast<const void*>(kernel), kBytes); st != hipSuccess) return st;
    const int pairs = std::min(p.a.max_rows, p.a.rows) * p.group, shares = p.few > 0 ? p.splits * p.few_tiles : 0;
    const int tiles = std::min((pairs + 32 * kColumnWaves - 1) / (32 * kColumnWaves), 65535 - shares);
    kernel<<<dim3(p.cache.key_value_heads, shares + tiles, p.a.sequences), 64 * kWaves, kBytes, stream>>>(p);
    return hipGetLastError();
}

template <int kFormat, int kPageGranules>
hipError_t launch_pages(const Params& p, hipStream_t stream) {
    const dim3 grid(p.cache.key_value_heads, p.splits * p.few_tiles, p.a.sequences);
    hipError_t st = hipSuccess;
    switch (p.many) {
        case kNone:
            if (p.waves == 1) kv8_few_rows_kernel<kFormat, kPageGranules, 1><<<grid, 64, 0, stream>>>(p);
            else kv8_few_rows_kernel<kFormat, kPageGranules, kFewWaves><<<grid, 64 * kFewWaves, 0, stream>>>(p);
            st = hipGetLastError();
            break;
        case kWide: st = launch_all_rows<kFormat, kPageGranules, 4, 1>(p, stream); break;
        case kHalved: st = launch_all_rows<kFormat, kPageGranules, 4, 2>(p, stream); break;
        default: st = launch_all_rows<kFormat, kPageGranules, 2, 4>(p, stream); break;
    }
    if (st != hipSuccess || p.splits == 1) return st;
    kv8_join_kernel<<<dim3(p.columns, p.cache.key_value_heads, p.a.sequences), 32 * kJoinGroups, 0, stream>>>(p);
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
    int many = kNone;  // where sequences of many rows may be among them
    int few = INT_MAX, columns = 0, few_tiles = 1;  // as in Params
    int splits = 1;
    int waves = kFewWaves;
};
constexpr int kBytesOfPartial = (kDim + 2) * 4;

Dealt dealt_of(const Kv8Cache& cache, const Kv8AttentionArgs& a, size_t workspace_bytes) {
    Dealt d;
    const int group = a.query_heads / cache.key_value_heads;
    const int rows = std::max(1, std::min(a.max_rows, a.rows));
    const int reach = static_cast<int>(std::min<long long>(a.window > 0 ? static_cast<long long>(a.window) + rows : INT_MAX, a.max_length));
    const long long blocks = static_cast<long long>(std::max(a.sequences, 1)) * cache.key_value_heads;
    const int tile = 16 / group;  // rows of a tile of few rows
    const long long pairs = static_cast<long long>(rows) * group;
    const auto tiles_of = [&](long long n) { return static_cast<int>((n / group + tile - 1) / tile); };
    // Tiles of 16 pairs and blocks of 128 that the rows make at least, and the
    // tokens that a row attends to on average where all lengths are the longest.
    const long long few_tiles = std::max(blocks, static_cast<long long>(a.rows) * a.query_heads / 16);
    const long long many_blocks = std::max(blocks, static_cast<long long>(a.rows) * a.query_heads / 128);
    const auto tokens_of = [&](int tile_rows) -> double {
        return a.window > 0 ? std::min<long long>(static_cast<long long>(a.window) + tile_rows, reach) : reach - std::min(rows, reach) / 2;
    };
    const double chain = a.window > 0 ? tokens_of(128 / group) : reach;
    // All rows in tiles of 16, whose shares fill the chip, or in blocks of 128,
    // which read and convert keys and values once for all columns?  us, fitted to
    // one layer of 1 to 100 sequences: tiles 6.5 and 1 for each 33000 tokens of a
    // tile, which has 120 more to start; blocks 11 and the longer of a chain, 0.0116 a
    // token, and of the whole chip's work, 0.08 for 1000 tokens of a block.  Measured,
    // 16 / 8 heads, blocks / tiles: 32 rows over 4000 tokens 56 / 13, 256 over 16000
    // 197 / 117, 512 over 16000 197 / 217; prompts of 256 rows 13.0 / 6.9, 801 22.3 / 20.8,
    // 1024 23.9 / 25.1; eight sequences' 128 over 4000 70 / 112; forty's 16 over 2000
    // 113 / 57.  Not where most sequences would find no tile of theirs.
    const bool tiles_win = few_tiles * (tokens_of(tile) + 120) / 33000 < 4.5 + std::max(0.0116 * chain, 8e-5 * many_blocks * tokens_of(128 / group));
    if (pairs <= 16 || (tiles_win && blocks * tiles_of(pairs) <= 4 * few_tiles + 1024)) {
        d.columns = pairs <= 16 ? static_cast<int>(pairs) : tiles_of(pairs) * tile * group;
    } else {
        // Blocks of 128 columns where that makes one a CU, or where a chain of
        // steps is short anyway; else the tokens of a step are dealt to two or
        // four key groups, for the chain's sake.  One layer, 16 / 8 heads, us
        // with 1 / 2 / 4 groups: prompts of 512 rows 20.4 / 18.3 / 16.5, 1024 33.8 /
        // 28.0 / 23.5, 2048 62 / 48 / 48, 4096 119 / 98 / 139; four prompts of 512 25.7
        // / 23.7 / 36.0, of 801 40.7 / 43.0 / 59.6, of 2048 118 / 121 / 182.
        const bool one = a.sequences == 1;
        d.many = many_blocks > (one ? 512 : 256) || reach <= 192 ? kWide
                 : many_blocks <= 128 && reach >= 384            ? kQuartered
                                                                 : kHalved;
        // sequences of few rows among them: up to two tiles, four while those are not many
        d.few = one ? 0 : blocks <= 64 ? 64 : 32;
        if (one) return d;
        d.columns = static_cast<int>(std::min<long long>(d.few / group, rows)) * group;
    }
    d.few_tiles = d.many == kNone ? tiles_of(d.columns) : 1;
    // Contexts are shared among workgroups until there is one a CU, or two
    // where a workgroup would have more than 4096 tokens: then lengths differ
    // most (16 sequences of 100..16000 tokens, two splits 72 us, four 62; 32 of
    // 1000, one 15.8, two 18.9; one of 65521, 32 splits 28.5, 64 32.0).  A share
    // is a step of every wave at least.
    const long long there = d.many == kNone ? std::min(blocks * d.few_tiles, few_tiles) : blocks;
    const auto for_blocks = [&](long long n) { return (n + there - 1) / there; };
    const auto for_tokens = [&](int n) { return (static_cast<long long>(reach) + n - 1) / n; };
    long long wanted = std::max(for_blocks(256), std::min(for_blocks(512), for_tokens(4096)));
    // Where tiles fill the chip by the caller's sizes, a step of few of them still
    // finds shares (not where the second launch costs more: forty's 16 rows 57, with it 71).
    if (d.many == kNone && d.few_tiles > 1 && there <= 512) wanted = std::max(wanted, std::min(2LL, for_tokens(1024)));
    const long long fits = static_cast<long long>(workspace_bytes / (static_cast<size_t>(blocks) * d.columns * kBytesOfPartial));
    d.splits = static_cast<int>(std::max<long long>(1, std::min<long long>({wanted, for_tokens(kFewWaves * kStep), fits, kMostSplits, 65535 / d.few_tiles})));
    // Short contexts of many sequences: a wave a workgroup, none waits at the
    // end for waves that had no step (256 sequences of 100 tokens 24.9 us, now
    // 15.7; of 1111..8192 tokens 445, a wave each 499).
    if (reach <= 512 && there >= 1024) d.waves = 1;
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
    p.scale2 = std::fabs(a.scale) * kLog2E;
    p.flip = a.scale < 0 ? 0x80008000u : 0u;
    const Dealt d = dealt_of(cache, a, a.workspace_bytes);
    p.columns = d.columns;
    p.splits = d.splits;
    p.waves = d.waves;
    p.many = d.many;
    p.few = d.few;
    p.few_tiles = d.few_tiles;
    p.few_rows = d.few / p.group;
    p.shared_rows = d.columns / p.group;
    p.tile_rows = 16 / p.group;
    const size_t slots = static_cast<size_t>(a.sequences) * cache.key_value_heads * d.columns * d.splits;
    p.partial_out = a.workspace;
    p.partial_sums = reinterpret_cast<float2*>(a.workspace + slots * kDim);
    return cache.format == kKv8Int8 ? launch_format<kKv8Int8>(p, stream) : launch_format<kKv8E4m3>(p, stream);
}

}  // namespace q3
