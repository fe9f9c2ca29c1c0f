// The paged key and value cache as the kernels see it, and what the attention kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace nf4 {

// n / d for n < 2^31 and a d that the host knows: a multiplication and a shift.  mul = ceil(2^(31 + s) / d) with 2^s >= d > 2^(s - 1) is
// below 2^32, and off by less than d / 2^(31 + s) <= 2^-31 for every unit of n.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor), mul(0), shift(0) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << (31 + shift)) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> 31 >> shift); }
};

struct CacheView {
    const void *k, *v;
    const float *k_scales, *v_scales;
    uint32_t pages, page_size, heads;
    FastDiv by_page;
};
struct BatchView {
    const int32_t *table, *lengths, *starts;
    uint32_t sequences, width, rows;  // width: pages to a sequence
};

// A sequence of the call: its rows and its tokens, cut to what the buffers hold whatever the device memory says.
struct Sequence {
    uint32_t row0, rows, length;
};
__device__ __forceinline__ Sequence sequence_of(const CacheView &c, const BatchView &b, uint32_t s) {
    const int32_t from = max(__ldg(b.starts + s), 0), to = max(__ldg(b.starts + s + 1), 0), len = max(__ldg(b.lengths + s), 0);
    Sequence q;
    q.row0 = min((uint32_t)from, b.rows);
    q.rows = max(min((uint32_t)to, b.rows), q.row0) - q.row0;
    q.length = (uint32_t)min((uint64_t)len, (uint64_t)b.width * c.page_size);
    return q;
}

// kv_cache.cu: a call's arguments looked over, with a message that begins with `what`.  check_rows also fills in the row stride.
int32_t check_cache(const char *what, const nf4_cache *c, const nf4_cache_batch *b);
int32_t check_rows(const char *what, const char *name, const void *p, uint64_t *ld, uint64_t width, int32_t io_dtype);
CacheView view_of(const nf4_cache &c);
BatchView view_of(const nf4_cache_batch &b);

// Eight values of the cache as they are stored, to f32: of bf16 words, or of a word of codes and their block's scale.
__device__ __forceinline__ void values_of_bf16(const uint4 &w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void values_of_codes(uint32_t w, float scale, const float *levels, float (&v)[8]) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(levels[(w >> (4 * i)) & 15u], scale);
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The token of a call's row, and where the cache has it (for head 0, counted in rows of a head).  The first sequence that starts behind
// the row is looked for among `held` of the batch's starts, every step-th, then among those between two of them.
constexpr int64_t kNowhere = -1, kNoRow = -2;  // in no page; the row belongs to no sequence
__device__ __forceinline__ int64_t place_of_row(const CacheView &c, const BatchView &b, const int32_t *held, uint32_t step, uint32_t row, int64_t &token) {
    uint32_t low = 0, high = (b.sequences + step - 1) / step;
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (held[mid] <= (int32_t)row) low = mid + 1;
        else high = mid;
    }
    if (low == 0) return kNoRow;
    high = min(low * step, b.sequences);
    low = (low - 1) * step + 1;
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (__ldg(b.starts + mid) <= (int32_t)row) low = mid + 1;
        else high = mid;
    }
    const uint32_t s = low - 1;
    const Sequence q = sequence_of(c, b, s);
    if (row - q.row0 >= q.rows) return kNoRow;
    token = (int64_t)q.length - q.rows + (row - q.row0);
    if (token < 0) return kNowhere;
    const uint32_t at = c.by_page.of((uint32_t)token);
    const int32_t page = __ldg(b.table + (uint64_t)s * b.width + at);
    if (page < 0 || (uint32_t)page >= c.pages) return kNowhere;
    return (int64_t)page * c.heads * c.page_size + ((uint32_t)token - at * c.page_size);
}

// ---- attention ------------------------------------------------------------------------------------
// f16 holds the levels times kLevelUnit: it rounds each, always the same way, and a sum over many tokens keeps the rounding
// errors' mean, which at 131072 tokens was 4.5e-3 of the result.  In this unit (found by search over [1, 2)) that mean is 1.7e-6 of a
// block's scale, a sixth of what it is without one, for normal values and heavy tails alike.
constexpr float kLevelUnit = 1.4589462280273438f;
__device__ __forceinline__ uint32_t level_pair_f16(uint32_t byte) {  // of a byte's two codes
    const __half2 h = __floats2half2_rn(__uint_as_float(c_level_bits[byte & 15u]) * kLevelUnit, __uint_as_float(c_level_bits[byte >> 4]) * kLevelUnit);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// A call's arguments as the kernels take them.  The rows that one head of the cache serves are numbered token by token,
// the query heads of a token side by side: row r is token r / group, query head head * group + r % group.
struct AttentionView {
    const void *q;
    void *out;
    uint64_t ldq, ldo;
    uint32_t group;
    FastDiv by_group;
    float scale_log2;  // the scale times log2(e): weights are powers of two
    // Where the keys of a row tile are shared out between several CTAs each leaves its part here: the sums of weights times
    // values [part][row * heads * group + head][dim], and {largest exponent, sum of weights} beside them.
    float *part_o;
    float2 *part_ml;
    uint32_t parts;
    const uint32_t *masks;  // of trees: [rows][words], else null
    uint32_t words;
};

// How many tokens a row sees; of a tile's rows the last sees most.
__device__ __forceinline__ uint32_t visible_end(const Sequence &s, const FastDiv &by_group, uint32_t row) {
    const int32_t token = (int32_t)s.length - (int32_t)s.rows + (int32_t)by_group.of(row);
    return (uint32_t)max(token, -1) + 1;
}

// Of trees: the first token of the nodes, and 32 bits of what a row sees, of the nodes from number `first` on (the tokens ahead of the nodes are seen).
__device__ __forceinline__ int32_t first_node(const Sequence &s) { return (int32_t)s.length - (int32_t)s.rows; }
__device__ __forceinline__ uint32_t seen_nodes(const AttentionView &a, uint32_t row, int32_t first) {
    const int32_t w = first >> 5;
    if (w < -1) return ~0u;
    const uint32_t *const of_row = a.masks + (uint64_t)row * a.words;
    const uint32_t lo = w < 0 ? ~0u : (uint32_t)w < a.words ? __ldg(of_row + w) : 0u;
    const uint32_t hi = (uint32_t)(w + 1) < a.words ? __ldg(of_row + w + 1) : 0u;
    return __funnelshift_r(lo, hi, (uint32_t)first & 31u);
}
// The low `n` bits (all from 32 on).
__device__ __forceinline__ uint32_t low_bits(uint32_t n) { return n >= 32 ? ~0u : (1u << n) - 1; }

// How many tokens a row sees, or may see of a tree.
template <bool TREE>
__device__ __forceinline__ uint32_t seen_end(const Sequence &s, const FastDiv &by_group, uint32_t row) {
    return TREE ? s.length : visible_end(s, by_group, row);
}

struct AttentionCall {
    CacheView cache;
    BatchView batch;
    AttentionView view;
    bool nf4, f32, tree;
    uint32_t head_dim;
    uint32_t most_rows, most_tokens;  // of a sequence, as far as the host knows: rows of the call's tensors, tokens
};

constexpr uint64_t kAttentionFlagBytes = 4096;  // at the start of a workspace, as zeros

// attention_decode.cu: bf16 tensors, few rows to a head of a sequence
uint64_t attention_decode_bytes(const AttentionCall &c);
int32_t attention_decode(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream);

// attention_chunk.cu: bf16 tensors, many rows; where it can count the call's steps
bool attention_chunk_counts(const AttentionCall &c);
uint64_t attention_chunk_bytes(const AttentionCall &c);
int32_t attention_chunk(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream);

// attention_tree.cu: bf16 tensors whose rows are nodes of trees, likewise
bool attention_tree_counts(const AttentionCall &c);
uint64_t attention_tree_bytes(const AttentionCall &c);
int32_t attention_tree(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream);

}  // namespace nf4
