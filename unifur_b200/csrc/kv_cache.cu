// The paged key and value cache: writing rows to their places, and reading them back.
//
// Both are bound by HBM at sizes worth the name and by their launch at a decode step's: a thread has eight values of a
// row (a word of codes), eight neighbouring lanes a block of 64, as in the quantizer, whose arithmetic this is.
#include "kv_cache.cuh"
#include "ptx.cuh"

namespace nf4 {

// ---- checks ---------------------------------------------------------------------------------------

int32_t check_cache(const char *what, const nf4_cache *c, const nf4_cache_batch *b) {
    if (!c || c->struct_bytes != sizeof(nf4_cache)) return fail(NF4_ERR_INVALID_ARG, "%s: cache is null or its struct_bytes wrong", what);
    if (!b || b->struct_bytes != sizeof(nf4_cache_batch)) return fail(NF4_ERR_INVALID_ARG, "%s: batch is null or its struct_bytes wrong", what);
    if (c->form != NF4_CACHE_BF16 && c->form != NF4_CACHE_NF4) return fail(NF4_ERR_INVALID_ARG, "%s: unknown form %d of the cache", what, c->form);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(NF4_ERR_UNSUPPORTED, "%s: head_dim is %u; 64, 128 and 256 are supported", what, c->head_dim);
    if (c->page_size == 0 || c->page_size % 16 != 0 || c->page_size > 65536)
        return fail(NF4_ERR_UNSUPPORTED, "%s: page_size is %u; multiples of 16 up to 65536 are supported", what, c->page_size);
    if (c->heads == 0 || c->heads > 4096) return fail(NF4_ERR_UNSUPPORTED, "%s: %u heads; 1 to 4096 are supported", what, c->heads);
    if (c->num_pages == 0 || c->num_pages >= 1u << 31 || (uint64_t)c->num_pages * c->heads * c->page_size >= 1ull << 31)
        return fail(NF4_ERR_UNSUPPORTED, "%s: a pool of %u pages is empty or has 2^31 rows of a head or more", what, c->num_pages);
    if (!c->k || !c->v || (c->form == NF4_CACHE_NF4 && (!c->k_scales || !c->v_scales)))
        return fail(NF4_ERR_INVALID_ARG, "%s: null pointer in the cache", what);
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scales) || !aligned16(c->v_scales))
        return fail(NF4_ERR_INVALID_ARG, "%s: the cache's pools must be 16-byte aligned", what);
    if (b->sequences > 65535) return fail(NF4_ERR_UNSUPPORTED, "%s: %u sequences; 65535 are supported", what, b->sequences);
    if (b->rows >= 1u << 31 || b->pages_per_sequence >= 1u << 31 || (uint64_t)b->pages_per_sequence * c->page_size >= 1ull << 31)
        return fail(NF4_ERR_UNSUPPORTED, "%s: 2^31 rows or tokens of a sequence or more", what);
    if (b->sequences && (!b->lengths || !b->row_starts || (!b->page_table && b->pages_per_sequence)))
        return fail(NF4_ERR_INVALID_ARG, "%s: null pointer in the batch", what);
    return NF4_OK;
}

// A row stride in elements, or that of dense rows.
int32_t check_rows(const char *what, const char *name, const void *p, uint64_t *ld, uint64_t width, int32_t io_dtype) {
    if (io_dtype != NF4_DTYPE_BF16 && io_dtype != NF4_DTYPE_F32) return fail(NF4_ERR_INVALID_ARG, "%s: io_dtype must be NF4_DTYPE_BF16 or NF4_DTYPE_F32", what);
    if (*ld == 0) *ld = width;
    if (!p) return fail(NF4_ERR_INVALID_ARG, "%s: %s is null", what, name);
    const uint64_t whole = io_dtype == NF4_DTYPE_BF16 ? 8 : 4;
    if (!aligned16(p) || *ld % whole != 0) return fail(NF4_ERR_INVALID_ARG, "%s: %s and its row stride must be 16-byte aligned", what, name);
    if (*ld < width) return fail(NF4_ERR_INVALID_ARG, "%s: the row stride of %s is %llu, below a row's %llu values", what, name, (unsigned long long)*ld, (unsigned long long)width);
    if (*ld >= 1ull << 40) return fail(NF4_ERR_UNSUPPORTED, "%s: the row stride of %s is too large", what, name);
    return NF4_OK;
}

CacheView view_of(const nf4_cache &c) { return CacheView{c.k, c.v, c.k_scales, c.v_scales, c.num_pages, c.page_size, c.heads, FastDiv(c.page_size)}; }
BatchView view_of(const nf4_cache_batch &b) {
    return BatchView{b.page_table, b.lengths, b.row_starts, b.sequences, b.pages_per_sequence, b.rows};
}

namespace {

constexpr int kThreads = 256;

// The sequence that a row of the call belongs to, by bisection of row_starts; b.sequences where there is none.
__device__ __forceinline__ uint32_t sequence_at(const BatchView &b, uint32_t row) {
    uint32_t low = 0, high = b.sequences;  // the first sequence that starts behind the row is in [low, high]
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (__ldg(b.starts + mid) <= (int32_t)row) low = mid + 1;
        else high = mid;
    }
    return low ? low - 1 : b.sequences;
}

// Where the cache has the token of a row for head 0, counted in rows of a head; -1: nowhere.  `in`: whether the row belongs to a
// sequence.
__device__ __forceinline__ int64_t place_of(const CacheView &c, const BatchView &b, uint32_t row, bool *in) {
    const uint32_t s = sequence_at(b, row);
    *in = false;
    if (s >= b.sequences) return -1;
    const Sequence q = sequence_of(c, b, s);
    if (row - q.row0 >= q.rows) return -1;
    *in = true;
    const int64_t token = (int64_t)q.length - q.rows + (row - q.row0);
    if (token < 0) return -1;
    const uint32_t at = c.by_page.of((uint32_t)token);
    const int32_t page = __ldg(b.table + (uint64_t)s * b.width + at);
    if (page < 0 || (uint32_t)page >= c.pages) return -1;
    return (int64_t)page * c.heads * c.page_size + ((uint32_t)token - at * c.page_size);
}

__device__ __forceinline__ void ld8(const float *p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

struct Rows {  // the call's tensors: k and v
    const void *in[2];
    void *out[2];
    uint64_t ld[2];
};

// A thread's group of eight values: row, keys or values, head, and which eight of the head's row.
struct Group {
    uint32_t row, which, head, at;
};
// groups: 2 * heads * dim / 8 to a row
__device__ __forceinline__ Group group_at(uint32_t i, uint32_t groups, uint32_t dim8) {
    Group g;
    g.row = i / groups;
    uint32_t rest = i - g.row * groups;
    g.which = rest >= groups / 2 ? 1u : 0u;
    rest -= g.which * (groups / 2);
    g.head = rest / dim8;
    g.at = rest - g.head * dim8;
    return g;
}

template <bool NF4, bool BF16>
__global__ void __launch_bounds__(kThreads)
append_kernel(const CacheView c, const BatchView b, const Rows t, uint32_t groups, uint32_t dim8, uint32_t work) {
    __shared__ uint32_t s_cells[kCellWords], s_cells_bf16[kCellWords];
    if (NF4 && threadIdx.x < kCellWords) {
        s_cells[threadIdx.x] = c_cell_table[threadIdx.x];
        s_cells_bf16[threadIdx.x] = c_cell_bf16_table[threadIdx.x];
    }
    __syncthreads();
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    // (a head's row is 8, 16 or 32 groups, so the eight lanes of a block are in range together)
    const bool any = i < work;
    const Group g = group_at(any ? i : 0u, groups, dim8);
    bool in;
    const int64_t place = any ? place_of(c, b, g.row, &in) : -1;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint64_t from = (uint64_t)g.row * t.ld[g.which] + 8 * (g.head * dim8 + g.at);
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (place >= 0) {
        if (BF16) {
            raw = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(t.in[g.which]) + from));
            values_of_bf16(raw, v);
        } else {
            ld8(static_cast<const float *>(t.in[g.which]) + from, v);
        }
    }
    const uint64_t to = ((uint64_t)place + (uint64_t)g.head * c.page_size) * dim8 + g.at;  // in groups of eight values
    void *const pool = const_cast<void *>(g.which ? c.v : c.k);
    if (!NF4) {
        if (place >= 0) {
            if (!BF16) raw = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
            static_cast<uint4 *>(pool)[to] = raw;
        }
        return;
    }
    float m = 0.0f;  // the block's scale as the quantizer has it: NaNs drop out
    bool number = true;
    #pragma unroll
    for (int k = 0; k < 8; ++k) {
        m = fmaxf(m, fabsf(v[k]));
        number = number && v[k] == v[k];
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    if (place < 0) return;
    uint32_t w;
    if (BF16 && number && m >= 1e-30f && m <= 1e30f) {
        const float rcp = approx_rcp(m);
        w = codes_of_bf16(v, rcp * 2097152.0f, rcp * 64.0f, s_cells_bf16);
    } else {
        w = codes_of_group(v, m, s_cells);
    }
    static_cast<uint32_t *>(pool)[to] = w;
    if ((g.at & 7u) == 0) const_cast<float *>(g.which ? c.v_scales : c.k_scales)[to >> 3] = m;
}

template <bool NF4, bool BF16>
__global__ void __launch_bounds__(kThreads)
read_kernel(const CacheView c, const BatchView b, const Rows t, uint32_t groups, uint32_t dim8, uint32_t work) {
    __shared__ float s_levels[16];
    if (NF4 && threadIdx.x < 16) s_levels[threadIdx.x] = __uint_as_float(c_level_bits[threadIdx.x]);
    __syncthreads();
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= work) return;
    const Group g = group_at(i, groups, dim8);
    bool in;
    const int64_t place = place_of(c, b, g.row, &in);
    if (!in) return;
    const uint64_t from = ((uint64_t)(place < 0 ? 0 : place) + (uint64_t)g.head * c.page_size) * dim8 + g.at;
    const void *const pool = g.which ? c.v : c.k;
    float v[8];
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (place < 0) {
        #pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(0x7fc00000u);  // NaN
    } else if (NF4) {
        const uint32_t w = __ldg(static_cast<const uint32_t *>(pool) + from);
        values_of_codes(w, __ldg((g.which ? c.v_scales : c.k_scales) + (from >> 3)), s_levels, v);
    } else {
        raw = __ldg(static_cast<const uint4 *>(pool) + from);
        values_of_bf16(raw, v);
    }
    const uint64_t to = (uint64_t)g.row * t.ld[g.which] + 8 * (g.head * dim8 + g.at);
    if (BF16) {
        if (NF4 || place < 0) raw = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
        __stcs(reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(t.out[g.which]) + to), raw);
    } else {
        float4 *const out = reinterpret_cast<float4 *>(static_cast<float *>(t.out[g.which]) + to);
        __stcs(out, make_float4(v[0], v[1], v[2], v[3]));
        __stcs(out + 1, make_float4(v[4], v[5], v[6], v[7]));
    }
}

typedef void (*MoveKernel)(CacheView, BatchView, Rows, uint32_t, uint32_t, uint32_t);

int32_t move_rows(const char *what, const nf4_cache *cache, const nf4_cache_batch *batch, Rows t, MoveKernel kernel, cudaStream_t stream) {
    const uint32_t dim8 = cache->head_dim / 8, groups = 2 * cache->heads * dim8;
    if (!batch->rows || !batch->sequences) return NF4_OK;
    const uint64_t work = (uint64_t)batch->rows * groups;
    if (work >= 1ull << 32) return fail(NF4_ERR_UNSUPPORTED, "%s: %llu values in a call; split it", what, (unsigned long long)work * 8);
    const unsigned grid = (unsigned)((work + kThreads - 1) / kThreads);
    count_launch();
    return launch_maybe_overlapped(kernel, dim3(grid), dim3(kThreads), 0, stream, true, view_of(*cache), view_of(*batch), t, groups, dim8, (uint32_t)work);
}

template <bool NF4>
MoveKernel append_of(bool bf16) { return bf16 ? append_kernel<NF4, true> : append_kernel<NF4, false>; }
template <bool NF4>
MoveKernel read_of(bool bf16) { return bf16 ? read_kernel<NF4, true> : read_kernel<NF4, false>; }

}  // namespace

}  // namespace nf4

using namespace nf4;

extern "C" {

int32_t nf4_cache_append_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const void *k, uint64_t ldk, const void *v,
                             uint64_t ldv, int32_t io_dtype, void *stream) {
    const char *const what = "nf4_cache_append_dev";
    NF4_TRY(check_cache(what, cache, batch));
    const uint64_t width = (uint64_t)cache->heads * cache->head_dim;
    if (batch->rows) {
        NF4_TRY(check_rows(what, "k", k, &ldk, width, io_dtype));
        NF4_TRY(check_rows(what, "v", v, &ldv, width, io_dtype));
    }
    const bool bf16 = io_dtype == NF4_DTYPE_BF16;
    return move_rows(what, cache, batch, Rows{{k, v}, {nullptr, nullptr}, {ldk, ldv}},
                     cache->form == NF4_CACHE_NF4 ? append_of<true>(bf16) : append_of<false>(bf16), static_cast<cudaStream_t>(stream));
}

int32_t nf4_cache_read_dev(const nf4_cache *cache, const nf4_cache_batch *batch, void *k, uint64_t ldk, void *v, uint64_t ldv,
                           int32_t io_dtype, void *stream) {
    const char *const what = "nf4_cache_read_dev";
    NF4_TRY(check_cache(what, cache, batch));
    const uint64_t width = (uint64_t)cache->heads * cache->head_dim;
    if (batch->rows) {
        NF4_TRY(check_rows(what, "k", k, &ldk, width, io_dtype));
        NF4_TRY(check_rows(what, "v", v, &ldv, width, io_dtype));
    }
    const bool bf16 = io_dtype == NF4_DTYPE_BF16;
    return move_rows(what, cache, batch, Rows{{nullptr, nullptr}, {k, v}, {ldk, ldv}},
                     cache->form == NF4_CACHE_NF4 ? read_of<true>(bf16) : read_of<false>(bf16), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
