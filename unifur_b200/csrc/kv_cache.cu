// The paged key and value cache: writing rows to their places, and reading them back.
//
// Both are bound by HBM at sizes worth the name and by their launch at a decode step's: a thread has eight values of a
// row at a time (a word of codes), eight neighbouring lanes a block of 64, as in the quantizer, whose arithmetic this is.
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
// Rows to a thread at most, all asked for before the first is used.  Measured with 1, 2, 4 and 8 for both: 7,300 rows of four heads of 128
// quantized and then read back as f32 in 22.4, 19.7, 20.5 and 26.7 us, 26,900 read as bf16 in 27.7, 19.4, 15.8 and 15.0 us (4.5 TB/s;
// bound by instructions as much as by HBM).
constexpr uint32_t kAppendBatch = 2, kReadBatch = 4;
constexpr uint32_t kMostRows = 4 * kThreads / 16;    // of a CTA: a row has 16 groups at least
constexpr uint32_t kStarts = 1024;                   // row_starts that a CTA holds; of more, every second, third, ...

struct Rows {  // the call's tensors
    void *k, *v;
    uint64_t ldk, ldv;
};

// A token's row is 2 * heads * dim / 8 groups of eight values: keys, then values, heads one after the other.  CTAs take `width` of them each
// (blockIdx.y: which; a multiple of eight, so that a block of 64 is eight neighbouring lanes') of batch * abreast rows (blockIdx.x).  A thread has
// the same group of `batch` rows: what it is and where it lies in a row is worked out once.
struct Move {
    uint32_t groups, shift;  // to a row; log2(dim / 8)
    uint32_t width, abreast, batch;
    __host__ __device__ uint32_t rows() const { return abreast * batch; }
};

// Where a CTA's rows have their token in the cache, for head 0 and counted in rows of a head.
struct Places {
    int32_t starts[kStarts];
    int64_t of[kMostRows];
};

// The whole CTA finds its rows' places, once for all of a row's groups.
__device__ __forceinline__ void find_places(const CacheView &c, const BatchView &b, const Move &m, uint32_t row0, Places &p) {
    const uint32_t tid = threadIdx.x, step = (b.sequences + kStarts - 1) / kStarts;
    for (uint32_t i = tid; i * step < b.sequences; i += kThreads) p.starts[i] = __ldg(b.starts + i * step);
    __syncthreads();
    int64_t token;
    if (tid < m.rows()) p.of[tid] = row0 + tid < b.rows ? place_of_row(c, b, p.starts, step, row0 + tid, token) : kNoRow;
    __syncthreads();
}

// A thread's group: its first row (of the CTA's), keys or values, where it is in a head's row of the pool (in groups, from the first head's
// row on) and in a row of the call's tensor (in values).  `any`: there is one for this thread.
struct Group {
    uint32_t row, at;
    bool any, v;
    uint64_t in_pool, in_row;
};
__device__ __forceinline__ Group group_at(const CacheView &c, const Move &m) {
    Group g;
    g.row = threadIdx.x / m.width;
    const uint32_t of_width = threadIdx.x - g.row * m.width, i = blockIdx.y * m.width + of_width;
    g.any = g.row < m.abreast && i < m.groups;
    g.v = i >= m.groups / 2;
    const uint32_t rest = i - (g.v ? m.groups / 2 : 0u), head = rest >> m.shift;
    g.at = rest & ((1u << m.shift) - 1);
    g.in_pool = ((uint64_t)head * c.page_size << m.shift) + g.at;
    g.in_row = 8ull * rest;
    return g;
}

template <bool NF4, bool BF16>
__global__ void __launch_bounds__(kThreads)
append_kernel(const CacheView c, const BatchView b, const Rows t, const Move move) {
    __shared__ uint32_t s_cells[kCellWords], s_cells_bf16[kCellWords];
    __shared__ Places s_places;
    if (NF4 && threadIdx.x < kCellWords) {
        s_cells[threadIdx.x] = c_cell_table[threadIdx.x];
        s_cells_bf16[threadIdx.x] = c_cell_bf16_table[threadIdx.x];
    }
    const Group g = group_at(c, move);
    const uint32_t row0 = blockIdx.x * move.rows();
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    constexpr uint32_t kQuads = BF16 ? 1 : 2, kBytes = BF16 ? 2 : 4;
    uint4 raw[kAppendBatch][kQuads];
    const uint64_t ld = g.v ? t.ldv : t.ldk;
    const uint8_t *const from = static_cast<const uint8_t *>(g.v ? t.v : t.k) + ((uint64_t)(row0 + g.row) * ld + g.in_row) * kBytes;
    #pragma unroll
    for (uint32_t u = 0; u < kAppendBatch; ++u)
        if (g.any && u < move.batch && row0 + g.row + u * move.abreast < b.rows)
            #pragma unroll
            for (uint32_t k = 0; k < kQuads; ++k) raw[u][k] = __ldcs(reinterpret_cast<const uint4 *>(from + u * move.abreast * ld * kBytes) + k);
    find_places(c, b, move, row0, s_places);  // (while the values come)
    void *const pool = const_cast<void *>(g.v ? c.v : c.k);
    float *const scales = const_cast<float *>(g.v ? c.v_scales : c.k_scales);
    #pragma unroll
    for (uint32_t u = 0; u < kAppendBatch; ++u) {
        if (u >= move.batch) break;
        const int64_t place = g.any ? s_places.of[g.row + u * move.abreast] : kNoRow;
        const uint64_t to = ((uint64_t)place << move.shift) + g.in_pool;  // in groups
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (place >= 0) {
            if constexpr (BF16) {
                values_of_bf16(raw[u][0], v);
            } else {
                #pragma unroll
                for (uint32_t k = 0; k < kQuads; ++k) {
                    v[4 * k] = __uint_as_float(raw[u][k].x); v[4 * k + 1] = __uint_as_float(raw[u][k].y);
                    v[4 * k + 2] = __uint_as_float(raw[u][k].z); v[4 * k + 3] = __uint_as_float(raw[u][k].w);
                }
            }
        }
        if (!NF4) {
            if (place >= 0)
                static_cast<uint4 *>(pool)[to] =
                    BF16 ? raw[u][0] : make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
            continue;
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
        if (place >= 0) {
            uint32_t w;
            if (BF16 && number && m >= 1e-30f && m <= 1e30f) {
                const float rcp = approx_rcp(m);
                w = codes_of_bf16(v, rcp * 2097152.0f, rcp * 64.0f, s_cells_bf16);
            } else {
                w = codes_of_group(v, m, s_cells);
            }
            static_cast<uint32_t *>(pool)[to] = w;
            if ((g.at & 7u) == 0) scales[to >> 3] = m;
        }
        __syncwarp();
    }
}

template <bool NF4, bool BF16>
__global__ void __launch_bounds__(kThreads)
read_kernel(const CacheView c, const BatchView b, const Rows t, const Move move) {
    __shared__ float s_levels[16];
    __shared__ Places s_places;
    if (NF4 && threadIdx.x < 16) s_levels[threadIdx.x] = __uint_as_float(c_level_bits[threadIdx.x]);
    const Group g = group_at(c, move);
    const uint32_t row0 = blockIdx.x * move.rows();
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    find_places(c, b, move, row0, s_places);
    if (!g.any) return;
    const void *const pool = g.v ? c.v : c.k;
    const float *const scales = g.v ? c.v_scales : c.k_scales;
    uint4 raw[kReadBatch];
    float scale[kReadBatch];
    #pragma unroll
    for (uint32_t u = 0; u < kReadBatch; ++u) {
        if (u >= move.batch) break;
        const int64_t place = s_places.of[g.row + u * move.abreast];
        if (place < 0) continue;
        const uint64_t from = ((uint64_t)place << move.shift) + g.in_pool;
        if (NF4) {
            raw[u].x = __ldg(static_cast<const uint32_t *>(pool) + from);
            scale[u] = __ldg(scales + (from >> 3));
        } else {
            raw[u] = __ldg(static_cast<const uint4 *>(pool) + from);
        }
    }
    constexpr uint32_t kBytes = BF16 ? 2 : 4;
    const uint64_t ld = g.v ? t.ldv : t.ldk;
    uint8_t *const to = static_cast<uint8_t *>(g.v ? t.v : t.k) + ((uint64_t)(row0 + g.row) * ld + g.in_row) * kBytes;
    #pragma unroll
    for (uint32_t u = 0; u < kReadBatch; ++u) {
        if (u >= move.batch) break;
        const int64_t place = s_places.of[g.row + u * move.abreast];
        if (place == kNoRow) continue;
        float v[8];
        if (place < 0) {
            #pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(0x7fc00000u);  // NaN
        } else if (NF4) {
            values_of_codes(raw[u].x, scale[u], s_levels, v);
        } else {
            values_of_bf16(raw[u], v);
        }
        uint8_t *const here = to + u * move.abreast * ld * kBytes;
        if (BF16) {
            if (NF4 || place < 0) raw[u] = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
            __stcs(reinterpret_cast<uint4 *>(here), raw[u]);
        } else {
            __stcs(reinterpret_cast<float4 *>(here), make_float4(v[0], v[1], v[2], v[3]));
            __stcs(reinterpret_cast<float4 *>(here) + 1, make_float4(v[4], v[5], v[6], v[7]));
        }
    }
}

typedef void (*MoveKernel)(CacheView, BatchView, Rows, Move);

int32_t move_rows(const char *what, const nf4_cache *cache, const nf4_cache_batch *batch, Rows t, MoveKernel kernel, uint32_t rows_of_thread, cudaStream_t stream) {
    if (!batch->rows || !batch->sequences) return NF4_OK;
    const uint32_t dim8 = cache->head_dim / 8, groups = 2 * cache->heads * dim8;
    const uint32_t across = (groups + kThreads - 1) / kThreads;  // CTAs to a row
    Move move{groups, dim8 == 8 ? 3u : dim8 == 16 ? 4u : 5u, ((groups + across - 1) / across + 7) / 8 * 8, 0, rows_of_thread};
    move.abreast = kThreads / move.width;
    // One row to a thread where that leaves no SM more than two CTAs: such a call takes what its chain of loads takes.
    if ((uint64_t)batch->rows * groups <= 2ull * kNumSMs * kThreads) move.batch = 1;
    const dim3 grid((unsigned)((batch->rows + move.rows() - 1) / move.rows()), across);
    count_launch();
    return launch_maybe_overlapped(kernel, grid, dim3(kThreads), 0, stream, true, view_of(*cache), view_of(*batch), t, move);
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
    return move_rows(what, cache, batch, Rows{const_cast<void *>(k), const_cast<void *>(v), ldk, ldv},
                     cache->form == NF4_CACHE_NF4 ? append_of<true>(bf16) : append_of<false>(bf16), kAppendBatch, static_cast<cudaStream_t>(stream));
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
    return move_rows(what, cache, batch, Rows{k, v, ldk, ldv},
                     cache->form == NF4_CACHE_NF4 ? read_of<true>(bf16) : read_of<false>(bf16), kReadBatch, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
