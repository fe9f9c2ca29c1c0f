// Trees of drafted tokens over the paged cache, beside their attention: masks and positions of the nodes' parents, and the move of an accepted
// path to the places behind the context.  Both are index work on a few kilobytes: they take what a launch and their chains of loads take.
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"

namespace nf4 {

namespace {

// ---- masks and positions ----------------------------------------------------------------------------
// A parent comes before its children, so a node's ancestors within its own word of 32 nodes follow from that word alone: a warp finds
// them for its lanes' nodes by doubling (after k exchanges a lane has its 2^k nearest ancestors and knows the next one), and the ancestor
// at which the way leaves the word.  A thread to a row then goes up a word at a time, and writes words from the highest down.
// (A node at a time, lanes leaving their words at different steps: 118 ns a node of the way, chains of 64 / 250 / 1000 nodes 7.7 / 27 / 113 us;
// so 1.7 / 2.4 / 6.7, and trees with two children to a node 1.7 / 2.4 / 6.8 where they took 1.9 / 2.8 / 4.9.)
// Nodes are prepared kWindow at a time, from the highest that the CTA's rows have, until no row has a way left.
constexpr uint32_t kTreeThreads = 256, kWindow = 2048;
static_assert(kWindow % 32 == 0);

__global__ void __launch_bounds__(kTreeThreads)
tree_kernel(const CacheView c, const BatchView b, const int32_t *const parents, uint32_t *const masks, uint32_t words, int32_t *const positions) {
    __shared__ uint2 s_nodes[kWindow];  // itself and its ancestors in its word; the parent of the first of them, or -1
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const Sequence s = sequence_of(c, b, blockIdx.x);
    for (uint32_t r0 = blockIdx.y * kTreeThreads; r0 < s.rows; r0 += gridDim.y * kTreeThreads) {
        const uint32_t i = r0 + tid, end = min(s.rows, r0 + kTreeThreads);
        uint32_t *const mask = masks && i < end ? masks + (uint64_t)(s.row0 + i) * words : nullptr;
        int32_t node = i < end ? (int32_t)i : -1;
        uint32_t met = 0, done = words;  // nodes on the way so far; words from here on are written
        for (int32_t w0 = (int32_t)((end - 1) / kWindow * kWindow); w0 >= 0; w0 -= (int32_t)kWindow) {
            if (!__syncthreads_or(node >= 0)) break;
            const uint32_t last = min(end, (uint32_t)w0 + kWindow);
            for (uint32_t at = (uint32_t)w0 + tid; at - lane < last; at += kTreeThreads) {
                int32_t up = at < last ? __ldg(parents + s.row0 + at) : -1;
                if (up < 0 || (uint32_t)up >= at) up = -1;
                uint32_t bits = 1u << lane, next = up >= (int32_t)(at - lane) ? (uint32_t)up & 31u : lane;
                #pragma unroll
                for (uint32_t k = 0; k < 5; ++k) {
                    bits |= __shfl_sync(0xffffffffu, bits, next);
                    next = __shfl_sync(0xffffffffu, next, next);
                }
                s_nodes[at - (uint32_t)w0] = make_uint2(bits, (uint32_t)__shfl_sync(0xffffffffu, up, next));
            }
            __syncthreads();
            while (node >= w0) {
                const uint2 of = s_nodes[node - w0];
                const uint32_t word = (uint32_t)node / 32;
                if (mask) {
                    for (uint32_t w = word + 1; w < done; ++w) mask[w] = 0;
                    if (word < done) mask[word] = of.x;
                }
                done = min(done, word);
                met += __popc(of.x);
                node = (int32_t)of.y;
            }
        }
        if (mask)
            for (uint32_t w = 0; w < done; ++w) mask[w] = 0;
        if (positions && i < end) positions[s.row0 + i] = (int32_t)s.length - (int32_t)s.rows + (int32_t)met - 1;
    }
}

// ---- keeping a path ---------------------------------------------------------------------------------
// A CTA to a sequence: its length is read before anything is written, so that the lengths may change in place.  A thread has a piece (16 bytes, or
// a block's scale) of every token of the path, and moves them in the path's order, kAhead loads before their stores: a path increases, so no token comes
// to a place that a later one is still to be read from, and one that an earlier was read from is written by the thread that read it.
constexpr uint32_t kKeepThreads = 512, kStep = 256, kAhead = 8;

template <class T>
__device__ __forceinline__ void move_path(T *pool, uint64_t pitch, uint64_t at, const int64_t (*places)[2], uint32_t n) {
    for (uint32_t j0 = 0; j0 < n; j0 += kAhead) {
        T v[kAhead];
        #pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j)
            if (j0 + j < n && places[j0 + j][0] >= 0) v[j] = pool[(uint64_t)places[j0 + j][0] * pitch + at];
        #pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j)
            if (j0 + j < n && places[j0 + j][0] >= 0) pool[(uint64_t)places[j0 + j][1] * pitch + at] = v[j];
    }
}

template <bool NF4>
__global__ void __launch_bounds__(kKeepThreads)
keep_kernel(const CacheView c, const BatchView b, uint32_t dim, const int32_t *const kept, uint32_t most, const int32_t *const counts, int32_t *const lengths_out) {
    __shared__ int64_t s_places[kStep][2];  // from, to; from -1: not moved
    __shared__ uint32_t s_count;
    const uint32_t tid = threadIdx.x, seq = blockIdx.x;
    if (tid == 0) s_count = 0xffffffffu;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const Sequence s = sequence_of(c, b, seq);
    const int32_t *const path = kept + (uint64_t)seq * most;
    const uint32_t asked = min((uint32_t)max(__ldg(counts + seq), 0), min(most, s.rows));
    __syncthreads();
    for (uint32_t j = tid; j < asked; j += kKeepThreads) {
        const int32_t node = __ldg(path + j), before = j ? __ldg(path + j - 1) : -1;
        if (node < 0 || (uint32_t)node >= s.rows || node <= before) atomicMin(&s_count, j);
    }
    __syncthreads();
    const uint32_t count = min(asked, s_count);
    const int64_t context = (int64_t)s.length - s.rows;
    if (lengths_out && tid == 0) lengths_out[seq] = (int32_t)max(context + (int64_t)count, (int64_t)0);
    auto place = [&](int64_t token) -> int64_t {
        if (token < 0) return kNowhere;
        const uint32_t at = c.by_page.of((uint32_t)token);
        const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at);
        if (page < 0 || (uint32_t)page >= c.pages) return kNowhere;
        return (int64_t)page * c.heads * c.page_size + ((uint32_t)token - at * c.page_size);
    };
    // pieces: of 16 bytes of a head's row of keys, of values, then scales likewise
    const uint32_t chunks = NF4 ? dim / 32 : dim / 8, blocks = NF4 ? dim / 64 : 0, all = 2 * c.heads * chunks, pieces = all + 2 * c.heads * blocks;
    for (uint32_t j0 = 0; j0 < count; j0 += kStep) {
        const uint32_t n = min(kStep, count - j0);
        __syncthreads();
        for (uint32_t j = tid; j < n; j += kKeepThreads) {
            const int64_t from = place(context + __ldg(path + j0 + j)), to = place(context + j0 + j);
            s_places[j][0] = to < 0 || from == to ? -1 : from;
            s_places[j][1] = to;
        }
        __syncthreads();
        for (uint32_t i = tid; i < pieces; i += kKeepThreads) {
            if (i < all) {
                const uint32_t r = i % (c.heads * chunks), head = r / chunks;
                uint4 *const pool = static_cast<uint4 *>(const_cast<void *>(i < c.heads * chunks ? c.k : c.v));
                move_path(pool, chunks, (uint64_t)head * c.page_size * chunks + r % chunks, s_places, n);
            } else if (NF4) {
                const uint32_t r = (i - all) % (c.heads * blocks), head = r / blocks;
                float *const pool = const_cast<float *>(i - all < c.heads * blocks ? c.k_scales : c.v_scales);
                move_path(pool, blocks, (uint64_t)head * c.page_size * blocks + r % blocks, s_places, n);
            }
        }
    }
}

}  // namespace

}  // namespace nf4

using namespace nf4;

extern "C" {

int32_t nf4_cache_tree_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const int32_t *parents, uint32_t *masks, uint32_t mask_words,
                           int32_t *positions, void *stream) {
    const char *const what = "nf4_cache_tree_dev";
    NF4_TRY(check_cache(what, cache, batch));
    if (mask_words > 1u << 26) return fail(NF4_ERR_UNSUPPORTED, "%s: masks of %u words; 2^26 are supported", what, mask_words);
    if (!batch->rows || !batch->sequences || (!masks && !positions)) return NF4_OK;
    if (!parents) return fail(NF4_ERR_INVALID_ARG, "%s: parents is null", what);
    // rows side by side, as far as the host knows of them
    const uint32_t most = batch->max_rows ? std::min(batch->max_rows, batch->rows) : batch->rows;
    const uint32_t across = std::max(1u, std::min((most + kTreeThreads - 1) / kTreeThreads, 8u * kNumSMs / batch->sequences));
    count_launch();
    return launch_maybe_overlapped(tree_kernel, dim3(batch->sequences, across), dim3(kTreeThreads), 0, static_cast<cudaStream_t>(stream), true, view_of(*cache),
                                   view_of(*batch), parents, masks, mask_words, positions);
}

int32_t nf4_cache_keep_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const int32_t *kept, uint32_t most_kept, const int32_t *counts,
                           int32_t *lengths_out, void *stream) {
    const char *const what = "nf4_cache_keep_dev";
    NF4_TRY(check_cache(what, cache, batch));
    if (most_kept >= 1u << 31) return fail(NF4_ERR_UNSUPPORTED, "%s: paths of 2^31 nodes or more", what);
    if (!batch->sequences) return NF4_OK;
    if (!counts || (!kept && most_kept)) return fail(NF4_ERR_INVALID_ARG, "%s: kept or counts is null", what);
    count_launch();
    return launch_maybe_overlapped(cache->form == NF4_CACHE_NF4 ? keep_kernel<true> : keep_kernel<false>, dim3(batch->sequences), dim3(kKeepThreads), 0,
                                   static_cast<cudaStream_t>(stream), true, view_of(*cache), view_of(*batch), cache->head_dim, kept, most_kept, counts, lengths_out);
}

}  // extern "C"
