// Appending keys and values to the paged cache with the positions' rotation on the way, and the queries rotated beside them.
//
// A row is q_heads + 2 * heads vectors of dim values; dim / 16 lanes have a vector, two groups of eight values each, which are those that the rotation
// takes together: groups g and g + rotary_dim / 16 for halves (value i with value i + rotary_dim / 2), any two for neighbours.  So a thread turns what
// it has loaded, and its cosines and sines serve all vectors of the row that it takes.  Bound by HBM at sizes worth the name: rows in, rows and
// what the cache holds out, 4 * rotary_dim bytes of the table a row.
// Products and sums are each rounded, with no FMA, so that a turned key is a defined f32 value whose codes are the quantizer's.
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"

namespace nf4 {

namespace {

constexpr uint32_t kMostThreads = 256;
constexpr uint32_t kStarts = 1024;                 // row_starts that a CTA holds; of more, every second, third, ...
constexpr uint32_t kMostRows = 96;                 // of a CTA

struct Rotated {
    const void *k, *v, *q;
    void *q_out;
    uint64_t ldk, ldv, ldq, ldo;
    const float *table;
    const int32_t *positions;
    uint32_t table_positions, rotary_dim, q_heads;
    bool pairs;
    // CTAs take `rounds` times `abreast` rows (blockIdx.x) and of each `width` vectors at a time, BATCH times (blockIdx.y: which)
    uint32_t width, abreast, rounds;
};

// Two groups of eight values turned.  pairs: neighbours, with four cosines and sines to a group.
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float was = a;
    a = __fsub_rn(__fmul_rn(was, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(was, s));
}

template <int D, bool NF4, bool BF16, uint32_t BATCH>
__global__ void __launch_bounds__(kMostThreads)
append_rotated_kernel(const CacheView c, const BatchView b, const Rotated t) {
    constexpr uint32_t L = D / 16, kBlocks = D / 64, kBytes = BF16 ? 2 : 4, kQuads = BF16 ? 1 : 2;
    __shared__ uint32_t s_cells[kCellWords];
    __shared__ int32_t s_starts[kStarts];
    __shared__ int64_t s_places[kMostRows];
    __shared__ int32_t s_positions[kMostRows];
    const uint32_t tid = threadIdx.x, lane = tid % L, slot = tid / L, of_cta = slot / t.width, first = blockIdx.y * t.width * BATCH + (slot - of_cta * t.width);
    const uint32_t rows = t.abreast * t.rounds, row0 = blockIdx.x * rows, vectors = t.q_heads + 2 * c.heads;
    const bool any = of_cta < t.abreast;
    if (NF4)
        for (uint32_t i = tid; i < kCellWords; i += blockDim.x) s_cells[i] = c_cell_table[i];
    // the thread's groups; turned[]: whether the rotation has them
    const uint32_t half = t.rotary_dim / 16;
    uint32_t group[2];
    bool turned[2];
    if (t.pairs || lane >= half) {
        const uint32_t from = t.pairs ? lane : 2 * half + (lane - half), apart = t.pairs ? L : L - half;
        group[0] = from;
        group[1] = from + apart;
        turned[0] = t.pairs && group[0] < 2 * half;
        turned[1] = t.pairs && group[1] < 2 * half;
    } else {
        group[0] = lane;
        group[1] = lane + half;
        turned[0] = turned[1] = true;
    }
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();

    // ---- all that the thread takes of a row is asked for: of the first ahead of the rows' places, of the next ones as registers become free ----
    uint4 raw[BATCH][2][kQuads];
    auto ask = [&](uint32_t u, uint32_t row) {
        const uint32_t vec = first + u * t.width;
        if (!any || vec >= vectors || row >= b.rows) return;
        const bool is_q = vec < t.q_heads, is_v = vec >= t.q_heads + c.heads;
        const uint32_t head = is_q ? vec : is_v ? vec - t.q_heads - c.heads : vec - t.q_heads;
        const uint8_t *const from = static_cast<const uint8_t *>(is_q ? t.q : is_v ? t.v : t.k) + ((uint64_t)row * (is_q ? t.ldq : is_v ? t.ldv : t.ldk) + (uint64_t)head * D) * kBytes;
        #pragma unroll
        for (int e = 0; e < 2; ++e)
            #pragma unroll
            for (uint32_t k = 0; k < kQuads; ++k) raw[u][e][k] = __ldcs(reinterpret_cast<const uint4 *>(from + group[e] * 8 * kBytes) + k);
    };
    #pragma unroll
    for (uint32_t u = 0; u < BATCH; ++u) ask(u, row0 + of_cta);
    // ---- the rows' places and positions (while the values come) ----
    const uint32_t step = (b.sequences + kStarts - 1) / kStarts;
    for (uint32_t i = tid; i * step < b.sequences; i += blockDim.x) s_starts[i] = __ldg(b.starts + i * step);
    __syncthreads();
    for (uint32_t i = tid; i < rows; i += blockDim.x) {
        int64_t place = kNoRow, token = -1;
        int32_t position = -1;
        if (row0 + i < b.rows) {
            if (t.positions) position = __ldg(t.positions + row0 + i);
            place = place_of_row(c, b, s_starts, step, row0 + i, token);
            if (!t.positions) position = (int32_t)token;
        }
        const bool there = position >= 0 && (uint32_t)position < t.table_positions;
        s_positions[i] = there ? position : -1;
        s_places[i] = there || place == kNoRow ? place : kNowhere;
    }
    __syncthreads();
    for (uint32_t round = 0; round < t.rounds; ++round) {  // (by all of a warp's threads)
        const uint32_t in_cta = of_cta + round * t.abreast, row = row0 + in_cta;
        if (__all_sync(0xffffffffu, row >= b.rows)) break;
        const int64_t place = any ? s_places[in_cta] : kNoRow;
        const int32_t position = any ? s_positions[in_cta] : -1;
        float cosines[8], sines[8];  // halves: of the two groups' pairs; neighbours: four to a group
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            cosines[i] = 1.f;
            sines[i] = 0.f;
        }
        if (position >= 0 && place != kNoRow) {
            const float *const angles = t.table + (uint64_t)position * t.rotary_dim;
            auto four = [&](float *to, const float *from) {
                const float4 w = __ldg(reinterpret_cast<const float4 *>(from));
                to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
            };
            if (t.pairs) {
                #pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (turned[e]) {
                        four(cosines + 4 * e, angles + 4 * group[e]);
                        four(sines + 4 * e, angles + t.rotary_dim / 2 + 4 * group[e]);
                    }
            } else if (turned[0]) {
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    four(cosines + 4 * e, angles + 8 * group[0] + 4 * e);
                    four(sines + 4 * e, angles + t.rotary_dim / 2 + 8 * group[0] + 4 * e);
                }
            }
        }

        #pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) {
            const uint32_t vec = first + u * t.width;
            const bool here = any && vec < vectors && place != kNoRow;
            const bool is_q = vec < t.q_heads, is_v = vec >= t.q_heads + c.heads;
            const uint32_t head = is_q ? vec : is_v ? vec - t.q_heads - c.heads : vec - t.q_heads;
            const bool turns = here && !is_v;
            float v[2][8];
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) v[e][i] = 0.f;
                if (!here) continue;
                if constexpr (BF16) {
                    values_of_bf16(raw[u][e][0], v[e]);
                } else {
                    #pragma unroll
                    for (uint32_t k = 0; k < kQuads; ++k) {
                        v[e][4 * k] = __uint_as_float(raw[u][e][k].x); v[e][4 * k + 1] = __uint_as_float(raw[u][e][k].y);
                        v[e][4 * k + 2] = __uint_as_float(raw[u][e][k].z); v[e][4 * k + 3] = __uint_as_float(raw[u][e][k].w);
                    }
                }
            }
            if (round + 1 < t.rounds) ask(u, row + t.abreast);
            if (turns) {
                if (t.pairs) {
                    #pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (turned[e])
                            #pragma unroll
                            for (int i = 0; i < 4; ++i) turn(v[e][2 * i], v[e][2 * i + 1], cosines[4 * e + i], sines[4 * e + i]);
                } else if (turned[0]) {
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) turn(v[0][i], v[1][i], cosines[i], sines[i]);
                }
            }
            if (here && is_q) {
                uint8_t *const to = static_cast<uint8_t *>(t.q_out) + ((uint64_t)row * t.ldo + (uint64_t)head * D) * kBytes;
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (position < 0)
                        #pragma unroll
                        for (int i = 0; i < 8; ++i) v[e][i] = __uint_as_float(0x7fc00000u);  // NaN
                    uint4 *const at = reinterpret_cast<uint4 *>(to + group[e] * 8 * kBytes);
                    if constexpr (BF16) {
                        *at = make_uint4(bf16_pair(v[e][0], v[e][1]), bf16_pair(v[e][2], v[e][3]), bf16_pair(v[e][4], v[e][5]), bf16_pair(v[e][6], v[e][7]));
                    } else {
                        #pragma unroll
                        for (int k = 0; k < 2; ++k)
                            reinterpret_cast<float4 *>(at)[k] = make_float4(v[e][4 * k], v[e][4 * k + 1], v[e][4 * k + 2], v[e][4 * k + 3]);
                    }
                }
            }
            const bool stored = here && !is_q && place >= 0;
            const uint64_t to = ((uint64_t)place + (uint64_t)head * c.page_size) * (D / 8);  // in groups
            void *const pool = const_cast<void *>(is_v ? c.v : c.k);
            if (!NF4) {
                #pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (stored)
                        static_cast<uint4 *>(pool)[to + group[e]] =
                            make_uint4(bf16_pair(v[e][0], v[e][1]), bf16_pair(v[e][2], v[e][3]), bf16_pair(v[e][4], v[e][5]), bf16_pair(v[e][6], v[e][7]));
                continue;
            }
            if (!__any_sync(0xffffffffu, stored)) continue;
            // a block's largest magnitude is its groups', which its vector's lanes have
            float most[kBlocks];
            #pragma unroll
            for (uint32_t k = 0; k < kBlocks; ++k) most[k] = 0.f;
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                float m = 0.f;  // (NaNs drop out)
                #pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[e][i]));
                #pragma unroll
                for (uint32_t k = 0; k < kBlocks; ++k)
                    if (group[e] / 8 == k) most[k] = fmaxf(most[k], m);
            }
            #pragma unroll
            for (uint32_t k = 0; k < kBlocks; ++k)
                #pragma unroll
                for (uint32_t d = 1; d < L; d <<= 1) most[k] = fmaxf(most[k], __shfl_xor_sync(0xffffffffu, most[k], d));
            if (!stored) continue;
            float *const scales = const_cast<float *>(is_v ? c.v_scales : c.k_scales);
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                float m = most[0];
                #pragma unroll
                for (uint32_t k = 1; k < kBlocks; ++k) m = group[e] / 8 == k ? most[k] : m;
                static_cast<uint32_t *>(pool)[to + group[e]] = codes_of_group(v[e], m, s_cells);
                if ((group[e] & 7u) == 0) scales[(to + group[e]) / 8] = m;
            }
        }
    }
}

typedef void (*RotatedKernel)(CacheView, BatchView, Rotated);

template <int D, uint32_t BATCH>
RotatedKernel kernel_of(bool nf4, bool bf16) {
    if (nf4) return bf16 ? append_rotated_kernel<D, true, true, BATCH> : append_rotated_kernel<D, true, false, BATCH>;
    return bf16 ? append_rotated_kernel<D, false, true, BATCH> : append_rotated_kernel<D, false, false, BATCH>;
}
template <int D>
RotatedKernel kernel_of(bool nf4, bool bf16, uint32_t batch) { return batch == 1 ? kernel_of<D, 1>(nf4, bf16) : kernel_of<D, 4>(nf4, bf16); }

}  // namespace

}  // namespace nf4

using namespace nf4;

extern "C" {

int32_t nf4_cache_append_rotated_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const nf4_rotation *rotation, const void *k, uint64_t ldk,
                                     const void *v, uint64_t ldv, const void *q, uint64_t ldq, uint32_t q_heads, void *q_out, uint64_t ldo, int32_t io_dtype,
                                     void *stream) {
    const char *const what = "nf4_cache_append_rotated_dev";
    NF4_TRY(check_cache(what, cache, batch));
    if (!rotation || rotation->struct_bytes != sizeof(nf4_rotation)) return fail(NF4_ERR_INVALID_ARG, "%s: rotation is null or its struct_bytes wrong", what);
    if (rotation->rotary_dim == 0 || rotation->rotary_dim % 16 != 0 || rotation->rotary_dim > cache->head_dim)
        return fail(NF4_ERR_UNSUPPORTED, "%s: rotary_dim is %u; multiples of 16 up to head_dim are supported", what, rotation->rotary_dim);
    if (rotation->table_positions >= 1u << 31) return fail(NF4_ERR_UNSUPPORTED, "%s: a table of 2^31 positions or more", what);
    if (rotation->table_positions && !rotation->table) return fail(NF4_ERR_INVALID_ARG, "%s: the rotation's table is null", what);
    if (!aligned16(rotation->table)) return fail(NF4_ERR_INVALID_ARG, "%s: the rotation's table must be 16-byte aligned", what);
    if (q_heads > 65535) return fail(NF4_ERR_UNSUPPORTED, "%s: %u query heads; 65535 are supported", what, q_heads);
    if (!batch->rows || !batch->sequences) return NF4_OK;
    const uint64_t width = (uint64_t)cache->heads * cache->head_dim, q_width = (uint64_t)q_heads * cache->head_dim;
    NF4_TRY(check_rows(what, "k", k, &ldk, width, io_dtype));
    NF4_TRY(check_rows(what, "v", v, &ldv, width, io_dtype));
    if (q_heads) {
        NF4_TRY(check_rows(what, "q", q, &ldq, q_width, io_dtype));
        NF4_TRY(check_rows(what, "q_out", q_out, &ldo, q_width, io_dtype));
        if (q == q_out && ldq != ldo) return fail(NF4_ERR_INVALID_ARG, "%s: q_out is q with another row stride", what);
    }
    Rotated t{k, v, q, q_out, ldk, ldv, ldq, ldo, rotation->table, rotation->positions, rotation->table_positions, rotation->rotary_dim, q_heads, rotation->pairs != 0, 0, 0, 1};
    const uint32_t lanes = cache->head_dim / 16, slots = kMostThreads / lanes, vectors = q_heads + 2 * cache->heads;
    // One vector to a thread where that leaves no SM more than two CTAs: such a call takes what its chain of loads takes.  Else four.
    const uint32_t batch_of = (uint64_t)batch->rows * vectors <= 2ull * kNumSMs * slots ? 1 : 4;
    const uint32_t across = (vectors + slots * batch_of - 1) / (slots * batch_of);  // CTAs to a row
    t.width = (vectors + across * batch_of - 1) / (across * batch_of);
    t.abreast = std::max(1u, slots / t.width);
    // A CTA finds its rows' places once, a chain of four loads: so many rounds that the CTAs which an SM has registers for (128 a thread) do all (measured with 7,345
    // rows of 28 + 8 heads of 128, NF4 / bf16: one round to a CTA 42 / 36 us, as many as that 29 / 25)
    const uint32_t threads = (t.abreast * t.width * lanes + 31) / 32 * 32, ctas = kNumSMs * std::max(1u, 512u / threads);
    const uint64_t in_turn = ((uint64_t)batch->rows + t.abreast - 1) / t.abreast * across;
    t.rounds = (uint32_t)std::min<uint64_t>(kMostRows / t.abreast, (in_turn + ctas - 1) / ctas);
    const uint32_t rows_of_cta = t.abreast * t.rounds;
    const dim3 grid((batch->rows + rows_of_cta - 1) / rows_of_cta, across);
    const bool nf4 = cache->form == NF4_CACHE_NF4, bf16 = io_dtype == NF4_DTYPE_BF16;
    count_launch();
    return launch_maybe_overlapped(cache->head_dim == 64 ? kernel_of<64>(nf4, bf16, batch_of) : cache->head_dim == 128 ? kernel_of<128>(nf4, bf16, batch_of) : kernel_of<256>(nf4, bf16, batch_of),
                                   grid, dim3(threads), 0, static_cast<cudaStream_t>(stream), true, view_of(*cache), view_of(*batch), t);
}

}  // extern "C"
