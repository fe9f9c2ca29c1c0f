// Attention of a call's rows over the paged cache: the entry points, the kernel for f32 tensors, and the join of parts.
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"

namespace nf4 {

namespace {

// ---- f32 throughout ---------------------------------------------------------------------------------
// A CTA has a tile of 64 rows of one head of the cache and goes over its tokens 32 at a time: scores 2 x 4 to a thread,
// weights through shared memory, values times weights 2 x dim / 8 to a thread, with the running largest exponent and sum of a
// softmax that is never held whole.  A row's scores are eight neighbouring lanes'.  Bound by FMAs: 32 of them to six
// 16-byte reads of shared memory.
constexpr int kThreads = 256;
constexpr uint32_t kRows = 64, kTokens = 32;

template <int D>
struct F32Shape {
    static constexpr uint32_t kPitch = D + 4, kPPitch = kTokens + 4;
    static constexpr uint32_t kSmem = 4 * (kRows * kPitch + 2 * kTokens * kPitch + kRows * kPPitch);
};

template <int D, bool NF4>
__global__ void __launch_bounds__(kThreads)
attention_f32_kernel(const CacheView c, const BatchView b, const AttentionView a) {
    using S = F32Shape<D>;
    extern __shared__ __align__(16) float smem[];
    float *const sq = smem, *const sk = sq + kRows * S::kPitch, *const sv = sk + kTokens * S::kPitch, *const sp = sv + kTokens * S::kPitch;
    __shared__ float s_levels[16];
    const uint32_t tid = threadIdx.x, tx = tid & 7u, ty = tid >> 3;
    if (tid < 16) s_levels[tid] = __uint_as_float(c_level_bits[tid]);
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const uint32_t part = blockIdx.x, head = blockIdx.y % c.heads, seq = blockIdx.z;
    const Sequence s = sequence_of(c, b, seq);
    const uint64_t rows = (uint64_t)s.rows * a.group;
    const uint32_t q_heads = c.heads * a.group;
    for (uint64_t r0 = (uint64_t)(blockIdx.y / c.heads) * kRows; r0 < rows; r0 += (uint64_t)(gridDim.y / c.heads) * kRows) {
        const uint32_t n = (uint32_t)min((uint64_t)kRows, rows - r0);
        __syncthreads();
        for (uint32_t i = tid; i < kRows * (D / 4); i += kThreads) {
            const uint32_t r = i / (D / 4), d = 4 * (i % (D / 4));
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < n) {
                const uint32_t token = (uint32_t)((r0 + r) / a.group), h = (uint32_t)((r0 + r) % a.group);
                v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + (uint64_t)(s.row0 + token) * a.ldq + (uint64_t)(head * a.group + h) * D + d);
            }
            *reinterpret_cast<float4 *>(sq + r * S::kPitch + d) = v;
        }
        // the tokens that this thread's two rows see, and those that any row of the tile does
        uint32_t sees[2];
        #pragma unroll
        for (int i = 0; i < 2; ++i) sees[i] = 2 * ty + i < n ? visible_end(s, a.by_group, (uint32_t)(r0 + 2 * ty + i)) : 0u;
        const uint32_t end = visible_end(s, a.by_group, (uint32_t)(r0 + n - 1)), tiles = (end + kTokens - 1) / kTokens;
        const uint32_t tile0 = (uint32_t)((uint64_t)tiles * part / a.parts), tile1 = (uint32_t)((uint64_t)tiles * (part + 1) / a.parts);
        float most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        float acc[2][D / 8] = {};
        for (uint32_t tile = tile0; tile < tile1; ++tile) {
            const uint32_t t0 = tile * kTokens;
            __syncthreads();
            for (uint32_t i = tid; i < 2 * kTokens * (D / 8); i += kThreads) {
                const uint32_t which = i / (kTokens * (D / 8)), j = i % (kTokens * (D / 8)), t = j / (D / 8), g = j % (D / 8);
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                const uint32_t token = t0 + t;
                if (token < end) {
                    const uint32_t at = c.by_page.of(token);
                    const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at);
                    if (page < 0 || (uint32_t)page >= c.pages) {
                        #pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(0x7fc00000u);  // NaN
                    } else {
                        const uint64_t from = (((uint64_t)page * c.heads + head) * c.page_size + (token - at * c.page_size)) * (D / 8) + g;
                        const void *const pool = which ? c.v : c.k;
                        if (NF4) values_of_codes(__ldg(static_cast<const uint32_t *>(pool) + from), __ldg((which ? c.v_scales : c.k_scales) + (from >> 3)), s_levels, v);
                        else values_of_bf16(__ldg(static_cast<const uint4 *>(pool) + from), v);
                    }
                }
                float *const to = (which ? sv : sk) + t * S::kPitch + 8 * g;
                *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
            __syncthreads();
            float x[2][4] = {};
            #pragma unroll 4
            for (uint32_t d = 0; d < D; d += 4) {
                float4 q[2], k[4];
                #pragma unroll
                for (int i = 0; i < 2; ++i) q[i] = *reinterpret_cast<const float4 *>(sq + (2 * ty + i) * S::kPitch + d);
                #pragma unroll
                for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4 *>(sk + (tx + 8 * j) * S::kPitch + d);
                #pragma unroll
                for (int i = 0; i < 2; ++i)
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[i][j] = fmaf(q[i].w, k[j].w, fmaf(q[i].z, k[j].z, fmaf(q[i].y, k[j].y, fmaf(q[i].x, k[j].x, x[i][j]))));
            }
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = most[i];
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[i][j] = t0 + tx + 8 * j < sees[i] ? x[i][j] * a.scale_log2 : -INFINITY;
                    top = fmaxf(top, x[i][j]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                const float base = top == -INFINITY ? 0.f : top;  // (nothing seen so far: every weight is 0)
                const float keep = exp2f(most[i] - base);
                most[i] = top;
                sum[i] *= keep;
                #pragma unroll
                for (int k = 0; k < D / 8; ++k) acc[i][k] *= keep;
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float w = exp2f(x[i][j] - base);
                    sum[i] += w;
                    sp[(2 * ty + i) * S::kPPitch + tx + 8 * j] = w;
                }
            }
            __syncwarp();  // (a row's weights are written and read by the same eight lanes)
            #pragma unroll 4
            for (uint32_t t = 0; t < kTokens; ++t) {
                const float w0 = sp[2 * ty * S::kPPitch + t], w1 = sp[(2 * ty + 1) * S::kPPitch + t];
                #pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const float4 v = *reinterpret_cast<const float4 *>(sv + t * S::kPitch + 4 * tx + 32 * j);
                    acc[0][4 * j] = fmaf(w0, v.x, acc[0][4 * j]); acc[0][4 * j + 1] = fmaf(w0, v.y, acc[0][4 * j + 1]);
                    acc[0][4 * j + 2] = fmaf(w0, v.z, acc[0][4 * j + 2]); acc[0][4 * j + 3] = fmaf(w0, v.w, acc[0][4 * j + 3]);
                    acc[1][4 * j] = fmaf(w1, v.x, acc[1][4 * j]); acc[1][4 * j + 1] = fmaf(w1, v.y, acc[1][4 * j + 1]);
                    acc[1][4 * j + 2] = fmaf(w1, v.z, acc[1][4 * j + 2]); acc[1][4 * j + 3] = fmaf(w1, v.w, acc[1][4 * j + 3]);
                }
            }
        }
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 4);
            if (2 * ty + i >= n) continue;
            const uint64_t r = r0 + 2 * ty + i;
            const uint32_t row = s.row0 + (uint32_t)(r / a.group), h = head * a.group + (uint32_t)(r % a.group);
            if (a.parts > 1) {
                const uint64_t at = ((uint64_t)part * b.rows + row) * q_heads + h;
                if (tx == 0) a.part_ml[at] = make_float2(most[i], sum[i]);
                #pragma unroll
                for (int j = 0; j < D / 32; ++j)
                    *reinterpret_cast<float4 *>(a.part_o + at * D + 4 * tx + 32 * j) =
                        make_float4(acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]);
                continue;
            }
            const float f = sum[i] == 0.f ? 0.f : 1.f / sum[i];
            float *const out = static_cast<float *>(a.out) + (uint64_t)row * a.ldo + (uint64_t)h * D;
            #pragma unroll
            for (int j = 0; j < D / 32; ++j)
                *reinterpret_cast<float4 *>(out + 4 * tx + 32 * j) = make_float4(acc[i][4 * j] * f, acc[i][4 * j + 1] * f, acc[i][4 * j + 2] * f, acc[i][4 * j + 3] * f);
        }
    }
}

// ---- the join of parts ------------------------------------------------------------------------------
// A warp to a row of a query head: parts by their largest exponents, in their order, so that the result does not depend on
// which was ready first.  Rows of no sequence have no parts and are left alone.
template <int D>
__global__ void __launch_bounds__(kThreads)
join_kernel(const BatchView b, const AttentionView a, uint32_t q_heads) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const uint64_t i = (uint64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32, all = (uint64_t)b.rows * q_heads;
    const uint32_t lane = threadIdx.x & 31u;
    if (i >= all) return;
    const uint32_t row = (uint32_t)(i / q_heads), h = (uint32_t)(i % q_heads);
    if ((int32_t)row < __ldg(b.starts) || (int32_t)row >= __ldg(b.starts + b.sequences)) return;
    float top = -INFINITY;
    for (uint32_t p = lane; p < a.parts; p += 32) top = fmaxf(top, __ldg(&a.part_ml[p * all + i].x));
    #pragma unroll
    for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc[D / 32] = {};
    #pragma unroll 4
    for (uint32_t p = 0; p < a.parts; ++p) {
        const float2 ml = __ldg(a.part_ml + p * all + i);
        const float f = ml.y == 0.f ? 0.f : exp2f(ml.x - base);  // (a NaN stays one)
        sum = fmaf(f, ml.y, sum);
        const float *const o = a.part_o + (p * all + i) * D + lane * (D / 32);
        #pragma unroll
        for (int j = 0; j < D / 32; j += 2) {
            const float2 v = ml.y == 0.f ? make_float2(0.f, 0.f) : __ldg(reinterpret_cast<const float2 *>(o + j));
            acc[j] = fmaf(f, v.x, acc[j]);
            acc[j + 1] = fmaf(f, v.y, acc[j + 1]);
        }
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    float *const out = static_cast<float *>(a.out) + (uint64_t)row * a.ldo + (uint64_t)h * D + lane * (D / 32);
    #pragma unroll
    for (int j = 0; j < D / 32; j += 2) *reinterpret_cast<float2 *>(out + j) = make_float2(acc[j] * f, acc[j + 1] * f);
}

// ---- how a call is carried out -----------------------------------------------------------------------
// Few rows to a head of a sequence: the kernel that streams the cache; its tiles have 16 rows, four of them read the tokens four times.
bool takes_decode(const AttentionCall &c) { return !c.f32 && (uint64_t)c.most_rows * c.view.group <= 64; }

struct Plan {
    uint32_t row_tiles, parts;  // CTAs to a head of a sequence: row tiles side by side, and parts of the tokens
};

Plan plan_of(const AttentionCall &c) {
    Plan p;
    const uint64_t tiles = std::max<uint64_t>(1, ((uint64_t)c.most_rows * c.view.group + kRows - 1) / kRows);
    p.row_tiles = (uint32_t)std::min<uint64_t>(tiles, 65535 / c.cache.heads);
    // two CTAs to an SM; a part has two token tiles at least
    const uint64_t ctas = (uint64_t)p.row_tiles * c.cache.heads * std::max(1u, c.batch.sequences);
    const uint64_t most = std::max<uint64_t>(1, c.most_tokens / (2 * kTokens));
    p.parts = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(64, most), std::max<uint64_t>(1, 2 * kNumSMs / ctas));
    return p;
}

uint64_t part_ml_bytes(const AttentionCall &c, uint32_t parts) {
    return ((uint64_t)parts * c.batch.rows * c.cache.heads * c.view.group * sizeof(float2) + 255) / 256 * 256;
}
uint64_t workspace_bytes_of(const AttentionCall &c, const Plan &p) {
    if (!c.f32) return takes_decode(c) ? attention_decode_bytes(c) : attention_chunk_bytes(c);
    if (p.parts == 1) return kAttentionFlagBytes;
    return kAttentionFlagBytes + part_ml_bytes(c, p.parts) + (uint64_t)p.parts * c.batch.rows * c.cache.heads * c.view.group * c.head_dim * sizeof(float);
}

template <int D, bool NF4>
int32_t launch_f32(const AttentionCall &c, const Plan &p, cudaStream_t stream) {
    auto kernel = attention_f32_kernel<D, NF4>;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), F32Shape<D>::kSmem));
    count_launch();
    return launch_maybe_overlapped(kernel, dim3(p.parts, p.row_tiles * c.cache.heads, c.batch.sequences), dim3(kThreads), F32Shape<D>::kSmem,
                                   stream, true, c.cache, c.batch, c.view);
}
template <int D>
int32_t launch_of(const AttentionCall &c, const Plan &p, cudaStream_t stream) {
    NF4_TRY((c.nf4 ? launch_f32<D, true>(c, p, stream) : launch_f32<D, false>(c, p, stream)));
    if (p.parts == 1) return NF4_OK;
    const uint32_t q_heads = c.cache.heads * c.view.group;
    const uint64_t warps = (uint64_t)c.batch.rows * q_heads;
    count_launch();
    return launch_maybe_overlapped(join_kernel<D>, dim3((unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32))),
                                   dim3(kThreads), 0, stream, true, c.batch, c.view, q_heads);
}

AttentionCall call_of(const nf4_cache &cache, const nf4_cache_batch &batch, uint32_t q_heads, int32_t io_dtype) {
    AttentionCall c{};
    c.cache = view_of(cache);
    c.batch = view_of(batch);
    c.view.group = q_heads / cache.heads;
    c.view.by_group = FastDiv(c.view.group);
    c.nf4 = cache.form == NF4_CACHE_NF4;
    c.f32 = io_dtype == NF4_DTYPE_F32;
    c.head_dim = cache.head_dim;
    const uint64_t table = (uint64_t)batch.pages_per_sequence * cache.page_size;
    c.most_rows = batch.max_rows ? std::min(batch.max_rows, batch.rows) : batch.rows;
    c.most_tokens = (uint32_t)(batch.max_length ? std::min<uint64_t>(batch.max_length, table) : table);
    return c;
}

int32_t check_heads(const char *what, const nf4_cache &cache, const nf4_cache_batch &batch, uint32_t q_heads) {
    if (q_heads == 0 || q_heads % cache.heads != 0)
        return fail(NF4_ERR_INVALID_ARG, "%s: %u query heads are no multiple of the cache's %u", what, q_heads, cache.heads);
    if (q_heads > 65535 || (uint64_t)batch.rows * q_heads >= 1ull << 31)
        return fail(NF4_ERR_UNSUPPORTED, "%s: rows times query heads are 2^31 or more, or the heads above 65535", what);
    return NF4_OK;
}

}  // namespace

}  // namespace nf4

using namespace nf4;

extern "C" {

uint64_t nf4_cache_attention_flag_bytes(void) { return kAttentionFlagBytes; }

uint64_t nf4_cache_attention_workspace_bytes(const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype) {
    const char *const what = "nf4_cache_attention_workspace_bytes";
    if (check_cache(what, cache, batch) != NF4_OK || check_heads(what, *cache, *batch, q_heads) != NF4_OK) return 0;
    const AttentionCall c = call_of(*cache, *batch, q_heads, io_dtype);
    return workspace_bytes_of(c, plan_of(c));
}

int32_t nf4_cache_attention_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const nf4_attention_args *args, void *stream) {
    const char *const what = "nf4_cache_attention_dev";
    NF4_TRY(check_cache(what, cache, batch));
    if (!args || args->struct_bytes != sizeof(nf4_attention_args)) return fail(NF4_ERR_INVALID_ARG, "%s: args is null or its struct_bytes wrong", what);
    NF4_TRY(check_heads(what, *cache, *batch, args->q_heads));
    if (!(args->scale - args->scale == 0.0f)) return fail(NF4_ERR_INVALID_ARG, "%s: scale is not finite", what);
    if (!batch->rows || !batch->sequences) return NF4_OK;
    const uint64_t width = (uint64_t)args->q_heads * cache->head_dim;
    uint64_t ldq = args->ldq, ldo = args->ldo;
    NF4_TRY(check_rows(what, "q", args->q, &ldq, width, args->io_dtype));
    NF4_TRY(check_rows(what, "out", args->out, &ldo, width, args->io_dtype));
    AttentionCall c = call_of(*cache, *batch, args->q_heads, args->io_dtype);
    c.view.q = args->q;
    c.view.out = args->out;
    c.view.ldq = ldq;
    c.view.ldo = ldo;
    c.view.scale_log2 = args->scale * 1.44269504088896340736f;
    const Plan p = plan_of(c);
    const uint64_t need = workspace_bytes_of(c, p);
    if (!args->workspace || args->workspace_bytes < need)
        return fail(NF4_ERR_INVALID_ARG, "%s: the workspace has %llu bytes, this call needs %llu", what,
                    (unsigned long long)(args->workspace ? args->workspace_bytes : 0), (unsigned long long)need);
    if (reinterpret_cast<uintptr_t>(args->workspace) & 255u) return fail(NF4_ERR_INVALID_ARG, "%s: the workspace must be 256-byte aligned", what);
    uint8_t *const ws = static_cast<uint8_t *>(args->workspace) + kAttentionFlagBytes;
    c.view.parts = p.parts;
    c.view.part_ml = reinterpret_cast<float2 *>(ws);
    c.view.part_o = reinterpret_cast<float *>(ws + part_ml_bytes(c, p.parts));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!c.f32) {
        uint8_t *const workspace = static_cast<uint8_t *>(args->workspace);
        return takes_decode(c) ? attention_decode(c, workspace, s) : attention_chunk(c, workspace, s);
    }
    return c.head_dim == 64 ? launch_of<64>(c, p, s) : c.head_dim == 128 ? launch_of<128>(c, p, s) : launch_of<256>(c, p, s);
}

}  // extern "C"
