// Attention of a call's rows over the paged cache: the entry points, the kernel for f32 tensors, and the join of parts.
#include <algorithm>
#include <type_traits>

#include "kv_cache.cuh"
#include "ptx.cuh"

namespace nf4 {

namespace {

// ---- f32 throughout ---------------------------------------------------------------------------------
// A CTA has a tile of 64 rows of one head of the cache (32 in the same four warps, 16 or 8 in one, where there are no more) and goes over its
// tokens 32 at a time (16 with one warp or a dim of 256, 8 with both): four or two rows to a thread, by every eighth token for the scores and by
// dim / 8 values for the results, weights from one to the other through shared memory, with the running largest exponent and sum of a
// softmax that is never held whole.  A row's scores are eight neighbouring lanes'.  FMAs are done in pairs.  Bound by shared
// memory, which gives registers 128 bytes a clock, so that 16 bytes to a lane take four whatever is broadcast: with four rows 8 such reads
// to 32 pairs of FMAs for the scores and 5 to 32 for the results (of 128), 24 to 32 TFLOP/s over long prompts.  (16 sequences of 4096 tokens, 7 rows of
// four heads of 128, the cache in L2: 110 us; with tiles of 64 rows 280, of 16 rows in four warps, one to a thread, 174.)
constexpr int kThreads = 256;

constexpr uint32_t tokens_of_tile(uint32_t dim, uint32_t warps) { return (dim == 256 ? 16 : 32) / (warps == 1 ? 2 : 1); }

// R: rows to a thread; W: warps, of 4 R rows each
template <int D, int R, int W>
struct F32Shape {
    static constexpr uint32_t kThreads = 32 * W, kRows = 4 * R * W, kTokens = tokens_of_tile(D, W), kPitch = D + 4, kPPitch = kRows + 4;
    static constexpr uint32_t kSmem = 4 * (kRows * kPitch + 2 * kTokens * kPitch + kTokens * kPPitch);
};

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 c, a, b, c;\n mov.b64 {%0, %1}, c;}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

template <int R>
__device__ __forceinline__ void put(float *to, const float (&v)[R]) {
    if constexpr (R == 4) *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2 *>(to) = make_float2(v[0], v[1]);
}
template <int R>
__device__ __forceinline__ void get(const float *from, float (&v)[R]) {
    if constexpr (R == 4) {
        const float4 w = *reinterpret_cast<const float4 *>(from);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
        const float2 w = *reinterpret_cast<const float2 *>(from);
        v[0] = w.x; v[1] = w.y;
    }
}

// TREE: rows are nodes of trees, which see their sequence's tokens ahead of the nodes and those nodes that their masks have
template <int D, bool NF4, int R, int W, bool TREE>
__global__ void __launch_bounds__(32 * W)
attention_f32_kernel(const CacheView c, const BatchView b, const AttentionView a) {
    using S = F32Shape<D, R, W>;
    constexpr uint32_t kCtaThreads = S::kThreads, kRows = S::kRows, kTokens = S::kTokens, kOwn = kTokens / 8;  // kOwn: tokens of a tile that a thread has scores of
    extern __shared__ __align__(16) float smem[];
    float *const sq = smem, *const sk = sq + kRows * S::kPitch, *const sv = sk + kTokens * S::kPitch, *const sp = sv + kTokens * S::kPitch;
    __shared__ float s_levels[16];
    const uint32_t tid = threadIdx.x, tx = tid & 7u, ty = tid >> 3;
    if (tid < 16) s_levels[tid] = __uint_as_float(c_level_bits[tid]);
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const uint32_t part = blockIdx.x, head = blockIdx.y % c.heads, seq = blockIdx.z;
    const Sequence s = sequence_of(c, b, seq);
    const uint32_t rows = s.rows * a.group;  // (below 2^31: the call's rows times its heads are)
    const uint32_t q_heads = c.heads * a.group;
    for (uint32_t r0 = blockIdx.y / c.heads * kRows; r0 < rows; r0 += gridDim.y / c.heads * kRows) {
        const uint32_t n = min(kRows, rows - r0);
        __syncthreads();
        for (uint32_t i = tid; i < kRows * (D / 4); i += kCtaThreads) {
            const uint32_t r = i / (D / 4), d = 4 * (i % (D / 4));
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < n) {
                const uint32_t token = a.by_group.of(r0 + r), h = r0 + r - token * a.group;
                v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + (uint64_t)(s.row0 + token) * a.ldq + (uint64_t)(head * a.group + h) * D + d);
            }
            *reinterpret_cast<float4 *>(sq + r * S::kPitch + d) = v;
        }
        // the tokens that this thread's rows see (TREE: the rows' numbers, kBlind where they see nothing), and those that any row of the tile does
        constexpr uint32_t kBlind = 0xffffffffu;
        uint32_t sees[R];
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            if (TREE) {
                const uint32_t token = a.by_group.of(r0 + min(R * ty + i, n - 1));
                sees[i] = R * ty + i < n && first_node(s) + (int32_t)token >= 0 ? s.row0 + token : kBlind;
            } else {
                sees[i] = R * ty + i < n ? visible_end(s, a.by_group, r0 + R * ty + i) : 0u;
            }
        }
        const uint32_t end = seen_end<TREE>(s, a.by_group, r0 + n - 1), tiles = (end + kTokens - 1) / kTokens;
        const uint32_t tile0 = (uint32_t)((uint64_t)tiles * part / a.parts), tile1 = (uint32_t)((uint64_t)tiles * (part + 1) / a.parts);
        float most[R], sum[R] = {};
        float2 acc[R][D / 16] = {};
        #pragma unroll
        for (int i = 0; i < R; ++i) most[i] = -INFINITY;
        // a tile's keys and values, kLoads groups of eight to a thread, asked for while the tile before is worked on
        constexpr uint32_t kLoads = 2 * kTokens * (D / 8) / kCtaThreads;
        uint4 raw[kLoads];
        float scale[kLoads];
        uint32_t state = 0;  // two bits to a group: 1 behind the last token, 2 in a page that there is not
        auto ask = [&](uint32_t tile) {
            state = 0;
            #pragma unroll
            for (uint32_t l = 0; l < kLoads; ++l) {
                const uint32_t i = tid + l * kCtaThreads, which = i / (kTokens * (D / 8)), j = i % (kTokens * (D / 8)), g = j % (D / 8);
                const uint32_t token = tile * kTokens + j / (D / 8);
                if (token >= end) {
                    state |= 1u << 2 * l;
                    continue;
                }
                const uint32_t at = c.by_page.of(token);
                const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at);
                if (page < 0 || (uint32_t)page >= c.pages) {
                    state |= 2u << 2 * l;
                    continue;
                }
                const uint64_t from = (((uint64_t)page * c.heads + head) * c.page_size + (token - at * c.page_size)) * (D / 8) + g;
                const void *const pool = which ? c.v : c.k;
                if (NF4) {
                    raw[l].x = __ldg(static_cast<const uint32_t *>(pool) + from);
                    scale[l] = __ldg((which ? c.v_scales : c.k_scales) + (from >> 3));
                } else {
                    raw[l] = __ldg(static_cast<const uint4 *>(pool) + from);
                }
            }
        };
        if (tile0 < tile1) ask(tile0);
        for (uint32_t tile = tile0; tile < tile1; ++tile) {
            const uint32_t t0 = tile * kTokens;
            __syncthreads();
            #pragma unroll
            for (uint32_t l = 0; l < kLoads; ++l) {
                const uint32_t i = tid + l * kCtaThreads, which = i / (kTokens * (D / 8)), j = i % (kTokens * (D / 8)), t = j / (D / 8), g = j % (D / 8);
                const uint32_t is = state >> 2 * l & 3u;
                float v[8];
                if (is) {
                    #pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = is == 1 ? 0.f : __uint_as_float(0x7fc00000u);  // NaN
                } else if (NF4) {
                    values_of_codes(raw[l].x, scale[l], s_levels, v);
                } else {
                    values_of_bf16(raw[l], v);
                }
                float *const to = (which ? sv : sk) + t * S::kPitch + 8 * g;
                const uint32_t half = g & 4u;  // (which comes first: so that eight lanes' stores hit all banks)
                *reinterpret_cast<float4 *>(to + half) = half ? make_float4(v[4], v[5], v[6], v[7]) : make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(to + (half ^ 4u)) = half ? make_float4(v[0], v[1], v[2], v[3]) : make_float4(v[4], v[5], v[6], v[7]);
            }
            if (tile + 1 < tile1) ask(tile + 1);
            __syncthreads();
            float2 pairs[R][kOwn] = {};  // the scores' sums over even and odd places
            #pragma unroll 4
            for (uint32_t d = 0; d < D; d += 4) {
                float4 q[R], k[kOwn];
                #pragma unroll
                for (int i = 0; i < R; ++i) q[i] = *reinterpret_cast<const float4 *>(sq + (R * ty + i) * S::kPitch + d);
                #pragma unroll
                for (int j = 0; j < kOwn; ++j) k[j] = *reinterpret_cast<const float4 *>(sk + (tx + 8 * j) * S::kPitch + d);
                #pragma unroll
                for (int i = 0; i < R; ++i)
                    #pragma unroll
                    for (int j = 0; j < kOwn; ++j) {
                        pairs[i][j] = fma2(make_float2(q[i].x, q[i].y), make_float2(k[j].x, k[j].y), pairs[i][j]);
                        pairs[i][j] = fma2(make_float2(q[i].z, q[i].w), make_float2(k[j].z, k[j].w), pairs[i][j]);
                    }
            }
            float x[kOwn][R];
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                float top = most[i];
                uint32_t window = ~0u;  // TREE: bit k: the row sees token t0 + k
                if (TREE) {
                    if ((int32_t)(t0 + kTokens) > first_node(s) && sees[i] != kBlind) window = seen_nodes(a, sees[i], (int32_t)t0 - first_node(s));
                    window = sees[i] == kBlind ? 0u : window & low_bits(end - t0);
                }
                #pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    x[j][i] = (TREE ? window >> (tx + 8 * j) & 1u : t0 + tx + 8 * j < sees[i]) ? (pairs[i][j].x + pairs[i][j].y) * a.scale_log2 : -INFINITY;
                    top = fmaxf(top, x[j][i]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                const float base = top == -INFINITY ? 0.f : top;  // (nothing seen so far: every weight is 0)
                const float keep = exp2f(most[i] - base);
                most[i] = top;
                sum[i] *= keep;
                #pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    acc[i][k].x *= keep;
                    acc[i][k].y *= keep;
                }
                #pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    x[j][i] = exp2f(x[j][i] - base);
                    sum[i] += x[j][i];
                }
            }
            #pragma unroll
            for (int j = 0; j < kOwn; ++j) put<R>(sp + (tx + 8 * j) * S::kPPitch + R * ty, x[j]);
            __syncwarp();  // (a row's weights are written and read by the same eight lanes)
            #pragma unroll 4
            for (uint32_t t = 0; t < kTokens; ++t) {
                float w[R];
                get<R>(sp + t * S::kPPitch + R * ty, w);
                #pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const float4 v = *reinterpret_cast<const float4 *>(sv + t * S::kPitch + 4 * tx + 32 * j);
                    #pragma unroll
                    for (int i = 0; i < R; ++i) {
                        acc[i][2 * j] = fma2(make_float2(w[i], w[i]), make_float2(v.x, v.y), acc[i][2 * j]);
                        acc[i][2 * j + 1] = fma2(make_float2(w[i], w[i]), make_float2(v.z, v.w), acc[i][2 * j + 1]);
                    }
                }
            }
        }
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 4);
            if (R * ty + i >= n) continue;
            const uint32_t r = r0 + R * ty + i, token = a.by_group.of(r), row = s.row0 + token, h = head * a.group + (r - token * a.group);
            if (a.parts > 1) {
                const uint64_t at = ((uint64_t)part * b.rows + row) * q_heads + h;
                if (tx == 0) a.part_ml[at] = make_float2(most[i], sum[i]);
                #pragma unroll
                for (int j = 0; j < D / 32; ++j)
                    *reinterpret_cast<float4 *>(a.part_o + at * D + 4 * tx + 32 * j) =
                        make_float4(acc[i][2 * j].x, acc[i][2 * j].y, acc[i][2 * j + 1].x, acc[i][2 * j + 1].y);
                continue;
            }
            const float f = sum[i] == 0.f ? 0.f : 1.f / sum[i];
            float *const out = static_cast<float *>(a.out) + (uint64_t)row * a.ldo + (uint64_t)h * D;
            #pragma unroll
            for (int j = 0; j < D / 32; ++j)
                *reinterpret_cast<float4 *>(out + 4 * tx + 32 * j) = make_float4(acc[i][2 * j].x * f, acc[i][2 * j].y * f, acc[i][2 * j + 1].x * f, acc[i][2 * j + 1].y * f);
        }
    }
}

// ---- the join of parts ------------------------------------------------------------------------------
// A CTA to a row of a query head: a warp takes every eighth part, in their order, by the largest exponent so far; then the warps' sums
// are joined in theirs, so that the result does not depend on which was ready first.  Rows of no sequence have no parts and are left
// alone.  (A warp to a row took 20 us for 64 parts, a chain of their loads.)
template <int D>
__global__ void __launch_bounds__(kThreads)
join_kernel(const BatchView b, const AttentionView a, uint32_t q_heads) {
    constexpr uint32_t W = kThreads / 32;
    __shared__ float2 s_ml[W];
    __shared__ float s_acc[W][D];
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const uint32_t i = blockIdx.x, all = b.rows * q_heads, lane = threadIdx.x & 31u, warp = threadIdx.x / 32;  // (below 2^31)
    const uint32_t row = i / q_heads, h = i - row * q_heads;
    if ((int32_t)row < __ldg(b.starts) || (int32_t)row >= __ldg(b.starts + b.sequences)) return;
    float top = -INFINITY, sum = 0.f, acc[D / 32] = {};
    #pragma unroll 4
    for (uint32_t p = warp; p < a.parts; p += W) {
        const float2 ml = __ldg(a.part_ml + (uint64_t)p * all + i);
        const float *const o = a.part_o + ((uint64_t)p * all + i) * D + lane * (D / 32);
        float2 v[D / 64];
        #pragma unroll
        for (int j = 0; j < D / 64; ++j) v[j] = __ldg(reinterpret_cast<const float2 *>(o) + j);
        const float now = fmaxf(top, ml.x), base = now == -INFINITY ? 0.f : now;
        const float keep = exp2f(top - base), f = ml.y == 0.f ? 0.f : exp2f(ml.x - base);  // (a NaN stays one)
        top = now;
        sum = fmaf(f, ml.y, sum * keep);
        #pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            acc[2 * j] = fmaf(f, ml.y == 0.f ? 0.f : v[j].x, acc[2 * j] * keep);
            acc[2 * j + 1] = fmaf(f, ml.y == 0.f ? 0.f : v[j].y, acc[2 * j + 1] * keep);
        }
    }
    if (lane == 0) s_ml[warp] = make_float2(top, sum);
    #pragma unroll
    for (int j = 0; j < D / 32; ++j) s_acc[warp][lane * (D / 32) + j] = acc[j];
    __syncthreads();
    if (threadIdx.x >= D) return;
    top = -INFINITY;
    #pragma unroll
    for (uint32_t w = 0; w < W; ++w) top = fmaxf(top, s_ml[w].x);
    const float base = top == -INFINITY ? 0.f : top;
    float value = 0.f;
    sum = 0.f;
    #pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
        const float f = exp2f(s_ml[w].x - base);
        sum = fmaf(f, s_ml[w].y, sum);
        value = fmaf(f, s_acc[w][threadIdx.x], value);
    }
    static_cast<float *>(a.out)[(uint64_t)row * a.ldo + (uint64_t)h * D + threadIdx.x] = sum == 0.f ? 0.f : value * (1.f / sum);
}

// ---- how a call is carried out -----------------------------------------------------------------------
// Which of two kernels: the one that streams the cache reads a head's tokens once for every 16 rows, the one for many rows once for
// every 256 (128 with a dim of 256).  By what each takes, in tenths of a microsecond on an SM: a row tile's start, and 128 tokens of
// it; the second kernel's own start, its joins and the expansion ahead of it are 15 to 20 us more.  Measured on both sides (us, first / second):
// 16 sequences of 8192 tokens, 8 heads of 128, NF4: 16 rows 61 / 161, 48 rows 159 / 162, 64 rows 207 / 162; bf16: 16 rows 95 / 123, 32 rows
// 173 / 124; one such sequence, NF4: 96 rows 28 / 37, 128 rows 36 / 37, 192 rows 48 / 40; 4 sequences of 512, 4 heads, NF4: 384 rows 24 / 26, 768
// rows 43 / 34, bf16: 256 rows 24 / 23, 384 rows 29 / 23; 8 of 4096, 4 heads of 256, NF4: 16 rows 41 / 57, 32 rows 67 / 57; 8 heads of 64, NF4: 64
// rows 50 / 48, 96 rows 68 / 48, bf16: 64 rows 41 / 40, 96 rows 56 / 40.
bool takes_decode(const AttentionCall &c) {
    if (c.f32) return false;
    if (!(c.tree ? attention_tree_counts(c) : attention_chunk_counts(c))) return true;  // (the other counts in 64 bits)
    const int of_dim = c.head_dim == 64 ? 0 : c.head_dim == 128 ? 1 : 2;
    static constexpr double kStream[2][3] = {{5, 11, 32}, {7, 9, 45}}, kMany[2][3] = {{13, 18, 40}, {19, 25, 58}};  // [NF4][dim]
    // row tiles of all sequences: by the most rows of one, or by all rows where that says less
    auto tiles = [&](uint64_t rows) -> double {
        const uint64_t group = c.view.group, all = (uint64_t)c.batch.rows * group / rows + c.batch.sequences;
        return (double)std::min<uint64_t>(all, c.batch.sequences * (((uint64_t)c.most_rows * group + rows - 1) / rows));
    };
    const double steps = c.most_tokens / 128 + 1, heads = c.cache.heads;
    if (c.tree) {
        // Likewise, trees having a kernel of their own for many rows (us, first / second; 16 sequences of 8192 tokens, 8 heads of 128, NF4: 16 rows of a head 62 /
        // 97, 32 rows 112 / 97, 64 rows 209 / 97; bf16: 94 / 90, 174 / 90, 32 rows of 64 81 / 86 and 89 / 75; one sequence, 4 heads, 112 rows, NF4: 8192 tokens
        // 21 / 20, 65536 93 / 40, four of 512 10 / 18)
        static constexpr double kTreeStream[2][3] = {{7, 14, 36}, {7, 9, 45}}, kTreeMany[2][3] = {{11, 14, 50}, {13, 16, 55}};
        return tiles(16) * heads * (32 + steps * kTreeStream[c.nf4][of_dim]) <= tiles(128) * heads * (64 + steps * kTreeMany[c.nf4][of_dim]) + kNumSMs * 90;
    }
    const double stream = tiles(16) * heads * (32 + steps * kStream[c.nf4][of_dim]);
    const double many = tiles(c.head_dim == 256 ? 128 : 256) * heads * (90 + steps * kMany[c.nf4][of_dim]) + kNumSMs * (c.nf4 ? 200 : 150);
    return stream <= many;
}

struct Plan {
    uint32_t row_tiles, parts;  // CTAs to a head of a sequence: row tiles side by side, and parts of the tokens
    uint32_t rows, warps;       // rows to a thread, warps of a CTA
};

Plan plan_of(const AttentionCall &c) {
    Plan p;
    const uint64_t rows = (uint64_t)c.most_rows * c.view.group;
    p.warps = rows <= 16 ? 1 : 4;
    p.rows = rows <= 8 || (rows > 16 && rows <= 32) ? 2 : 4;
    const uint64_t of_tile = 4 * p.rows * p.warps, tiles = std::max<uint64_t>(1, (rows + of_tile - 1) / of_tile);
    p.row_tiles = (uint32_t)std::min<uint64_t>(tiles, 65535 / c.cache.heads);
    // four CTAs to an SM, of 32 rows eight, of one warp sixteen, as near as parts of equally many token tiles come to it (measured with two, three, four
    // and six: 29, 26, 23 and 27 us for three prompts of 100 rows over 700 tokens, two heads of 64; of one warp with 10, 16 and 24: 70, 53 and 68
    // us for 16 sequences of 4096 tokens, four heads of 64); 256 parts at most (with 32, 64, 128 and 256 one row over 65536 tokens took 711, 364, 226
    // and 132 us)
    const uint64_t ctas = (uint64_t)p.row_tiles * c.cache.heads * std::max(1u, c.batch.sequences);
    const uint64_t tokens = tokens_of_tile(c.head_dim, p.warps), token_tiles = std::max<uint64_t>(1, (c.most_tokens + tokens - 1) / tokens);
    const uint64_t parts = std::min<uint64_t>(std::min<uint64_t>(256, token_tiles), std::max<uint64_t>(1, (p.warps == 1 ? 16 : p.rows == 4 ? 4 : 8) * kNumSMs / ctas));
    const uint64_t tiles_of_part = (token_tiles + parts - 1) / parts;
    p.parts = (uint32_t)((token_tiles + tiles_of_part - 1) / tiles_of_part);
    return p;
}

uint64_t part_ml_bytes(const AttentionCall &c, uint32_t parts) {
    return ((uint64_t)parts * c.batch.rows * c.cache.heads * c.view.group * sizeof(float2) + 255) / 256 * 256;
}
uint64_t workspace_bytes_of(const AttentionCall &c, const Plan &p) {
    if (!c.f32) return takes_decode(c) ? attention_decode_bytes(c) : c.tree ? attention_tree_bytes(c) : attention_chunk_bytes(c);
    if (p.parts == 1) return kAttentionFlagBytes;
    return kAttentionFlagBytes + part_ml_bytes(c, p.parts) + (uint64_t)p.parts * c.batch.rows * c.cache.heads * c.view.group * c.head_dim * sizeof(float);
}

template <int D, bool NF4, int R, int W>
int32_t launch_f32(const AttentionCall &c, const Plan &p, cudaStream_t stream) {
    auto kernel = c.tree ? attention_f32_kernel<D, NF4, R, W, true> : attention_f32_kernel<D, NF4, R, W, false>;
    constexpr uint32_t kSmem = F32Shape<D, R, W>::kSmem;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), kSmem));
    count_launch();
    return launch_maybe_overlapped(kernel, dim3(p.parts, p.row_tiles * c.cache.heads, c.batch.sequences), dim3(32 * W), kSmem,
                                   stream, true, c.cache, c.batch, c.view);
}
template <int D>
int32_t launch_of(const AttentionCall &c, const Plan &p, cudaStream_t stream) {
    auto launch = [&](auto nf4) {
        constexpr bool kNf4 = decltype(nf4)::value;
        if (p.warps == 1) return p.rows == 2 ? launch_f32<D, kNf4, 2, 1>(c, p, stream) : launch_f32<D, kNf4, 4, 1>(c, p, stream);
        return p.rows == 2 ? launch_f32<D, kNf4, 2, 4>(c, p, stream) : launch_f32<D, kNf4, 4, 4>(c, p, stream);
    };
    NF4_TRY((c.nf4 ? launch(std::true_type()) : launch(std::false_type())));
    if (p.parts == 1) return NF4_OK;
    const uint32_t q_heads = c.cache.heads * c.view.group;
    count_launch();
    return launch_maybe_overlapped(join_kernel<D>, dim3(c.batch.rows * q_heads), dim3(kThreads), 0, stream, true, c.batch, c.view, q_heads);
}

AttentionCall call_of(const nf4_cache &cache, const nf4_cache_batch &batch, uint32_t q_heads, int32_t io_dtype, bool tree) {
    AttentionCall c{};
    c.tree = tree;
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

uint64_t call_flag_bytes(const char *what, const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype, bool tree) {
    if (check_cache(what, cache, batch) != NF4_OK || check_heads(what, *cache, *batch, q_heads) != NF4_OK) return kAttentionFlagBytes;
    return takes_decode(call_of(*cache, *batch, q_heads, io_dtype, tree)) ? kAttentionFlagBytes : 0;
}

uint64_t workspace_bytes(const char *what, const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype, bool tree) {
    if (check_cache(what, cache, batch) != NF4_OK || check_heads(what, *cache, *batch, q_heads) != NF4_OK) return 0;
    const AttentionCall c = call_of(*cache, *batch, q_heads, io_dtype, tree);
    return workspace_bytes_of(c, plan_of(c));
}

// tree: the rows are nodes that see what their masks say
int32_t attention(const char *what, const nf4_cache *cache, const nf4_cache_batch *batch, const uint32_t *masks, uint32_t mask_words, bool tree,
                  const nf4_attention_args *args, void *stream) {
    NF4_TRY(check_cache(what, cache, batch));
    if (!args || args->struct_bytes != sizeof(nf4_attention_args)) return fail(NF4_ERR_INVALID_ARG, "%s: args is null or its struct_bytes wrong", what);
    NF4_TRY(check_heads(what, *cache, *batch, args->q_heads));
    if (!(args->scale - args->scale == 0.0f)) return fail(NF4_ERR_INVALID_ARG, "%s: scale is not finite", what);
    if (mask_words > 1u << 26) return fail(NF4_ERR_UNSUPPORTED, "%s: masks of %u words; 2^26 are supported", what, mask_words);
    if (!batch->rows || !batch->sequences) return NF4_OK;
    if (tree && mask_words && !masks) return fail(NF4_ERR_INVALID_ARG, "%s: masks is null", what);
    const uint64_t width = (uint64_t)args->q_heads * cache->head_dim;
    uint64_t ldq = args->ldq, ldo = args->ldo;
    NF4_TRY(check_rows(what, "q", args->q, &ldq, width, args->io_dtype));
    NF4_TRY(check_rows(what, "out", args->out, &ldo, width, args->io_dtype));
    AttentionCall c = call_of(*cache, *batch, args->q_heads, args->io_dtype, tree);
    c.view.masks = masks;
    c.view.words = mask_words;
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
        return takes_decode(c) ? attention_decode(c, workspace, s) : c.tree ? attention_tree(c, workspace, s) : attention_chunk(c, workspace, s);
    }
    return c.head_dim == 64 ? launch_of<64>(c, p, s) : c.head_dim == 128 ? launch_of<128>(c, p, s) : launch_of<256>(c, p, s);
}

}  // namespace

}  // namespace nf4

using namespace nf4;

extern "C" {

uint64_t nf4_cache_attention_flag_bytes(void) { return kAttentionFlagBytes; }

uint64_t nf4_cache_attention_call_flag_bytes(const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype) {
    return call_flag_bytes("nf4_cache_attention_call_flag_bytes", cache, batch, q_heads, io_dtype, false);
}
uint64_t nf4_cache_tree_attention_call_flag_bytes(const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype) {
    return call_flag_bytes("nf4_cache_tree_attention_call_flag_bytes", cache, batch, q_heads, io_dtype, true);
}

uint64_t nf4_cache_attention_workspace_bytes(const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype) {
    return workspace_bytes("nf4_cache_attention_workspace_bytes", cache, batch, q_heads, io_dtype, false);
}
uint64_t nf4_cache_tree_attention_workspace_bytes(const nf4_cache *cache, const nf4_cache_batch *batch, uint32_t q_heads, int32_t io_dtype) {
    return workspace_bytes("nf4_cache_tree_attention_workspace_bytes", cache, batch, q_heads, io_dtype, true);
}

int32_t nf4_cache_attention_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const nf4_attention_args *args, void *stream) {
    return attention("nf4_cache_attention_dev", cache, batch, nullptr, 0, false, args, stream);
}
int32_t nf4_cache_tree_attention_dev(const nf4_cache *cache, const nf4_cache_batch *batch, const uint32_t *masks, uint32_t mask_words,
                                     const nf4_attention_args *args, void *stream) {
    return attention("nf4_cache_tree_attention_dev", cache, batch, masks, mask_words, true, args, stream);
}

}  // extern "C"
