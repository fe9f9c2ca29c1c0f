// Attention of many rows over the paged cache (chunks of prompts, whole prompts) on the tensor cores.
//
// Bound by the MMAs (4 * dim operations for a row and a token) and by the exponentials beside them.  A CTA has 256 rows of one
// head of the cache (a token's query heads are neighbouring rows), or 128 with a dim of 256, as one or two MMA tiles of 128, and goes over the
// tokens 128 (or 64) a step.  Keys and values are in shared memory in f16 or bf16 with 128-byte swizzle: brought there by TMA from a bf16
// cache; looked up by four warps from codes that came by bulk copies, times their block's scale, from a quantized one, once for all
// of the CTA's rows.  One elected thread issues tcgen05.mma:
//   S = Q K^T   both operands from shared memory, 128 x 128 f32 sums in tensor memory
//   O += P V    P from tensor memory, where the softmax warps have put it over S; V as it lies, MN-major
// A softmax thread owns a row: it reads S, keeps the row's largest exponent m and sum l, and writes P = 2^(S c - m + 7) back as f16
// (bf16 with a bf16 cache).  While one tile's softmax runs, the other's two products do.  m is the largest exponent so far or up to 8
// below it: O is rescaled only where a row rises above that, by the warps themselves, at a moment when
// no product is writing it.
// f16's range: K's and V's scales are divided by the power of two of the largest among the CTA's tokens, a row of Q by its own
// (exact); the powers come back in f32.  f16 is off by 2^-12 on average, bf16 would be by 2^-9.
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace nf4 {

namespace {

constexpr uint32_t kThreads = 512;
// Weights are 2^(S c - m + kRaise): up to 2^15, so that f16 holds those that are 2^-32 of a row's largest; their sum is raised alike.
constexpr float kRaise = 7.f;
constexpr uint32_t kGroup = 16;  // tokens that are in one page for sure
// warps 0-3 and 4-7: softmax of a tile; 8-11: codes to f16; 12: copies; 13: MMAs
constexpr uint32_t kExpandWarp = 8, kCopyWarp = 12, kMmaWarp = 13;
// Registers: 512 threads are launched with 128 each; the two softmax warpgroups take 160 and leave 96 to the other two (together the
// same 65536).
constexpr uint32_t kSoftmaxRegs = 160, kOtherRegs = 96;

template <int D, bool NF4>
struct Shape {
    static constexpr uint32_t kTiles = D == 256 ? 1 : 2, kRows = 128 * kTiles;
    static constexpr uint32_t kTokens = D == 256 ? 64 : 128;          // of a step
    static constexpr uint32_t kBlocks = D / 64;
    static constexpr uint32_t kQTile = 128 * D * 2, kTile = kTokens * D * 2, kBox = kTokens * 128;
    static constexpr uint32_t kRaw = NF4 ? kTokens * (D / 2 + 4 * kBlocks) : 0, kRawSlots = 3;
    static constexpr uint32_t kSlots = NF4 ? (D == 64 ? 4 : 3) : 4;
    // codes, then the table on a multiple of its 32 KB, then Q, then the ring (bf16: Q, then the ring)
    static constexpr uint32_t kSmem = (NF4 ? 65536 : 2048) - 1024 + kTiles * kQTile + kSlots * kTile;
    static constexpr uint32_t kS = 0, kO = 256;                       // columns of tensor memory
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// Two at a time: half the instructions of the FMA pipe
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint4 ld_shared_u4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared_u4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// A power of two (as a float) that no scale up to `most` (bits) exceeds, between 2^-100 and 2^126.
__device__ __forceinline__ float power_above(uint32_t most) {
    return __uint_as_float(min(max((most & 0x7f800000u) + 0x00800000u, 27u << 23), 253u << 23));
}
__device__ __forceinline__ float reciprocal_of_power(float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); }

// row_tiles: the most that the call's rows can make of one head
template <int D, bool NF4>
__global__ void __launch_bounds__(kThreads, 1)
attention_chunk_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const CacheView c, const BatchView b,
                       const AttentionView a, uint32_t row_tiles, const FailureRef failure) {
    using S = Shape<D, NF4>;
    constexpr uint32_t N = S::kTokens, kBlocks = S::kBlocks;
    extern __shared__ uint8_t smem_any[];
    __shared__ __align__(8) uint64_t s_bars[19];
    __shared__ uint32_t s_tmem, s_most[2], s_bad;
    __shared__ float s_qpower[S::kRows];
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
    const uint32_t base = ptx::smem_addr(smem_any);
    const uint32_t raw0 = (base + 15u) & ~15u, table = (raw0 + S::kRawSlots * S::kRaw + 32767u) & ~32767u;
    const uint32_t q0 = NF4 ? table + 32768u : (base + 1023u) & ~1023u, ring0 = q0 + S::kTiles * S::kQTile;
    const uint32_t bars = ptx::smem_addr(s_bars), full0 = bars, empty0 = bars + 32, raw_full0 = bars + 64, raw_empty0 = bars + 88, s_full0 = bars + 112,
                   p_ready0 = bars + 128, tail_bar = bars + 144;
    if (ring0 + S::kSlots * S::kTile > base + S::kSmem) {
        if (tid == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 22);
        return;
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < S::kSlots; ++i) {
            ptx::mbar_init(full0 + 8 * i, NF4 ? 4 : 1);
            ptx::mbar_init(empty0 + 8 * i, 1);
        }
        for (uint32_t i = 0; i < 3; ++i) {
            ptx::mbar_init(raw_full0 + 8 * i, 1);
            ptx::mbar_init(raw_empty0 + 8 * i, 4);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            ptx::mbar_init(s_full0 + 8 * i, 1);
            ptx::mbar_init(p_ready0 + 8 * i, 4);
        }
        ptx::mbar_init(tail_bar, 1);
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
        s_most[0] = s_most[1] = s_bad = 0;
    }
    if (NF4) {
        for (uint32_t i = tid; i < 256 * 8; i += kThreads) {  // the table: an entry's copy to a lane
            const uint32_t byte = i >> 3, entry = level_pair_f16(byte);
            st_shared_u4(table + byte * 128u + (i & 7u) * 16u, make_uint4(entry, entry, entry, entry));
        }
    }
    if (warp == kMmaWarp) {
        ptx::tmem_alloc(ptx::smem_addr(&s_tmem), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = s_tmem;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    // ---- which rows: the last tiles, which see most, first ----
    const uint32_t part = blockIdx.y, head = blockIdx.x % c.heads, want = row_tiles - 1 - blockIdx.x / c.heads;
    uint32_t seq = b.sequences, r0 = 0;
    {
        uint32_t before = 0;
        for (uint32_t s0 = 0; s0 < b.sequences; s0 += 32) {
            uint32_t own = 0;
            if (s0 + lane < b.sequences) own = (uint32_t)(((uint64_t)sequence_of(c, b, s0 + lane).rows * a.group + S::kRows - 1) / S::kRows);
            uint32_t upto = own;
            #pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, upto, k);
                if (lane >= (uint32_t)k) upto += o;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + upto > want);
            if (past) {
                const int l0 = __ffs(past) - 1;
                seq = s0 + l0;
                r0 = (want - (before + __shfl_sync(0xffffffffu, upto - own, l0))) * S::kRows;
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    bool ok = true;
    if (seq < b.sequences) {
        const Sequence s = sequence_of(c, b, seq);
        const uint32_t rows = (uint32_t)min((uint64_t)S::kRows, (uint64_t)s.rows * a.group - r0), live = (rows + 127) / 128;
        const uint32_t end = visible_end(s, a.by_group, r0 + rows - 1), all = (end + N - 1) / N;
        const uint32_t step0 = (uint32_t)((uint64_t)all * part / a.parts), steps = (uint32_t)((uint64_t)all * (part + 1) / a.parts) - step0;
        const uint32_t t_first = step0 * N, t_end = min(end, t_first + steps * N);  // this CTA's tokens
        const uint32_t q_heads = c.heads * a.group;

        // ---- Q to shared memory; the largest scales of the CTA's tokens ----
        if (steps) {
            constexpr uint32_t kLanes = D / 8;  // to a row: eight values each
            const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a scale below zero: the rows change sign, so that c is not)
            #pragma unroll 4
            for (uint32_t i = tid; i < live * 128 * kLanes; i += kThreads) {
                const uint32_t r = i / kLanes, x = i % kLanes;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (r < rows) {
                    const uint32_t row = r0 + r;
                    w = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.q) + (uint64_t)(s.row0 + row / a.group) * a.ldq +
                                                               (uint64_t)(head * a.group + row % a.group) * D) + x);
                    w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
                }
                if (NF4) {
                    uint32_t u[4] = {w.x, w.y, w.z, w.w}, most = 0;
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) most = max(most, max((u[k] << 16) & 0x7fffffffu, u[k] & 0x7fff0000u));
                    #pragma unroll
                    for (uint32_t k = 1; k < kLanes; k <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, k));
                    // the row's largest magnitude is left in [2^11, 2^12)
                    const int e = most ? min(max((int)(most >> 23) - 127 - 11, -100), 115) : 0;
                    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) u[k] = pack<true>(__uint_as_float(u[k] << 16) * down, __uint_as_float(u[k] & 0xffff0000u) * down);
                    w = make_uint4(u[0], u[1], u[2], u[3]);
                    if (x == 0) s_qpower[r] = __uint_as_float((uint32_t)(127 + e) << 23);
                }
                const uint32_t tile = r >> 7, rr = r & 127u;
                st_shared_u4(q0 + tile * S::kQTile + (x >> 3) * 16384u + rr * 128u + (((x & 7u) ^ (rr & 7u)) << 4), w);
            }
            ptx::fence_proxy_async();
            uint32_t most_k = 0, most_v = 0;
            bool bad = false;
            for (uint32_t t = t_first + (NF4 ? tid : tid * kGroup); t < t_end; t += NF4 ? kThreads : kThreads * kGroup) {
                const uint32_t at = c.by_page.of(t);
                const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at);
                if (page < 0 || (uint32_t)page >= c.pages) {
                    bad = true;
                } else if (NF4) {
                    const uint64_t row = ((uint64_t)page * c.heads + head) * c.page_size + (t - at * c.page_size);
                    #pragma unroll
                    for (uint32_t k = 0; k < kBlocks; ++k) {
                        most_k = max(most_k, __float_as_uint(__ldg(c.k_scales + row * kBlocks + k)));
                        most_v = max(most_v, __float_as_uint(__ldg(c.v_scales + row * kBlocks + k)));
                    }
                }
            }
            if (NF4) {
                most_k = __reduce_max_sync(0xffffffffu, most_k);
                most_v = __reduce_max_sync(0xffffffffu, most_v);
                if (lane == 0) {
                    atomicMax(&s_most[0], most_k);
                    atomicMax(&s_most[1], most_v);
                }
            }
            if (bad) s_bad = 1;
        }
        __syncthreads();
        const float k_power = NF4 ? power_above(s_most[0]) : 1.f, v_power = NF4 ? power_above(s_most[1]) : 1.f;

        if (warp < 8) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            const uint32_t tile = warp >> 2, r = tid & 127u, row = r0 + tile * 128 + r;  // this thread's row
            if (tile < live) {
                const bool real = tile * 128 + r < rows;
                const uint32_t sees = real ? visible_end(s, a.by_group, row) : 0u, sees_first = visible_end(s, a.by_group, r0 + tile * 128);
                const float factor = fmaxf(fabsf(a.scale_log2) * (NF4 ? s_qpower[tile * 128 + r] * k_power : 1.f), 1.2e-38f);
                const uint32_t lanes = (warp & 3u) << 21;  // a warp reaches its quarter of tensor memory's lanes
                const uint32_t ts = tmem + S::kS + tile * N + lanes, to = tmem + S::kO + tile * D + lanes;
                float m = -INFINITY, l = 0.f;
                for (uint32_t j = 0; j < steps; ++j) {
                    if (!__all_sync(0xffffffffu, ptx::mbar_wait_suspended(s_full0 + 8 * tile, j & 1u))) {
                        ok = false;
                        if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 23);
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t t0 = t_first + j * N, lim = sees > t0 ? sees - t0 : 0u;
                    const bool masked = t0 + N > sees_first;
                    // Weights by m as it is, and only then the look at the largest score: where it is out of reach, once or twice a
                    // row, they are made again.  So nothing waits for a maximum, and S need not be held whole.
                    uint32_t p[N / 2];
                    float2 sum;
                    for (;;) {
                        const float from = m == -INFINITY ? 0.f : kRaise - m;
                        float top[2] = {-INFINITY, -INFINITY};
                        sum = make_float2(0.f, 0.f);
                        uint32_t ahead[2][32];  // 32 scores come while 32 are worked on
                        tmem_ld32(ts, ahead[0]);
                        #pragma unroll
                        for (uint32_t k = 0; k < N; k += 32) {
                            uint32_t (&x)[32] = ahead[k / 32 & 1];
                            ptx::tmem_wait_ld();
                            if (k + 32 < N) tmem_ld32(ts + k + 32, ahead[k / 32 + 1 & 1]);
                            if (masked) {
                                #pragma unroll
                                for (uint32_t i = 0; i < 32; ++i) x[i] = k + i < lim ? x[i] : 0xff800000u;
                            }
                            #pragma unroll
                            for (uint32_t i = 0; i < 32; i += 2) {
                                top[(i >> 1) & 1] = fmaxf(fmaxf(top[(i >> 1) & 1], __uint_as_float(x[i])), __uint_as_float(x[i + 1]));
                                const float2 e = fma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), factor, from);
                                const float2 w = make_float2(exp2_approx(e.x), exp2_approx(e.y));
                                sum = add2(sum, w);
                                p[(k + i) / 2] = pack<NF4>(w.x, w.y);
                            }
                        }
                        const float high = fmaxf(top[0], top[1]) * factor;
                        if (!__any_sync(0xffffffffu, high > m + 8.f)) break;
                        const float now = fmaxf(m, high), keep = m == -INFINITY ? 0.f : exp2_approx(m - now);
                        m = now;
                        l *= keep;
                        if (j) {  // the products so far are done: the scores waited for came behind them
                            #pragma unroll 1
                            for (uint32_t k = 0; k < D; k += 32) {
                                uint32_t v[32];
                                tmem_ld32(to + k, v);
                                ptx::tmem_wait_ld();
                                #pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * keep);
                                tmem_st32(to + k, v);
                            }
                        }
                    }
                    l += sum.x + sum.y;
                    #pragma unroll
                    for (uint32_t k = 0; k < N / 2; k += 32) tmem_st32(ts + k, p + k);
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(p_ready0 + 8 * tile);
                }
                if (ok && steps && !__all_sync(0xffffffffu, ptx::mbar_wait_suspended(s_full0 + 8 * tile, steps & 1u))) {
                    ok = false;
                    if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 24);
                }
                ptx::tc_fence_after();
                if (s_bad || !ok) l = __uint_as_float(0x7fc00000u);  // NaN
                const uint32_t out_row = s.row0 + row / a.group, h = head * a.group + row % a.group;
                const uint64_t at = ((uint64_t)part * b.rows + out_row) * q_heads + h;
                if (a.parts > 1 && real) a.part_ml[at] = make_float2(m, l);
                const float f = (a.parts > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l) * v_power;
                #pragma unroll
                for (uint32_t k = 0; k < D; k += 32) {
                    uint32_t v[32];
                    __syncwarp();
                    if (steps) {
                        tmem_ld32(to + k, v);
                        ptx::tmem_wait_ld();
                    }
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = steps ? __float_as_uint(__uint_as_float(v[i]) * f) : 0u;
                    if (!real) continue;
                    if (a.parts > 1) {
                        if (!steps) continue;  // (a part without tokens is not read)
                        uint4 *const o = reinterpret_cast<uint4 *>(a.part_o + at * D + k);
                        #pragma unroll
                        for (int i = 0; i < 8; ++i) o[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    } else {
                        uint4 *const o = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)out_row * a.ldo + (uint64_t)h * D + k);
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t w[4];
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = bf16_pair(__uint_as_float(v[8 * i + 2 * e]), __uint_as_float(v[8 * i + 2 * e + 1]));
                            o[i] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                ptx::tc_fence_before();
            }
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
            if (NF4 && warp >= kExpandWarp && warp < kExpandWarp + 4) {
                // ---- codes to f16: a thread has 16 bytes of a token's row, 32 values ----
                constexpr uint32_t kLanes = D / 32, kPass = 128 / kLanes;
                const uint32_t th = tid - 32 * kExpandWarp, q = th % kLanes, lane_word = table | lane * 4u;
                // In which order a thread takes its four words: so that eight lanes' 16-byte stores hit all banks
                const uint32_t order = D == 128 ? (q >> 1) * 2 : D == 256 ? q >> 1 : 0u;
                for (uint32_t i = 0; i < 2 * steps; ++i) {
                    const uint32_t rs = i % S::kRawSlots, slot = i % S::kSlots, raw = raw0 + rs * S::kRaw, to = ring0 + slot * S::kTile + (q >> 1) * S::kBox;
                    bool got = ptx::mbar_wait_suspended(raw_full0 + 8 * rs, (i / S::kRawSlots) & 1u);
                    if (got && i >= S::kSlots) got = ptx::mbar_wait_suspended(empty0 + 8 * slot, (i / S::kSlots + 1) & 1u);
                    if (!__all_sync(0xffffffffu, got)) {
                        ok = false;
                        if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 25);
                        break;
                    }
                    const float unit = reciprocal_of_power(i & 1u ? v_power : k_power) * (1.f / kLevelUnit);
                    const uint32_t t0 = t_first + (i >> 1) * N;
                    #pragma unroll
                    for (uint32_t pass = 0; pass < N / kPass; ++pass) {
                        const uint32_t t = pass * kPass + th / kLanes;
                        uint4 w = ld_shared_u4(raw + t * (D / 2) + q * 16);
                        float scale;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(scale) : "r"(raw + N * (D / 2) + (t * kBlocks + (q >> 1)) * 4) : "memory");
                        scale = t0 + t < t_end ? scale * unit : 0.f;  // (behind the last token anything may stand)
                        const uint32_t s2 = pack<true>(scale, scale);
                        if (order & 2u) w = make_uint4(w.z, w.w, w.x, w.y);
                        if (order & 1u) w = make_uint4(w.y, w.x, w.w, w.z);
                        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                        #pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) {
                            uint32_t v[4];
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t word = words[k], at = ((e == 0 ? word << 7 : word >> (8 * e - 7)) & 0x7f80u) | lane_word;
                                asm("ld.shared.u32 %0, [%1];" : "=r"(v[e]) : "r"(at));  // (free to move: the table stands)
                                v[e] = mul_f16x2(v[e], s2);
                            }
                            const uint32_t chunk = (q & 1u) * 4 + (k ^ order);
                            st_shared_u4(to + t * 128 + ((chunk ^ (t & 7u)) << 4), make_uint4(v[0], v[1], v[2], v[3]));
                        }
                    }
                    ptx::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive(full0 + 8 * slot);
                        ptx::mbar_arrive(raw_empty0 + 8 * rs);
                    }
                }
            } else if (warp == kCopyWarp) {
                constexpr uint32_t kGroups = N / kGroup;
                const uint32_t stored = min(s.length, t_first + steps * N);  // tokens that there are
                for (uint32_t j = 0; j < steps; ++j) {
                    const uint32_t t0 = t_first + j * N, g = lane % kGroups, box = lane / kGroups, t = t0 + g * kGroup;
                    const uint32_t groups = min(kGroups, (stored - t0 + kGroup - 1) / kGroup);
                    uint32_t place = 0;
                    if (g < groups) {
                        const uint32_t at = c.by_page.of(t);
                        const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at);
                        if (page >= 0 && (uint32_t)page < c.pages) place = ((uint32_t)page * c.heads + head) * c.page_size + (t - at * c.page_size);
                    }
                    for (uint32_t which = 0; which < 2; ++which) {
                        const uint32_t i = 2 * j + which;
                        bool got = true;
                        if (NF4) {
                            const uint32_t rs = i % S::kRawSlots, bar = raw_full0 + 8 * rs, to = raw0 + rs * S::kRaw;
                            if (i >= S::kRawSlots) got = ptx::mbar_wait_suspended(raw_empty0 + 8 * rs, (i / S::kRawSlots + 1) & 1u);
                            got = __all_sync(0xffffffffu, got);
                            if (got) {
                                if (lane == 0) ptx::mbar_arrive_expect_tx(bar, groups * (kGroup * (D / 2) + kGroup * kBlocks * 4));
                                __syncwarp();
                                if (box == 0 && g < groups) {
                                    ptx::bulk_g2s(to + g * kGroup * (D / 2), static_cast<const uint8_t *>(which ? c.v : c.k) + (uint64_t)place * (D / 2), kGroup * (D / 2), bar);
                                    ptx::bulk_g2s(to + N * (D / 2) + g * kGroup * kBlocks * 4, (which ? c.v_scales : c.k_scales) + (uint64_t)place * kBlocks,
                                                  kGroup * kBlocks * 4, bar);
                                }
                            }
                        } else {
                            const uint32_t slot = i % S::kSlots, to = ring0 + slot * S::kTile;
                            if (i >= S::kSlots) got = ptx::mbar_wait_suspended(empty0 + 8 * slot, (i / S::kSlots + 1) & 1u);
                            got = __all_sync(0xffffffffu, got);
                            const bool tail = which && t0 + N > s.length;  // values that anything may stand behind: zeros, for weights of zero
                            const uint32_t bar = tail ? tail_bar : full0 + 8 * slot;
                            if (got) {
                                if (lane == 0) ptx::mbar_arrive_expect_tx(bar, groups * (kGroup * 128) * (D / 64));
                                __syncwarp();
                                if (g < groups && box < D / 64)
                                    ptx::tma_load_2d(to + box * S::kBox + g * (kGroup * 128), which ? &tmap_v : &tmap_k, (int32_t)(64 * box), (int32_t)place, bar);
                            }
                            if (got && tail) {
                                got = __all_sync(0xffffffffu, ptx::mbar_wait_suspended(tail_bar, 0));  // (once in a CTA's life)
                                for (uint32_t k = (s.length - t0) * 8 + lane; k < N * 8; k += 32)
                                    #pragma unroll
                                    for (uint32_t x = 0; x < D / 64; ++x) st_shared_u4(to + x * S::kBox + k * 16, make_uint4(0u, 0u, 0u, 0u));
                                ptx::fence_proxy_async();
                                __syncwarp();
                                if (lane == 0) ptx::mbar_arrive(full0 + 8 * slot);
                            }
                        }
                        if (!got) {
                            ok = false;
                            if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 26);
                            break;
                        }
                    }
                    if (!ok) break;
                }
            } else if (warp == kMmaWarp && steps) {
                constexpr uint32_t fmt = NF4 ? 0 : 1;
                constexpr uint32_t idesc_s = ptx::f16_idesc(fmt, 128, N, false, false), idesc_o = ptx::f16_idesc(fmt, 128, D, false, true);
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    if (!ok) return;
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_suspended(bar, parity));
                    if (!ok && lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 27);
                };
                auto wait_full = [&](uint32_t i) { wait(full0 + 8 * (i % S::kSlots), (i / S::kSlots) & 1u); };
                auto scores = [&](uint32_t tile, uint32_t i) {  // of the keys in ring place i
                    const uint64_t qd = ptx::sw128_desc(q0 + tile * S::kQTile), kd = ptx::sw128_desc(ring0 + i % S::kSlots * S::kTile);
                    #pragma unroll
                    for (uint32_t k = 0; k < D / 16; ++k)
                        ptx::mma_ss_f16(tmem + S::kS + tile * N, qd + (k >> 2) * (16384 >> 4) + (k & 3u) * 2, kd + (k >> 2) * (S::kBox >> 4) + (k & 3u) * 2, idesc_s, k != 0);
                    ptx::tc_commit(s_full0 + 8 * tile);
                };
                auto products = [&](uint32_t tile, uint32_t i, bool add) {
                    const uint64_t vd = ptx::sw128_desc(ring0 + i % S::kSlots * S::kTile, S::kBox);
                    #pragma unroll
                    for (uint32_t k = 0; k < N / 16; ++k) ptx::mma_ts_f16(tmem + S::kO + tile * D, tmem + S::kS + tile * N + 8 * k, vd + 128 * k, idesc_o, add || k != 0);
                };
                wait_full(0);
                ptx::tc_fence_after();
                if (ok && ptx::elect_one()) {
                    for (uint32_t t = 0; t < live; ++t) scores(t, 0);
                    ptx::tc_commit(empty0);
                }
                __syncwarp();
                for (uint32_t j = 0; j < steps && ok; ++j) {
                    const uint32_t iv = 2 * j + 1, ik = 2 * j + 2;
                    const bool more = j + 1 < steps;
                    wait_full(iv);
                    for (uint32_t t = 0; t < live; ++t) {
                        wait(p_ready0 + 8 * t, j & 1u);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        if (ptx::elect_one()) {
                            products(t, iv, j != 0);
                            if (t + 1 == live) ptx::tc_commit(empty0 + 8 * (iv % S::kSlots));
                            if (!more) ptx::tc_commit(s_full0 + 8 * t);
                        }
                        __syncwarp();
                        if (!more) continue;
                        if (t == 0) wait_full(ik);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        if (ptx::elect_one()) {
                            scores(t, ik);
                            if (t + 1 == live) ptx::tc_commit(empty0 + 8 * (ik % S::kSlots));
                        }
                        __syncwarp();
                    }
                }
            }
        }
    }
    if (!ok) ptx::let_flights_land();
    __syncwarp();
    __syncthreads();
    if (warp == kMmaWarp) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

template <int D, bool NF4>
int32_t launch(const AttentionCall &c, cudaStream_t stream) {
    using S = Shape<D, NF4>;
    auto kernel = attention_chunk_kernel<D, NF4>;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kSmem));
    const uint64_t pool = (uint64_t)c.cache.pages * c.cache.heads * c.cache.page_size;
    CUtensorMap map_k{}, map_v{};
    if (!NF4) {
        NF4_TRY(make_map(&map_k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.cache.k, pool, D, 2 * D, kGroup, 64, CU_TENSOR_MAP_SWIZZLE_128B));
        NF4_TRY(make_map(&map_v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.cache.v, pool, D, 2 * D, kGroup, 64, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    FailureRef failure;
    NF4_TRY(prefill_failure_ref(&failure));
    const uint32_t tiles = attention_chunk_tiles(c);
    if ((uint64_t)tiles * c.cache.heads >= 1ull << 31) return fail(NF4_ERR_UNSUPPORTED, "attention: too many rows in a call");
    count_launch();
    return launch_maybe_overlapped(kernel, dim3(tiles * c.cache.heads, c.view.parts), dim3(kThreads), S::kSmem, stream, true, map_k, map_v, c.cache, c.batch,
                                   c.view, tiles, failure);
}

}  // namespace

uint32_t attention_chunk_tiles(const AttentionCall &c) {
    const uint32_t rows = c.head_dim == 256 ? 128 : 256;
    return (uint32_t)((uint64_t)c.batch.rows * c.view.group / rows) + c.batch.sequences;
}

int32_t attention_chunk(const AttentionCall &c, cudaStream_t stream) {
    switch (c.head_dim) {
        case 64: return c.nf4 ? launch<64, true>(c, stream) : launch<64, false>(c, stream);
        case 128: return c.nf4 ? launch<128, true>(c, stream) : launch<128, false>(c, stream);
        default: return c.nf4 ? launch<256, true>(c, stream) : launch<256, false>(c, stream);
    }
}

}  // namespace nf4
