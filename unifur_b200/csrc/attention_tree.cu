// Attention of trees of drafted tokens over the paged cache on the tensor cores: rows are a tree's nodes, which see their sequence's context and those
// nodes that their masks have.
//
// A tree has some tens of nodes, so that a head of the cache serves 20 to 500 rows, and reading the cache, expanding a quantized one, the exponentials
// and the MMAs take about as long as one another.  A row tile is one MMA tile of 128 rows (a token's query heads are neighbouring rows), which goes over its
// tokens 128 (a dim of 256: 64) a step.  The line of steps, its shares, pieces and their join are those of the kernel for many rows (attention_steps.cuh).
//
// S = Q K^T has two places in tensor memory, so that a step's scores come while the last one's weights are made.  Two softmax warpgroups have
// half of a step's tokens each, of the same rows (a thread has a row's 64 scores of a step): with largest exponents, sums and an accumulator of
// results of their own, which become one when a piece ends, so that they have nothing to say to one another before.  (One warpgroup: 2000 cycles a step of 128
// tokens over a bf16 cache, where the exponentials and the MMAs are 1024 each, and 2400 to 4000 beside eight warps that expand; two: 1700 and 2500.)  With a
// dim of 256 tensor memory has no room for a second accumulator: one warpgroup, and 64 tokens a step.
//
// A quantized cache's codes come to shared memory by 16-byte copies of three warps (bulk copies of a page's sixteen tokens take 135 cycles each whoever
// waits, 40 a step: 5300 cycles), which find the powers of two for the scales as well and ask the L2 for the tile after; eight warps expand them.  Where nine
// row tiles or more of a head read the cache it is expanded ahead, as for many rows.  Masks are looked at only in the steps that reach behind the
// context.
//
// Measured (16 sequences of 8192 tokens, 8 heads of 128): bf16, 16 to 64 rows of a head, 89 us = 6.0 TB/s; NF4, 16 to 128 rows, 97 to 99 us, 2800 cycles a step,
// in which a scheduler issues 2000 instructions for two softmax and two expanding warps.  Tried for those, with no gain: a fourth of the words expanded by byte permutes of
// the levels' bytes in place of lookups, half of the exponentials by FMA, a step's first scores asked for during the last one's weights, up to 64 rows in
// the tile twice with a softmax warp to each scheduler.  Everything else (weights, f16's range, the order of sums) is as in the kernel for many rows, and said there,
// but for the unit of a row's sums over a quantized cache: a step that a row sees nothing of may hold far larger values, of other branches, and has no say in it.
#include <algorithm>

#include "attention_steps.cuh"
#include "tmap.cuh"

namespace nf4 {

namespace {

constexpr uint32_t kThreads = 640;
// warps 0-3 and 4-7: softmax; 8-15: codes to f16 (a bf16 cache: the first of them copy, all where pages are small); 16, 18, 19: codes' copies; 17: MMAs
constexpr uint32_t kExpandWarp = 8, kExpandWarps = 4, kCopyWarp = 16, kMmaWarp = 17, kLoaders = 3;  // kExpandWarps: to a tile

template <int D, bool NF4>
struct Shape {
    static constexpr uint32_t kRows = 128, kTokens = D == 256 ? 64 : 128;  // of a step
    static constexpr uint32_t kHalves = D == 256 ? 1 : 2, kHalf = kTokens / kHalves, kSoftmaxWarps = 4 * kHalves;
    static constexpr uint32_t kBlocks = D / 64;
    static constexpr uint32_t kQTile = 128 * D * 2, kTile = kTokens * D * 2, kBox = kTokens * 128;
    static constexpr uint32_t kCodes = kTokens * D / 2, kRaw = NF4 ? kCodes + kTokens * kBlocks * 4 : 0, kRawSlots = kLoaders;  // codes, then scales
    // A table entry's copies to the lanes are 256 bytes apart where there is room, so that a byte permute makes a whole address (a dim of 128: 3 % of the
    // time, though the ring has a place less), else 128.
    static constexpr bool kApart = NF4 && D <= 128;
    static constexpr uint32_t kStride = kApart ? 256 : 128, kTable = 256 * kStride;
    static constexpr uint32_t kSlots = D == 64 ? (NF4 ? 6 : 7) : D == 128 ? (NF4 ? 3 : 6) : NF4 ? 3 : 5;  // of the ring; one more where the table is not needed
    // Q and codes, then the table on a multiple of its 64 KB, then the ring; or codes, then the table on a multiple of its 32 KB, then Q, then the ring;
    // or (bf16) Q, then the ring
    static constexpr uint32_t kSmem = (kApart ? 131072 : (NF4 ? 65536 : 2048) + kQTile) - 1024 + kSlots * kTile;
    static constexpr uint32_t kS = 0, kO = 256;  // columns of tensor memory: S's two places, then the halves' O's
    // 640 threads are launched with 96 registers each; what the softmax warpgroups take more the others leave (480 to a thread of each warpgroup together)
    static constexpr uint32_t kSoftmaxRegs = kHalves == 2 ? 128 : 152, kOtherRegs = kHalves == 2 ? 72 : 80;
    static_assert(kHalves * kSoftmaxRegs + (5 - kHalves) * kOtherRegs <= 480 && kSlots + 1 <= 8);
};

// kWhole: up to that many steps more than a share, and a share's twelfth but no more than four, row tiles stay whole.  Measured on both sides, tiles of one length,
// as many as given for 148 CTAs, us divided / whole (heads of 128, 64 rows).  NF4: 8 steps, 144 tiles 30 / 25, 80 27.5 / 24.5; 16 steps, 112 40 / 36, 96 35 / 36; 32 steps, 120 59 / 59,
// 112 56 / 58; 64 steps, 136 110 / 106, 128 104 / 105; 128 steps, 140 199 / 196, 136 195 / 196; 256 steps, 140 390 / 386, 128 355 / 377: as long at 5.5 to 7, 7, 7, 8, 10 and 20 steps
// more than a share.  A bf16 cache, bound by its bytes, could go on for longer: 16 steps, 96 tiles 35 / 30, 80 28 / 29; 64 steps, 112 92 / 83, 96 81 / 82.
constexpr uint32_t kStart = 4, kLeast = 3, kWhole = 6;  // (see Walker)
constexpr uint32_t kMostLess = 4;  // by how many powers of two a step may be below a row's unit

// The row of the n-th chunk that a lane of a softmax warp takes of the results: its warp's 32 rows, its half's values.
template <uint32_t LANES>  // to a row
__device__ __forceinline__ uint32_t row_of_chunk(uint32_t warp, uint32_t lane, uint32_t n) { return (warp & 3u) * 32 + n * (32 / LANES) + lane / LANES; }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.f : __uint_as_float((uint32_t)(127 + e) << 23); }  // up to 127
__device__ __forceinline__ void take_columns(uint32_t taddr, uint32_t (&r)[16]) { ptx::tmem_ld16(taddr, r); }
__device__ __forceinline__ void take_columns(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void cp_async_16_upto(uint32_t dst_smem, const void *src, uint32_t bytes) {  // of the sixteen, and zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {  // once this thread's copies so far have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

template <int D, bool NF4>
__global__ void __launch_bounds__(kThreads, 1)
attention_tree_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const CacheView c, const BatchView b,
                      const AttentionView a, const Dense dense, uint32_t box_rows, Split *const splits, const FailureRef failure) {
    using S = Shape<D, NF4>;
    using Walk = Walker<S::kRows, S::kTokens, kStart, kLeast, kWhole, true>;
    constexpr uint32_t kCopies = !NF4 && D >= 128 ? 2 : 1;  // (as in the kernel for many rows)
    constexpr uint32_t kSmallCopies = 4;               // warps to a tile whose pages are of sixteen tokens
    const bool small_pages = !NF4 && box_rows == kGroup;
    constexpr uint32_t N = S::kTokens, kBlocks = S::kBlocks, kHalves = S::kHalves, kHalf = S::kHalf;
    extern __shared__ uint8_t smem_any[];
    __shared__ __align__(8) uint64_t s_bars[40];
    __shared__ uint32_t s_tmem, s_bad[8], s_first[6];  // s_bad: of the last eight pieces, its number + 1 where a page was not there (it is marked up to six pieces ahead)
    __shared__ Share s_share;
    __shared__ float s_qpower[NF4 ? 128 : 1];
    __shared__ float2 s_powers[8];  // of the last steps' K and V, for the softmax (who writes them is fewer steps ahead of who reads)
    __shared__ float s_raw_powers[S::kRawSlots];  // of the tiles in the raw ring
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
    const uint32_t base = ptx::smem_addr(smem_any);
    const uint32_t aligned = (base + 1023u) & ~1023u, raw0 = S::kApart ? aligned + S::kQTile : (base + 15u) & ~15u;
    const uint32_t table = (raw0 + S::kRawSlots * S::kRaw + S::kTable - 1) & ~(S::kTable - 1);
    const uint32_t q0 = NF4 && !S::kApart ? table + S::kTable : aligned, ring0 = S::kApart ? table + S::kTable : q0 + S::kQTile;
    // s_full, p_ready: of S's places; pv_done: products that a rescaling waits for; pair: the two warps that have the same rows
    const uint32_t bars = ptx::smem_addr(s_bars), full0 = bars, empty0 = bars + 64, raw_full0 = bars + 128, raw_empty0 = bars + 176, s_full0 = bars + 200,
                   p_ready0 = bars + 216, pv_done = bars + 232, q_ready = bars + 240, o_done = bars + 248, tail0 = bars + 256, pair0 = bars + 272;
    if (ring0 + S::kSlots * S::kTile > base + S::kSmem) {
        ptx::pdl_wait();
        if (tid == 0) {
            NF4_REPORT_FAILURE(*failure.flag, *failure.host, 30);
            splits[blockIdx.x].rows = 0;
        }
        return;
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < 8; ++i) {  // (a place more than kSlots may be in use)
            ptx::mbar_init(full0 + 8 * i, NF4 ? kExpandWarps : small_pages ? kSmallCopies : kCopies);
            ptx::mbar_init(empty0 + 8 * i, 1);
        }
        for (uint32_t i = 0; i < S::kRawSlots; ++i) {
            ptx::mbar_init(raw_full0 + 16 * i, 33);  // each lane's copies, and the powers
            ptx::mbar_init(raw_full0 + 16 * i + 8, 33);
            ptx::mbar_init(raw_empty0 + 8 * i, kExpandWarps);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            ptx::mbar_init(s_full0 + 8 * i, 1);
            ptx::mbar_init(p_ready0 + 8 * i, S::kSoftmaxWarps);
            ptx::mbar_init(tail0 + 8 * i, 1);
        }
        ptx::mbar_init(pv_done, 1);
        ptx::mbar_init(q_ready, S::kSoftmaxWarps);
        ptx::mbar_init(o_done, 1);
        for (uint32_t i = 0; i < 4; ++i) ptx::mbar_init(pair0 + 8 * i, 2);
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
    }
    if (tid < 8) s_bad[tid] = 0;
    if (NF4) {
        for (uint32_t i = tid; i < 256 * 8; i += kThreads) {  // the table: an entry's copy to a lane
            const uint32_t byte = i >> 3, entry = level_pair_f16(byte);
            st_shared_u4(table + byte * S::kStride + (i & 7u) * 16u, make_uint4(entry, entry, entry, entry));
        }
        ptx::fence_proxy_async();  // (copies may come to this place instead)
    }
    if (warp == kMmaWarp) {
        ptx::tmem_alloc(ptx::smem_addr(&s_tmem), 512);
        ptx::tmem_relinquish();
    }
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    // ---- this CTA's share of the line, and where in it begins ----
    if (warp == 0) {
        const Share share = share_out<Walk>(c, b, a, s_first);
        if (lane == 0) {
            s_share = share;
            splits[blockIdx.x].rows = 0;
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = s_tmem;
    bool ok = true;
    const bool expanded = NF4 && dense.capacity && __ldg(dense.bases + b.sequences) <= dense.capacity;  // (more tokens than the host knew of: not)
    const uint32_t slots = S::kSlots + (expanded ? 1u : 0u);
    auto place_of = [&](uint32_t slot) -> uint32_t { return slot < S::kSlots ? ring0 + slot * S::kTile : table; };
    // codes: 30 shared memory; 31 scores, 32 sums to be rescaled, 33 results, 37 the warp of the same rows; 34 expanding; 35 copies; 36 MMAs
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_suspended(bar, parity))) {
            ok = false;
            if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, code);
        }
    };
    if (s_first[4] < s_first[5]) {
        Walk walk{sequence_of(c, b, s_first[0]), s_first[0], s_first[1], s_first[2], s_first[3], s_first[4], s_first[5], s_share.whole};
        Piece p;
        if (warp < S::kSoftmaxWarps) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
            const uint32_t half = warp >> 2, r = tid & 127u;
            const uint32_t lanes = (warp & 3u) << 21;  // a warp reaches its quarter of tensor memory's lanes
            const uint32_t ts0 = tmem + S::kS + half * kHalf + lanes, to0 = tmem + S::kO + lanes, to = to0 + half * D;
            constexpr uint32_t kWide = D / kHalves, kLanes = kWide / 8;  // values of a row's results that a warp takes; lanes to them
            uint32_t scores = 0, finished = 0, step = 0, piece = 0;  // steps and pieces so far
            // The two warps that have the same rows meet three times a piece.  left: they are still to meet behind the results.
            const uint32_t pair = pair0 + 8 * (warp & 3u);
            uint32_t meets = 0;
            bool left = false;
            auto come = [&] {
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(pair);
            };
            auto meet = [&] { wait(pair, meets++ & 1u, 37); };
            for (; ok && walk.next(c, b, a, p); step += p.steps, ++piece) {
                // ---- Q to shared memory: half of the pair's rows, as they are, and beside a quantized cache then divided by a power of two ----
                // (Short loops: code that runs once a piece comes from the L2.  Unrolled, with the loads in registers, this took 11000 cycles.)
                if (left) meet();  // the other warp has taken its results from these rows' places
                left = false;
                constexpr uint32_t kRowLanes = D / 8, kRounds = kRowLanes / kHalves, kRowsOfRound = 32 / kRowLanes;
                const uint32_t first_row = (warp & 3u) * 32 + half * (32 / kHalves) + lane / kRowLanes, chunk = lane % kRowLanes;
                #pragma unroll 2
                for (uint32_t i = 0; i < kRounds; ++i) {
                    const uint32_t of_tile = first_row + i * kRowsOfRound;
                    const bool real = of_tile < p.rows;
                    const uint32_t row = real ? p.r0 + of_tile : p.r0, token = a.by_group.of(row);
                    const __nv_bfloat16 *const from = static_cast<const __nv_bfloat16 *>(a.q) + (uint64_t)(p.s.row0 + token) * a.ldq + (uint64_t)(p.head * a.group + row - token * a.group) * D;
                    ptx::cp_async_16_or_zero(q0 + chunk_place(of_tile, chunk), from + 8 * chunk, real);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (NF4 || a.scale_log2 < 0.f) {
                    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a scale below zero: the rows change sign, so that c is not)
                    #pragma unroll 2
                    for (uint32_t i = 0; i < kRounds; ++i) {  // (a thread changes what it has brought)
                        const uint32_t of_tile = first_row + i * kRowsOfRound, at = q0 + chunk_place(of_tile, chunk);
                        const uint4 w = ld_shared_u4(at);
                        uint32_t u[4] = {w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip};
                        if (NF4) {
                            constexpr uint32_t kSize = 0x7fff7fffu;  // (bf16 magnitudes go by their bits)
                            uint32_t two = __vmaxu2(__vmaxu2(u[0] & kSize, u[1] & kSize), __vmaxu2(u[2] & kSize, u[3] & kSize));
                            #pragma unroll
                            for (uint32_t d = 1; d < kRowLanes; d <<= 1) two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, d));
                            const uint32_t most = max(two << 16, two & 0xffff0000u);
                            // the row's largest magnitude is left in [2^11, 2^12)
                            const int e2 = most ? min(max((int)(most >> 23) - 127 - 11, -100), 115) : 0;
                            const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) u[e] = pack<true>(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
                            if (chunk == 0) s_qpower[of_tile] = __uint_as_float((uint32_t)(127 + e2) << 23);
                        }
                        st_shared_u4(at, make_uint4(u[0], u[1], u[2], u[3]));
                    }
                }
                ptx::fence_proxy_async();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(q_ready);

                // ---- the steps ----
                const bool idle = (warp & 3u) * 32 >= p.rows;  // none of the warp's rows is one: its part of S is never looked at
                const bool real = r < p.rows;
                const uint32_t token = a.by_group.of(real ? p.r0 + r : p.r0), node_row = p.s.row0 + token;
                const int32_t nodes0 = first_node(p.s);
                const uint32_t sees = real && nodes0 + (int32_t)token >= 0 ? p.s.length : 0u;  // (a node with a negative token sees nothing)
                const uint32_t context = (uint32_t)max(nodes0, 0);
                float row_factor = fabsf(a.scale_log2);
                float m = -INFINITY, l = 0.f;
                int unit = 0, top_unit = 0;  // NF4: exponents of what the row's sums are in units of, and of the largest of a step that it saw something of
                for (uint32_t j = 0; j < p.steps; ++j, ++scores) {
                    const uint32_t place = scores & 1u, ts = ts0 + place * N;
                    wait(s_full0 + 8 * place, (scores / 2) & 1u, 31);
                    if (!ok) break;
                    if (idle) {
                        if (lane == 0) ptx::mbar_arrive(p_ready0 + 8 * place);
                        continue;
                    }
                    ptx::tc_fence_after();
                    uint32_t x[2][32];  // the row's scores
                    static_assert(kHalf == 64);
                    tmem_ld32(ts, x[0]);
                    tmem_ld32(ts + 32, x[1]);
                    if (NF4 && j == 0) row_factor *= s_qpower[r];  // (the scores are behind both warps' queries)
                    const uint32_t t0 = (p.step0 + j) * N + half * kHalf, lim = sees > t0 ? sees - t0 : 0u;
                    // (written before the keys' arrival was made known, which the scores are behind)
                    const float2 powers = NF4 ? ld_shared_f2(ptx::smem_addr(s_powers + ((step + j) & 7u))) : make_float2(1.f, 1.f);
                    const float factor = fmaxf(row_factor * powers.x, 1.2e-38f);
                    ptx::tmem_wait_ld();
                    if (t0 + kHalf > context) {
                        #pragma unroll
                        for (uint32_t u = 0; u < 2; ++u) {
                            const uint32_t seen = seen_nodes(a, node_row, (int32_t)(t0 + 32 * u) - nodes0) & low_bits(lim > 32 * u ? lim - 32 * u : 0u);
                            #pragma unroll
                            for (uint32_t i = 0; i < 32; ++i) x[u][i] = seen >> i & 1u ? x[u][i] : 0xff800000u;
                        }
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    #pragma unroll
                    for (uint32_t i = 0; i < 64; i += 2) top[i / 2 % 4] = fmaxf(fmaxf(top[i / 2 % 4], __uint_as_float(x[i / 32][i % 32])), __uint_as_float(x[i / 32][i % 32 + 1]));
                    const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * factor;
                    // The step's values are in units of powers.y, a row's sums in units of 2^unit of which that is 2^-less.  A step that the row sees nothing of leaves its
                    // unit, and one whose power is below it or far above takes it along, so that `less` costs a weight few of its bits (no further down than
                    // 2^-60 of the largest, so that the sums do not overflow; from there on weights lose theirs, and a value below 2^-120 of the largest is made that).
                    int shift = 0, less = 0;
                    if (NF4) {
                        const int of_step = (int)(__float_as_uint(powers.y) >> 23);
                        if ((uint32_t)(unit - of_step) > kMostLess && high != -INFINITY) {
                            top_unit = max(top_unit, of_step);
                            const int now = max(of_step, top_unit - 60);
                            shift = unit - now;
                            unit = now;
                        }
                        less = min(max(unit - of_step, 0), 60);
                    }
                    // m stays up to 8 below the largest score: once or twice a row it is out of reach
                    if (__any_sync(0xffffffffu, high > m + 8.f || shift)) {
                        const float now = fmaxf(m, high);
                        float keep = m == -INFINITY ? 0.f : exp2_approx(m - now);
                        m = now;
                        l *= keep;
                        if (NF4) keep *= power_of_two(shift);
                        if (j) {  // once the products so far are done
                            wait(pv_done, (scores - 1) & 1u, 32);
                            if (!ok) break;
                            ptx::tc_fence_after();
                            #pragma unroll 1
                            for (uint32_t k = 0; k < D; k += 16) {
                                uint32_t v[16];
                                ptx::tmem_ld16(to + k, v);
                                ptx::tmem_wait_ld();
                                #pragma unroll
                                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * keep);
                                tmem_st16(to + k, v);
                            }
                        }
                    }
                    const float from = m == -INFINITY ? 0.f : kRaise<NF4> - m - (float)less;
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    #pragma unroll
                    for (uint32_t u = 0; u < 2; ++u) {
                        uint32_t pw[16];
                        #pragma unroll
                        for (uint32_t i = 0; i < 32; i += 2) {
                            const float2 e = fma2(make_float2(__uint_as_float(x[u][i]), __uint_as_float(x[u][i + 1])), factor, from);
                            const float2 w = make_float2(exp2_approx(e.x), exp2_approx(e.y));
                            sum[i / 2 % 2] = add2(sum[i / 2 % 2], w);
                            pw[i / 2] = pack<NF4>(w.x, w.y);
                        }
                        tmem_st16(ts + 16 * u, pw);  // (over scores that all of the row's are read of)
                    }
                    sum[0] = add2(sum[0], sum[1]);
                    l += (sum[0].x + sum[0].y) * (NF4 ? __uint_as_float((uint32_t)(127 + less) << 23) : 1.f);
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(p_ready0 + 8 * place);
                }
                wait(o_done, finished & 1u, 33);
                ++finished;
                if (idle) continue;
                ptx::tc_fence_after();

                // ---- the row's results, through the place of this warp's part of Q (the products are done) so that whole rows go out ----
                const bool whole = p.steps == p.all;
                float w0 = 1.f, w1 = 0.f;  // what the halves' results count
                if (kHalves == 2) {  // this one's largest exponent and sum to the other's warp, and its to this one
                    st_shared_u4(q0 + chunk_place(r, half * kLanes), make_uint4(__float_as_uint(m), __float_as_uint(l), (uint32_t)unit, 0u));
                    come();
                    meet();
                    const uint4 got = ld_shared_u4(q0 + chunk_place(r, (1 - half) * kLanes));
                    const float2 theirs = make_float2(__uint_as_float(got.x), __uint_as_float(got.y));
                    come();
                    meet();  // (both have read: results come to these places)
                    const float now = fmaxf(m, theirs.x), from = now == -INFINITY ? 0.f : now;
                    w0 = exp2_approx((half ? theirs.x : m) - from);
                    w1 = exp2_approx((half ? m : theirs.x) - from);
                    l = fmaf(half ? l : theirs.y, w1, (half ? theirs.y : l) * w0);
                    m = now;
                    if (NF4) {  // and to one unit
                        const int larger = max(unit, (int)got.z), mine = unit - larger, other = (int)got.z - larger;
                        w0 *= power_of_two(half ? other : mine);
                        w1 *= power_of_two(half ? mine : other);
                        unit = larger;
                    }
                }
                if (s_bad[piece & 7u] == piece + 1 || !ok) l = __uint_as_float(0x7fc00000u);  // NaN
                const uint64_t part = (uint64_t)(2 * blockIdx.x + (p.step0 ? 0 : 1)) * S::kRows;
                if (!whole && half == 0) a.part_ml[part + r] = make_float2(m, l * kLower<NF4>);
                const float f = (whole ? l == 0.f ? 0.f : 1.f / l : kLower<NF4>) * (NF4 ? __uint_as_float((uint32_t)unit << 23) : 1.f);
                #pragma unroll 1
                for (uint32_t pass = 0; pass < (whole ? 1u : 2u); ++pass) {  // bf16 results, or half of the f32 sums at a time
                    const uint32_t columns = whole ? kWide : kWide / 2, first = half * kWide + pass * columns;
                    constexpr uint32_t kTake = kWide == 32 ? 16 : 32;  // columns at a time
                    __syncwarp();
                    #pragma unroll 1
                    for (uint32_t k = 0; k < columns; k += kTake) {
                        uint32_t x[kTake], y[kTake];
                        take_columns(to0 + first + k, x);
                        if (kHalves == 2) take_columns(to0 + D + first + k, y);
                        ptx::tmem_wait_ld();
                        #pragma unroll
                        for (uint32_t i = 0; i < kTake; ++i) {
                            float v = __uint_as_float(x[i]);
                            if (kHalves == 2) v = fmaf(__uint_as_float(y[i]), w1, v * w0);
                            x[i] = __float_as_uint(v * f);
                        }
                        const uint32_t at = half * kLanes + (whole ? k / 8 : k / 4);
                        if (whole) {
                            #pragma unroll
                            for (uint32_t i = 0; i < kTake / 8; ++i) {
                                uint32_t u[4];
                                #pragma unroll
                                for (int e = 0; e < 4; ++e) u[e] = bf16_pair(__uint_as_float(x[8 * i + 2 * e]), __uint_as_float(x[8 * i + 2 * e + 1]));
                                st_shared_u4(q0 + chunk_place(r, at + i), make_uint4(u[0], u[1], u[2], u[3]));
                            }
                        } else {
                            #pragma unroll
                            for (uint32_t i = 0; i < kTake / 4; ++i) st_shared_u4(q0 + chunk_place(r, at + i), make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
                        }
                    }
                    __syncwarp();
                    #pragma unroll 4
                    for (uint32_t i = 0; i < kLanes; ++i) {
                        const uint32_t of_tile = row_of_chunk<kLanes>(warp, lane, i), xx = lane % kLanes;
                        const uint4 v = ld_shared_u4(q0 + chunk_place(of_tile, half * kLanes + xx));
                        if (of_tile >= p.rows) continue;
                        if (whole) {
                            const uint32_t q_row = p.r0 + of_tile, of = a.by_group.of(q_row);
                            *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)(p.s.row0 + of) * a.ldo +
                                                       (uint64_t)(p.head * a.group + q_row - of * a.group) * D + first + 8 * xx) = v;
                        } else {
                            *reinterpret_cast<uint4 *>(a.part_o + (part + of_tile) * D + first + 4 * xx) = v;
                        }
                    }
                }
                if (kHalves == 2) {  // (the next queries come to the same places)
                    come();
                    left = true;
                }
                __syncwarp();
                if (!whole && p.step0 == 0 && tid == 0) {
                    const uint32_t more = min(s_share.cta_of(p.line0 + kStart + p.all - 1) - blockIdx.x, gridDim.x - 1 - blockIdx.x);
                    splits[blockIdx.x] = Split{p.s.row0, p.r0, p.rows, p.head, more};
                }
                ptx::tc_fence_before();
            }
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegs));
            if (warp == kMmaWarp) {
                constexpr uint32_t fmt = NF4 ? 0 : 1;
                constexpr uint32_t idesc_s = ptx::f16_idesc(fmt, 128, N, false, false), idesc_o = ptx::f16_idesc(fmt, 128, D, false, true);
                uint32_t made = 0, used = 0, rows_in = 0;  // scores, weights and Q's so far
                Ring ring;  // the next tile of K or V
                // (by the elected thread) of the keys in a place of the ring, to the place of the n-th
                auto scores = [&](uint32_t at, uint32_t n) {
                    const uint64_t qd = ptx::sw128_desc(q0), kd = ptx::sw128_desc(place_of(at));
                    #pragma unroll
                    for (uint32_t k = 0; k < D / 16; ++k)
                        ptx::mma_ss_f16(tmem + S::kS + (n & 1u) * N, qd + (k >> 2) * (16384 >> 4) + (k & 3u) * 2, kd + (k >> 2) * (S::kBox >> 4) + (k & 3u) * 2, idesc_s, k != 0);
                    ptx::tc_commit(s_full0 + 8 * (n & 1u));
                    ptx::tc_commit(empty0 + 8 * at);
                };
                while (ok && walk.next(c, b, a, p)) {
                    for (uint32_t j = 0; j < min(2u, p.steps) && ok; ++j, ring.on(slots)) {  // the first scores
                        wait(full0 + 8 * ring.slot, ring.round & 1u, 36);
                        if (j == 0) wait(q_ready, rows_in++ & 1u, 36);
                        ptx::tc_fence_after();
                        if (ok && ptx::elect_one()) scores(ring.slot, made);
                        ++made;
                        __syncwarp();
                    }
                    for (uint32_t j = 0; j < p.steps && ok; ++j) {
                        const Ring v = ring;
                        ring.on(slots);
                        wait(full0 + 8 * v.slot, v.round & 1u, 36);
                        wait(p_ready0 + 8 * (used & 1u), (used / 2) & 1u, 36);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        if (ptx::elect_one()) {
                            const uint64_t vd = ptx::sw128_desc(place_of(v.slot), S::kBox);
                            #pragma unroll
                            for (uint32_t k = 0; k < N / 16; ++k) {
                                const uint32_t half = k / (kHalf / 16), of_half = k % (kHalf / 16);
                                ptx::mma_ts_f16(tmem + S::kO + half * D, tmem + S::kS + (used & 1u) * N + half * kHalf + 8 * of_half, vd + 128 * k, idesc_o, j != 0 || of_half != 0);
                            }
                            ptx::tc_commit(pv_done);
                            ptx::tc_commit(empty0 + 8 * v.slot);
                            if (j + 1 == p.steps) ptx::tc_commit(o_done);
                        }
                        ++used;
                        __syncwarp();
                        if (j + 2 >= p.steps) continue;
                        wait(full0 + 8 * ring.slot, ring.round & 1u, 36);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        if (ptx::elect_one()) scores(ring.slot, made);
                        ++made;
                        __syncwarp();
                        ring.on(slots);
                    }
                }
            } else if (NF4 && !expanded && warp >= kExpandWarp && warp < kCopyWarp) {
                // ---- codes to f16: a thread has 16 bytes of some tokens' rows, 32 values each ----
                // Two groups of four warps take every second tile (of a piece, whose tiles are an even number): a tile takes a group as long in
                // accesses' and barriers' latency as in lookups, which the other's then fill.  (Eight warps to a tile: 126 us in place of 120 for the case above, as it was then.)
                constexpr uint32_t kLanes = D / 32, kPass = 32 * kExpandWarps / kLanes, kOwn = N / kPass;
                const uint32_t group = (warp - kExpandWarp) / kExpandWarps, th = tid % (32 * kExpandWarps), q = th % kLanes, row = th / kLanes, lane_word = table | lane * 4u;
                // In which order a thread takes its four words: so that eight lanes' 16-byte stores hit all banks
                const uint32_t order = D == 128 ? (q >> 1) * 2 : D == 256 ? q >> 1 : 0u;
                uint32_t raw6 = group, raw_round = 0;  // the tile's number modulo two rounds of the raw ring
                Ring ring;
                if (group) ring.on(slots);
                while (ok && walk.next(c, b, a, p)) {
                    #pragma unroll 1
                    for (uint32_t turn = group; ok && turn < 2 * p.steps; turn += 2) {
                        const uint32_t rs = raw6 % S::kRawSlots, full = raw_full0 + 16 * rs + 8 * (raw6 & 1u);
                        const uint32_t slot = ring.slot, raw = raw0 + rs * S::kRaw, dst = place_of(slot) + (q >> 1) * S::kBox;
                        wait(full, raw_round & 1u, 34);
                        const float unit = reciprocal_of_power(s_raw_powers[rs]) * (1.f / kLevelUnit);
                        uint32_t from = raw + row * (D / 2) + q * 16, scale_at = raw + S::kCodes + (row * kBlocks + (q >> 1)) * 4, to = dst + row * 128;
                        uint4 next = ld_shared_u4(from);
                        float scale;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(scale) : "r"(scale_at) : "memory");
                        if (ring.round) wait(empty0 + 8 * slot, (ring.round + 1) & 1u, 34);
                        if (!ok) break;
                        #pragma unroll 1
                        for (uint32_t pass = 0; pass < kOwn; ++pass) {
                            const uint32_t s2 = pack<true>(scale * unit, scale * unit);
                            uint4 w = next;
                            from += kPass * (D / 2);
                            scale_at += kPass * kBlocks * 4;
                            if (pass + 1 < kOwn) {
                                next = ld_shared_u4(from);
                                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(scale) : "r"(scale_at) : "memory");
                            }
                            if (order & 2u) w = make_uint4(w.z, w.w, w.x, w.y);
                            if (order & 1u) w = make_uint4(w.y, w.x, w.w, w.z);
                            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                            // (all lookups ahead of the stores, which none could pass: four at a time took the latency of one each)
                            uint32_t v[4][4];
                            #pragma unroll
                            for (uint32_t k = 0; k < 4; ++k)
                                #pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t word = words[k], at = S::kApart ? __byte_perm(word, lane_word, 0x7604u | ((uint32_t)e << 4))
                                                                                   : ((e == 0 ? word << 7 : word >> (8 * e - 7)) & 0x7f80u) | lane_word;
                                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[k][e]) : "r"(at));
                                }
                            #pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) {
                                const uint32_t chunk = (q & 1u) * 4 + (k ^ order);
                                st_shared_u4(to + ((chunk ^ (row & 7u)) << 4),
                                             make_uint4(mul_f16x2(v[k][0], s2), mul_f16x2(v[k][1], s2), mul_f16x2(v[k][2], s2), mul_f16x2(v[k][3], s2)));
                            }
                            to += kPass * 128;
                        }
                        ptx::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            ptx::mbar_arrive(full0 + 8 * slot);
                            ptx::mbar_arrive(raw_empty0 + 8 * rs);
                        }
                        raw6 += 2;
                        if (raw6 >= 2 * S::kRawSlots) {
                            raw6 -= 2 * S::kRawSlots;
                            ++raw_round;
                        }
                        ring.on(slots);
                        ring.on(slots);
                    }
                }
            } else if (NF4 && !expanded && warp >= kCopyWarp) {
                // ---- codes and scales to shared memory: a warp has every third tile, and a slot of its own ----
                const uint32_t own = warp == kCopyWarp ? 0u : warp - kMmaWarp, raw = raw0 + own * S::kRaw, empty = raw_empty0 + 8 * own;
                uint32_t turn = own, step = 0, piece = 0;
                bool more = walk.next(c, b, a, p);
                struct Tile {
                    bool real, values, scarce;  // scarce: a page that there is not
                    uint32_t info, t0, stored, place, piece;  // place: of group `lane`
                };
                // the next tile of this warp, and where its tokens are
                auto look = [&]() -> Tile {
                    while (more && turn >= 2 * p.steps) {
                        turn -= 2 * p.steps;
                        step += p.steps;
                        ++piece;
                        more = walk.next(c, b, a, p);
                    }
                    Tile t{more, false, false, 0, 0, 0, 0, piece};
                    if (!more) return t;
                    const Turn<2> of(turn, p.steps);
                    turn += kLoaders;
                    t.values = of.values;
                    t.info = step + of.step;
                    t.t0 = (p.step0 + of.step) * N;
                    t.stored = p.s.length > t.t0 ? min(p.s.length - t.t0, N) : 0u;
                    if (lane < N / kGroup && lane * kGroup < t.stored) {
                        const uint32_t token = t.t0 + lane * kGroup, at = c.by_page.of(token);
                        const int32_t page = __ldg(b.table + (uint64_t)p.seq * b.width + at);
                        t.scarce = page < 0 || (uint32_t)page >= c.pages;
                        t.place = t.scarce ? 0u : ((uint32_t)page * c.heads + p.head) * c.page_size + (token - at * c.page_size);
                    }
                    return t;
                };
                // The scales of a step's tokens, of K and of V; with the keys for both, whose powers the softmax takes, and with the values again for theirs:
                // the step's keys may be another warp's, of which this one knows nothing.
                constexpr uint32_t kQuads = N * kBlocks / 128;
                uint4 scales[2][kQuads];
                auto ask_scales = [&](const Tile &t) {
                    #pragma unroll
                    for (uint32_t i = 0; i < kQuads; ++i) {
                        constexpr uint32_t kOfGroup = 4 * kBlocks;
                        const uint32_t ch = i * 32 + lane;
                        const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, t.place, ch / kOfGroup) * kBlocks + (ch % kOfGroup) * 4;
                        #pragma unroll
                        for (int e = 0; e < 2; ++e)
                            scales[e][i] = ch * 4 < t.stored * kBlocks && (e || !t.values) ? __ldg(reinterpret_cast<const uint4 *>((e ? c.v_scales : c.k_scales) + at)) : make_uint4(0u, 0u, 0u, 0u);
                    }
                };
                Tile t = look();
                if (t.real) ask_scales(t);
                for (uint32_t n = 0; ok && t.real; ++n) {
                    uint32_t most[2] = {0, 0};
                    #pragma unroll
                    for (uint32_t i = 0; i < kQuads; ++i)
                        #pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t bits[4] = {scales[e][i].x, scales[e][i].y, scales[e][i].z, scales[e][i].w};
                            #pragma unroll
                            for (uint32_t x = 0; x < 4; ++x) most[e] = max(most[e], (i * 32 + lane) * 4 + x < t.stored * kBlocks ? bits[x] : 0u);
                        }
                    const float2 powers = make_float2(power_for(__reduce_max_sync(0xffffffffu, most[0])), power_for(__reduce_max_sync(0xffffffffu, most[1])));
                    if (t.scarce) s_bad[t.piece & 7u] = t.piece + 1;
                    const Tile next = look();
                    if (n) wait(empty, (n + 1) & 1u, 35);
                    if (!ok) break;
                    // A slot's rounds have two barriers in turn: a group that takes every second tile comes to every second of them, and one barrier's
                    // parity would show an earlier round as well.
                    const uint32_t full = raw_full0 + 16 * own + 8 * ((own + n) & 1u);  // (tile own + 3 n)
                    const uint8_t *const pool = static_cast<const uint8_t *>(t.values ? c.v : c.k);
                    const float *const pool_scales = t.values ? c.v_scales : c.k_scales;
                    #pragma unroll
                    for (uint32_t i = 0; i < S::kCodes / 512; ++i) {
                        constexpr uint32_t kOfGroup = D / 2;  // 16-byte pieces
                        const uint32_t ch = i * 32 + lane, g = ch / kOfGroup;
                        const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, t.place, g) * (D / 2) + (ch % kOfGroup) * 16;
                        cp_async_16_upto(raw + ch * 16, pool + at, ch * 16 / (D / 2) < t.stored ? 16u : 0u);  // (behind the last token anything may stand: zeros)
                    }
                    #pragma unroll
                    for (uint32_t i = 0; i < N * kBlocks / 128; ++i) {
                        constexpr uint32_t kOfGroup = 4 * kBlocks;
                        const uint32_t ch = i * 32 + lane, first = ch * 4;  // scales of the tile
                        const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, t.place, ch / kOfGroup) * kBlocks + (ch % kOfGroup) * 4;
                        const uint32_t there = t.stored * kBlocks;
                        cp_async_16_upto(raw + S::kCodes + ch * 16, pool_scales + at, there > first ? min((there - first) * 4, 16u) : 0u);
                    }
                    cp_async_arrive(full);
                    __syncwarp();  // (another lane's s_bad is ahead of the arrival)
                    if (lane == 0) {
                        s_raw_powers[own] = t.values ? powers.y : powers.x;
                        if (!t.values) s_powers[t.info & 7u] = powers;
                        ptx::mbar_arrive(full);
                    }
                    // the L2 asked for the next tile's codes
                    #pragma unroll
                    for (uint32_t i = 0; i < S::kCodes / 4096; ++i) {
                        constexpr uint32_t kOfGroup = D / 16;  // lines
                        const uint32_t line = i * 32 + lane;
                        const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, next.place, line / kOfGroup) * (D / 2) + (line % kOfGroup) * 128;
                        if (line * 128 / (D / 2) < next.stored) asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t *>(next.values ? c.v : c.k) + at));
                    }
                    if (next.real) ask_scales(next);
                    t = next;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
            } else if (!NF4 && small_pages) {
                // ---- a bf16 cache whose pages hold sixteen tokens (or an odd number of them): 16-byte copies of four warps to K's tiles and four to V's ----
                // (With TMA, boxes of sixteen tokens: 16 sequences of 8192 tokens, 8 heads of 128, pages of 16, 64 rows a head 106 to 109 us,
                // so 96 to 98; heads of 64 98 to 121 us, so 76 to 90; pages of 48 are as fast either way, larger boxes stay with TMA.)
                if (warp < kCopyWarp && warp >= kExpandWarp) {
                    constexpr uint32_t kRows = N / kSmallCopies, kChunks = D / 8, kRound = 32 / kChunks;  // tokens of a warp; 16-byte pieces of a row; tokens at a time
                    const uint32_t own = warp & 1u, first = ((warp - kExpandWarp) >> 1) * kRows, x = lane % kChunks;
                    const __nv_bfloat16 *const pool = static_cast<const __nv_bfloat16 *>(own ? c.v : c.k);
                    uint32_t pending = 0;  // the barrier of the tile whose copies are under way, or 0
                    auto deliver = [&] {   // (its copies are done)
                        ptx::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive(pending);
                        pending = 0;
                    };
                    Ring ring;
                    for (uint32_t piece = 0; ok && walk.next(c, b, a, p); ++piece) {
                        #pragma unroll 1
                        for (uint32_t turn = 0; ok && turn < 2 * p.steps; ++turn, ring.on(slots)) {
                            const Turn<2> of(turn, p.steps);
                            if (of.values != own) continue;
                            const uint32_t t0 = (p.step0 + of.step) * N + first, slot = ring.slot, dst = place_of(slot);
                            const uint32_t stored = p.s.length > t0 ? min(p.s.length - t0, kRows) : 0u;  // of the warp's tokens
                            uint32_t place = 0;  // of group `lane`
                            if (lane * kGroup < stored) {
                                const uint32_t t = t0 + lane * kGroup, at = c.by_page.of(t);
                                const int32_t page = __ldg(b.table + (uint64_t)p.seq * b.width + at);
                                if (page >= 0 && (uint32_t)page < c.pages) place = ((uint32_t)page * c.heads + p.head) * c.page_size + (t - at * c.page_size);
                                else s_bad[piece & 7u] = piece + 1;
                            }
                            __syncwarp();
                            if (ring.round && !__all_sync(0xffffffffu, ptx::mbar_try_wait(empty0 + 8 * slot, (ring.round + 1) & 1u))) {
                                if (pending) {  // (before a wait that may be for what it holds back)
                                    asm volatile("cp.async.wait_all;" ::: "memory");
                                    deliver();
                                }
                                wait(empty0 + 8 * slot, (ring.round + 1) & 1u, 35);
                            }
                            if (!ok) break;
                            #pragma unroll
                            for (uint32_t i = 0; i < kRows / kRound; ++i) {
                                const uint32_t t = i * kRound + lane / kChunks, row = first + t;
                                const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, place, i * kRound / kGroup) + t % kGroup;
                                ptx::cp_async_16_or_zero(dst + (x >> 3) * S::kBox + row * 128 + (((x & 7u) ^ (row & 7u)) << 4), pool + at * D + x * 8, t < stored);
                            }
                            asm volatile("cp.async.commit_group;" ::: "memory");
                            if (pending) {
                                asm volatile("cp.async.wait_group 1;" ::: "memory");
                                deliver();
                            }
                            pending = full0 + 8 * slot;
                        }
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    if (ok && pending) deliver();
                }
            } else if (NF4 ? warp == kCopyWarp : warp >= kExpandWarp && warp < kExpandWarp + 2 * kCopies) {
                // ---- tiles as they are: of a bf16 cache's pages, or of what was expanded ahead ----
                const uint32_t own = NF4 ? 0u : (warp - kExpandWarp) & 1u, part = NF4 ? 0u : (warp - kExpandWarp) >> 1;  // bf16: K or V, and which columns
                const uint32_t unit = box_rows, units = N / unit;  // tokens that come together, being in one page
                uint32_t tails = 0, step = 0;
                Ring ring;
                for (uint32_t piece = 0; ok && walk.next(c, b, a, p); ++piece, step += p.steps) {
                    const uint32_t tile0 = expanded ? __ldg(dense.bases + p.seq) + p.step0 : 0u;
                    const uint32_t stored = min(p.s.length, (p.step0 + p.steps) * N);  // tokens that there are
                    #pragma unroll 1
                    for (uint32_t turn = 0; ok && turn < 2 * p.steps; ++turn, ring.on(slots)) {
                        const Turn<2> of(turn, p.steps);
                        const uint32_t which = of.values, j = of.step;
                        if (!NF4 && which != own) continue;
                        const uint32_t t0 = (p.step0 + j) * N, g = lane % units, box = lane / units, t = t0 + g * unit;
                        const uint32_t groups = stored > t0 ? min(units, (stored - t0 + unit - 1) / unit) : 0u;
                        const uint32_t slot = ring.slot, dst = place_of(slot);
                        uint32_t place = 0;
                        if (NF4) {
                            if (!which) {
                                const float2 powers = __ldg(dense.powers + (uint64_t)(tile0 + j) * c.heads + p.head);
                                if (powers.x == 0.f) s_bad[piece & 7u] = piece + 1;  // (a page that there is not)
                                if (lane == 0) s_powers[(step + j) & 7u] = powers;
                            }
                        } else if (g < groups) {
                            const uint32_t at = c.by_page.of(t);
                            const int32_t page = __ldg(b.table + (uint64_t)p.seq * b.width + at);
                            if (page >= 0 && (uint32_t)page < c.pages) place = ((uint32_t)page * c.heads + p.head) * c.page_size + (t - at * c.page_size);
                            else s_bad[piece & 7u] = piece + 1;
                        }
                        __syncwarp();
                        if (ring.round) wait(empty0 + 8 * slot, (ring.round + 1) & 1u, 35);
                        if (!ok) break;
                        if (NF4) {
                            const uint32_t bar = full0 + 8 * slot;
                            if (lane == 0) {
                                ptx::mbar_arrive_expect_tx(bar, S::kTile);
                                const int32_t row = (int32_t)(((tile0 + j) * c.heads + p.head) * N);
                                #pragma unroll
                                for (uint32_t x = 0; x < D / 64; ++x) ptx::tma_load_2d(dst + x * S::kBox, which ? &tmap_v : &tmap_k, (int32_t)(64 * x), row, bar);
                                for (uint32_t e = 1; e < kExpandWarps; ++e) ptx::mbar_arrive(bar);  // (for the warps that expand)
                            }
                        } else {
                            const bool tail = which && t0 + N > p.s.length;  // values that anything may stand behind: zeros, for weights of zero
                            const uint32_t bar = tail ? tail0 + 8 * part : full0 + 8 * slot;
                            constexpr uint32_t kColumns = D / 64 / kCopies;  // boxes of 64
                            if (lane == 0) ptx::mbar_arrive_expect_tx(bar, groups * (unit * 128) * kColumns);
                            __syncwarp();
                            if (g < groups && box < kColumns) {
                                const uint32_t x = part * kColumns + box;
                                ptx::tma_load_2d(dst + x * S::kBox + g * (unit * 128), which ? &tmap_v : &tmap_k, (int32_t)(64 * x), (int32_t)place, bar);
                            }
                            if (tail) {
                                wait(bar, tails & 1u, 35);
                                ++tails;
                                for (uint32_t k = (p.s.length > t0 ? p.s.length - t0 : 0u) * 8 + lane; k < N * 8; k += 32)
                                    #pragma unroll
                                    for (uint32_t x = 0; x < kColumns; ++x) st_shared_u4(dst + (part * kColumns + x) * S::kBox + k * 16, make_uint4(0u, 0u, 0u, 0u));
                                ptx::fence_proxy_async();
                                __syncwarp();
                                if (lane == 0) ptx::mbar_arrive(full0 + 8 * slot);
                            }
                        }
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

constexpr uint64_t kTileRows = 128;
uint64_t tokens_of(const AttentionCall &c) { return c.head_dim == 256 ? 64 : 128; }

// Tiles to a head to be expanded ahead: where the host's bounds say that nine row tiles or more of a head go over most tokens.  Expanding 128 tokens of a head
// ahead takes 29 ns, and saves 3.5 of a row tile's 10.
uint64_t dense_tiles(const AttentionCall &c) {
    if (!c.nf4 || (uint64_t)c.most_rows * c.view.group <= 8 * kTileRows) return 0;
    return attention_expanded_tiles(c);
}

// The row tiles that several CTAs had: a warp to a row.  Its parts' largest exponents and sums come together, a lane to each, and then their results, eight
// parts asked for at a time and added in the order of the tokens.
constexpr uint32_t kJoinWarpsOfTree = 8;
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarpsOfTree)
join_rows_kernel(const AttentionView a, const Split *const splits) {
    constexpr uint32_t kWide = D / 32, kAtOnce = 8;  // values of a row to a lane; parts in flight
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const Split s = splits[blockIdx.x];
    const uint32_t lane = threadIdx.x & 31u, parts = s.more + 1;
    const uint32_t r = blockIdx.y * kJoinWarpsOfTree + threadIdx.x / 32;
    if (r >= s.rows) return;
    auto part = [&](uint32_t i) { return (uint64_t)(2 * (blockIdx.x + i) + (i ? 0 : 1)) * kTileRows + r; };
    float m = -INFINITY;
    for (uint32_t i = lane; i < parts; i += 32) m = fmaxf(m, __ldg(&a.part_ml[part(i)].x));
    #pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float from = m == -INFINITY ? 0.f : m;  // (nothing seen: 2^-inf)
    float sum = 0.f, acc[kWide] = {};
    for (uint32_t i0 = 0; i0 < parts; i0 += 32) {
        const float2 ml = i0 + lane < parts ? __ldg(a.part_ml + part(i0 + lane)) : make_float2(-INFINITY, 0.f);
        const float counts = exp2_approx(ml.x - from);
        sum = fmaf(counts, ml.y, sum);
        for (uint32_t i = i0; i < min(parts, i0 + 32); i += kAtOnce) {
            float v[kAtOnce][kWide];
            #pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                if (i + k >= parts) continue;
                const float2 *const o = reinterpret_cast<const float2 *>(a.part_o + part(i + k) * D + lane * kWide);
                #pragma unroll
                for (uint32_t j = 0; j < kWide; j += 2) {
                    const float2 w = __ldg(o + j / 2);
                    v[k][j] = w.x;
                    v[k][j + 1] = w.y;
                }
            }
            #pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                if (i + k >= parts) continue;
                const float f = __shfl_sync(0xffffffffu, counts, (i + k) & 31u);
                #pragma unroll
                for (uint32_t j = 0; j < kWide; ++j) acc[j] = fmaf(f, v[k][j], acc[j]);
            }
        }
    }
    #pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const uint32_t q_row = s.r0 + r, token = a.by_group.of(q_row);
    __nv_bfloat16 *const out = static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)(s.row0 + token) * a.ldo + (uint64_t)(s.head * a.group + q_row - token * a.group) * D + lane * kWide;
    #pragma unroll
    for (uint32_t j = 0; j < kWide; j += 2) *reinterpret_cast<uint32_t *>(out + j) = bf16_pair(acc[j] * f, acc[j + 1] * f);
}

struct Layout {  // of the workspace
    uint64_t splits, ml, o, bases, powers, k, v, bytes;
    explicit Layout(const AttentionCall &c) {
        uint64_t at = kAttentionFlagBytes;
        auto take = [&](uint64_t n) {
            const uint64_t from = at;
            at += (n + 255) / 256 * 256;
            return from;
        };
        const uint64_t tiles = dense_tiles(c), expanded = tiles * c.cache.heads * tokens_of(c) * c.head_dim * 2;
        splits = take(kNumSMs * sizeof(Split));
        ml = take(2ull * kNumSMs * kTileRows * sizeof(float2));
        o = take(2ull * kNumSMs * kTileRows * c.head_dim * sizeof(float));
        bases = take(tiles ? (c.batch.sequences + 1ull) * sizeof(uint32_t) : 0);
        powers = take(tiles * c.cache.heads * sizeof(float2));
        k = take(expanded);
        v = take(expanded);
        bytes = at;
    }
};

template <int D, bool NF4>
int32_t launch(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    using S = Shape<D, NF4>;
    auto kernel = attention_tree_kernel<D, NF4>;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kSmem));
    const uint64_t pool = (uint64_t)c.cache.pages * c.cache.heads * c.cache.page_size;
    CUtensorMap map_k{}, map_v{};
    uint32_t box_rows = kGroup;  // tokens of a page that come in one copy
    while (box_rows < S::kTokens && c.cache.page_size % (2 * box_rows) == 0) box_rows *= 2;
    if (!NF4) {
        NF4_TRY(make_map(&map_k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.cache.k, pool, D, 2 * D, box_rows, 64, CU_TENSOR_MAP_SWIZZLE_128B));
        NF4_TRY(make_map(&map_v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.cache.v, pool, D, 2 * D, box_rows, 64, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    FailureRef failure;
    NF4_TRY(prefill_failure_ref(&failure));
    const Layout at(c);
    Split *const splits = reinterpret_cast<Split *>(workspace + at.splits);
    AttentionView view = c.view;
    view.part_ml = reinterpret_cast<float2 *>(workspace + at.ml);
    view.part_o = reinterpret_cast<float *>(workspace + at.o);
    Dense dense{};
    if (NF4) {
        dense.capacity = (uint32_t)dense_tiles(c);
        if (dense.capacity) {
            uint32_t *const bases = reinterpret_cast<uint32_t *>(workspace + at.bases);
            float2 *const powers = reinterpret_cast<float2 *>(workspace + at.powers);
            dense.bases = bases;
            dense.powers = powers;
            NF4_TRY(attention_expand(c, dense.capacity, workspace + at.k, workspace + at.v, bases, powers, &map_k, &map_v, stream));
        }
    }
    const uint32_t ctas = persistent_ctas();
    count_launch(2);
    NF4_TRY(launch_maybe_overlapped(kernel, dim3(ctas), dim3(kThreads), S::kSmem, stream, true, map_k, map_v, c.cache, c.batch, view, dense, box_rows, splits, failure));
    return launch_maybe_overlapped(join_rows_kernel<D>, dim3(ctas, S::kRows / kJoinWarpsOfTree), dim3(32 * kJoinWarpsOfTree), 0, stream, true, view,
                                   static_cast<const Split *>(splits));
}

}  // namespace

uint64_t attention_tree_bytes(const AttentionCall &c) {
    return Layout(c).bytes;
}

// The line of steps is counted in 32 bits, and what the page table has room for bounds it.
bool attention_tree_counts(const AttentionCall &c) {
    const uint64_t tiles = ((uint64_t)c.batch.rows * c.view.group / kTileRows + c.batch.sequences) * c.cache.heads;
    const uint64_t steps = ((uint64_t)c.batch.width * c.cache.page_size + tokens_of(c) - 1) / tokens_of(c);
    return tiles * (steps + 1 + kStart) < 1ull << 31;
}

int32_t attention_tree(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    switch (c.head_dim) {
        case 64: return c.nf4 ? launch<64, true>(c, workspace, stream) : launch<64, false>(c, workspace, stream);
        case 128: return c.nf4 ? launch<128, true>(c, workspace, stream) : launch<128, false>(c, workspace, stream);
        default: return c.nf4 ? launch<256, true>(c, workspace, stream) : launch<256, false>(c, workspace, stream);
    }
}

}  // namespace nf4
