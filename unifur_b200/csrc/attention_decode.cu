// Attention of few rows over the paged cache (decode steps, drafted tokens): up to sixteen rows of a head at a time.
//
// Bound by the bytes of the cache, and for a quantized one by its lookups as well.  A CTA has an SM to itself; the groups of
// sixteen tokens of all sequences, heads and row tiles form one line that the CTAs share out evenly, whatever the sequences'
// lengths.  In a CTA every warp takes every W-th group of its share, which it has brought to shared memory by TMA into a
// ring of its own (three groups in flight: no barrier between warps while tokens stream), with its own running largest exponent,
// sum and accumulator.  At the end of a head's share the warps' results are joined through shared memory, and where the
// tokens of a head were several CTAs', the CTA that is done last joins theirs out of the workspace, in the order of the tokens.
//
// Mathematics, per group of sixteen tokens t and eight rows r (one MMA tile):
//   x[t][r] = scale * log2(e) * sum_b ks[t][b] (levels_b[t] . q_b[r]),  w = 2^(x - m[r] + 8),  l[r] += w,
//   o[d][r] += sum_t levels[t][d] (w[t][r] vs[t][block of d])
// Tokens are on the MMA's M side in the first product and on its K side in the second, so the weights go from one to the other by a
// transposition of 8 x 8 tiles (movmatrix) and nothing is padded to sixteen rows.  A quantized cache's codes are
// looked up in a table of pairs of f16 levels, a copy to a lane, as in the decode GEMV: a byte of K holds neighbouring d, and for V the
// nibbles of two tokens are put side by side first.  Block scales never touch f16 on their own: K's multiply the f32 sums of a
// block, V's the weights.  The weights enter the second product in f16 (2^-11 of each; bf16 with a bf16 cache: 2^-8, half of the
// result's own rounding on average), times V's scale divided by a power of two `ref` that no scale so far exceeds.
// m is the largest exponent seen or up to 8 below it: while no score exceeds m by more than 8 nothing has to be
// rescaled, which spares the maximum over the tokens in nearly every group.
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace nf4 {

namespace {

// Weights are 2^(x - m + kRaise), and times V's scales up to 2^15, so that f16 holds those that are 2^-31 of a row's largest; their sum is
// raised alike.
constexpr float kRaise = 8.f;
constexpr uint32_t kGroup = 16;   // tokens to a group: pages are multiples of it
constexpr uint32_t kStages = 3;   // groups in flight, a warp
constexpr uint32_t kPassRegs = 16;  // accumulator registers of a thread that go through shared memory at a time

template <int D, bool NF4, int NT>
struct Shape {
    // what an SM holds: registers for the accumulators, and three groups to a warp in about 100 KB (192 KB without the table)
    static constexpr uint32_t kWarps = NF4 ? (D == 256 || (D == 128 && NT == 2) ? 8 : 16) : D == 64 ? 12 : 1024 / D;
    static constexpr uint32_t kThreads = 32 * kWarps;
    static constexpr uint32_t kRows = 8 * NT, kBlocks = D / 64;
    static constexpr uint32_t kRowBytes = NF4 ? D / 2 : 2 * D;       // a token's stored row
    static constexpr uint32_t kTile = kGroup * kRowBytes;              // a group's codes or values, of K or of V
    static constexpr uint32_t kScaleTile = NF4 ? kGroup * kBlocks * 4 : 0;  // its scales, likewise
    static constexpr uint32_t kAcc = D / 16 * 4 * NT;                  // accumulator registers of a thread
    // where the warps' results meet, and in a join every CTA's factors
    static constexpr uint32_t kMerge = kWarps * kPassRegs * 32 * 4 > 10240 ? kWarps * kPassRegs * 32 * 4 : 10240;
    static constexpr uint32_t kScaleRing = kWarps * kStages * 2 * kScaleTile;
    static constexpr uint32_t kFirst = kMerge + kScaleRing;            // ahead of the table
    static constexpr uint32_t kRing = kWarps * kStages * 2 * kTile;
    // the table lies on a multiple of its size, so that a byte permute makes a whole address: the second 64 KB of shared memory
    static constexpr uint32_t kSmem = NF4 ? 131072 - 1024 + kRing : kFirst + kRing + 1024;
    static constexpr uint32_t kPartFloats = kRows * D + 2 * kRows;    // a share's result in the workspace
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// Which token of a group an MMA's row or k stands for: an order in which eight lanes' reads of K (rows 0..3 at a time) and of V
// (rows 0, 2, 4, 6) both hit all banks with the TMA's swizzle.
__device__ __forceinline__ uint32_t token_of(uint32_t i) { return ((i ^ (i >> 2)) & 1u) << 2 | (i & 1u) << 1 | ((i >> 1) & 1u) | (i & 8u); }

struct Share {
    uint64_t total;
    uint32_t ctas;
    bool whole;  // heads are not divided
    __device__ uint64_t start(uint32_t cta) const { return total * cta / ctas; }
    __device__ uint32_t cta_of(uint64_t g) const { return (uint32_t)(((g + 1) * ctas - 1) / total); }
};

struct Line {  // a sequence's part of the line of groups
    uint32_t groups;  // to a head and row tile
    uint32_t items;   // heads times row tiles
};
__device__ __forceinline__ Line line_of(const CacheView &c, const BatchView &b, uint32_t group, uint32_t rows_of_tile, uint32_t s) {
    Line l{0, 0};
    if (s >= b.sequences) return l;
    const Sequence q = sequence_of(c, b, s);
    l.groups = max(1u, (q.length + kGroup - 1) / kGroup);
    l.items = (uint32_t)(((uint64_t)q.rows * group + rows_of_tile - 1) / rows_of_tile) * c.heads;
    return l;
}

template <int D, bool NF4, int NT>
__global__ void __launch_bounds__(Shape<D, NF4, NT>::kThreads, 1)
attention_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const CacheView c, const BatchView b,
                        const AttentionView a, uint32_t *const counters, float *const parts, const FailureRef failure) {
    using S = Shape<D, NF4, NT>;
    constexpr uint32_t W = S::kWarps, kBlocks = S::kBlocks;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bars[W * kStages];
    __shared__ float2 s_ml[W][S::kRows];
    __shared__ float2 s_fin[S::kRows];
    __shared__ uint32_t s_last;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
    const uint32_t base = ptx::smem_addr(smem);
    const uint32_t table = NF4 ? (base + S::kFirst + 65535u) & ~65535u : 0;
    const uint32_t ring0 = (NF4 ? table + 65536u : (base + S::kFirst + 1023u) & ~1023u) + warp * (kStages * 2 * S::kTile);
    const uint32_t scales0 = base + S::kMerge + warp * (kStages * 2 * S::kScaleTile);
    float *const merge = reinterpret_cast<float *>(smem);
    const uint32_t bars = ptx::smem_addr(s_bars) + 8 * kStages * warp;
    if (NF4 && table + 65536u + S::kRing > base + S::kSmem) {
        if (tid == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 20);
        return;
    }
    if (lane == 0) {
        for (uint32_t i = 0; i < kStages; ++i) ptx::mbar_init(bars + 8 * i, 1);
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
    }
    if (NF4) {
        for (uint32_t i = tid; i < 256 * 8; i += S::kThreads) {  // a thread writes four lanes' copies of an entry
            const uint32_t byte = i >> 3, entry = c_level_f16_bits[byte & 15u] | c_level_f16_bits[byte >> 4] << 16;
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(table + byte * 256u + (i & 7u) * 16u), "r"(entry) : "memory");
        }
    }
    __syncthreads();
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    // ---- this CTA's share of the line ----
    Share share{0, 1, false};
    {
        uint64_t groups = 0;
        uint32_t items = 0;
        for (uint32_t s = lane; s < b.sequences; s += 32) {
            const Line l = line_of(c, b, a.group, S::kRows, s);
            groups += (uint64_t)l.groups * l.items;
            items += l.items;
        }
        #pragma unroll
        for (int k = 1; k < 32; k <<= 1) {
            groups += __shfl_xor_sync(0xffffffffu, groups, k);
            items += __shfl_xor_sync(0xffffffffu, items, k);
        }
        if (groups == 0) return;
        share.total = groups;
        share.ctas = (uint32_t)min((uint64_t)gridDim.x, groups);
        // a head whose tokens are two groups to a warp is not worth dividing: the join costs about as much
        share.whole = groups <= (uint64_t)items * (2 * W);
    }
    if (blockIdx.x >= share.ctas) return;
    const uint64_t first = share.start(blockIdx.x), end = share.start(blockIdx.x + 1);

    // the sequence that `first` is in, and how far into it
    uint32_t seq = 0;
    Line line{0, 0};
    uint64_t at = 0;  // groups into the sequence's part of the line
    {
        uint64_t before = 0;
        for (uint32_t s0 = 0; s0 < b.sequences; s0 += 32) {
            const Line l = line_of(c, b, a.group, S::kRows, s0 + lane);
            const uint64_t own = (uint64_t)l.groups * l.items;
            uint64_t upto = own;
            #pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const uint64_t o = __shfl_up_sync(0xffffffffu, upto, k);
                if (lane >= (uint32_t)k) upto += o;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + upto > first);
            if (past) {
                const int l0 = __ffs(past) - 1;
                seq = s0 + l0;
                line.groups = __shfl_sync(0xffffffffu, l.groups, l0);
                line.items = __shfl_sync(0xffffffffu, l.items, l0);
                at = first - (before + __shfl_sync(0xffffffffu, upto - own, l0));
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    uint64_t now = first;
    uint32_t item = (uint32_t)(at / line.groups), off = (uint32_t)(at % line.groups);
    if (share.whole && off) {  // a head belongs to the CTA in whose share it begins
        now += line.groups - off;
        off = 0;
        ++item;
    }

    // ---- what a lane has of every group ----
    const uint32_t lane_word = table | lane * 4u;
    auto pair_at = [&](uint32_t word, int byte) -> uint32_t {  // the levels of a byte's two codes: {table's upper half, byte, lane * 4}
        return ld_shared_u32(__byte_perm(word, lane_word, 0x7604u | ((uint32_t)byte << 4)));
    };
    constexpr uint32_t kRB = S::kRowBytes;
    // the 16-byte chunk of a row that TMA puts at chunk i of it is i ^ twist(row)
    auto twist = [](uint32_t row) -> uint32_t { return !NF4 || D == 256 ? row & 7u : D == 128 ? (row >> 1) & 3u : (row >> 2) & 1u; };
    const uint32_t krow = token_of(g), vrow0 = token_of(2 * t4), vrow1 = token_of(2 * t4 + 1);

    uint32_t used = 0;  // groups that this warp has taken from its ring
    bool ok = true;
    const uint32_t pages16 = c.page_size / kGroup;

    while (now < end) {
        while (item >= line.items) {  // on to the next sequence with rows
            ++seq;
            if (seq >= b.sequences) break;
            line = line_of(c, b, a.group, S::kRows, seq);
            item = 0;
        }
        if (seq >= b.sequences) break;
        const Sequence s = sequence_of(c, b, seq);
        const uint32_t tiles = line.items / c.heads, head = item / tiles, tile = item - head * tiles;
        const uint32_t n = share.whole ? line.groups : (uint32_t)min((uint64_t)(line.groups - off), end - now);
        const uint64_t item_first = now - off;
        const uint32_t r0 = tile * S::kRows, rows = min((uint64_t)S::kRows, (uint64_t)s.rows * a.group - r0);
        const uint32_t stored = (s.length + kGroup - 1) / kGroup;  // groups that there are (none in an empty sequence)
        const uint32_t mine = off + warp < min(off + n, stored) ? (min(off + n, stored) - off - warp + W - 1) / W : 0;

        // the places of 32 of this warp's groups at a time, one to a lane, in rows of the pool
        uint32_t place = 0;
        bool lost = false;  // a page that there is not
        auto look_up = [&](uint32_t k) {
            const uint32_t i = k + lane;
            place = 0;
            if (i < mine) {
                const uint32_t group = off + warp + i * W, at_page = group / pages16;
                const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at_page);
                if (page < 0 || (uint32_t)page >= c.pages) lost = true;
                else place = ((uint32_t)page * c.heads + head) * c.page_size + (group - at_page * pages16) * kGroup;
            }
            lost = __any_sync(0xffffffffu, lost);
        };
        auto ask = [&](uint32_t k) {  // for this warp's group number k
            const uint32_t row = __shfl_sync(0xffffffffu, place, k & 31u);
            if (lane == 0) {
                const uint32_t slot = (used + k) % kStages, bar = bars + 8 * slot, to = ring0 + slot * (2 * S::kTile);
                ptx::mbar_arrive_expect_tx(bar, 2 * S::kTile + 2 * S::kScaleTile);
                if (NF4) {
                    const uint32_t st = scales0 + slot * (2 * S::kScaleTile);
                    ptx::tma_load_2d(to, &tmap_k, 0, (int32_t)row, bar);
                    ptx::bulk_g2s(st, c.k_scales + (uint64_t)row * kBlocks, S::kScaleTile, bar);
                    ptx::tma_load_2d(to + S::kTile, &tmap_v, 0, (int32_t)row, bar);
                    ptx::bulk_g2s(st + S::kScaleTile, c.v_scales + (uint64_t)row * kBlocks, S::kScaleTile, bar);
                } else {
                    #pragma unroll
                    for (uint32_t x = 0; x < D / 64; ++x) ptx::tma_load_2d(to + x * 2048, &tmap_k, (int32_t)(64 * x), (int32_t)row, bar);
                    #pragma unroll
                    for (uint32_t x = 0; x < D / 64; ++x) ptx::tma_load_2d(to + S::kTile + x * 2048, &tmap_v, (int32_t)(64 * x), (int32_t)row, bar);
                }
            }
        };
        look_up(0);
        #pragma unroll
        for (uint32_t k = 0; k < kStages; ++k)
            if (ok && k < mine) ask(k);

        // ---- the rows' queries, as the first product's B operand ----
        uint32_t q[NT][D / 16][2];
        float factor[NT][2];       // of columns 2 t4 and 2 t4 + 1: scale, log2(e), and the power of two the row was divided by
        uint32_t sees[NT][2];
        const uint32_t sees_first = visible_end(s, a.group, r0);
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t r = r0 + 8 * nt + g;
            const bool real = 8 * nt + g < rows;
            const __nv_bfloat16 *const p = static_cast<const __nv_bfloat16 *>(a.q) + (uint64_t)(s.row0 + (real ? r / a.group : 0u)) * a.ldq +
                                           (uint64_t)(head * a.group + (real ? r % a.group : 0u)) * D;
            float f = a.scale_log2;
            if (NF4) {
                uint32_t raw[kBlocks][8];
                uint32_t most = 0;  // the largest magnitude's bits
                #pragma unroll
                for (uint32_t k = 0; k < kBlocks; ++k) {
                    const uint4 *const from = reinterpret_cast<const uint4 *>(p + 64 * k + 16 * t4);
                    const uint4 zero = make_uint4(0u, 0u, 0u, 0u), lo = real ? __ldg(from) : zero, hi = real ? __ldg(from + 1) : zero;
                    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        raw[k][i] = w[i];
                        most = max(most, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
                    }
                }
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // the row is divided by a power of two that leaves its largest magnitude in [2^11, 2^12), exact for all that counts
                const int e = most ? min(max((int)(most >> 23) - 127 - 11, -100), 115) : 0;
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                f *= __uint_as_float((uint32_t)(127 + e) << 23);
                #pragma unroll
                for (uint32_t k = 0; k < kBlocks; ++k)
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        q[nt][4 * k + i / 2][i & 1] = f16_pair(__uint_as_float(raw[k][i] << 16) * down, __uint_as_float(raw[k][i] & 0xffff0000u) * down);
            } else {
                const uint32_t *const from = reinterpret_cast<const uint32_t *>(p);
                #pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    q[nt][i][0] = real ? __ldg(from + 8 * i + t4) : 0u;
                    q[nt][i][1] = real ? __ldg(from + 8 * i + 4 + t4) : 0u;
                }
            }
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                factor[nt][j] = __shfl_sync(0xffffffffu, f, 4 * (2 * t4 + j));
                const uint32_t col = 8 * nt + 2 * t4 + j;
                sees[nt][j] = col < rows ? visible_end(s, a.group, r0 + col) : s.length;
            }
        }

        float o[D / 16][NT][4] = {};
        float m[NT][2], l[NT][2] = {};
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY;
        float ref = 0.f, unref = 0.f;  // the power of two that V's scales are divided by, and its reciprocal
        #pragma unroll 1
        for (uint32_t k = 0; k < mine; ++k) {
            const uint32_t slot = (used + k) % kStages, kt = ring0 + slot * (2 * S::kTile), vt = kt + S::kTile;
            const uint32_t t0 = (off + warp + k * W) * kGroup;
            if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bars + 8 * slot, ((used + k) / kStages) & 1u))) {
                ok = false;
                if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 21);
            }
            // ---- scores ----
            float x[NT][4];
            if (NF4) {
                const uint32_t ksc = scales0 + slot * (2 * S::kScaleTile) + krow * (4 * kBlocks);
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
                #pragma unroll
                for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                    const uint32_t from = kt + krow * kRB + ((2 * kb + (t4 >> 1)) ^ twist(krow)) * 16 + (t4 & 1u) * 8;
                    const uint2 lo = ptx::ld_shared_v2(from), hi = ptx::ld_shared_v2(from + 8 * kRB);
                    const float s_lo = __uint_as_float(ld_shared_u32(ksc + 4 * kb)), s_hi = __uint_as_float(ld_shared_u32(ksc + 4 * kb + 32 * kBlocks));
                    float acc[NT][4] = {};
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t wl = i < 2 ? lo.x : lo.y, wh = i < 2 ? hi.x : hi.y;
                        const int by = 2 * (i & 1);
                        const uint32_t a0 = pair_at(wl, by), a1 = pair_at(wh, by), a2 = pair_at(wl, by + 1), a3 = pair_at(wh, by + 1);
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt) ptx::mma_16816_f16(acc[nt], a0, a1, a2, a3, q[nt][4 * kb + i][0], q[nt][4 * kb + i][1]);
                    }
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        x[nt][0] = fmaf(s_lo, acc[nt][0], x[nt][0]);
                        x[nt][1] = fmaf(s_lo, acc[nt][1], x[nt][1]);
                        x[nt][2] = fmaf(s_hi, acc[nt][2], x[nt][2]);
                        x[nt][3] = fmaf(s_hi, acc[nt][3], x[nt][3]);
                    }
                }
            } else {
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
                const uint32_t row = (lane & 7u) + ((lane >> 3) & 1u) * 8, half = lane >> 4;
                #pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    uint32_t af[4];
                    ptx::ldmatrix_x4(af, kt + (i >> 2) * 2048 + row * 128 + (((2 * (i & 3) + half) ^ (row & 7u)) << 4));
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) ptx::mma_16816_bf16(x[nt], af[0], af[1], af[2], af[3], q[nt][i][0], q[nt][i][1]);
                }
            }
            const uint32_t tok_lo = t0 + (NF4 ? krow : g), tok_hi = tok_lo + 8;
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                x[nt][0] *= factor[nt][0];
                x[nt][1] *= factor[nt][1];
                x[nt][2] *= factor[nt][0];
                x[nt][3] *= factor[nt][1];
            }
            const bool tail = t0 + kGroup > sees_first;  // some row does not see all of the group
            if (tail) {
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    x[nt][0] = tok_lo < sees[nt][0] ? x[nt][0] : -INFINITY;
                    x[nt][1] = tok_lo < sees[nt][1] ? x[nt][1] : -INFINITY;
                    x[nt][2] = tok_hi < sees[nt][0] ? x[nt][2] : -INFINITY;
                    x[nt][3] = tok_hi < sees[nt][1] ? x[nt][3] : -INFINITY;
                }
            }
            // ---- weights ----
            bool above = false;
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int j = 0; j < 2; ++j) above = above || fmaxf(x[nt][j], x[nt][j + 2]) > m[nt][j] + 8.f;
            if (__any_sync(0xffffffffu, above)) {
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = fmaxf(x[nt][j], x[nt][j + 2]);
                        #pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        top = fmaxf(top, m[nt][j]);
                        const float keep = m[nt][j] == -INFINITY ? 0.f : exp2_approx(m[nt][j] - top);
                        m[nt][j] = top;
                        l[nt][j] *= keep;
                        #pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            o[i][nt][j] *= keep;
                            o[i][nt][j + 2] *= keep;
                        }
                    }
            }
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float from = m[nt][j] == -INFINITY ? 0.f : m[nt][j] - kRaise;
                    x[nt][j] = exp2_approx(x[nt][j] - from);
                    x[nt][j + 2] = exp2_approx(x[nt][j + 2] - from);
                    l[nt][j] += x[nt][j] + x[nt][j + 2];
                }
            // ---- weights times values ----
            if (NF4) {
                const uint32_t vsc = scales0 + slot * (2 * S::kScaleTile) + S::kScaleTile + krow * (4 * kBlocks);
                float s_lo[kBlocks], s_hi[kBlocks];
                uint32_t most = 0;
                #pragma unroll
                for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                    // (behind the sequence's last token anything may stand)
                    s_lo[kb] = tok_lo < s.length ? __uint_as_float(ld_shared_u32(vsc + 4 * kb)) : 0.f;
                    s_hi[kb] = tok_hi < s.length ? __uint_as_float(ld_shared_u32(vsc + 4 * kb + 32 * kBlocks)) : 0.f;
                    most = max(most, max(__float_as_uint(s_lo[kb]), __float_as_uint(s_hi[kb])));
                }
                most = __reduce_max_sync(0xffffffffu, most);
                if (most > __float_as_uint(ref)) {
                    // the next power of two but one, between 2^-100 and 2^126
                    const uint32_t bits = min(max((most & 0x7f800000u) + 0x01000000u, 27u << 23), 253u << 23);
                    const float keep = ref * __uint_as_float(0x7f000000u - bits);
                    ref = __uint_as_float(bits);
                    unref = __uint_as_float(0x7f000000u - bits);
                    #pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            #pragma unroll
                            for (int j = 0; j < 4; ++j) o[i][nt][j] *= keep;
                }
                #pragma unroll
                for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                    const float f_lo = s_lo[kb] * unref, f_hi = s_hi[kb] * unref;
                    uint32_t w[NT][2];
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        w[nt][0] = movmatrix(f16_pair(x[nt][0] * f_lo, x[nt][1] * f_lo));
                        w[nt][1] = movmatrix(f16_pair(x[nt][2] * f_hi, x[nt][3] * f_hi));
                    }
                    const uint32_t in0 = ((2 * kb + (g >> 2)) ^ twist(vrow0)) * 16 + (g & 3u) * 4, in1 = ((2 * kb + (g >> 2)) ^ twist(vrow1)) * 16 + (g & 3u) * 4;
                    const uint32_t u0 = ld_shared_u32(vt + vrow0 * kRB + in0), u1 = ld_shared_u32(vt + vrow1 * kRB + in1);
                    const uint32_t u2 = ld_shared_u32(vt + (vrow0 + 8) * kRB + in0), u3 = ld_shared_u32(vt + (vrow1 + 8) * kRB + in1);
                    constexpr uint32_t kLow = 0x0f0f0f0fu;
                    const uint32_t even = (u0 & kLow) | (u1 << 4 & ~kLow), odd = (u0 >> 4 & kLow) | (u1 & ~kLow);
                    const uint32_t even8 = (u2 & kLow) | (u3 << 4 & ~kLow), odd8 = (u2 >> 4 & kLow) | (u3 & ~kLow);
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a0 = pair_at(even, i), a1 = pair_at(odd, i), a2 = pair_at(even8, i), a3 = pair_at(odd8, i);
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt) ptx::mma_16816_f16(o[4 * kb + i][nt], a0, a1, a2, a3, w[nt][0], w[nt][1]);
                    }
                }
            } else {
                if (t0 + kGroup > s.length) {  // behind the last token anything may stand: zeros, for the product with weights of zero
                    for (uint32_t i = lane; i < kGroup * (D / 8); i += 32) {
                        const uint32_t row = i / (D / 8), chunk = i % (D / 8);
                        if (t0 + row >= s.length)
                            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vt + (chunk >> 3) * 2048 + row * 128 + ((chunk & 7u) << 4)), "r"(0u) : "memory");
                    }
                    ptx::fence_proxy_async();
                    __syncwarp();
                }
                uint32_t w[NT][2];
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    w[nt][0] = movmatrix(bf16_pair(x[nt][0], x[nt][1]));
                    w[nt][1] = movmatrix(bf16_pair(x[nt][2], x[nt][3]));
                }
                const uint32_t row = (lane & 7u) + (lane >> 4) * 8, half = (lane >> 3) & 1u;
                #pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    uint32_t af[4];
                    ptx::ldmatrix_x4_trans(af, vt + (i >> 2) * 2048 + row * 128 + (((2 * (i & 3) + half) ^ (row & 7u)) << 4));
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) ptx::mma_16816_bf16(o[i][nt], af[0], af[1], af[2], af[3], w[nt][0], w[nt][1]);
                }
            }
            __syncwarp();
            if (k + kStages < mine) {
                if (((k + kStages) & 31u) == 0) look_up(k + kStages);
                if (ok) ask(k + kStages);
            }
        }
        used += mine;

        // ---- the warps' results become the share's ----
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
                if (lost || !ok) l[nt][j] = __uint_as_float(0x7fc00000u);  // NaN, and the results with it
                if (g == 0) s_ml[warp][8 * nt + 2 * t4 + j] = make_float2(m[nt][j], l[nt][j]);
            }
        __syncthreads();
        if (warp == 0 && lane < S::kRows) {
            float top = -INFINITY, sum = 0.f;
            #pragma unroll
            for (uint32_t w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][lane].x);
            #pragma unroll
            for (uint32_t w = 0; w < W; ++w) sum += s_ml[w][lane].y * (s_ml[w][lane].x == -INFINITY ? 0.f : exp2_approx(s_ml[w][lane].x - top));
            s_fin[lane] = make_float2(top, sum);
        }
        {
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = -INFINITY;
                    #pragma unroll
                    for (uint32_t w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][8 * nt + 2 * t4 + j].x);
                    const float keep = (m[nt][j] == -INFINITY ? 0.f : exp2_approx(m[nt][j] - top)) * (NF4 ? ref : 1.f);
                    #pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        o[i][nt][j] *= keep;
                        o[i][nt][j + 2] *= keep;
                    }
                }
        }
        const uint32_t c0 = share.whole ? blockIdx.x : share.cta_of(item_first), c1 = share.whole ? blockIdx.x : share.cta_of(item_first + line.groups - 1);
        const bool whole = c0 == c1;
        float *const part = parts + (uint64_t)(2 * blockIdx.x + (off ? 0 : 1)) * S::kPartFloats;
        // an accumulator register pair (j, j + 2) of (i, nt), lane: row 8 nt + 2 t4 + j, values `value_at` and the next
        auto value_at = [](uint32_t i, uint32_t ln) -> uint32_t {
            return NF4 ? (i >> 2) * 64 + (ln >> 2) * 8 + (i & 3u) * 2 : 16 * i + (ln >> 2);
        };
        auto deliver = [&](uint32_t pr, uint32_t ln, float lo, float hi) {  // pr: register pair number
            const uint32_t i = pr / (2 * NT), nt = pr / 2 % NT, j = pr & 1u, row = 8 * nt + 2 * (ln & 3u) + j;
            if (row >= rows) return;
            const float sum = s_fin[row].y, f = sum == 0.f ? 0.f : 1.f / sum;
            const uint32_t r = r0 + row, d = value_at(i, ln);
            __nv_bfloat16 *const to = static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)(s.row0 + r / a.group) * a.ldo + (uint64_t)(head * a.group + r % a.group) * D + d;
            if (NF4) {
                *reinterpret_cast<uint32_t *>(to) = bf16_pair(lo * f, hi * f);
            } else {  // (of m-tile i: d and d + 8)
                to[0] = __float2bfloat16_rn(lo * f);
                to[8] = __float2bfloat16_rn(hi * f);
            }
        };
        constexpr uint32_t kPasses = S::kAcc / kPassRegs, kPairs = kPassRegs / 2;
        #pragma unroll
        for (uint32_t pass = 0; pass < kPasses; ++pass) {
            #pragma unroll
            for (uint32_t x = 0; x < kPassRegs; ++x) {
                const uint32_t reg = pass * kPassRegs + x, pr = reg / 2, i = pr / (2 * NT), nt = pr / 2 % NT, j = pr & 1u;
                merge[(warp * kPassRegs + x) * 32 + lane] = o[i][nt][j + 2 * (reg & 1u)];
            }
            __syncthreads();
            for (uint32_t e = tid; e < kPairs * 32; e += S::kThreads) {
                const uint32_t pr = e >> 5, ln = e & 31u;
                float lo = 0.f, hi = 0.f;
                #pragma unroll
                for (uint32_t w = 0; w < W; ++w) {
                    lo += merge[(w * kPassRegs + 2 * pr) * 32 + ln];
                    hi += merge[(w * kPassRegs + 2 * pr + 1) * 32 + ln];
                }
                if (whole) deliver(pass * kPairs + pr, ln, lo, hi);
                else __stcg(reinterpret_cast<float2 *>(part) + (pass * kPairs * 32 + e), make_float2(lo, hi));
            }
            __syncthreads();
        }
        if (!whole) {
            if (tid < S::kRows) __stcg(reinterpret_cast<float2 *>(part + S::kRows * D) + tid, s_fin[tid]);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t done = atomicAdd(counters + c0, 1u);
                s_last = done == c1 - c0;
                if (s_last) counters[c0] = 0;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                // the parts lie in CTA c0's place for a head that begins, in the others' for one that goes on
                auto part_of = [&](uint32_t cta) -> const float * { return parts + (uint64_t)(2 * cta + (cta == c0 ? 1 : 0)) * S::kPartFloats; };
                float *const f = merge;  // [part][row]: 2^(its largest exponent - the largest)
                if (tid < S::kRows) {
                    float top = -INFINITY, sum = 0.f;
                    for (uint32_t cta = c0; cta <= c1; ++cta) top = fmaxf(top, __ldcg(reinterpret_cast<const float2 *>(part_of(cta) + S::kRows * D) + tid).x);
                    for (uint32_t cta = c0; cta <= c1; ++cta) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part_of(cta) + S::kRows * D) + tid);
                        const float keep = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
                        sum += ml.y * keep;
                        f[(cta - c0) * S::kRows + tid] = keep;
                    }
                    s_fin[tid] = make_float2(top, sum);
                }
                __syncthreads();
                for (uint32_t e = tid; e < S::kAcc / 2 * 32; e += S::kThreads) {
                    const uint32_t pr = e >> 5, ln = e & 31u, row = 8 * (pr / 2 % NT) + 2 * (ln & 3u) + (pr & 1u);
                    float lo = 0.f, hi = 0.f;
                    #pragma unroll 4
                    for (uint32_t cta = c0; cta <= c1; ++cta) {
                        const float2 v = __ldcg(reinterpret_cast<const float2 *>(part_of(cta)) + e);
                        const float keep = f[(cta - c0) * S::kRows + row];
                        lo = fmaf(v.x, keep, lo);
                        hi = fmaf(v.y, keep, hi);
                    }
                    deliver(pr, ln, lo, hi);
                }
                __syncthreads();
            }
        }
        now += n;
        off = 0;
        ++item;
    }
    if (!ok) ptx::let_flights_land();
}

template <int D, bool NF4, int NT>
int32_t launch(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    using S = Shape<D, NF4, NT>;
    static_assert(S::kMerge / 4 / S::kRows >= kNumSMs && kNumSMs * 4 <= kAttentionFlagBytes);
    auto kernel = attention_decode_kernel<D, NF4, NT>;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kSmem));
    const uint64_t rows = (uint64_t)c.cache.pages * c.cache.heads * c.cache.page_size;
    CUtensorMap map_k, map_v;
    auto of = [&](CUtensorMap *map, const void *pool) {
        if (!NF4) return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, pool, rows, D, 2 * D, kGroup, 64, CU_TENSOR_MAP_SWIZZLE_128B);
        return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, pool, rows, D / 2, D / 2, kGroup, D / 2,
                        D == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : D == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
    };
    NF4_TRY(of(&map_k, c.cache.k));
    NF4_TRY(of(&map_v, c.cache.v));
    FailureRef failure;
    NF4_TRY(prefill_failure_ref(&failure));
    count_launch();
    return launch_maybe_overlapped(kernel, dim3(persistent_ctas()), dim3(S::kThreads), S::kSmem, stream, true, map_k, map_v, c.cache, c.batch, c.view,
                                   reinterpret_cast<uint32_t *>(workspace), reinterpret_cast<float *>(workspace + kAttentionFlagBytes), failure);
}

template <int NT>
int32_t launch_of(const AttentionCall &c, uint8_t *ws, cudaStream_t s) {
    switch (c.head_dim) {
        case 64: return c.nf4 ? launch<64, true, NT>(c, ws, s) : launch<64, false, NT>(c, ws, s);
        case 128: return c.nf4 ? launch<128, true, NT>(c, ws, s) : launch<128, false, NT>(c, ws, s);
        default: return c.nf4 ? launch<256, true, NT>(c, ws, s) : launch<256, false, NT>(c, ws, s);
    }
}

bool one_tile(const AttentionCall &c) { return (uint64_t)c.most_rows * c.view.group <= 8; }

}  // namespace

uint64_t attention_decode_bytes(const AttentionCall &c) {
    const uint64_t rows = one_tile(c) ? 8 : 16;
    return kAttentionFlagBytes + 2ull * kNumSMs * (rows * c.head_dim + 2 * rows) * sizeof(float);
}

int32_t attention_decode(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    return one_tile(c) ? launch_of<1>(c, workspace, stream) : launch_of<2>(c, workspace, stream);
}

}  // namespace nf4
