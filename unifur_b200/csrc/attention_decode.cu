// Attention of few rows, or over few tokens, of the paged cache (decode steps, drafted tokens, short prompts): up to sixteen rows of a head at a time.
//
// Bound by the bytes of the cache, and for a quantized one by its lookups as well.  A CTA has an SM to itself; the units
// (16 or 32 tokens) of all sequences, heads and row tiles, and their starts, form one line that the CTAs share out evenly, whatever the sequences'
// lengths.  In a CTA every warp takes every W-th unit of its share, which it has brought to shared memory by TMA into a
// ring of its own (two or three units in flight: no barrier between warps while tokens stream), with its own running largest exponent,
// sum and accumulator.  At the end of a head's share the warps' results are joined through shared memory, and where the
// tokens of a head were several CTAs', the CTA that is done last joins theirs out of the workspace, in the order of the tokens.
//
// Mathematics, per group of sixteen tokens t and eight rows r (one MMA tile):
//   x[t][r] = scale * log2(e) * sum_b ks[t][b] (levels_b[t] . q_b[r]),  w = 2^(x - m[r] + raise),  l[r] += w,
//   o[d][r] += sum_t levels[t][d] (w[t][r] vs[t][block of d])
// Tokens are on the MMA's M side in the first product and on its K side in the second, so the weights go from one to the other by a
// transposition of 8 x 8 tiles (movmatrix) and nothing is padded to sixteen rows.  A quantized cache's codes are
// looked up in a table of pairs of f16 levels, a copy to a lane, as in the decode GEMV: a byte of K holds neighbouring d, and for V the
// nibbles of two tokens are put side by side first.  Block scales never touch f16 on their own: K's multiply the f32 sums of a
// block, V's the weights.  The weights enter the second product in f16 (2^-11 of each; bf16 with a bf16 cache: 2^-8, half of the
// result's own rounding on average), times V's scale divided by a power of two `ref` that no scale so far exceeds, of the tokens that some row of the tile sees.
// m is the largest exponent seen or up to 8 below it: while no score exceeds m by more than 8 nothing has to be
// rescaled, which spares the maximum over the tokens in nearly every group.
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace nf4 {

namespace {

// Weights are 2^(x - m + raise).  With a quantized cache raised by 8, and times V's scales up to 2^15, so that f16 holds those that are 2^-31 of a
// row's largest; they are up to 2^16, which sums and results lose again (kLower) before V's power of two comes back, so that no value overflows
// them that would not overflow a sum of weights up to one.  bf16 has the range: weights up to one.
template <bool NF4>
constexpr float kRaise = NF4 ? 8.f : -8.f;
constexpr float kLower = 1.f / 65536.f;
constexpr float kNothing = -3e38f;  // the largest exponent of a row that has seen no token: all but the lowest number, so that weights of -inf are zeros
constexpr uint32_t kGroup = 16;   // tokens to a group: pages are multiples of it

template <int D, bool NF4, int NT>
struct Shape {
    // What an SM holds: registers for the accumulators (168 a thread with twelve warps, 255 with eight), and stages of kPer groups to a
    // warp in 96 KB (192 KB without the table).  Two groups at a time leave less to do for each: the wait, the request for the next, the
    // looks at the largest score and scale.
    static constexpr uint32_t kPer = NF4 && D <= 128 ? 2 : 1;
    static constexpr uint32_t kWarps = NF4 ? (D == 64 ? 16 : D == 128 && NT == 1 ? 12 : 8) : D == 64 ? 12 : 1024 / D;
    static constexpr uint32_t kThreads = 32 * kWarps;
    static constexpr uint32_t kRows = 8 * NT, kBlocks = D / 64;
    static constexpr uint32_t kRowBytes = NF4 ? D / 2 : 2 * D;       // a token's stored row
    static constexpr uint32_t kTile = kGroup * kRowBytes;              // a group's codes or values, of K or of V
    static constexpr uint32_t kScaleTile = NF4 ? kGroup * kBlocks * 4 : 0;  // its scales, likewise
    static constexpr uint32_t kFit = 98304 / (kWarps * kPer * 2 * kTile), kStages = !NF4 || kFit > 3 ? 3 : kFit;
    static constexpr uint32_t kAcc = D / 16 * 4 * NT;                  // accumulator registers of a thread
    // A head's start and end in a CTA (its queries, the first copies, the warps' results) take about as long as two units of every warp: 3.7 us
    // where a unit in the stream takes 0.155 (128, NF4), 2.6 and 0.2 (128, bf16).  63 sequences of one token beside one of 120,000 (four heads) take 33
    // and 62 us; 387 and 654 when only units counted, the CTAs that had the single tokens being last by far.
    static constexpr uint32_t kStart = 2 * kWarps;
    // accumulator registers of a thread that go through shared memory at a time: what the space ahead of the table holds
    static constexpr uint32_t kPassRegs = kAcc >= 32 && NF4 && kWarps <= 12 ? 32 : 16;
    static constexpr uint32_t kMerge = kWarps * kPassRegs * 32 * 4;    // where the warps' results meet
    static constexpr uint32_t kScaleRing = kWarps * kStages * kPer * 2 * kScaleTile;
    static constexpr uint32_t kFirst = kMerge + kScaleRing;            // ahead of the table
    static constexpr uint32_t kRing = kWarps * kStages * kPer * 2 * kTile;
    // the table lies on a multiple of its size, so that a byte permute makes a whole address: the second 64 KB of shared memory
    static constexpr uint32_t kSmem = NF4 ? 131072 - 1024 + kRing : kFirst + kRing + 1024;
    static_assert((!NF4 || kFirst <= 61440) && kSmem <= 232448 - 3200);  // (up to 3200 bytes are static)
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

template <uint32_t N>
__device__ __forceinline__ void ld_scales(uint32_t addr, float (&v)[N]) {
    if constexpr (N == 1) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory");
    else if constexpr (N == 2) asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
    else asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}

// Which token of a group an MMA's row or k stands for: an order in which eight lanes' reads of K (rows 0..3 at a time) and of V
// (rows 0, 2, 4, 6) both hit all banks with the TMA's swizzle.
__device__ __forceinline__ uint32_t token_of(uint32_t i) { return ((i ^ (i >> 2)) & 1u) << 2 | (i & 1u) << 1 | ((i >> 1) & 1u) | (i & 8u); }

__device__ __forceinline__ uint64_t divided(uint64_t a, uint64_t b) {  // a / b, mostly of small numbers
    return (a | b) >> 32 ? a / b : (uint64_t)((uint32_t)a / (uint32_t)b);
}

// How the line is shared out: of every head and row tile its start, which counts as much as kStart units, and behind it its units (kPer groups
// each).  quota 0: `per` places to a CTA, one more to the first `more` of them, whatever head they are of.  Otherwise a CTA has units of one head only, and a head as many CTAs as it takes for none to have more than `quota`.
struct Share {
    uint64_t per;
    uint32_t more, quota;
    bool whole;  // quota 0: heads are not divided
    __device__ uint64_t start(uint32_t cta) const { return per * cta + min(cta, more); }
    __device__ uint32_t cta_of(uint64_t u) const {
        const uint64_t first = (per + 1) * more;  // places of the CTAs that have one more
        return u < first ? (uint32_t)divided(u, per + 1) : more + (uint32_t)divided(u - first, per);
    }
};

struct Line {  // a sequence's part of the line
    Sequence s;
    uint32_t units;  // to a head and row tile
    uint32_t tiles, items;  // row tiles, and heads times row tiles
    __device__ uint64_t all(uint32_t start) const { return (uint64_t)(units + start) * items; }
};
__device__ __forceinline__ Line line_of(const CacheView &c, const BatchView &b, uint32_t group, uint32_t rows_of_tile, uint32_t tokens_of_unit, uint32_t s) {
    Line l{{0, 0, 0}, 0, 0, 0};
    if (s >= b.sequences) return l;
    l.s = sequence_of(c, b, s);
    l.units = max(1u, (l.s.length + tokens_of_unit - 1) / tokens_of_unit);
    l.tiles = (uint32_t)(((uint64_t)l.s.rows * group + rows_of_tile - 1) / rows_of_tile);
    l.items = l.tiles * c.heads;
    return l;
}

// TREE: rows are nodes of trees, which see their sequence's tokens ahead of the nodes and those nodes that their masks have
template <int D, bool NF4, int NT, bool TREE>
__global__ void __launch_bounds__(Shape<D, NF4, NT>::kThreads, 1)
attention_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const CacheView c, const BatchView b,
                        const AttentionView a, uint32_t *const counters, float *const parts, const FailureRef failure) {
    using S = Shape<D, NF4, NT>;
    constexpr uint32_t W = S::kWarps, kBlocks = S::kBlocks, kStages = S::kStages, G = S::kPer, kUnit = G * kGroup, kStart = S::kStart;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bars[W * kStages];
    __shared__ float2 s_ml[W][S::kRows];
    __shared__ float2 s_fin[S::kRows];
    __shared__ uint32_t s_last;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
    const uint32_t base = ptx::smem_addr(smem);
    const uint32_t table = NF4 ? (base + S::kFirst + 65535u) & ~65535u : 0;
    const uint32_t ring0 = (NF4 ? table + 65536u : (base + S::kFirst + 1023u) & ~1023u) + warp * (kStages * G * 2 * S::kTile);
    const uint32_t scales0 = base + S::kMerge + warp * (kStages * G * 2 * S::kScaleTile);
    float2 *const merge = reinterpret_cast<float2 *>(smem);
    const uint32_t bars = ptx::smem_addr(s_bars) + 8 * kStages * warp;
    if (NF4 && table + 65536u + S::kRing > base + S::kSmem) {
        ptx::pdl_wait();
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
            const uint32_t byte = i >> 3, entry = level_pair_f16(byte);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(table + byte * 256u + (i & 7u) * 16u), "r"(entry) : "memory");
        }
    }
    __syncthreads();
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    // ---- this CTA's share of the line ----
    const Line line0 = line_of(c, b, a.group, S::kRows, kUnit, lane);  // of the first 32 sequences
    Share share;
    {
        uint64_t units = line0.all(0);
        uint32_t items = line0.items, longest = line0.items ? line0.units : 0u;
        for (uint32_t s = lane + 32; s < b.sequences; s += 32) {
            const Line l = line_of(c, b, a.group, S::kRows, kUnit, s);
            units += l.all(0);
            items += l.items;
            longest = max(longest, l.items ? l.units : 0u);
        }
        #pragma unroll
        for (int k = 1; k < 32; k <<= 1) units += __shfl_xor_sync(0xffffffffu, units, k);
        items = __reduce_add_sync(0xffffffffu, items);
        longest = __reduce_max_sync(0xffffffffu, longest);
        if (units == 0) return;  // nothing to do
        const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, units);
        if (blockIdx.x >= ctas) return;
        const uint64_t each = divided(units, ctas);
        // heads whose tokens are two units to a warp are not worth dividing: the join costs about as much.  It goes by the longest, which its CTA may
        // come to last (200 sequences of one token beside one of 5000, four heads of 128, NF4: 33 us; undivided, as they were by their mean, 46).
        share.whole = longest <= 2 * W;
        // A CTA with two heads' units starts and ends twice, which takes about as long as two units of every warp.  So where the heads can
        // be given CTAs of their own with a quota that is not longer by more, they are.  Quotas of all units over fewer CTAs: with as many
        // fewer as there are heads every head's last CTA may have next to nothing, so that one always serves.
        share.quota = 0;
        if (!share.whole && items < ctas && b.sequences <= 32 && units < 1ull << 31) {
            uint32_t quota[4], need[4];
            #pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                quota[k] = ((uint32_t)units - 1) / (ctas - items * (k + 1) / 4) + 1;
                need[k] = line0.items * ((line0.units + quota[k] - 1) / quota[k]);
            }
            #pragma unroll
            for (uint32_t k = 0; k < 4; ++k) need[k] = __reduce_add_sync(0xffffffffu, need[k]);
            #pragma unroll
            for (uint32_t k = 4; k-- > 0;)
                if (need[k] <= ctas && quota[k] <= each + 2 * W) share.quota = quota[k];
        }
        if (!share.quota) {
            const uint64_t places = units + (uint64_t)items * kStart;
            share.per = divided(places, ctas);
            share.more = (uint32_t)(places - share.per * ctas);
        }
    }

    // the sequence that this CTA begins in, and how far into it: first, in the line (places, or with a quota CTAs)
    uint64_t first = share.quota ? blockIdx.x : share.start(blockIdx.x), end = share.quota ? 0 : share.start(blockIdx.x + 1);
    uint32_t seq = b.sequences;
    Line line = line0;
    uint64_t at = 0;
    {
        uint64_t before = 0;
        for (uint32_t s0 = 0; s0 < b.sequences; s0 += 32) {
            const Line l = s0 ? line_of(c, b, a.group, S::kRows, kUnit, s0 + lane) : line0;
            const uint64_t own = share.quota ? (uint64_t)l.items * ((l.units + share.quota - 1) / share.quota) : l.all(kStart);
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
                line.units = __shfl_sync(0xffffffffu, l.units, l0);
                line.tiles = __shfl_sync(0xffffffffu, l.tiles, l0);
                line.items = __shfl_sync(0xffffffffu, l.items, l0);
                line.s.row0 = __shfl_sync(0xffffffffu, l.s.row0, l0);
                line.s.rows = __shfl_sync(0xffffffffu, l.s.rows, l0);
                line.s.length = __shfl_sync(0xffffffffu, l.s.length, l0);
                at = first - (before + __shfl_sync(0xffffffffu, upto - own, l0));
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (seq >= b.sequences) return;  // (with a quota the last CTAs may have nothing)
    uint64_t now;
    uint32_t item, off, c0, c1;  // off: the first of a head's units that is this CTA's; c0, c1: the CTAs that they are shared by
    uint32_t lead;               // places of the head's start that are this CTA's too
    if (share.quota) {
        const uint32_t ways = (line.units + share.quota - 1) / share.quota, way = (uint32_t)at % ways;
        item = (uint32_t)at / ways;
        // `ways` shares that differ by one at most; the line is this share
        const uint32_t each = line.units / ways, rest = line.units - each * ways;
        off = way * each + min(way, rest);
        lead = 0;
        now = off;
        end = off + each + (way < rest ? 1 : 0);
        c0 = blockIdx.x - way;
        c1 = c0 + ways - 1;
    } else {
        now = first;
        item = (uint32_t)divided(at, line.units + kStart);
        const uint32_t in = (uint32_t)(at - (uint64_t)item * (line.units + kStart));  // how far into the head
        off = in > kStart ? in - kStart : 0u;
        lead = in > kStart ? 0u : kStart - in;
        if (share.whole && in) {  // a head belongs to the CTA in whose share it begins
            now += line.units + kStart - in;
            lead = kStart;
            off = 0;
            ++item;
        }
    }

    // ---- what a lane has of every group ----
    const uint32_t lane_word = table | lane * 4u;
    auto pair_at = [&](uint32_t word, int byte) -> uint32_t {  // the levels of a byte's two codes: {table's upper half, byte, lane * 4}
        uint32_t v;
        asm("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(__byte_perm(word, lane_word, 0x7604u | ((uint32_t)byte << 4))));  // (free to move: the table stands)
        return v;
    };
    constexpr uint32_t kRB = S::kRowBytes;
    // the 16-byte chunk of a row that TMA puts at chunk i of it is i ^ twist(row)
    auto twist = [](uint32_t row) -> uint32_t { return !NF4 || D == 256 ? row & 7u : D == 128 ? (row >> 1) & 3u : (row >> 2) & 1u; };
    const uint32_t krow = token_of(g);
    uint32_t k_at[kBlocks], v_at[kBlocks][2];  // where in a group's tile the lane reads codes of K and of V
    #pragma unroll
    for (uint32_t kb = 0; kb < kBlocks; ++kb) {
        k_at[kb] = krow * kRB + ((2 * kb + (t4 >> 1)) ^ twist(krow)) * 16 + (t4 & 1u) * 8;
        #pragma unroll
        for (uint32_t i = 0; i < 2; ++i) v_at[kb][i] = token_of(2 * t4 + i) * kRB + ((2 * kb + (g >> 2)) ^ twist(token_of(2 * t4 + i))) * 16 + (g & 3u) * 4;
    }

    uint32_t slot = 0, phase = 0;  // the next stage of this warp's ring, and its barrier's parity
    bool ok = true;
    const bool split = G == 2 && c.page_size % kUnit != 0;  // a unit's two groups may be in two pages, and come apart

    while (now < end) {
        while (item >= line.items) {  // on to the next sequence with rows
            ++seq;
            if (seq >= b.sequences) break;
            line = line_of(c, b, a.group, S::kRows, kUnit, seq);
            item = 0;
        }
        if (seq >= b.sequences) break;
        const Sequence s = line.s;
        const uint32_t head = line.tiles == 1 ? item : item / line.tiles, tile = item - head * line.tiles;
        now += lead;
        if (!share.whole && now >= end) break;  // the share ends ahead of the head's units
        const uint32_t n = share.whole ? line.units : (uint32_t)min((uint64_t)(line.units - off), end - now);
        const uint64_t item_first = now - off;
        const uint32_t r0 = tile * S::kRows, rows = min((uint64_t)S::kRows, (uint64_t)s.rows * a.group - r0);
        // the first token that is not this share's, or that none of the tile's rows sees
        const uint32_t limit = min(seen_end<TREE>(s, a.by_group, r0 + rows - 1), (off + n) * kUnit);
        const uint32_t here = limit > off * kUnit ? (limit - off * kUnit + kUnit - 1) / kUnit : 0u;  // units with tokens
        const uint32_t mine = warp < here ? (here - warp + W - 1) / W : 0u;

        // ---- the rows' queries are asked for ----
        uint32_t q[NT][D / 16][2];
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t r = r0 + 8 * nt + g;
            const bool real = 8 * nt + g < rows;
            const uint32_t token = real ? a.by_group.of(r) : 0u;
            const __nv_bfloat16 *const p = static_cast<const __nv_bfloat16 *>(a.q) + (uint64_t)(s.row0 + token) * a.ldq + (uint64_t)(head * a.group + (real ? r - token * a.group : 0u)) * D;
            if (NF4) {
                #pragma unroll
                for (uint32_t k = 0; k < kBlocks; ++k) {
                    const uint4 *const from = reinterpret_cast<const uint4 *>(p + 64 * k + 16 * t4);
                    const uint4 zero = make_uint4(0u, 0u, 0u, 0u), lo = real ? __ldg(from) : zero, hi = real ? __ldg(from + 1) : zero;
                    q[nt][4 * k][0] = lo.x; q[nt][4 * k][1] = lo.y; q[nt][4 * k + 1][0] = lo.z; q[nt][4 * k + 1][1] = lo.w;
                    q[nt][4 * k + 2][0] = hi.x; q[nt][4 * k + 2][1] = hi.y; q[nt][4 * k + 3][0] = hi.z; q[nt][4 * k + 3][1] = hi.w;
                }
            } else {
                const uint32_t *const from = reinterpret_cast<const uint32_t *>(p);
                #pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    q[nt][i][0] = real ? __ldg(from + 8 * i + t4) : 0u;
                    q[nt][i][1] = real ? __ldg(from + 8 * i + 4 + t4) : 0u;
                }
            }
        }

        // ---- the first units ----
        // the places of this warp's next boxes (a unit, or its two groups), one to a lane, in rows of the pool
        const uint32_t boxes = split ? 2 : 1, ahead = 32 / boxes;  // ahead: units
        uint32_t place = 0;
        bool lost = false;  // a page that there is not
        auto look_up = [&](uint32_t k) {
            const uint32_t token = (off + warp + (k + (split ? lane >> 1 : lane)) * W) * kUnit + (split ? (lane & 1u) * kGroup : 0u);
            place = 0;
            if (token < limit) {
                const uint32_t at_page = c.by_page.of(token);
                const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at_page);
                if (page < 0 || (uint32_t)page >= c.pages) lost = true;
                else place = ((uint32_t)page * c.heads + head) * c.page_size + (token - at_page * c.page_size);
            }
        };
        auto ask = [&](uint32_t k, uint32_t to_slot) {  // for this warp's unit number k
            const uint32_t row0 = __shfl_sync(0xffffffffu, place, (boxes * k) & 31u), row1 = split ? __shfl_sync(0xffffffffu, place, (boxes * k + 1) & 31u) : 0u;
            if (lane == 0) {
                const uint32_t bar = bars + 8 * to_slot, to = ring0 + to_slot * (2 * G * S::kTile);
                if (NF4) {
                    const uint32_t st = scales0 + to_slot * (2 * G * S::kScaleTile), part = split ? 1u : G;
                    const bool two = split && (off + warp + k * W) * kUnit + kGroup < limit;
                    ptx::mbar_arrive_expect_tx(bar, (two ? 2u : part) * (2 * S::kTile + 2 * S::kScaleTile));
                    ptx::tma_load_2d(to, &tmap_k, 0, (int32_t)row0, bar);
                    ptx::bulk_g2s(st, c.k_scales + (uint64_t)row0 * kBlocks, part * S::kScaleTile, bar);
                    ptx::tma_load_2d(to + G * S::kTile, &tmap_v, 0, (int32_t)row0, bar);
                    ptx::bulk_g2s(st + G * S::kScaleTile, c.v_scales + (uint64_t)row0 * kBlocks, part * S::kScaleTile, bar);
                    if (two) {
                        ptx::tma_load_2d(to + S::kTile, &tmap_k, 0, (int32_t)row1, bar);
                        ptx::bulk_g2s(st + S::kScaleTile, c.k_scales + (uint64_t)row1 * kBlocks, S::kScaleTile, bar);
                        ptx::tma_load_2d(to + (G + 1) * S::kTile, &tmap_v, 0, (int32_t)row1, bar);
                        ptx::bulk_g2s(st + (G + 1) * S::kScaleTile, c.v_scales + (uint64_t)row1 * kBlocks, S::kScaleTile, bar);
                    }
                } else {
                    ptx::mbar_arrive_expect_tx(bar, 2 * S::kTile);
                    #pragma unroll
                    for (uint32_t x = 0; x < D / 64; ++x) ptx::tma_load_2d(to + x * 2048, &tmap_k, (int32_t)(64 * x), (int32_t)row0, bar);
                    #pragma unroll
                    for (uint32_t x = 0; x < D / 64; ++x) ptx::tma_load_2d(to + S::kTile + x * 2048, &tmap_v, (int32_t)(64 * x), (int32_t)row0, bar);
                }
            }
        };
        if (mine) look_up(0);
        #pragma unroll
        for (uint32_t k = 0; k < kStages; ++k)
            if (ok && k < mine) ask(k, slot + k < kStages ? slot + k : slot + k - kStages);

        // ---- the queries as the first product's B operand ----
        float factor[NT][2];       // of columns 2 t4 and 2 t4 + 1: scale, log2(e), and the power of two the row was divided by
        uint32_t sees[NT][2];      // the first token that the columns' rows do not see; TREE: the rows' numbers, kBlind where they see nothing
        constexpr uint32_t kBlind = 0xffffffffu;
        const uint32_t sees_first = min(TREE ? (uint32_t)max(first_node(s), 0) : visible_end(s, a.by_group, r0), limit);
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float f = a.scale_log2;
            if (NF4) {
                uint32_t most = 0;  // the largest magnitude's bits
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const uint32_t w = q[nt][i / 2][i & 1];
                    most = max(most, max((w << 16) & 0x7fffffffu, w & 0x7fff0000u));
                }
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // the row is divided by a power of two that leaves its largest magnitude in [2^11, 2^12), exact for all that counts
                const int e = most ? min(max((int)(most >> 23) - 127 - 11, -100), 115) : 0;
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                f *= __uint_as_float((uint32_t)(127 + e) << 23) * (1.f / kLevelUnit);
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const uint32_t w = q[nt][i / 2][i & 1];
                    q[nt][i / 2][i & 1] = f16_pair(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
                }
            }
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                factor[nt][j] = __shfl_sync(0xffffffffu, f, 4 * (2 * t4 + j));
                const uint32_t col = 8 * nt + 2 * t4 + j;
                if (TREE) {
                    const uint32_t token = a.by_group.of(r0 + min(col, rows - 1));
                    sees[nt][j] = col < rows && first_node(s) + (int32_t)token >= 0 ? s.row0 + token : kBlind;
                } else {
                    sees[nt][j] = col < rows ? min(visible_end(s, a.by_group, r0 + col), limit) : limit;
                }
            }
        }

        float o[D / 16][NT][4] = {};
        float m[NT][2], l[NT][2] = {};
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = kNothing;
        float ref = 0.f, unref = 0.f;  // the power of two that V's scales are divided by, and its reciprocal
        auto go_on = [&](uint32_t k) {  // the stage of unit k is read: another unit may come to it
            __syncwarp();
            if (k + kStages < mine) {
                if (((k + kStages) & (ahead - 1)) == 0) look_up(k + kStages);
                if (ok) ask(k + kStages, slot);
            }
        };
        #pragma unroll 1
        for (uint32_t k = 0; k < mine; ++k) {
            const uint32_t kt = ring0 + slot * (G * 2 * S::kTile), t0 = (off + warp + k * W) * kUnit;
            if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bars + 8 * slot, phase))) {
                ok = false;
                if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 21);
            }
            // ---- what the lane has of the groups ----
            uint2 kw[G][kBlocks][2];
            uint32_t vw[G][kBlocks][4];
            float ks[G][2][kBlocks], vs[G][2][kBlocks];
            if (NF4) {
                #pragma unroll
                for (uint32_t u = 0; u < G; ++u) {
                    const uint32_t ksc = scales0 + slot * (2 * G * S::kScaleTile) + u * S::kScaleTile + krow * (4 * kBlocks), from0 = kt + u * S::kTile,
                                   vt = from0 + G * S::kTile;
                    #pragma unroll
                    for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                        const uint32_t from = from0 + k_at[kb];
                        kw[u][kb][0] = ptx::ld_shared_v2(from);
                        kw[u][kb][1] = ptx::ld_shared_v2(from + 8 * kRB);
                        vw[u][kb][0] = ld_shared_u32(vt + v_at[kb][0]);
                        vw[u][kb][1] = ld_shared_u32(vt + v_at[kb][1]);
                        vw[u][kb][2] = ld_shared_u32(vt + v_at[kb][0] + 8 * kRB);
                        vw[u][kb][3] = ld_shared_u32(vt + v_at[kb][1] + 8 * kRB);
                    }
                    #pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        ld_scales<kBlocks>(ksc + h * 32 * kBlocks, ks[u][h]);
                        ld_scales<kBlocks>(ksc + G * S::kScaleTile + h * 32 * kBlocks, vs[u][h]);
                    }
                }
            }
            if (NF4) go_on(k);  // (all that the stage had is in registers)
            // ---- scores ----
            float x[G][NT][4];
            #pragma unroll
            for (uint32_t u = 0; u < G; ++u) {
                if (NF4) {
                    #pragma unroll
                    for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                        float acc[NT][4];
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t wl = i < 2 ? kw[u][kb][0].x : kw[u][kb][0].y, wh = i < 2 ? kw[u][kb][1].x : kw[u][kb][1].y;
                            const int by = 2 * (i & 1);
                            const uint32_t a0 = pair_at(wl, by), a1 = pair_at(wh, by), a2 = pair_at(wl, by + 1), a3 = pair_at(wh, by + 1);
                            #pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (i == 0) ptx::mma_16816_f16_zero(acc[nt], a0, a1, a2, a3, q[nt][4 * kb][0], q[nt][4 * kb][1]);
                                else ptx::mma_16816_f16(acc[nt], a0, a1, a2, a3, q[nt][4 * kb + i][0], q[nt][4 * kb + i][1]);
                            }
                        }
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) x[u][nt][e] = kb ? fmaf(ks[u][e >> 1][kb], acc[nt][e], x[u][nt][e]) : ks[u][e >> 1][kb] * acc[nt][e];
                    }
                } else {
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) x[u][nt][0] = x[u][nt][1] = x[u][nt][2] = x[u][nt][3] = 0.f;
                    const uint32_t row = (lane & 7u) + ((lane >> 3) & 1u) * 8, half = lane >> 4;
                    #pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        uint32_t af[4];
                        ptx::ldmatrix_x4(af, kt + (i >> 2) * 2048 + row * 128 + (((2 * (i & 3) + half) ^ (row & 7u)) << 4));
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt) ptx::mma_16816_bf16(x[u][nt], af[0], af[1], af[2], af[3], q[nt][i][0], q[nt][i][1]);
                    }
                }
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][nt][e] *= factor[nt][e & 1];
            }
            if (t0 + G * kGroup > sees_first) {  // some row does not see all of it
                uint32_t window[NT][2], some = 0;  // TREE: bit i: the column's row sees token t0 + i; some row of the tile does
                if (TREE) {
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        #pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            window[nt][j] = sees[nt][j] == kBlind ? 0u : seen_nodes(a, sees[nt][j], (int32_t)t0 - first_node(s)) & low_bits(limit - t0);
                            some |= window[nt][j];
                        }
                    if (NF4) {
                        some |= __shfl_xor_sync(0xffffffffu, some, 1);
                        some |= __shfl_xor_sync(0xffffffffu, some, 2);
                    }
                }
                #pragma unroll
                for (uint32_t u = 0; u < G; ++u) {
                    const uint32_t tok = t0 + u * kGroup + (NF4 ? krow : g);
                    #pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            #pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const bool seen = TREE ? window[nt][j] >> (tok + 8 * h - t0) & 1u : tok + 8 * h < sees[nt][j];
                                x[u][nt][2 * h + j] = seen ? x[u][nt][2 * h + j] : -INFINITY;
                            }
                        #pragma unroll
                        for (uint32_t kb = 0; NF4 && kb < kBlocks; ++kb)  // (anything may stand behind; a node that the tile's rows do not see has no say in `ref`)
                            vs[u][h][kb] = (TREE ? some >> (tok + 8 * h - t0) & 1u : tok + 8 * h < limit) ? vs[u][h][kb] : 0.f;
                    }
                }
            }
            // ---- weights ----
            bool above = false;
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(x[0][nt][j], x[0][nt][j + 2]);
                    #pragma unroll
                    for (uint32_t u = 1; u < G; ++u) top = fmaxf(top, fmaxf(x[u][nt][j], x[u][nt][j + 2]));
                    above = above || top > m[nt][j] + 8.f;
                }
            if (__any_sync(0xffffffffu, above)) {
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = m[nt][j];
                        #pragma unroll
                        for (uint32_t u = 0; u < G; ++u) top = fmaxf(top, fmaxf(x[u][nt][j], x[u][nt][j + 2]));
                        #pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const float keep = exp2_approx(m[nt][j] - top);
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
                    const float from = kRaise<NF4> - m[nt][j];
                    #pragma unroll
                    for (uint32_t u = 0; u < G; ++u) {
                        x[u][nt][j] = exp2_approx(x[u][nt][j] + from);
                        x[u][nt][j + 2] = exp2_approx(x[u][nt][j + 2] + from);
                        l[nt][j] += x[u][nt][j] + x[u][nt][j + 2];
                    }
                }
            // ---- weights times values ----
            if (NF4) {
                uint32_t most = 0;
                #pragma unroll
                for (uint32_t u = 0; u < G; ++u)
                    #pragma unroll
                    for (uint32_t kb = 0; kb < kBlocks; ++kb) most = max(most, max(__float_as_uint(vs[u][0][kb]), __float_as_uint(vs[u][1][kb])));
                if (__any_sync(0xffffffffu, most > __float_as_uint(ref))) {
                    most = __reduce_max_sync(0xffffffffu, most);
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
                for (uint32_t u = 0; u < G; ++u)
                    #pragma unroll
                    for (uint32_t kb = 0; kb < kBlocks; ++kb) {
                        const float f_lo = vs[u][0][kb] * unref, f_hi = vs[u][1][kb] * unref;
                        uint32_t w[NT][2];
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            w[nt][0] = movmatrix(f16_pair(x[u][nt][0] * f_lo, x[u][nt][1] * f_lo));
                            w[nt][1] = movmatrix(f16_pair(x[u][nt][2] * f_hi, x[u][nt][3] * f_hi));
                        }
                        const uint32_t u0 = vw[u][kb][0], u1 = vw[u][kb][1], u2 = vw[u][kb][2], u3 = vw[u][kb][3];
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
                const uint32_t vt = kt + S::kTile;
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
                    w[nt][0] = movmatrix(bf16_pair(x[0][nt][0], x[0][nt][1]));
                    w[nt][1] = movmatrix(bf16_pair(x[0][nt][2], x[0][nt][3]));
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
            if (!NF4) go_on(k);
            if (++slot == kStages) {
                slot = 0;
                phase ^= 1u;
            }
        }

        // ---- the warps' results become one ----
        if (!share.quota) {
            c0 = share.whole ? blockIdx.x : share.cta_of(item_first);
            c1 = share.whole ? blockIdx.x : share.cta_of(item_first + line.units - 1);
        }
        float *const part = parts + (uint64_t)(2 * blockIdx.x + (off ? 0 : 1)) * S::kPartFloats;
        // A register pair (j, j + 2) of (i, nt) in a lane is of row 8 nt + 2 t4 + j, values value_at and the next (bf16: the eighth from it).
        auto deliver = [&](uint32_t pr, uint32_t ln, float lo, float hi) {  // pr: register pair number
            const uint32_t i = pr / (2 * NT), nt = pr / 2 % NT, j = pr & 1u, row = 8 * nt + 2 * (ln & 3u) + j;
            if (row >= rows) return;
            const float sum = s_fin[row].y, f = sum == 0.f ? 0.f : 1.f / sum;
            const uint32_t r = r0 + row, token = a.by_group.of(r), d = NF4 ? (i >> 2) * 64 + (ln >> 2) * 8 + (i & 3u) * 2 : 16 * i + (ln >> 2);
            __nv_bfloat16 *const to = static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)(s.row0 + token) * a.ldo + (uint64_t)(head * a.group + r - token * a.group) * D + d;
            if (NF4) {
                *reinterpret_cast<uint32_t *>(to) = bf16_pair(lo * f, hi * f);
            } else {
                to[0] = __float2bfloat16_rn(lo * f);
                to[8] = __float2bfloat16_rn(hi * f);
            }
        };
        // Each lane's l is a part of its columns' sums.  `last`: to the call's output, else to the workspace.
        auto meet = [&](float unit, bool last) {
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    #pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
                    if (g == 0) s_ml[warp][8 * nt + 2 * t4 + j] = make_float2(m[nt][j], l[nt][j]);
                }
            __syncthreads();
            if (warp == 0 && lane < S::kRows) {
                float top = kNothing, sum = 0.f;
                #pragma unroll
                for (uint32_t w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][lane].x);
                #pragma unroll
                for (uint32_t w = 0; w < W; ++w) sum += s_ml[w][lane].y * exp2_approx(s_ml[w][lane].x - top);
                s_fin[lane] = make_float2(top, sum);
            }
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = kNothing;
                    #pragma unroll
                    for (uint32_t w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][8 * nt + 2 * t4 + j].x);
                    const float keep = exp2_approx(m[nt][j] - top) * unit;
                    #pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        o[i][nt][j] *= keep;
                        o[i][nt][j + 2] *= keep;
                    }
                }
            constexpr uint32_t kPasses = S::kAcc / S::kPassRegs, kPairs = S::kPassRegs / 2;
            #pragma unroll
            for (uint32_t pass = 0; pass < kPasses; ++pass) {
                #pragma unroll
                for (uint32_t x = 0; x < kPairs; ++x) {
                    const uint32_t pr = pass * kPairs + x, i = pr / (2 * NT), nt = pr / 2 % NT, j = pr & 1u;
                    merge[(warp * kPairs + x) * 32 + lane] = make_float2(o[i][nt][j], o[i][nt][j + 2]);
                }
                __syncthreads();
                if (pass == 0 && !last && tid < S::kRows) __stcg(reinterpret_cast<float2 *>(part + S::kRows * D) + tid, s_fin[tid]);
                for (uint32_t e = tid; e < kPairs * 32; e += S::kThreads) {
                    const uint32_t pr = e >> 5, ln = e & 31u;
                    float lo = 0.f, hi = 0.f;
                    #pragma unroll
                    for (uint32_t w = 0; w < W; ++w) {
                        const float2 v = merge[(w * kPairs + pr) * 32 + ln];
                        lo += v.x;
                        hi += v.y;
                    }
                    if (last) deliver(pass * kPairs + pr, ln, lo, hi);
                    else __stcg(reinterpret_cast<float2 *>(part) + (pass * kPairs * 32 + e), make_float2(lo, hi));
                }
                __syncthreads();
            }
        };
        if (__any_sync(0xffffffffu, lost) || !ok) l[0][0] = l[0][1] = l[NT - 1][0] = l[NT - 1][1] = __uint_as_float(0x7fc00000u);  // NaN, and the results with it
        const bool divided = c0 != c1;
        if (NF4) {
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                l[nt][0] *= kLower;
                l[nt][1] *= kLower;
            }
        }
        meet(NF4 ? ref * (kLower / kLevelUnit) : 1.f, !divided);
        if (divided) {
            if (tid == 0) {  // (behind the barrier that `meet` ends with: its release is for what all threads stored)
                uint32_t done;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(done) : "l"(counters + c0) : "memory");
                s_last = done == c1 - c0;
                if (s_last) counters[c0] = 0;
            }
            __syncthreads();
            if (s_last) {
                // Every warp takes the parts of some CTAs as it took groups, in their order.  They lie in CTA c0's place for a head that
                // begins, in the others' for one that goes on.
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    m[nt][0] = m[nt][1] = kNothing;
                    l[nt][0] = l[nt][1] = 0.f;
                    #pragma unroll
                    for (int i = 0; i < D / 16; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
                }
                #pragma unroll 2
                for (uint32_t cta = c0 + warp; cta <= c1; cta += W) {
                    const float2 *const from = reinterpret_cast<const float2 *>(parts + (uint64_t)(2 * cta + (cta == c0 ? 1 : 0)) * S::kPartFloats);
                    float2 ml[NT][2], v[NT][2][D / 16];
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        #pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            ml[nt][j] = __ldcg(from + S::kRows * D / 2 + 8 * nt + 2 * t4 + j);
                            #pragma unroll
                            for (int i = 0; i < D / 16; ++i) v[nt][j][i] = __ldcg(from + ((i * NT + nt) * 2 + j) * 32 + lane);
                        }
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        #pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float top = fmaxf(m[nt][j], ml[nt][j].x), keep = exp2_approx(m[nt][j] - top), f = exp2_approx(ml[nt][j].x - top);
                            m[nt][j] = top;
                            l[nt][j] = l[nt][j] * keep + (g == 0 ? ml[nt][j].y * f : 0.f);
                            #pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                o[i][nt][j] = o[i][nt][j] * keep + v[nt][j][i].x * f;
                                o[i][nt][j + 2] = o[i][nt][j + 2] * keep + v[nt][j][i].y * f;
                            }
                        }
                }
                meet(1.f, true);
            }
        }
        now += n;
        off = 0;
        lead = kStart;
        ++item;
    }
    if (!ok) ptx::let_flights_land();
}

template <int D, bool NF4, int NT, bool TREE>
int32_t launch(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    using S = Shape<D, NF4, NT>;
    static_assert(kNumSMs * 4 <= kAttentionFlagBytes);
    auto kernel = attention_decode_kernel<D, NF4, NT, TREE>;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kSmem));
    const uint64_t rows = (uint64_t)c.cache.pages * c.cache.heads * c.cache.page_size;
    CUtensorMap map_k, map_v;
    const uint32_t box = c.cache.page_size % (S::kPer * kGroup) == 0 ? S::kPer * kGroup : kGroup;  // a unit, or one of its groups
    auto of = [&](CUtensorMap *map, const void *pool) {
        if (!NF4) return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, pool, rows, D, 2 * D, kGroup, 64, CU_TENSOR_MAP_SWIZZLE_128B);
        return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, pool, rows, D / 2, D / 2, box, D / 2,
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

template <int NT, bool TREE>
int32_t launch_of(const AttentionCall &c, uint8_t *ws, cudaStream_t s) {
    switch (c.head_dim) {
        case 64: return c.nf4 ? launch<64, true, NT, TREE>(c, ws, s) : launch<64, false, NT, TREE>(c, ws, s);
        case 128: return c.nf4 ? launch<128, true, NT, TREE>(c, ws, s) : launch<128, false, NT, TREE>(c, ws, s);
        default: return c.nf4 ? launch<256, true, NT, TREE>(c, ws, s) : launch<256, false, NT, TREE>(c, ws, s);
    }
}

bool one_tile(const AttentionCall &c) { return (uint64_t)c.most_rows * c.view.group <= 8; }

}  // namespace

uint64_t attention_decode_bytes(const AttentionCall &c) {
    const uint64_t rows = one_tile(c) ? 8 : 16;
    return kAttentionFlagBytes + 2ull * kNumSMs * (rows * c.head_dim + 2 * rows) * sizeof(float);
}

int32_t attention_decode(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    if (c.tree) return one_tile(c) ? launch_of<1, true>(c, workspace, stream) : launch_of<2, true>(c, workspace, stream);
    return one_tile(c) ? launch_of<1, false>(c, workspace, stream) : launch_of<2, false>(c, workspace, stream);
}

}  // namespace nf4
