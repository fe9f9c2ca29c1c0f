// Attention of many rows over the paged cache (chunks of prompts, whole prompts) on the tensor cores.
//
// Bound by the MMAs (4 * dim operations for a row and a token) and by the exponentials beside them.  A row tile is 256 rows of one
// head of the cache (a token's query heads are neighbouring rows), or 128 with a dim of 256: one or two MMA tiles of 128.  It goes over the
// tokens that it sees 128 (or 64) a step.  The steps of all sequences, heads and row tiles form one line that the CTAs, one to an SM, share
// out evenly: a CTA has pieces of the line, and a row tile that is in several CTAs leaves its parts in the workspace for the join.
//
// Keys and values are in shared memory in f16 or bf16 with 128-byte swizzle: brought there by TMA from a bf16 cache; looked up by four warps
// from codes that came by bulk copies, times their block's scale, from a quantized one, once for all of a tile's rows.  One elected thread
// issues tcgen05.mma:
//   S = Q K^T   both operands from shared memory, 128 x 128 f32 sums in tensor memory
//   O += P V    P from tensor memory, where the softmax warps have put it over S; V as it lies, MN-major
// A softmax thread owns a row: it reads S, keeps the row's largest exponent m and sum l, and writes P = 2^(S c - m + raise) back as f16
// (bf16 with a bf16 cache).  While one tile's softmax runs, the other's two products do.  (64 tokens a step and two places for S, so that a step's scores are
// there when the last one's weights are done, were tried: a first product of 64 columns takes as long as one of 128, A's rows being read for half
// the work, and 128 tokens of two tiles took 6100 cycles instead of 4270.)  m is the largest exponent so far or up to 8
// below it: O is rescaled only where a row rises above that, by the warps themselves, at a moment when
// no product is writing it.  Copies and lookups run ahead into the next piece while a row tile's results are written.
// f16's range: K's and V's scales are divided by a power of two that brings a step's largest next to the upper end of it, a row of Q by its own
// (exact).  K's comes back as a factor of the step's scores; V's goes into the step's weights, relative to the largest so far (`ref`), which
// comes back at the end.  f16 is off by 2^-12 on average, bf16 would be by 2^-9.  A step's tokens share the power, those that a row does not see
// among them: a value has all of its bits down to 2^-29 of the step's largest scale, and is off by 2^-37 of that below.  (The sums are f32 and
// take any size.)
#include <algorithm>

#include "kv_cache.cuh"
#include "ptx.cuh"
#include "tmap.cuh"

namespace nf4 {

namespace {

constexpr uint32_t kThreads = 512;
// Weights are 2^(S c - m + raise).  In f16 up to 2^15, so that it holds those that are 2^-32 of a row's largest; their sum is raised alike, and where
// sums go to the workspace both are lowered by that again, so that no value overflows them that would not overflow a sum of weights up to
// one.  bf16 has the range: weights up to one.
template <bool NF4>
constexpr float kRaise = NF4 ? 7.f : -8.f;
template <bool NF4>
constexpr float kLower = NF4 ? 1.f / 32768.f : 1.f;
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
    // S's places to a tile: with a dim of 256 there is room for two, so that the next step's scores come while weights are made
    static constexpr uint32_t kPlaces = D == 256 ? 2 : 1;
    static constexpr uint32_t kBlocks = D / 64;
    static constexpr uint32_t kQTile = 128 * D * 2, kTile = kTokens * D * 2, kBox = kTokens * 128;
    static constexpr uint32_t kScales = kTokens * kBlocks * 4;
    // a tile's codes and scales, and with K's the V's scales of the step: their power goes to the softmax ahead of V
    static constexpr uint32_t kRaw = NF4 ? kTokens * D / 2 + 2 * kScales : 0, kRawSlots = D == 64 ? 5 : 2;
    static constexpr uint32_t kSlots = D == 64 ? (NF4 ? 6 : 7) : NF4 ? 3 : 5;  // of the ring; one more where the table is not needed
    // codes, then the table on a multiple of its 32 KB, then Q, then the ring (bf16: Q, then the ring)
    static constexpr uint32_t kSmem = (NF4 ? 65536 : 2048) - 1024 + kTiles * kQTile + kSlots * kTile;
    static constexpr uint32_t kS = 0, kO = 256;                       // columns of tensor memory: the tiles' S's, then O's
};

// A tile's 128 rows of queries, as the MMA reads them, and in their place later the tile's results: a box of 128 rows to every 64 values (128
// bytes), 16-byte chunks swizzled.  Each of the tile's four warps has the 32 rows whose softmax is its own, for both, so that a warp which
// writes its next queries has nothing to wait for from one that still reads its results out.
__host__ __device__ constexpr uint32_t chunk_place(uint32_t row, uint32_t x) { return (x >> 3) * 16384u + row * 128u + (((x & 7u) ^ (row & 7u)) << 4); }
// The n-th chunk (of dim / 8) that a lane of one of the four warps brings of the queries, and that it takes of the results.
struct RowChunk {
    uint32_t row, x;
};
__host__ __device__ constexpr RowChunk chunk_of(uint32_t dim, uint32_t warp, uint32_t lane, uint32_t n) {
    const uint32_t lanes = dim / 8;  // of a row
    return RowChunk{warp * 32 + n * (32 / lanes) + lane / lanes, lane % lanes};
}

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
__device__ __forceinline__ float2 ld_shared_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared_u4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// The power of two that scales up to `most` (bits) are divided by, to be below 2^15: 2^-126 or more.
constexpr int kTop = 15;
__device__ __forceinline__ float power_for(uint32_t most) { return __uint_as_float((uint32_t)max((int)(most >> 23) + 1 - kTop, 1) << 23); }
__device__ __forceinline__ float reciprocal_of_power(float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); }

// How the line of steps is shared out: `per` to a CTA, one more to the first `more` of them.
struct Share {
    uint32_t per, more, ctas;
    __device__ uint32_t start(uint32_t cta) const { return per * cta + min(cta, more); }
    __device__ uint32_t cta_of(uint32_t u) const {
        const uint32_t first = (per + 1) * more;
        return u < first ? u / (per + 1) : more + (u - first) / per;
    }
};

// A run of steps of one row tile.
struct Piece {
    Sequence s;
    uint32_t seq, head, r0, rows, live;  // rows of the tile; MMA tiles that have some
    uint32_t step0, steps, all;          // of the `all` steps that the tile has
    uint32_t line0;                      // where the tile's steps begin in the line
};

// Steps' worth of time that a row tile takes beside its steps (its queries in, its results out): counted in the line, or the CTAs that have
// a prompt's first tiles, of one step each, would be done last.
constexpr uint32_t kStart = 4;

template <uint32_t R, uint32_t N>
struct Walker {  // through a CTA's pieces; every warp goes its own way
    Sequence s;
    uint32_t seq, head, tile, off, now, end;

    static __device__ __forceinline__ uint32_t tiles_of(const Sequence &s, uint32_t group) { return (uint32_t)(((uint64_t)s.rows * group + R - 1) / R); }
    // (a tile that sees nothing has one step all the same: its results are zeros)
    static __device__ __forceinline__ uint32_t steps_of(const Sequence &s, const AttentionView &a, uint32_t tile) {
        const uint32_t last = (uint32_t)min((uint64_t)(tile + 1) * R, (uint64_t)s.rows * a.group) - 1;
        return max(1u, (visible_end(s, a.by_group, last) + N - 1) / N);
    }
    __device__ __forceinline__ bool next(const CacheView &c, const BatchView &b, const AttentionView &a, Piece &p) {
        do {
            if (!one(c, b, a, p)) return false;
        } while (p.steps == 0);  // (the end of a share that lies ahead of a tile's first step)
        return true;
    }
    __device__ __forceinline__ bool one(const CacheView &c, const BatchView &b, const AttentionView &a, Piece &p) {
        if (now >= end) return false;
        while (tile >= tiles_of(s, a.group)) {  // on to the next head, or the next sequence with rows
            tile = 0;
            if (s.rows == 0 || ++head >= c.heads) {
                head = 0;
                if (++seq >= b.sequences) return false;
                s = sequence_of(c, b, seq);
            }
        }
        p.s = s;
        p.seq = seq;
        p.head = head;
        p.r0 = tile * R;
        p.rows = (uint32_t)min((uint64_t)R, (uint64_t)s.rows * a.group - p.r0);
        p.live = (p.rows + 127) / 128;
        p.all = steps_of(s, a, tile);
        p.line0 = now - off;
        // of the tile's place in the line [line0, line0 + kStart + all) the steps are behind kStart
        const uint32_t upto = min(p.all + kStart, end - p.line0);
        p.step0 = off > kStart ? off - kStart : 0u;
        p.steps = (upto > kStart ? upto - kStart : 0u) - p.step0;
        now = p.line0 + upto;
        off = 0;
        ++tile;
        return true;
    }
};

// A quantized cache's keys and values expanded to f16 once for all row tiles, by a kernel ahead: a step's tokens of a head are a tile of
// kTokens rows, zeros behind the sequence's last token.
struct Dense {
    uint32_t capacity;        // tiles to a head that there is room for; 0: codes are expanded where they are used
    const uint32_t *bases;    // [sequences] a sequence's first tile, and behind them [sequences]: all tiles
    const float2 *powers;     // [tile][head] what K's and V's scales are divided by
};

// What the join has to know of a row tile that several CTAs have: written by the CTA in whose share it begins, rows 0 by the others.
struct Split {
    uint32_t row0, r0, rows, head, more;  // more: CTAs behind the first
};

// A place in the ring of tiles, and the parity of its barriers' round.
struct Ring {
    uint32_t slot = 0, round = 0;
    __device__ __forceinline__ void on(uint32_t slots) {
        if (++slot == slots) {
            slot = 0;
            ++round;
        }
    }
};

// In which order a piece's tiles of K and V come: K 0, V 0, K 1, V 1, ...; with two places for S K 0, K 1, V 0, K 2, V 1, ..., V n - 1.
template <uint32_t kPlaces>
struct Turn {
    uint32_t values, step;
    __device__ __forceinline__ Turn(uint32_t turn, uint32_t steps) {
        if (kPlaces == 1) {
            values = turn & 1u;
            step = turn / 2;
            return;
        }
        const bool last = turn + 1 == 2 * steps;
        values = last || (turn && !(turn & 1u)) ? 1 : 0;
        step = last ? steps - 1 : values ? turn / 2 - 1 : (turn + 1) / 2;
    }
};

template <int D, bool NF4>
__global__ void __launch_bounds__(kThreads, 1)
attention_chunk_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const CacheView c, const BatchView b,
                       const AttentionView a, const Dense dense, uint32_t box_rows, Split *const splits, const FailureRef failure) {
    using S = Shape<D, NF4>;
    using Walk = Walker<S::kRows, S::kTokens>;
    // A bf16 cache's pages may be of sixteen tokens, and a warp asks for boxes one after another: four warps share the asking, a tile's
    // columns between two of them (with one, 137 cycles to a box of 2 KB, the MMAs waited for copies)
    constexpr uint32_t kCopies = !NF4 && D >= 128 ? 2 : 1;
    constexpr uint32_t N = S::kTokens, kBlocks = S::kBlocks, kPlaces = S::kPlaces;
    extern __shared__ uint8_t smem_any[];
    __shared__ __align__(8) uint64_t s_bars[42];
    __shared__ uint32_t s_tmem, s_bad[8], s_first[6];  // s_bad: of the last eight pieces, its number + 1 where a page was not there
    __shared__ Share s_share;
    __shared__ Walk s_walk[8];
    __shared__ Piece s_piece[8];
    __shared__ float s_qpower[NF4 ? S::kRows : 1];
    __shared__ float2 s_powers[8];  // of the last steps' K and V (who writes them is at most four steps ahead of who reads)
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
    const uint32_t base = ptx::smem_addr(smem_any);
    const uint32_t raw0 = (base + 15u) & ~15u, table = (raw0 + S::kRawSlots * S::kRaw + 32767u) & ~32767u;
    const uint32_t q0 = NF4 ? table + 32768u : (base + 1023u) & ~1023u, ring0 = q0 + S::kTiles * S::kQTile;
    // s_full, p_ready: of a tile's places; pv_done: products that a rescaling waits for
    const uint32_t bars = ptx::smem_addr(s_bars), full0 = bars, empty0 = bars + 64, raw_full0 = bars + 128, raw_empty0 = bars + 168, s_full0 = bars + 208,
                   p_ready0 = bars + 240, pv_done0 = bars + 272, q_ready0 = bars + 288, tail0 = bars + 304, o_done0 = bars + 320;
    if (ring0 + S::kSlots * S::kTile > base + S::kSmem) {
        ptx::pdl_wait();
        if (tid == 0) {
            NF4_REPORT_FAILURE(*failure.flag, *failure.host, 22);
            splits[blockIdx.x].rows = 0;
        }
        return;
    }
    if (tid == 0) {
        static_assert(S::kSlots + 1 <= 8);
        for (uint32_t i = 0; i < 8; ++i) {  // (a place more than kSlots may be in use)
            ptx::mbar_init(full0 + 8 * i, NF4 ? 4 : kCopies);
            ptx::mbar_init(empty0 + 8 * i, 1);
        }
        for (uint32_t i = 0; i < S::kRawSlots; ++i) {
            ptx::mbar_init(raw_full0 + 8 * i, 1);
            ptx::mbar_init(raw_empty0 + 8 * i, 4);
        }
        for (uint32_t i = 0; i < 4; ++i) {
            ptx::mbar_init(s_full0 + 8 * i, 1);
            ptx::mbar_init(p_ready0 + 8 * i, 4);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            ptx::mbar_init(pv_done0 + 8 * i, 1);
            ptx::mbar_init(q_ready0 + 8 * i, 4);
            ptx::mbar_init(o_done0 + 8 * i, 1);
        }
        for (uint32_t i = 0; i < 2; ++i) ptx::mbar_init(tail0 + 8 * i, 1);
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
    }
    if (tid < 8) s_bad[tid] = 0;
    if (NF4) {
        for (uint32_t i = tid; i < 256 * 8; i += kThreads) {  // the table: an entry's copy to a lane
            const uint32_t byte = i >> 3, entry = level_pair_f16(byte);
            st_shared_u4(table + byte * 128u + (i & 7u) * 16u, make_uint4(entry, entry, entry, entry));
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
        // a lane a sequence: its steps, all heads
        auto steps_of = [&](uint32_t s0, Sequence &s) -> uint32_t {
            s = Sequence{0, 0, 0};
            if (s0 + lane < b.sequences) s = sequence_of(c, b, s0 + lane);
            const uint32_t tiles = Walk::tiles_of(s, a.group);
            uint32_t sum = 0;
            if (tiles <= 8)
                for (uint32_t t = 0; t < tiles; ++t) sum += kStart + Walk::steps_of(s, a, t);
            for (uint32_t many = __ballot_sync(0xffffffffu, tiles > 8); many; many &= many - 1) {  // with the whole warp
                const int l = __ffs(many) - 1;
                const Sequence o{__shfl_sync(0xffffffffu, s.row0, l), __shfl_sync(0xffffffffu, s.rows, l), __shfl_sync(0xffffffffu, s.length, l)};
                uint32_t part = 0;
                for (uint32_t t = lane; t < Walk::tiles_of(o, a.group); t += 32) part += kStart + Walk::steps_of(o, a, t);
                part = __reduce_add_sync(0xffffffffu, part);
                if ((int)lane == l) sum = part;
            }
            return sum * c.heads;
        };
        Sequence s0;
        const uint32_t own0 = steps_of(0, s0);
        uint32_t total = own0;
        for (uint32_t k = 32; k < b.sequences; k += 32) {
            Sequence s;
            total += steps_of(k, s);
        }
        total = __reduce_add_sync(0xffffffffu, total);
        Share share;
        share.ctas = min(gridDim.x, (total + kStart + 1) / (kStart + 2));  // two steps at least
        share.per = share.ctas ? total / share.ctas : 0;
        share.more = share.ctas ? total - share.per * share.ctas : 0;
        const uint32_t first = share.start(blockIdx.x);
        uint32_t last = blockIdx.x < share.ctas ? share.start(blockIdx.x + 1) : first, before = 0;
        bool found = false;
        for (uint32_t k = 0; first < last && k < b.sequences; k += 32) {
            Sequence s = s0;
            const uint32_t own = k ? steps_of(k, s) : own0;
            uint32_t upto = own;
            #pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= (uint32_t)d) upto += o;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + upto > first);
            if (past) {
                const int l = __ffs(past) - 1;
                const Sequence o{__shfl_sync(0xffffffffu, s.row0, l), __shfl_sync(0xffffffffu, s.rows, l), __shfl_sync(0xffffffffu, s.length, l)};
                const uint32_t at = first - before - __shfl_sync(0xffffffffu, upto - own, l), of_head = __shfl_sync(0xffffffffu, own, l) / c.heads;
                const uint32_t head = of_head ? at / of_head : c.heads;
                uint32_t left = at - head * of_head, tile = 0;
                for (uint32_t t0 = 0;; t0 += 32) {
                    const uint32_t mine = t0 + lane < Walk::tiles_of(o, a.group) ? kStart + Walk::steps_of(o, a, t0 + lane) : 0u;
                    uint32_t sum = mine;
                    #pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const uint32_t v = __shfl_up_sync(0xffffffffu, sum, d);
                        if (lane >= (uint32_t)d) sum += v;
                    }
                    const uint32_t in = __ballot_sync(0xffffffffu, sum > left);
                    if (in) {
                        const int t = __ffs(in) - 1;
                        tile = t0 + t;
                        left -= __shfl_sync(0xffffffffu, sum - mine, t);
                        found = head < c.heads;
                        break;
                    }
                    if (t0 + 32 >= Walk::tiles_of(o, a.group)) break;  // (not reached where row starts do not decrease: the head has that many steps)
                    left -= __shfl_sync(0xffffffffu, sum, 31);
                }
                if (lane == 0) {
                    s_first[0] = k + l;
                    s_first[1] = head;
                    s_first[2] = tile;
                    s_first[3] = left;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (!found) last = first;  // (row starts that decrease, whose rows are more than the line is counted for: no access by what is not there)
        if (lane == 0) {
            s_first[4] = first;
            s_first[5] = last;
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
    if (s_first[4] < s_first[5]) {
        Walk walk{sequence_of(c, b, s_first[0]), s_first[0], s_first[1], s_first[2], s_first[3], s_first[4], s_first[5]};
        Piece p;
        if (warp < 8) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            const uint32_t tile = warp >> 2, r = tid & 127u;
            const uint32_t lanes = (warp & 3u) << 21;  // a warp reaches its quarter of tensor memory's lanes
            const uint32_t ts0 = tmem + S::kS + kPlaces * tile * N + lanes, to = tmem + S::kO + tile * D + lanes;
            const uint32_t q_tile = q0 + tile * S::kQTile;
            uint32_t scores = 0, finished = 0, step = 0, piece = 0;  // steps and pieces of this tile, steps and pieces of the CTA, so far
            for (; ok && walk.next(c, b, a, p); step += p.steps, ++piece) {
                if (tile >= p.live) continue;
                // (what the steps do not need waits in shared memory: registers are short there)
                if (lane == 0) {
                    s_walk[warp] = walk;
                    s_piece[warp] = p;
                }
                // ---- Q to shared memory ----
                constexpr uint32_t kLanes = D / 8, kBatch = kLanes < 16 ? kLanes : 16;  // lanes to a row, eight values each; loads in flight
                const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a scale below zero: the rows change sign, so that c is not)
                #pragma unroll 1
                for (uint32_t i0 = 0; i0 < kLanes; i0 += kBatch) {
                    uint4 w[kBatch];
                    #pragma unroll
                    for (uint32_t k = 0; k < kBatch; ++k) {
                        const RowChunk own = chunk_of(D, warp & 3u, lane, i0 + k);
                        const uint32_t row = p.r0 + tile * 128 + own.row, token = a.by_group.of(row);
                        w[k] = make_uint4(0u, 0u, 0u, 0u);
                        if (tile * 128 + own.row < p.rows)
                            w[k] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(a.q) + (uint64_t)(p.s.row0 + token) * a.ldq +
                                                                         (uint64_t)(p.head * a.group + row - token * a.group) * D) + own.x);
                    }
                    #pragma unroll
                    for (uint32_t k = 0; k < kBatch; ++k) {
                        const RowChunk own = chunk_of(D, warp & 3u, lane, i0 + k);
                        uint32_t u[4] = {w[k].x ^ flip, w[k].y ^ flip, w[k].z ^ flip, w[k].w ^ flip};
                        if (NF4) {
                            constexpr uint32_t kSize = 0x7fff7fffu;  // (bf16 magnitudes go by their bits)
                            uint32_t two = __vmaxu2(__vmaxu2(u[0] & kSize, u[1] & kSize), __vmaxu2(u[2] & kSize, u[3] & kSize));
                            #pragma unroll
                            for (uint32_t d = 1; d < kLanes; d <<= 1) two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, d));
                            const uint32_t most = max(two << 16, two & 0xffff0000u);
                            // the row's largest magnitude is left in [2^11, 2^12)
                            const int e2 = most ? min(max((int)(most >> 23) - 127 - 11, -100), 115) : 0;
                            const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) u[e] = pack<true>(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
                            if (own.x == 0) s_qpower[tile * 128 + own.row] = __uint_as_float((uint32_t)(127 + e2) << 23);
                        }
                        st_shared_u4(q_tile + chunk_place(own.row, own.x), make_uint4(u[0], u[1], u[2], u[3]));
                    }
                }
                ptx::fence_proxy_async();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(q_ready0 + 8 * tile);

                // ---- the steps ----
                const uint32_t row = p.r0 + tile * 128 + r, t_first = p.step0 * N;
                const bool real = tile * 128 + r < p.rows;
                const uint32_t sees = real ? visible_end(p.s, a.by_group, row) : 0u, sees_first = visible_end(p.s, a.by_group, p.r0 + tile * 128);
                const uint32_t steps = p.steps;
                const float row_factor = fabsf(a.scale_log2) * (NF4 ? s_qpower[tile * 128 + r] : 1.f);
                float m = -INFINITY, l = 0.f, ref = 0.f;
                for (uint32_t j = 0; j < steps; ++j, ++scores) {
                    const uint32_t place = kPlaces * tile + scores % kPlaces, ts = ts0 + scores % kPlaces * N;
                    if (!__all_sync(0xffffffffu, ptx::mbar_wait_suspended(s_full0 + 8 * place, (scores / kPlaces) & 1u))) {
                        ok = false;
                        if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 23);
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t t0 = t_first + j * N, lim = sees > t0 ? sees - t0 : 0u;
                    const bool masked = t0 + N > sees_first;
                    // (written before the keys' arrival was made known, which the scores are behind)
                    const float2 powers = NF4 ? ld_shared_f2(ptx::smem_addr(s_powers + ((step + j) & 7u))) : make_float2(1.f, 1.f);
                    const float factor = fmaxf(row_factor * powers.x, 1.2e-38f);
                    const float ref_was = ref;
                    if (NF4) ref = fmaxf(ref, powers.y);
                    // the step's values are in units of powers.y, the sums in units of ref: 2^-less of that (a difference that is no more
                    // than 2^-60 of the largest is made that)
                    const int less = NF4 ? min((int)(__float_as_uint(ref) >> 23) - (int)(__float_as_uint(powers.y) >> 23), 60) : 0;
                    bool grown = NF4 && ref != ref_was && j;
                    // Weights by m as it is, and only then the look at the largest score: where it is out of reach, once or twice a
                    // row, they are made again.  So nothing waits for a maximum, and S need not be held whole.
                    uint32_t pw[N / 2];
                    float2 sum;
                    for (;;) {
                        const float from = m == -INFINITY ? 0.f : kRaise<NF4> - m - (float)less;
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
                                pw[(k + i) / 2] = pack<NF4>(w.x, w.y);
                            }
                        }
                        const float high = fmaxf(top[0], top[1]) * factor;
                        const bool above = __any_sync(0xffffffffu, high > m + 8.f);
                        if (!above && !grown) break;
                        float keep = 1.f;
                        if (above) {
                            const float now = fmaxf(m, high);
                            keep = m == -INFINITY ? 0.f : exp2_approx(m - now);
                            m = now;
                            l *= keep;
                        }
                        if (grown) keep *= ref_was * reciprocal_of_power(ref);
                        grown = false;
                        if (j) {  // once the products so far are done: the last step's were, with one place, ahead of these scores
                            if (kPlaces > 1 && !__all_sync(0xffffffffu, ptx::mbar_wait_suspended(pv_done0 + 8 * tile, (scores - 1) & 1u))) {
                                ok = false;
                                if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 28);
                                break;
                            }
                            ptx::tc_fence_after();
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
                        if (!above) break;
                    }
                    if (!ok) break;
                    l += (sum.x + sum.y) * (NF4 ? __uint_as_float((uint32_t)(127 + less) << 23) : 1.f);
                    #pragma unroll
                    for (uint32_t k = 0; k < N / 2; k += 32) tmem_st32(ts + k, pw + k);
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(p_ready0 + 8 * place);
                }
                if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_suspended(o_done0 + 8 * tile, finished & 1u))) {
                    ok = false;
                    if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 24);
                }
                ++finished;
                ptx::tc_fence_after();
                walk = s_walk[warp];
                p = s_piece[warp];

                // ---- the row's results, through the place of this warp's rows of Q (the products are done) so that whole rows go out ----
                if (s_bad[piece & 7u] == piece + 1 || !ok) l = __uint_as_float(0x7fc00000u);  // NaN
                const bool whole = p.steps == p.all;
                const uint64_t part = (uint64_t)(2 * blockIdx.x + (p.step0 ? 0 : 1)) * S::kRows + tile * 128;
                if (!whole) a.part_ml[part + r] = make_float2(m, l * kLower<NF4>);
                const float f = (whole ? l == 0.f ? 0.f : 1.f / l : kLower<NF4>) * (NF4 ? ref : 1.f);
                constexpr uint32_t kChunks = D / 8;  // of a staged row: bf16 results, or half of a row's f32 sums
                #pragma unroll 1
                for (uint32_t half = 0; half < (whole ? 1u : 2u); ++half) {
                    const uint32_t columns = whole ? D : D / 2;
                    __syncwarp();
                    uint32_t v[2][32];
                    tmem_ld32(to + half * columns, v[0]);
                    #pragma unroll
                    for (uint32_t k = 0; k < D; k += 32) {
                        if (k >= columns) break;
                        uint32_t (&x)[32] = v[k / 32 & 1];
                        ptx::tmem_wait_ld();
                        if (k + 32 < columns) tmem_ld32(to + half * columns + k + 32, v[k / 32 + 1 & 1]);
                        #pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                        if (whole) {
                            #pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) {
                                uint32_t w[4];
                                #pragma unroll
                                for (int e = 0; e < 4; ++e) w[e] = bf16_pair(__uint_as_float(x[8 * i + 2 * e]), __uint_as_float(x[8 * i + 2 * e + 1]));
                                st_shared_u4(q_tile + chunk_place(r, k / 8 + i), make_uint4(w[0], w[1], w[2], w[3]));
                            }
                        } else {
                            #pragma unroll
                            for (uint32_t i = 0; i < 8; ++i)
                                st_shared_u4(q_tile + chunk_place(r, k / 4 + i), make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
                        }
                    }
                    __syncwarp();
                    #pragma unroll 8
                    for (uint32_t i = 0; i < kChunks; ++i) {
                        const RowChunk own = chunk_of(D, warp & 3u, lane, i);
                        const uint4 w = ld_shared_u4(q_tile + chunk_place(own.row, own.x));
                        const bool here = tile * 128 + own.row < p.rows;
                        if (whole) {
                            const uint32_t q_row = p.r0 + tile * 128 + own.row, token = a.by_group.of(q_row);
                            if (here)
                                *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)(p.s.row0 + token) * a.ldo +
                                                           (uint64_t)(p.head * a.group + q_row - token * a.group) * D + 8 * own.x) = w;
                        } else if (here) {
                            *reinterpret_cast<uint4 *>(a.part_o + (part + own.row) * D + half * (D / 2) + 4 * own.x) = w;
                        }
                    }
                }
                __syncwarp();  // (the next queries come to the same place)
                if (!whole && p.step0 == 0 && tid == 0) {
                    const uint32_t more = min(s_share.cta_of(p.line0 + kStart + p.all - 1) - blockIdx.x, gridDim.x - 1 - blockIdx.x);
                    splits[blockIdx.x] = Split{p.s.row0, p.r0, p.rows, p.head, more};
                }
                ptx::tc_fence_before();
            }
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
            if (NF4 && !expanded && warp >= kExpandWarp && warp < kExpandWarp + 4) {
                // ---- codes to f16: a thread has 16 bytes of a token's row, 32 values ----
                constexpr uint32_t kLanes = D / 32, kPass = 128 / kLanes;
                const uint32_t th = tid - 32 * kExpandWarp, q = th % kLanes, lane_word = table | lane * 4u;
                // In which order a thread takes its four words: so that eight lanes' 16-byte stores hit all banks
                const uint32_t order = D == 128 ? (q >> 1) * 2 : D == 256 ? q >> 1 : 0u;
                uint32_t i = 0, step = 0;  // tiles and steps so far
                Ring ring;
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_suspended(bar, parity))) {
                        ok = false;
                        if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 25);
                    }
                };
                for (; ok && walk.next(c, b, a, p); step += p.steps) {
                    const uint32_t t_end = min(visible_end(p.s, a.by_group, p.r0 + p.rows - 1), (p.step0 + p.steps) * N);
                    #pragma unroll 1
                    for (uint32_t turn = 0; ok && turn < 2 * p.steps; ++turn, ++i, ring.on(slots)) {
                        const Turn<kPlaces> of(turn, p.steps);
                        const uint32_t which = of.values, j = of.step, t0 = (p.step0 + j) * N;
                        const uint32_t rs = i % S::kRawSlots, slot = ring.slot, raw = raw0 + rs * S::kRaw, dst = place_of(slot) + (q >> 1) * S::kBox;
                        wait(raw_full0 + 8 * rs, (i / S::kRawSlots) & 1u);
                        // the power for the tile's largest scale
                        auto power_of = [&](uint32_t from) {
                            uint32_t most = 0;
                            #pragma unroll
                            for (uint32_t k = 0; k < N * kBlocks / 64; ++k) {
                                const uint32_t at = 2 * (k * 32 + lane);  // (a token's blocks, or tokens, together)
                                const float2 v = ld_shared_f2(from + 4 * at);
                                most = max(most, t0 + at / kBlocks < t_end ? __float_as_uint(v.x) : 0u);
                                most = max(most, t0 + (at + 1) / kBlocks < t_end ? __float_as_uint(v.y) : 0u);
                            }
                            return power_for(__reduce_max_sync(0xffffffffu, most));
                        };
                        const float power = power_of(raw + N * (D / 2));
                        if (!which) {
                            const float v_power = power_of(raw + N * (D / 2) + S::kScales);
                            if (tid == 32 * kExpandWarp) s_powers[(step + j) & 7u] = make_float2(power, v_power);
                        }
                        if (ring.round) wait(empty0 + 8 * slot, (ring.round + 1) & 1u);
                        if (!ok) break;
                        {
                            const float unit = reciprocal_of_power(power) * (1.f / kLevelUnit);
                            uint4 raws[N / kPass];
                            uint32_t factors[N / kPass];
                            #pragma unroll
                            for (uint32_t pass = 0; pass < N / kPass; ++pass) {
                                const uint32_t t = pass * kPass + th / kLanes;
                                raws[pass] = ld_shared_u4(raw + t * (D / 2) + q * 16);
                                float scale;
                                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(scale) : "r"(raw + N * (D / 2) + (t * kBlocks + (q >> 1)) * 4) : "memory");
                                scale = t0 + t < t_end ? scale * unit : 0.f;  // (behind the last token anything may stand)
                                factors[pass] = pack<true>(scale, scale);
                            }
                            #pragma unroll
                            for (uint32_t pass = 0; pass < N / kPass; ++pass) {
                                const uint32_t t = pass * kPass + th / kLanes, s2 = factors[pass];
                                uint4 w = raws[pass];
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
                                    st_shared_u4(dst + t * 128 + ((chunk ^ (t & 7u)) << 4), make_uint4(v[0], v[1], v[2], v[3]));
                                }
                            }
                            ptx::fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) {
                                ptx::mbar_arrive(full0 + 8 * slot);
                                ptx::mbar_arrive(raw_empty0 + 8 * rs);
                            }
                        }
                    }
                }
            } else if (NF4 ? warp == kCopyWarp : warp < kExpandWarp + 2 * kCopies) {
                const uint32_t own = NF4 ? 0u : (warp - kExpandWarp) & 1u, part = NF4 ? 0u : (warp - kExpandWarp) >> 1;  // bf16: K or V, and which columns
                const uint32_t unit = NF4 ? kGroup : box_rows, units = N / unit;  // tokens that come together, being in one page
                uint32_t i = 0, tails = 0, step = 0;
                Ring ring;
                for (uint32_t piece = 0; ok && walk.next(c, b, a, p); ++piece, step += p.steps) {
                    const uint32_t tile0 = expanded ? __ldg(dense.bases + p.seq) + p.step0 : 0u;
                    const uint32_t stored = min(p.s.length, (p.step0 + p.steps) * N);  // tokens that there are
                    #pragma unroll 1
                    for (uint32_t turn = 0; ok && turn < 2 * p.steps; ++turn, ++i, ring.on(slots)) {
                        const Turn<kPlaces> of(turn, p.steps);
                        const uint32_t which = of.values, j = of.step;
                        if (!NF4 && which != own) continue;
                        const uint32_t t0 = (p.step0 + j) * N, g = lane % units, box = lane / units, t = t0 + g * unit;
                        const uint32_t groups = stored > t0 ? min(units, (stored - t0 + unit - 1) / unit) : 0u;
                        const uint32_t rs = i % S::kRawSlots, slot = ring.slot;
                        uint32_t place = 0;
                        if (expanded) {
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
                        bool got = true;
                        if (NF4 && !expanded) {
                            if (i >= S::kRawSlots) got = ptx::mbar_wait_suspended(raw_empty0 + 8 * rs, (i / S::kRawSlots + 1) & 1u);
                        } else if (ring.round) {
                            got = ptx::mbar_wait_suspended(empty0 + 8 * slot, (ring.round + 1) & 1u);
                        }
                        got = __all_sync(0xffffffffu, got);
                        const uint32_t dst = place_of(slot);
                        if (!got) {
                        } else if (NF4 && expanded) {
                            const uint32_t bar = full0 + 8 * slot;
                            if (lane == 0) {
                                ptx::mbar_arrive_expect_tx(bar, S::kTile);
                                const int32_t row = (int32_t)(((tile0 + j) * c.heads + p.head) * N);
                                #pragma unroll
                                for (uint32_t x = 0; x < D / 64; ++x) ptx::tma_load_2d(dst + x * S::kBox, which ? &tmap_v : &tmap_k, (int32_t)(64 * x), row, bar);
                                for (int e = 0; e < 3; ++e) ptx::mbar_arrive(bar);  // (for the four warps that expand)
                            }
                        } else if (NF4) {
                            const uint32_t bar = raw_full0 + 8 * rs, raw = raw0 + rs * S::kRaw;
                            if (lane == 0) ptx::mbar_arrive_expect_tx(bar, groups * (kGroup * (D / 2) + (which ? 1u : 2u) * kGroup * kBlocks * 4));
                            __syncwarp();
                            if (box == 0 && g < groups) {
                                ptx::bulk_g2s(raw + g * kGroup * (D / 2), static_cast<const uint8_t *>(which ? c.v : c.k) + (uint64_t)place * (D / 2), kGroup * (D / 2), bar);
                                ptx::bulk_g2s(raw + N * (D / 2) + g * kGroup * kBlocks * 4, (which ? c.v_scales : c.k_scales) + (uint64_t)place * kBlocks, kGroup * kBlocks * 4, bar);
                                if (!which)
                                    ptx::bulk_g2s(raw + N * (D / 2) + S::kScales + g * kGroup * kBlocks * 4, c.v_scales + (uint64_t)place * kBlocks, kGroup * kBlocks * 4, bar);
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
                                got = __all_sync(0xffffffffu, ptx::mbar_wait_suspended(bar, tails & 1u));
                                ++tails;
                                for (uint32_t k = (p.s.length > t0 ? p.s.length - t0 : 0u) * 8 + lane; k < N * 8; k += 32)
                                    #pragma unroll
                                    for (uint32_t x = 0; x < kColumns; ++x) st_shared_u4(dst + (part * kColumns + x) * S::kBox + k * 16, make_uint4(0u, 0u, 0u, 0u));
                                ptx::fence_proxy_async();
                                __syncwarp();
                                if (lane == 0) ptx::mbar_arrive(full0 + 8 * slot);
                            }
                        }
                        if (!got) {
                            ok = false;
                            if (lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 26);
                        }
                    }
                }
            } else if (warp == kMmaWarp + 1) {
                // (idle otherwise) the L2 asked for the queries of all of the CTA's pieces
                while (walk.next(c, b, a, p))
                    for (uint32_t i = lane; i < p.rows * (D / 64); i += 32) {
                        const uint32_t row = p.r0 + i / (D / 64), token = a.by_group.of(row);
                        const __nv_bfloat16 *const q = static_cast<const __nv_bfloat16 *>(a.q) + (uint64_t)(p.s.row0 + token) * a.ldq +
                                                       (uint64_t)(p.head * a.group + row - token * a.group) * D + i % (D / 64) * 64;
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
                    }
            } else if (warp == kMmaWarp) {
                constexpr uint32_t fmt = NF4 ? 0 : 1;
                constexpr uint32_t idesc_s = ptx::f16_idesc(fmt, 128, N, false, false), idesc_o = ptx::f16_idesc(fmt, 128, D, false, true);
                uint32_t made[2] = {0, 0}, used[2] = {0, 0}, rows_in[2] = {0, 0};  // scores, weights and Q's so far
                Ring ring;  // the next tile of K or V
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    if (!ok) return;
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_suspended(bar, parity));
                    if (!ok && lane == 0) NF4_REPORT_FAILURE(*failure.flag, *failure.host, 27);
                };
                auto wait_full = [&](const Ring &at) { wait(full0 + 8 * at.slot, at.round & 1u); };
                // (these two by the elected thread)
                auto scores = [&](uint32_t tile, uint32_t at, uint32_t n) {  // of the keys in ring place `at`, to the place of the tile's n-th
                    const uint64_t qd = ptx::sw128_desc(q0 + tile * S::kQTile), kd = ptx::sw128_desc(place_of(at));
                    #pragma unroll
                    for (uint32_t k = 0; k < D / 16; ++k)
                        ptx::mma_ss_f16(tmem + S::kS + (kPlaces * tile + n % kPlaces) * N, qd + (k >> 2) * (16384 >> 4) + (k & 3u) * 2, kd + (k >> 2) * (S::kBox >> 4) + (k & 3u) * 2,
                                        idesc_s, k != 0);
                    ptx::tc_commit(s_full0 + 8 * (kPlaces * tile + n % kPlaces));
                };
                auto products = [&](uint32_t tile, uint32_t at, uint32_t n, bool add) {
                    const uint64_t vd = ptx::sw128_desc(place_of(at), S::kBox);
                    #pragma unroll
                    for (uint32_t k = 0; k < N / 16; ++k)
                        ptx::mma_ts_f16(tmem + S::kO + tile * D, tmem + S::kS + (kPlaces * tile + n % kPlaces) * N + 8 * k, vd + 128 * k, idesc_o, add || k != 0);
                    if (kPlaces > 1) ptx::tc_commit(pv_done0 + 8 * tile);
                };
                while (ok && walk.next(c, b, a, p)) {
                    for (uint32_t j = 0; j < min(kPlaces, p.steps) && ok; ++j, ring.on(slots)) {  // the first scores
                        wait_full(ring);
                        for (uint32_t t = 0; t < p.live; ++t) {
                            if (j == 0) {
                                wait(q_ready0 + 8 * t, rows_in[t] & 1u);
                                ++rows_in[t];
                            }
                            ptx::tc_fence_after();
                            if (ok && ptx::elect_one()) {
                                scores(t, ring.slot, made[t]);
                                if (t + 1 == p.live) ptx::tc_commit(empty0 + 8 * ring.slot);
                            }
                            ++made[t];
                            __syncwarp();
                        }
                    }
                    for (uint32_t j = 0; j < p.steps && ok; ++j) {
                        const bool more = j + kPlaces < p.steps;
                        const Ring v = ring;
                        ring.on(slots);
                        const Ring k = ring;
                        if (more) ring.on(slots);
                        wait_full(v);
                        for (uint32_t t = 0; t < p.live; ++t) {
                            wait(p_ready0 + 8 * (kPlaces * t + used[t] % kPlaces), (used[t] / kPlaces) & 1u);
                            if (!ok) break;
                            ptx::tc_fence_after();
                            if (ptx::elect_one()) {
                                products(t, v.slot, used[t], j != 0);
                                if (t + 1 == p.live) ptx::tc_commit(empty0 + 8 * v.slot);
                                if (j + 1 == p.steps) ptx::tc_commit(o_done0 + 8 * t);
                            }
                            ++used[t];
                            __syncwarp();
                            if (!more) continue;
                            if (t == 0) wait_full(k);
                            if (!ok) break;
                            ptx::tc_fence_after();
                            if (ptx::elect_one()) {
                                scores(t, k.slot, made[t]);
                                if (t + 1 == p.live) ptx::tc_commit(empty0 + 8 * k.slot);
                            }
                            ++made[t];
                            __syncwarp();
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

// ---- a quantized cache expanded once --------------------------------------------------------------
// Where several row tiles of a head go over the same tokens.  A CTA has a tile of N tokens of one head: the power of two
// for its largest scale, then levels times scales in f16, eight values to a thread at a time.  Bound by what it writes.
template <int D>
__global__ void __launch_bounds__(256)
expand_kernel(const CacheView c, const BatchView b, uint4 *const k_out, uint4 *const v_out, uint32_t *const bases, float2 *const powers) {
    constexpr uint32_t N = Shape<D, true>::kTokens, kBlocks = D / 64, kGroups = D / 8;  // eight values each
    __shared__ uint32_t s_pairs[256], s_most[2], s_place[N], s_bad;
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    s_pairs[tid] = level_pair_f16(tid);
    if (tid < 2) s_most[tid] = 0;
    if (tid == 2) s_bad = 0;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    // which sequence the tile is of (every warp finds it); the first CTA writes down where each begins
    const uint32_t head = blockIdx.x % c.heads, want = blockIdx.x / c.heads;
    uint32_t seq = b.sequences, tile = 0;
    uint64_t before = 0;
    Sequence s{0, 0, 0};
    for (uint32_t s0 = 0; s0 < b.sequences && (seq == b.sequences || blockIdx.x == 0); s0 += 32) {
        Sequence o{0, 0, 0};
        if (s0 + lane < b.sequences) o = sequence_of(c, b, s0 + lane);
        const uint32_t own = s0 + lane < b.sequences ? max(1u, (o.length + N - 1) / N) : 0u;
        uint32_t upto = own;
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= (uint32_t)d) upto += v;
        }
        if (blockIdx.x == 0 && tid < 32 && s0 + lane < b.sequences) bases[s0 + lane] = (uint32_t)before + upto - own;
        const uint32_t past = __ballot_sync(0xffffffffu, before + upto > want);
        if (past && seq == b.sequences) {
            const int l = __ffs(past) - 1;
            seq = s0 + l;
            tile = want - (uint32_t)before - __shfl_sync(0xffffffffu, upto - own, l);
            s = Sequence{__shfl_sync(0xffffffffu, o.row0, l), __shfl_sync(0xffffffffu, o.rows, l), __shfl_sync(0xffffffffu, o.length, l)};
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (blockIdx.x == 0 && tid == 0) bases[b.sequences] = (uint32_t)min(before, (uint64_t)0xffffffffu);
    if (seq == b.sequences) return;
    __syncthreads();
    const uint32_t t0 = tile * N, tokens = s.length > t0 ? min(N, s.length - t0) : 0u;
    if (tid < N) {
        uint32_t place = 0;
        if (tid < tokens) {
            const uint32_t at = c.by_page.of(t0 + tid);
            const int32_t page = __ldg(b.table + (uint64_t)seq * b.width + at);
            if (page < 0 || (uint32_t)page >= c.pages) s_bad = 1;
            else place = ((uint32_t)page * c.heads + head) * c.page_size + (t0 + tid - at * c.page_size);
            uint32_t most[2] = {0, 0};
            #pragma unroll
            for (uint32_t k = 0; k < kBlocks; ++k) {
                most[0] = max(most[0], __float_as_uint(__ldg(c.k_scales + (uint64_t)place * kBlocks + k)));
                most[1] = max(most[1], __float_as_uint(__ldg(c.v_scales + (uint64_t)place * kBlocks + k)));
            }
            atomicMax(&s_most[0], most[0]);
            atomicMax(&s_most[1], most[1]);
        }
        s_place[tid] = place;
    }
    __syncthreads();
    const float power[2] = {power_for(s_most[0]), power_for(s_most[1])};
    const uint64_t out0 = ((uint64_t)want * c.heads + head) * N * kGroups;
    if (tid == 0) powers[(uint64_t)want * c.heads + head] = s_bad ? make_float2(0.f, 0.f) : make_float2(power[0], power[1]);
    #pragma unroll
    for (uint32_t which = 0; which < 2; ++which) {
        const uint32_t *const codes = static_cast<const uint32_t *>(which ? c.v : c.k);
        const float *const scales = which ? c.v_scales : c.k_scales;
        const float unit = reciprocal_of_power(power[which]) * (1.f / kLevelUnit);
        #pragma unroll 4
        for (uint32_t i = tid; i < N * kGroups; i += 256) {
            const uint32_t t = i / kGroups, g = i % kGroups;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (t < tokens) {
                const uint64_t row = s_place[t];
                const uint32_t w = __ldg(codes + row * kGroups + g);
                const float scale = __ldg(scales + row * kBlocks + g / 8) * unit;
                const uint32_t s2 = pack<true>(scale, scale);
                v = make_uint4(mul_f16x2(s_pairs[w & 255u], s2), mul_f16x2(s_pairs[w >> 8 & 255u], s2), mul_f16x2(s_pairs[w >> 16 & 255u], s2), mul_f16x2(s_pairs[w >> 24], s2));
            }
            (which ? v_out : k_out)[out0 + i] = v;
        }
    }
}

// The row tiles that several CTAs had: a warp to four rows at a time, the parts in the order of the tokens.
constexpr uint32_t kJoinRows = 4, kJoinWarps = 8;
template <int D, bool NF4>
__global__ void __launch_bounds__(32 * kJoinWarps)
join_pieces_kernel(const AttentionView a, const Split *const splits) {
    constexpr uint32_t kRows = Shape<D, NF4>::kRows, kWide = D / 32;  // values of a row to a lane
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    const Split s = splits[blockIdx.x];
    const uint32_t r0 = (blockIdx.y * kJoinWarps + threadIdx.x / 32) * kJoinRows, lane = threadIdx.x & 31u;
    if (r0 >= s.rows) return;
    auto part = [&](uint32_t i) { return (uint64_t)(2 * (blockIdx.x + i) + (i ? 0 : 1)) * kRows + r0; };
    float m[kJoinRows], sum[kJoinRows], acc[kJoinRows][kWide];
    #pragma unroll
    for (uint32_t r = 0; r < kJoinRows; ++r) {
        m[r] = -INFINITY;
        sum[r] = 0.f;
        #pragma unroll
        for (uint32_t j = 0; j < kWide; ++j) acc[r][j] = 0.f;
    }
    #pragma unroll 2
    for (uint32_t i = 0; i <= s.more; ++i) {
        #pragma unroll
        for (uint32_t r = 0; r < kJoinRows; ++r) {  // (a tile's rows behind its last hold anything; they are not written)
            const float2 ml = __ldg(a.part_ml + part(i) + r);
            float v[kWide];
            const float *const o = a.part_o + (part(i) + r) * D + lane * kWide;
            #pragma unroll
            for (uint32_t j = 0; j < kWide; j += 2) {
                const float2 w = __ldg(reinterpret_cast<const float2 *>(o + j));
                v[j] = w.x;
                v[j + 1] = w.y;
            }
            const float top = fmaxf(m[r], ml.x), base = top == -INFINITY ? 0.f : top;
            const float keep = exp2_approx(m[r] - base), f = exp2_approx(ml.x - base);  // (nothing seen: 2^-inf)
            m[r] = top;
            sum[r] = fmaf(f, ml.y, sum[r] * keep);
            #pragma unroll
            for (uint32_t j = 0; j < kWide; ++j) acc[r][j] = fmaf(f, v[j], acc[r][j] * keep);
        }
    }
    #pragma unroll
    for (uint32_t r = 0; r < kJoinRows; ++r) {
        if (r0 + r >= s.rows) break;
        const float f = sum[r] == 0.f ? 0.f : 1.f / sum[r];
        const uint32_t q_row = s.r0 + r0 + r, token = a.by_group.of(q_row);
        __nv_bfloat16 *const out = static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)(s.row0 + token) * a.ldo + (uint64_t)(s.head * a.group + q_row - token * a.group) * D + lane * kWide;
        #pragma unroll
        for (uint32_t j = 0; j < kWide; j += 2) *reinterpret_cast<uint32_t *>(out + j) = bf16_pair(acc[r][j] * f, acc[r][j + 1] * f);
    }
}

uint64_t rows_of(const AttentionCall &c) { return c.head_dim == 256 ? 128 : 256; }
uint64_t tokens_of(const AttentionCall &c) { return c.head_dim == 256 ? 64 : 128; }

// Tiles to a head to be expanded ahead: where the host's bounds say that three row tiles or more of a head go over most tokens (with two
// the expansion in place, which is slower by half a step, costs what the kernel ahead does), up to 2 GB.
uint64_t dense_tiles(const AttentionCall &c) {
    if (!c.nf4 || (uint64_t)c.most_rows * c.view.group <= 2 * rows_of(c)) return 0;
    const uint64_t tiles = (uint64_t)c.batch.sequences * std::max<uint64_t>(1, (c.most_tokens + tokens_of(c) - 1) / tokens_of(c));
    return tiles * c.cache.heads * tokens_of(c) * c.head_dim * 4 <= 1ull << 31 && tiles * c.cache.heads * tokens_of(c) < 1ull << 31 ? tiles : 0;
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
        const uint64_t tiles = dense_tiles(c), dense = tiles * c.cache.heads * tokens_of(c) * c.head_dim * 2;
        splits = take(kNumSMs * sizeof(Split));
        ml = take(2ull * kNumSMs * rows_of(c) * sizeof(float2));
        o = take(2ull * kNumSMs * rows_of(c) * c.head_dim * sizeof(float));
        bases = take(tiles ? (c.batch.sequences + 1ull) * sizeof(uint32_t) : 0);
        powers = take(tiles * c.cache.heads * sizeof(float2));
        k = take(dense);
        v = take(dense);
        bytes = at;
    }
};

template <int D, bool NF4>
int32_t launch(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    using S = Shape<D, NF4>;
    auto kernel = attention_chunk_kernel<D, NF4>;
    NF4_TRY(ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::kSmem));
    const uint64_t pool = (uint64_t)c.cache.pages * c.cache.heads * c.cache.page_size;
    CUtensorMap map_k{}, map_v{};
    uint32_t box_rows = kGroup;  // tokens of a page that come in one copy
    if (!NF4) {
        while (box_rows < S::kTokens && c.cache.page_size % (2 * box_rows) == 0) box_rows *= 2;
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
    if constexpr (NF4) {
        dense.capacity = (uint32_t)dense_tiles(c);
        if (dense.capacity) {
            uint32_t *const bases = reinterpret_cast<uint32_t *>(workspace + at.bases);
            float2 *const powers = reinterpret_cast<float2 *>(workspace + at.powers);
            const uint64_t dense_rows = (uint64_t)dense.capacity * c.cache.heads * S::kTokens;
            NF4_TRY(make_map(&map_k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, workspace + at.k, dense_rows, D, 2 * D, S::kTokens, 64, CU_TENSOR_MAP_SWIZZLE_128B));
            NF4_TRY(make_map(&map_v, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, workspace + at.v, dense_rows, D, 2 * D, S::kTokens, 64, CU_TENSOR_MAP_SWIZZLE_128B));
            dense.bases = bases;
            dense.powers = powers;
            count_launch();
            NF4_TRY(launch_maybe_overlapped(expand_kernel<D>, dim3(dense.capacity * c.cache.heads), dim3(256), 0, stream, true, c.cache, c.batch,
                                            reinterpret_cast<uint4 *>(workspace + at.k), reinterpret_cast<uint4 *>(workspace + at.v), bases, powers));
        }
    }
    const uint32_t ctas = persistent_ctas();
    count_launch(2);
    NF4_TRY(launch_maybe_overlapped(kernel, dim3(ctas), dim3(kThreads), S::kSmem, stream, true, map_k, map_v, c.cache, c.batch, view, dense, box_rows, splits, failure));
    return launch_maybe_overlapped(join_pieces_kernel<D, NF4>, dim3(ctas, S::kRows / (kJoinRows * kJoinWarps)), dim3(32 * kJoinWarps), 0, stream, true, view,
                                   static_cast<const Split *>(splits));
}

}  // namespace

uint64_t attention_chunk_bytes(const AttentionCall &c) {
    return Layout(c).bytes;
}

// The line of steps is counted in 32 bits, and what the page table has room for bounds it.
bool attention_chunk_counts(const AttentionCall &c) {
    const uint64_t tiles = ((uint64_t)c.batch.rows * c.view.group / rows_of(c) + c.batch.sequences) * c.cache.heads;
    const uint64_t steps = ((uint64_t)c.batch.width * c.cache.page_size + tokens_of(c) - 1) / tokens_of(c);
    return tiles * (steps + 1 + kStart) < 1ull << 31;
}

int32_t attention_chunk(const AttentionCall &c, uint8_t *workspace, cudaStream_t stream) {
    switch (c.head_dim) {
        case 64: return c.nf4 ? launch<64, true>(c, workspace, stream) : launch<64, false>(c, workspace, stream);
        case 128: return c.nf4 ? launch<128, true>(c, workspace, stream) : launch<128, false>(c, workspace, stream);
        default: return c.nf4 ? launch<256, true>(c, workspace, stream) : launch<256, false>(c, workspace, stream);
    }
}

}  // namespace nf4

using namespace nf4;

extern "C" {

int32_t nf4_cache_attention_row_place(uint32_t head_dim, uint32_t thread, uint32_t chunk, int32_t results) {
    const char *const what = "nf4_cache_attention_row_place";
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(NF4_ERR_UNSUPPORTED, "%s: head_dim is %u; 64, 128 and 256 are supported", what, head_dim);
    if (thread >= 128 || chunk >= head_dim / 8) return fail(NF4_ERR_INVALID_ARG, "%s: no such thread or chunk", what);
    if (results) return (int32_t)chunk_place(thread, chunk);
    const RowChunk own = chunk_of(head_dim, thread / 32, thread % 32, chunk);
    return (int32_t)chunk_place(own.row, own.x);
}

}  // extern "C"
