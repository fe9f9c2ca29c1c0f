// What the attention kernels on the tensor cores share: how their steps are shared out between the CTAs, and how one walks through them.
#pragma once
#include <cuda.h>

#include "kv_cache.cuh"
#include "ptx.cuh"

namespace nf4 {

namespace {

// Weights are 2^(S c - m + raise).  In f16 up to 2^15, so that it holds those that are 2^-32 of a row's largest; their sum is raised alike, and where
// sums go to the workspace both are lowered by that again, so that no value overflows them that would not overflow a sum of weights up to
// one.  bf16 has the range: weights up to one.
template <bool NF4>
constexpr float kRaise = NF4 ? 7.f : -8.f;
template <bool NF4>
constexpr float kLower = NF4 ? 1.f / 32768.f : 1.f;
constexpr uint32_t kGroup = 16;  // tokens that are in one page for sure

// Where a chunk of 16 bytes of a tile's 128 rows is, of the queries as the MMA reads them: a box of 128 rows to every 64 values (128 bytes), chunks
// swizzled.
__host__ __device__ constexpr uint32_t chunk_place(uint32_t row, uint32_t x) { return (x >> 3) * 16384u + row * 128u + (((x & 7u) ^ (row & 7u)) << 4); }

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
    bool whole;  // a tile belongs to the CTA in whose share it begins
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

// Through a CTA's pieces; every warp goes its own way.  R rows to a tile, N tokens to a step; START: steps' worth of time that a row tile takes beside
// its steps (its queries in, its results out), counted in the line, or the CTAs that have a prompt's first tiles, of one step each, would be done
// last; LEAST: what a CTA has of the line at least; WHOLE: how much
// more than its share a CTA may have at least where no row tile is divided then, in place of the second start and the join (0: tiles are divided); TREE: rows
// are nodes of trees.
template <uint32_t R, uint32_t N, uint32_t START, uint32_t LEAST, uint32_t WHOLE, bool TREE>
struct Walker {
    static constexpr uint32_t kStart = START, kLeast = LEAST, kWhole = WHOLE;
    Sequence s;
    uint32_t seq, head, tile, off, now, end;
    bool whole;

    static __device__ __forceinline__ uint32_t tiles_of(const Sequence &s, uint32_t group) { return (uint32_t)(((uint64_t)s.rows * group + R - 1) / R); }
    // (a tile that sees nothing has one step all the same: its results are zeros)
    static __device__ __forceinline__ uint32_t steps_of(const Sequence &s, const AttentionView &a, uint32_t tile) {
        const uint32_t last = (uint32_t)min((uint64_t)(tile + 1) * R, (uint64_t)s.rows * a.group) - 1;
        return max(1u, (seen_end<TREE>(s, a.by_group, last) + N - 1) / N);
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
        const uint32_t upto = WHOLE && whole ? p.all + kStart : min(p.all + kStart, end - p.line0);
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


// By one warp of every CTA: the share of the line that each has, and where this CTA's begins: first_of {sequence, head, tile, place in the tile's part
// of the line, place in the line, end in the line}.
template <class Walk>
__device__ __forceinline__ Share share_out(const CacheView &c, const BatchView &b, const AttentionView &a, uint32_t *first_of) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t longest = 0, shortest = 0xffffffffu, all_tiles = 0;  // what a tile has of the line at most and at least
    // a lane a sequence: its steps, all heads
    auto steps_of = [&](uint32_t s0, Sequence &s) -> uint32_t {
        s = Sequence{0, 0, 0};
        if (s0 + lane < b.sequences) s = sequence_of(c, b, s0 + lane);
        const uint32_t tiles = Walk::tiles_of(s, a.group);
        if (Walk::kWhole && tiles) {
            longest = max(longest, Walk::kStart + Walk::steps_of(s, a, tiles - 1));
            shortest = min(shortest, Walk::kStart + Walk::steps_of(s, a, 0));
            all_tiles += tiles * c.heads;
        }
        uint32_t sum = 0;
        if (tiles <= 8)
            for (uint32_t t = 0; t < tiles; ++t) sum += Walk::kStart + Walk::steps_of(s, a, t);
        for (uint32_t many = __ballot_sync(0xffffffffu, tiles > 8); many; many &= many - 1) {  // with the whole warp
            const int l = __ffs(many) - 1;
            const Sequence o{__shfl_sync(0xffffffffu, s.row0, l), __shfl_sync(0xffffffffu, s.rows, l), __shfl_sync(0xffffffffu, s.length, l)};
            uint32_t part = 0;
            for (uint32_t t = lane; t < Walk::tiles_of(o, a.group); t += 32) part += Walk::kStart + Walk::steps_of(o, a, t);
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
    share.ctas = min(gridDim.x, (total + Walk::kLeast - 1) / Walk::kLeast);
    share.whole = false;
    if (Walk::kWhole) {
        longest = __reduce_max_sync(0xffffffffu, longest);
        shortest = __reduce_min_sync(0xffffffffu, shortest);
        all_tiles = __reduce_add_sync(0xffffffffu, all_tiles);
        // (no share is as long as a tile then, so that none has two that begin in it)
        const uint32_t of_share = share.ctas ? total / share.ctas : 0, more = Walk::kWhole + min(4u, of_share / 12);  // (measured: see kWhole)
        share.whole = all_tiles <= gridDim.x && (uint64_t)shortest * share.ctas >= total && (uint64_t)(longest - min(longest, more)) * share.ctas <= total;
    }
    share.per = share.ctas ? total / share.ctas : 0;
    share.more = share.ctas ? total - share.per * share.ctas : 0;
    const uint32_t first = share.start(blockIdx.x);
    uint32_t last = blockIdx.x < share.ctas ? share.start(blockIdx.x + 1) : first, before = 0, skipped = 0;
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
                const uint32_t mine = t0 + lane < Walk::tiles_of(o, a.group) ? Walk::kStart + Walk::steps_of(o, a, t0 + lane) : 0u;
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
            if (Walk::kWhole && share.whole && left) {  // on to the next tile's beginning
                skipped = Walk::kStart + Walk::steps_of(o, a, tile) - left;
                left = 0;
                ++tile;
            }
            if (lane == 0) {
                first_of[0] = k + l;
                first_of[1] = head;
                first_of[2] = tile;
                first_of[3] = left;
            }
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (!found) last = first;  // (row starts that decrease, whose rows are more than the line is counted for: no access by what is not there)
    if (lane == 0) {
        first_of[4] = first + skipped;
        first_of[5] = last;
    }
    return share;
}

}  // namespace

// attention_chunk.cu: a quantized cache expanded ahead (see Dense).  How many tiles to a head the workspace may have, 0 where there is no
// expanding; and the kernel ahead, with the tensor maps of what it leaves in k and v (each tiles * heads * kTokens rows of f16).
uint64_t attention_expanded_tiles(const AttentionCall &c);
int32_t attention_expand(const AttentionCall &c, uint32_t capacity, void *k, void *v, uint32_t *bases, float2 *powers, CUtensorMap *map_k, CUtensorMap *map_v,
                         cudaStream_t stream);

}  // namespace nf4
