// Paged decode attention over the cache in 4 bits (layout and meaning of codes and params: kv4.cu).
//
// One new token per sequence:  score_t = (q . k_t) / sqrt(D),  k_t = least_t + step_t * code_t,  p = softmax(score) over the
// sequence's tokens,  out = sum_t p_t (least_t + step_t * code_t).  Written with the codes n_t as they lie in memory:
//     q . k_t = least_t * sum(q) + step_t * (q . n_t)          out = sum_t p_t least_t + sum_t (p_t step_t) n_t
// so only the products with the codes touch every element, and the dequantised values are never formed (nor rounded).
//
// Bound: a token costs D / 2 + 4 bytes per KV head and side, a quarter of a 16-bit cache, at four times the tokens per byte.  What
// limits the kernel is therefore the number of instructions per element, and its layout follows from that:
//   * The tokens are the rows of mma.sync m16n8k16 and the query heads of a KV head's group its columns (S^T = K Q^T, O^T = V^T P^T), as
//     in the 16-bit kernel; a matrix unit at a few tens of per cent of its rate and no reduction over lanes per score.
//   * A code becomes an f16 operand with one logic instruction per two elements and no arithmetic: bits masked in place ARE a subnormal
//     f16, exact: the low four bits of a byte are n_even * 2^-24, the high four 16 n_odd * 2^-24, the whole byte their sum F (the high
//     byte of a half comes down with a byte permute that clears the rest).  The factors are powers of two and are put back into
//     the query fragments and the output.  Logic instructions run at half rate and are what binds, so V takes F
//     where it does not need the mask: the odd dimension is (F - even) / 16, taken from the accumulators at the end.  (K cannot: the
//     query fragment of the even element would be q_even - q_odd / 16, which f16 rounds; measured beyond the tolerance of f16 queries
//     with peaked scores.)
//   * K: a lane's 16-byte (D = 128) piece of a token holds its A fragments for all of the contraction, since the order of the contraction
//     is free: the query fragments are loaded in the order in which the masks deliver the elements.  V: two byte permutes pair the
//     words of two tokens, then the same masks.
//   * Up to four query heads per KV head (QUAD): the scores are integer products.  As bytes the codes need no conversion at all: F is the word
//     as it lies in memory and L one mask per word (16 logic instructions per step and lane where the f16 form needs 80), and
//     the four unused columns take the lower bytes of the queries' integers, so that a lane has whole scores of one head.  Two bytes hold a
//     query to 2^-16 of its largest element, three to 2^-24.  What two leave shows where one channel is far larger than the others (norm of
//     the output's error, channel 50 / 200 / 1000 times as large): bf16 1.8 / 2.5 / 3.5e-3 with two and 1.6 / 1.7 / 1.6e-3 with three, both below the
//     half step of its rounding (2^-8); f16 9 / 23 / 26e-4 with two, 2e-4 with three, its half step being 4.9e-4.  The third byte costs a product per
//     tile and 16 bytes of queries (64 sequences of 512 to 32768 tokens: bf16 110 -> 117 us, f16 132 -> 135).  So f16 takes three bytes, bf16
//     two.  More heads take the f16 form: queries as f16, scaled by a power of two per (sequence, head) so that a bf16 query of any size fits.
//   * The weights p_t * step_t enter as f16, relative to a running power of two about the largest step, which joins the running maximum of
//     the softmax in rescaling the accumulator.  Their rounding (half a step of 2^-11) multiplies codes of 0 .. 15, more than the
//     values themselves amount to: 2^-10 of the output, measured, unseen in a bf16 output and five times the rounding of an f16 one.  For
//     f16 the weights therefore come in two parts, the second in the unused columns (QUAD, free) or in products of its own, and V
//     enters as n - 8, one more 16-bit subtraction per operand: sums of n itself are far larger than what is left of them once
//     sum(p_t least_t) joins them, and the matrix unit cuts its sums off (100001 tokens, 16 heads: error 1.2e-3 of the output with
//     n, 2.1e-4, the rounding of the output, with n - 8; 46 -> 48 us).
// Sums, maxima and accumulators are float32.
// Measured (bf16, 32 heads of 128, page size 16): 64 sequences of 512 to 32768 tokens on 8 KV heads 109 us, 5.2 TB/s (86 us at the copy rate;
// the steps between the first and the last stream 6.1 TB/s, the rest is the start and the joins); two of 131072 tokens on 4 KV heads 44 us,
// on 2 KV heads 40; one of 1024 tokens 12 us, of which 2 are the launch, 2 the prefix, 3 the first copies, 3 the step itself, 2 the joins.
//
// Work: the tiles of 16 tokens of all (KV head, sequence) pairs in one list, every pair a few tiles longer for what its start costs, cut into
// equal contiguous ranges, one per CTA, and each CTA's range into equal ranges, one per warp.  A warp owns its pipeline (stages of 32
// tokens, copies running ahead across sequence boundaries, page entries one step further ahead), so there is no block-wide barrier
// before the end.  Where pages hold whole tiles the
// copies are bulk copies, four per tile (codes and params of K and V), each issued by a lane of its own: ~20 instructions per step where
// 16-byte copies with a page lookup per token take ~90.  A pair that lies inside a warp's range is written by the warp.  Otherwise the warps
// of a CTA put their partials (maximum, sum, accumulator) together, and the CTAs that share a pair join theirs together: each waits, bounded,
// for the pair's counter and takes its share of the output's 32-dimension slices (a cooperative launch makes all CTAs resident; where it
// is refused the CTA that arrives last joins everything).  Fixed order either way: the same bits from call to call.  One CTA joining 38
// others' parts of 16 heads took 18 us, all of them together 3.
#include <limits.h>
#include <math.h>
#include <stdlib.h>

#include "common.cuh"

namespace puter {

namespace q4d {

constexpr int kTile = 16;             // tokens per tile
constexpr int kPrefixSmem = 1024;     // sequences whose tile prefix sums fit shared memory
constexpr int kStageBytes = 209 * 1024;  // of shared memory for the copies in flight: three steps of 16 warps or of 8 with twice the tokens
constexpr int kWarpTiles = 2;         // tiles that a warp gets at least before another CTA takes part
constexpr int kMostTokens = INT_MAX - 255;  // of a context: places two steps behind its last token still fit 31 bits

struct Params {
    const uint16_t* q;
    const uint8_t *kCodes, *vCodes;
    const uint32_t *kParams, *vParams;
    const int32_t *table, *ctxLens;
    uint16_t* out;
    int* errorFlag;
    const int* tileStart;  // [batch + 3] exclusive prefix of tiles, the most and the fewest of one, or nullptr: scanned in shared memory
    float* acc;            // partial accumulators [slots, heads of a block, D]: one slot per warp, then two per CTA
    float2* ml;            // (maximum in the log2 domain, sum) [slots, heads of a block]
    int* counters;         // arrivals (and departures) per (unit, sequence): zero on entry and on exit
    int together;          // all CTAs run at the same time (cooperative launch): the owners of a pair join it together
    int batch, maxPages, pageCount, pageSize, pageShift, numHeads, kvHeads, group;
    int blocks, units;     // head blocks per KV head, KV heads * blocks
    float scaleLog2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes, uint64_t pol) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(pol) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// one bulk copy, counted by the mbarrier `bar`; addresses and size are multiples of 16 bytes
__device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t pol) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(pol) : "memory");
}
// false when the copies that `bar` counts have not landed after about a second
__device__ __forceinline__ bool landed(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < (1 << 22); i++) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t* r) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void lds64(uint32_t a, uint32_t* r) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same onto zero
__device__ __forceinline__ void mma0(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// codes as bytes (0 .. 255) times signed query bytes, exact sums
__device__ __forceinline__ void imma(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void imma0(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// low and high four bits of the lower byte of each half, less 8, as f16: 1024 + n and 64 + n are one logic instruction away
__device__ __forceinline__ uint32_t sub16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t low8(uint32_t x) { return sub16((x & 0x000F000Fu) | 0x64006400u, 0x64086408u); }
__device__ __forceinline__ uint32_t high8(uint32_t x) { return sub16((x & 0x00F000F0u) | 0x54005400u, 0x54805480u); }
// lowest signed byte of v; v is left with the rest: v = rest * 256 + byte
__device__ __forceinline__ uint32_t limb(int& v) {
    const int b = (int)(int8_t)v;
    v = (v - b) >> 8;
    return (uint32_t)b & 255u;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127

// tokens of sequence b: negative or over-long contexts are cut and flagged
__device__ __forceinline__ int seq_ctx(const Params& p, int b) {
    long long ctx = p.ctxLens[b];
    const long long cap = (long long)p.maxPages * p.pageSize;
    if (ctx < 0 || ctx > cap) {
        atomicExch(p.errorFlag, 1);
        ctx = ctx < 0 ? 0 : cap;
    }
    return (int)ctx;
}

// exclusive prefix sum of tiles per sequence: out[0 .. batch], the most tiles of one in out[batch + 1] and the fewest of one that is not
// empty in out[batch + 2]; lens (may be null): the cut contexts.  Every thread of the block calls it.
__device__ void block_prefix(const Params& p, int start, int* out, int* lens) {
    __shared__ int sums[32], tops[32], bottoms[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int carry = 0, top = 0, bottom = INT_MAX;
    for (int base = 0; base < p.batch; base += blockDim.x) {
        const int b = base + threadIdx.x, ctx = b < p.batch ? seq_ctx(p, b) : 0;
        const int tiles = ctx > 0 ? (int)(((long long)ctx + kTile - 1) / kTile) + start : 0;
        int incl = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += n;
        }
        const int most = __reduce_max_sync(0xffffffffu, tiles), fewest = __reduce_min_sync(0xffffffffu, tiles ? tiles : INT_MAX);
        if (lane == 31) {
            sums[warp] = incl;
            tops[warp] = most;
            bottoms[warp] = fewest;
        }
        __syncthreads();
        const int used = (min(p.batch - base, (int)blockDim.x) + 31) / 32;
        int before = carry;
        for (int w = 0; w < used; w++) {
            if (w < warp) before += sums[w];
            carry += sums[w];
            top = max(top, tops[w]);
            bottom = min(bottom, bottoms[w]);
        }
        if (b < p.batch) {
            out[b] = before + incl - tiles;
            if (lens) lens[b] = ctx;
        }
        if (base + (int)blockDim.x < p.batch) __syncthreads();  // the sums have been read
    }
    if (threadIdx.x == 0) {
        out[p.batch] = carry;
        out[p.batch + 1] = top;
        out[p.batch + 2] = bottom;
    }
    __syncthreads();
}
__global__ void __launch_bounds__(1024) prefix_kernel(Params p, int start, int* out) { block_prefix(p, start, out, nullptr); }

// a / b for b > 0; 64-bit divisions take a hundred instructions and are hardly ever needed
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((unsigned long long)(a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// `total` tiles cut into `parts` ranges: the first `more` of them have one tile more than `each`
struct Split {
    long long each, more;
    __device__ __forceinline__ Split(long long total, int parts) : each(quotient(total, parts)), more(total - each * parts) {}
    __device__ __forceinline__ long long begin(int i) const { return i * each + (i < more ? i : more); }
    __device__ __forceinline__ int holding(long long g) const {
        const long long edge = more * (each + 1);
        return (int)(g < edge ? quotient(g, each + 1) : more + quotient(g - edge, each));
    }
};

// NT: blocks of eight query heads that a warp serves with one pass over the codes, 0: a block of four with integer scores (QUAD);
// MT: tiles per step
template <int D_, int NT_, int WARPS_, int MT_>
struct Shape {
    static constexpr int D = D_, NT = NT_ ? NT_ : 1, WARPS = WARPS_, MT = MT_;
    static constexpr bool QUAD = NT_ == 0;
    static constexpr int STEP = 16 * MT;            // tokens per step of a warp
    // A pair counts this many tiles more than it has, which nobody works on: what a warp spends on another pair's queries, partial and cold
    // pipeline.  Two steps measured best of none, one, two and three (us, none against two): 256 sequences of up to 2000 tokens 51 : 32, 100 of up
    // to 4000 at 8 heads per KV head 46 : 26, 48 of up to 3000 with 12 KV heads of 64 23 : 17.5, 64 of 512 to 32768 tokens 114.9 : 110.9.
    static constexpr int START = 2 * MT;
    static constexpr int ROW = D / 2;               // bytes of a token's codes
    static constexpr int STAGE = 2 * STEP * ROW + 2 * STEP * 4;
    static constexpr int STAGES = kStageBytes / (WARPS * STAGE);
    static constexpr int SMEM = WARPS * STAGES * STAGE;
    static constexpr int HEADS = QUAD ? 4 : 8 * NT;
};

// weight of a part under the maximum M of all (a part without a finite score has sum 0, or NaN, which stays NaN)
__device__ __forceinline__ float weight(float2 ml, float M) { return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : exp2f(ml.x - M); }

// PAGED: pages hold whole tiles (page size a multiple of 16): bulk copies.  Otherwise 16-byte copies with a page lookup per token.
template <int DT, typename S, bool PAGED>
__global__ void __launch_bounds__(S::WARPS * 32, 1) decode_kernel(Params p) {
    constexpr int D = S::D, NT = S::NT, MT = S::MT, kStep = S::STEP, kStart = S::START;
    constexpr int WK = D / 32;   // words of a token's K codes in a lane
    constexpr int WV = D / 64;   // words of a token's V codes in a lane
    constexpr int ROW = S::ROW;
    constexpr bool QUAD = S::QUAD;
    constexpr bool SPLIT = DT == DT_F16;  // weights in two parts
    constexpr bool FINE = QUAD && DT == DT_F16;  // queries as integers of three bytes
    constexpr int J = QUAD ? 1 : 2;  // heads of a lane: t, or 8nt + 2t and 8nt + 2t + 1
    constexpr int kPart = S::HEADS * D * 4 + S::HEADS * 8;  // a partial in shared memory: accumulators, then (maximum, sum)
    static_assert(kPart <= S::STAGES * S::STAGE, "a warp's partial takes the place of its stages");
    extern __shared__ __align__(128) unsigned char smemRaw[];
    __shared__ int sStart[kPrefixSmem + 3], sCtx[kPrefixSmem];
    __shared__ int sSeg[32];       // entry 2w + i: the pair of warp w's partial i (0: it began before the warp's range, 1: it goes on behind it)
    __shared__ int sNear[S::WARPS];  // which of the two lies in shared memory
    __shared__ int sB[32], sUnit[32], sWhere[32];  // of an entry: sequence, unit; pair inside the CTA's range (2) or begun before it (0) or going on behind it (1)
    __shared__ int sShared[2], sFirst[2], sOwners[2], sGo[2];  // pairs shared with other CTAs: entry, first owner, owners, whether to join
    __shared__ __align__(8) uint64_t sBar[S::WARPS * S::STAGES];
    __shared__ uint4 sTop[FINE ? S::WARPS * 32 : 1];
    const int* ts = p.tileStart;
    if (!ts) {
        block_prefix(p, kStart, sStart, sCtx);
        ts = sStart;
    }
    auto ctx_of = [&](int b) { return p.tileStart ? seq_ctx(p, b) : sCtx[b]; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long long T = ts[p.batch], total = T * p.units;
    if (total == 0) return;
    // CTAs that take part: every one of them has work
    const long long most = (total + S::WARPS * kWarpTiles - 1) / (S::WARPS * kWarpTiles);
    const int parts = most < (long long)gridDim.x ? (int)most : (int)gridDim.x;
    if ((int)blockIdx.x >= parts) return;
    const Split split(total, parts);
    // Ranges end where a pair ends while no pair is large (12 tiles per warp, or a sixteenth of a range): the range may then grow by one pair,
    // but no pair is shared between CTAs, which would cost 4 us at the end.  One sequence of 1024 tokens 14.9 -> 11.8 us, 8 of 1000 19.3 -> 12.9.
    const bool aligned = ts[p.batch + 1] <= max((long long)(12 * S::WARPS), split.each / 16);
    auto edge = [&](int i) {
        const long long at = split.begin(i);
        if (!aligned || at >= total) return at;
        const long long unit = quotient(at, T);
        const int r = (int)(at - unit * T);
        int a = 0, z = p.batch;
        while (z - a > 1) {
            const int m = (a + z) >> 1;
            if (ts[m] <= r) a = m;
            else z = m;
        }
        return unit * T + (r - ts[a] < ts[a + 1] - r ? ts[a] : ts[a + 1]);
    };
    // Few large pairs (eight CTAs each at least) get whole CTAs, in proportion and rounded: a CTA that ends one pair and begins another is
    // 4 us late, and every owner of both waits for it.  What the rounding adds to a range, each^2 / (2 fewest) tiles or so, is kept
    // to some 64 (3 us of streaming).  Two sequences of 16384 tokens with 32 heads on 2 KV heads 23.7 -> 18.6 us, on 8 24.4 -> 22.0.
    // (each >= 2 kStart: the first CTA of a pair has tiles of its own; the products below fit 32 bits)
    const long long fewest = ts[p.batch + 2];
    const bool owned = !aligned && split.each >= 2 * kStart && fewest >= 8 * split.each && split.each * split.each <= 128 * fewest &&
                       total * (parts + 1ll) >> 32 == 0;
    // first CTA of the pair that begins at tile `at`
    auto owner = [&](long long at) { return (int)(((uint32_t)at * parts + (uint32_t)total / 2) / (uint32_t)total); };
    long long clo, chi, from = 0;  // from: where the warps' ranges begin
    if (owned) {
        // the last pair whose first CTA is not behind this one: at * parts + total / 2 < (i + 1) * total
        const uint32_t i = blockIdx.x, last = ((i + 1) * (uint32_t)total - (uint32_t)total / 2 - 1) / (uint32_t)parts, unit = last / (uint32_t)T;
        const int r = (int)(last - unit * (uint32_t)T);
        int a = 0, z = p.batch;
        while (z - a > 1) {
            const int m = (a + z) >> 1;
            if (ts[m] <= r) a = m;
            else z = m;
        }
        const long long at = unit * T + ts[a], tiles = ts[a + 1] - ts[a];
        const int first = owner(at);
        const Split inside(tiles, owner(at + tiles) - first);
        clo = at + inside.begin((int)i - first);
        chi = at + inside.begin((int)i - first + 1);
        from = (int)i == first ? clo + kStart : clo;
    } else {
        clo = edge(blockIdx.x);
        chi = edge(blockIdx.x + 1);
        from = aligned ? clo + kStart : clo;
    }
    if (clo >= chi) return;
    const long long lo = from + warp * (chi - from) / S::WARPS, hi = from + (warp + 1) * (chi - from) / S::WARPS;
    if (threadIdx.x < 32) sSeg[threadIdx.x] = -1;
    if (threadIdx.x < S::WARPS) sNear[threadIdx.x] = -1;
    if (threadIdx.x < 2) sShared[threadIdx.x] = -1;
    const uint32_t bars = smem_u32(sBar) + warp * S::STAGES * 8;
    if (PAGED && lane == 0) {
        for (int i = 0; i < S::STAGES; i++) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * i) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    unsigned char* const mine = smemRaw + warp * (S::STAGES * S::STAGE);
    const uint32_t base = smem_u32(mine);
    uint64_t pol;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));

    if (lo < hi) {
        // ---- the copies' own place in the range, ahead of the computation's ----
        long long iNext = lo;     // first tile behind the segment that is being copied
        int iUnit = (int)quotient(lo, T), ib = 0, iTok = 0, iEnd = 0, iStage = 0;
        {
            const int r = (int)(lo - iUnit * T);
            int a = 0, z = p.batch;
            while (z - a > 1) {
                const int m = (a + z) >> 1;
                if (ts[m] <= r) a = m;
                else z = m;
            }
            ib = a;
        }
        int cUnit = iUnit, cb = ib;
        constexpr int PL = PAGED ? 1 : MT / 2;  // look-ups of a lane
        int entryPage[PL] = {};       // page of this lane's tile (not PAGED: tokens lane + 32 i) of the step to be copied next
        uint32_t inPage[PL] = {};     // and its place in that page, plus the KV head's place in a page
        uint32_t headOff = (uint32_t)(iUnit / p.blocks) * (uint32_t)p.pageSize;
        const uint32_t pageSlots = (uint32_t)p.kvHeads * (uint32_t)p.pageSize;
        const int32_t* iTable = p.table;
        // PAGED: lanes 0 .. 4 MT - 1 issue one copy each: tile lane / 4 of the step, pool lane % 4
        const int part = lane & 3, tileOf = (lane >> 2) % MT;
        const unsigned char* const pool = part == 0 ? p.kCodes : part == 1 ? p.vCodes : (const unsigned char*)(part == 2 ? p.kParams : p.vParams);
        const uint32_t perSlot = part < 2 ? ROW : 4;
        const uint32_t dstOff = (part < 2 ? part * kStep * ROW : 2 * kStep * ROW + (part - 2) * kStep * 4) + tileOf * kTile * perSlot;
        // Moves to the next step and starts fetching its page entries.
        auto look_ahead = [&]() {
            while (iTok >= iEnd) {
                if (iNext >= hi) return;
                long long r = iNext - (long long)iUnit * T;
                if (r >= T) {
                    iUnit++;
                    ib = 0;
                    r -= T;
                    headOff = (uint32_t)(iUnit / p.blocks) * (uint32_t)p.pageSize;
                }
                while (ts[ib + 1] <= r) ib++;
                const long long s0 = ts[ib], s1 = ts[ib + 1], stop = hi - (long long)iUnit * T, e = s1 < stop ? s1 : stop;
                const int ctx = ctx_of(ib);
                const long long end = (e - s0 - kStart) * kTile;
                iTable = p.table + (size_t)ib * p.maxPages;
                iTok = r - s0 > kStart ? (int)((r - s0 - kStart) * kTile) : 0;
                iEnd = (int)(end < ctx ? end : ctx);
                iNext = (long long)iUnit * T + e;
            }
#pragma unroll
            for (int i = 0; i < PL; i++) {
                const int tok = PAGED ? iTok + tileOf * kTile : iTok + lane + 32 * i;
                const int entry = p.pageShift >= 0 ? tok >> p.pageShift : tok / p.pageSize;
                inPage[i] = (uint32_t)(tok - entry * p.pageSize) + headOff;
                entryPage[i] = tok < iEnd ? __ldg(iTable + entry) : 0;
            }
        };
        // Copies the step that look_ahead found and looks for the next.  PAGED copies whole tiles (a tile lies in one page), so tokens
        // behind the sequence come along and are masked; otherwise they are zero-filled.
        auto issue = [&]() {
            if (iTok < iEnd) {
                uint32_t slot[PL];
#pragma unroll
                for (int i = 0; i < PL; i++) {
                    if ((uint32_t)entryPage[i] >= (uint32_t)p.pageCount) {
                        atomicExch(p.errorFlag, 1);
                        entryPage[i] = 0;  // never dereferenced
                    }
                    slot[i] = (uint32_t)entryPage[i] * pageSlots + inPage[i];
                }
                const uint32_t st = base + iStage * S::STAGE;
                if (PAGED) {
                    const uint32_t bar = bars + 8 * iStage;
                    const int tiles = min((iEnd - iTok + kTile - 1) / kTile, MT);
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(tiles * (2 * kTile * ROW + 2 * kTile * 4)) : "memory");
                    __syncwarp();
                    if (lane < 4 * tiles) bulk(st + dstOff, pool + (size_t)slot[0] * perSlot, kTile * perSlot, bar, pol);
                } else {
#pragma unroll
                    for (int i = 0; i < PL; i++) {
                        const bool live = iTok + lane + 32 * i < iEnd;
                        if (!live) slot[i] = 0;
                        copy4(st + 2 * kStep * ROW + (lane + 32 * i) * 4, p.kParams + slot[i], live ? 4 : 0);
                        copy4(st + 2 * kStep * ROW + kStep * 4 + (lane + 32 * i) * 4, p.vParams + slot[i], live ? 4 : 0);
                    }
                    constexpr int PER = ROW / 16;  // 16-byte pieces of a token
#pragma unroll
                    for (int i = 0; i < PER * PL; i++) {
                        const int token = (lane + 32 * i) / PER, piece = (lane + 32 * i) % PER;
                        const uint32_t src = __shfl_sync(0xffffffffu, slot[i / PER], token & 31);
                        const uint32_t bytes = iTok + token < iEnd ? 16u : 0u;
                        const uint32_t dst = st + (lane + 32 * i) * 16;
                        copy16(dst, p.kCodes + (size_t)src * ROW + piece * 16, bytes, pol);
                        copy16(dst + kStep * ROW, p.vCodes + (size_t)src * ROW + piece * 16, bytes, pol);
                    }
                }
                iTok += kStep;
                look_ahead();
            }
            if (++iStage == S::STAGES) iStage = 0;
            if (!PAGED) asm volatile("cp.async.commit_group;" ::: "memory");
        };
        look_ahead();
        {  // the first pair's queries set out with the page entries instead of behind them
            const int kvh = cUnit / p.blocks, block = cUnit - kvh * p.blocks;
            const int head0 = kvh * p.group + block * S::HEADS, heads = min(p.group - block * S::HEADS, S::HEADS);
            constexpr int LINES = S::HEADS * D * 2 / 128;
            uint32_t unused;
            if (lane < LINES && lane * 64 < heads * D)
                asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(unused) : "l"(p.q + ((size_t)cb * p.numHeads + head0) * D + lane * 64));
        }
#pragma unroll 1
        for (int s = 0; s < S::STAGES - 1; s++) issue();

        // rows of a tile: row r is token rowTok(r): neighbouring rows differ in the lowest bit of their token, so the K loads of eight lanes
        // cover all banks, and even rows' tokens lie in both halves of 128 bytes (the V loads of D = 128 take two turns all the same)
        auto rowTok = [](int r) { return r < 4 ? r : r ^ 1; };
        const int tokG = rowTok(g);
        const uint32_t kOff = tokG * ROW + t * (ROW / 4);
        const uint32_t vOffA = rowTok(2 * t) * ROW + g * (ROW / 8), vOffB = rowTok(2 * t + 1) * ROW + g * (ROW / 8);

        int stage = 0;
        uint32_t parity = 0;  // of the stages' barriers
        bool okay = true;
        long long cur = lo;
        while (cur < hi) {
            long long r = cur - (long long)cUnit * T;
            if (r >= T) { cUnit++; cb = 0; r -= T; }
            while (ts[cb + 1] <= r) cb++;
            const int b = cb;
            const long long s0 = ts[b] + kStart, s1 = ts[b + 1], stop = hi - (long long)cUnit * T, e = s1 < stop ? s1 : stop;
            if (e <= s0) {
                cur = (long long)cUnit * T + e;
                continue;
            }
            const int ctx = ctx_of(b);
            const int tok0 = r > s0 ? (int)((r - s0) * kTile) : 0;
            const long long endTok = (e - s0) * kTile;
            const int tokEnd = (int)(endTok < ctx ? endTok : ctx);
            const int kvh = cUnit / p.blocks, block = cUnit % p.blocks;
            const int head0 = kvh * p.group + block * S::HEADS, heads = min(p.group - block * S::HEADS, S::HEADS);

            // ---- queries, and their sums for the least terms.
            // QUAD: integers Q = q kUnits / max |q|, in signed bytes.  With L and F as above, 16 q . n = sum (16 Q_even - Q_odd) L + Q_odd F:
            // three and two bytes, FINE four and three.  Column 2h takes byte 1 of head h and column 2h + 1 byte 0, so a lane finds both in its two
            // accumulators; bytes 2 and 3 have products of their own.
            // Otherwise: f16 fragments in the order of the masks, scaled by 2^-qe (and by 1/16 where the codes come 16-fold). ----
            constexpr float kUnits = FINE ? 8300000.f : 32600.f;  // three signed bytes hold 127 * 65793, two 127 * 257
            uint32_t qb[WK][NT][4];  // f16: [word][block of heads][dims (0,4), (2,6), (1,5), (3,7)]; QUAD: [word][0][bytes 1, 0 for L, bytes 2, 3 for L, bytes 1, 0 for F]
            uint32_t* const topF = (uint32_t*)(sTop + (FINE ? threadIdx.x : 0));  // FINE: byte 2 for F, this thread's words (there is no register for them)
            float qScale[NT][J], qSum[NT][J];
            if (QUAD) {
                float x[WK][8], big = 0.f, sum = 0.f;
                const int h = g >> 1;
                const uint16_t* row = p.q + ((size_t)b * p.numHeads + head0 + (h < heads ? h : 0)) * D + t * (D / 4);
#pragma unroll
                for (int w = 0; w < WK; w++) {
                    const uint4 raw = __ldg((const uint4*)(row + 8 * w));
                    unpack16_arith<DT>(raw.x, x[w][0], x[w][1]);
                    unpack16_arith<DT>(raw.y, x[w][2], x[w][3]);
                    unpack16_arith<DT>(raw.z, x[w][4], x[w][5]);
                    unpack16_arith<DT>(raw.w, x[w][6], x[w][7]);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (h >= heads) x[w][i] = 0.f;
                        big = fmaxf(big, fabsf(x[w][i]));
                        sum += x[w][i];
                    }
                }
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                big = fminf(fmaxf(big, 1e-34f), 3.38e38f);  // kUnits / big stays finite; smaller queries than that lose their lower bits
                const float toInt = kUnits / big;
#pragma unroll
                for (int w = 0; w < WK; w++) {
                    uint32_t last = 0;
                    qb[w][0][0] = qb[w][0][1] = qb[w][0][2] = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int even = __float2int_rn(x[w][2 * i] * toInt);
                        int odd = __float2int_rn(x[w][2 * i + 1] * toInt), mix = 16 * even - odd;
                        const uint32_t m0 = limb(mix), m1 = limb(mix), m2 = FINE ? limb(mix) : (uint32_t)mix & 255u, o0 = limb(odd), o1 = FINE ? limb(odd) : (uint32_t)odd & 255u;
                        qb[w][0][0] |= ((g & 1) ? m0 : m1) << (8 * i);
                        qb[w][0][1] |= ((g & 1) ? (FINE ? (uint32_t)mix & 255u : 0u) : m2) << (8 * i);
                        qb[w][0][2] |= ((g & 1) ? o0 : o1) << (8 * i);
                        last |= ((g & 1) ? 0u : (uint32_t)odd & 255u) << (8 * i);
                    }
                    if (FINE) topF[w] = last;
                }
                qScale[0][0] = __shfl_sync(0xffffffffu, big * (p.scaleLog2 / (16.f * kUnits)), 8 * t);
                qSum[0][0] = __shfl_sync(0xffffffffu, sum * p.scaleLog2, 8 * t);
            } else {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float x[WK][8], big = 0.f, sum = 0.f;
                const bool have = nt * 8 + g < heads;
                const uint16_t* row = p.q + ((size_t)b * p.numHeads + head0 + (have ? nt * 8 + g : 0)) * D + t * (D / 4);
#pragma unroll
                for (int w = 0; w < WK; w++) {
                    const uint4 raw = __ldg((const uint4*)(row + 8 * w));
                    unpack16_arith<DT>(raw.x, x[w][0], x[w][1]);
                    unpack16_arith<DT>(raw.y, x[w][2], x[w][3]);
                    unpack16_arith<DT>(raw.z, x[w][4], x[w][5]);
                    unpack16_arith<DT>(raw.w, x[w][6], x[w][7]);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (!have) x[w][i] = 0.f;
                        big = fmaxf(big, fabsf(x[w][i]));
                        sum += x[w][i];
                    }
                }
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                // the largest element to [2^14, 2^15): elements down to 2^-17 of it keep all bits of bf16, with the 1/16 too
                const int qe = big > 0.f ? min(max((int)(__float_as_uint(big) >> 23) - 141, -112), 112) : 0;
                const float down = pow2(-qe), odd = down * 0.0625f;
#pragma unroll
                for (int w = 0; w < WK; w++) {
                    float lo[4], hi[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        hi[i] = x[w][2 * i + 1] * odd;
                        lo[i] = x[w][2 * i] * down;
                    }
                    qb[w][nt][0] = pack16_arith<DT_F16>(lo[0], lo[2]);
                    qb[w][nt][1] = pack16_arith<DT_F16>(lo[1], lo[3]);
                    qb[w][nt][2] = pack16_arith<DT_F16>(hi[0], hi[2]);
                    qb[w][nt][3] = pack16_arith<DT_F16>(hi[1], hi[3]);
                }
                // (2^24 puts the subnormals' unit back: 2^136 at most in the two factors of a score together)
                const float up = pow2(qe) * p.scaleLog2 * 4096.f, scaled = sum * p.scaleLog2;
#pragma unroll
                for (int j = 0; j < 2; j++) {  // this lane's score columns: heads 2t, 2t + 1
                    qScale[nt][j % J] = __shfl_sync(0xffffffffu, up, (2 * t + j) * 4);
                    qSum[nt][j % J] = __shfl_sync(0xffffffffu, scaled, (2 * t + j) * 4);
                }
            }
            }

            // O^T in units of 2^-24 2^ve: word w, pair i: [0], [1] = dim base + 8w + 2i of heads 2t, 2t + 1; [2], [3] = that dim plus 16
            // times the one behind it; base = g * D / 8.  QUAD: [0], [2] of head t ([1], [3]: its weights'
            // second part, or zero)
            float o[WV][4][NT][4];
            float m[NT][J], l[NT][J], z[NT][J];
#pragma unroll
            for (int w = 0; w < WV; w++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) o[w][i][nt][0] = o[w][i][nt][1] = o[w][i][nt][2] = o[w][i][nt][3] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < J; j++) { m[nt][j] = -INFINITY; l[nt][j] = 0.f; z[nt][j] = 0.f; }
            // the weights are relative to m (per head) and to 2^ve: references that move only when the exponentials of a lane add up to more
            // than kMost or its steps to more than 2 MT 2^ve, so most steps neither reduce a maximum over the lanes nor touch the accumulators.  A
            // weight is then at most kMost 2 MT = 8192: inside f16, and float32 sums do not mind.
            int ve = -110;
            float veUp = pow2(-110), veInv = pow2(110);
            float from[NT][J];  // the reference in use: m, or 0 while there is none (nothing but scores of -inf)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) from[nt][0] = from[nt][J - 1] = 0.f;
            constexpr float kMost = 1024.f;
            float limit = -INFINITY;  // -inf until every head of this lane has a reference

            for (int tk = tok0; tk < tokEnd; tk += kStep) {
                if (PAGED) {
                    okay = okay && __all_sync(0xffffffffu, landed(bars + 8 * stage, parity));
                    if (!okay) {  // the range is gone through all the same, so that every arrival is counted; its rows are NaN
                        atomicExch(p.errorFlag, 3);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) l[nt][0] = l[nt][J - 1] = NAN;
                        break;
                    }
                } else {
                    asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
                }
                __syncwarp();
                issue();
                const uint32_t st = base + stage * S::STAGE;
                if (++stage == S::STAGES) {
                    stage = 0;
                    parity ^= 1;
                }
                // ---- scores ----
                float se[MT][NT][4];
                {
                    uint32_t rows[MT][2][4];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const uint32_t at = st + (mt * 16 + i * 8) * ROW + kOff;
                            if (WK == 4) lds128(at, rows[mt][i]);
                            else lds64(at, rows[mt][i]);
                        }
                    }
                    // (tiles innermost: the products of a tile wait for one another)
                    if (QUAD) {
                        int mid[MT][4], top[MT][4];  // 256 and 1 times a sum; 65536 and (FINE) 65536 * 256 times a sum
                        uint32_t qt[4] = {};
                        if (FINE && WK == 4) *(uint4*)qt = *(const uint4*)topF;
                        else if (FINE) *(uint2*)qt = *(const uint2*)topF;
#pragma unroll
                        for (int w = 0; w < WK; w += 2) {
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) {
                                const uint32_t* x = rows[mt][0] + w;
                                const uint32_t* y = rows[mt][1] + w;
                                const uint32_t x0 = x[0] & 0x0F0F0F0Fu, y0 = y[0] & 0x0F0F0F0Fu, x1 = x[1] & 0x0F0F0F0Fu, y1 = y[1] & 0x0F0F0F0Fu;
                                if (w == 0) {
                                    imma0(mid[mt], x0, y0, x1, y1, qb[w][0][0], qb[w + 1][0][0]);
                                    imma0(top[mt], x0, y0, x1, y1, qb[w][0][1], qb[w + 1][0][1]);
                                } else {
                                    imma(mid[mt], x0, y0, x1, y1, qb[w][0][0], qb[w + 1][0][0]);
                                    imma(top[mt], x0, y0, x1, y1, qb[w][0][1], qb[w + 1][0][1]);
                                }
                                imma(mid[mt], x[0], y[0], x[1], y[1], qb[w][0][2], qb[w + 1][0][2]);
                                if (FINE) imma(top[mt], x[0], y[0], x[1], y[1], qt[w], qt[w + 1]);
                            }
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
                            for (int i = 0; i < 4; i += 2)
                                // FINE: at most 64 * 128 * 270 * 257 < 2^30 in the lower half, 2^22 in the upper; otherwise 16 * 32600 * 15 * 128 < 2^30 in all
                                se[mt][0][i] = FINE ? fmaf((float)(top[mt][i + 1] * 256 + top[mt][i]), 65536.f, (float)(mid[mt][i] * 256 + mid[mt][i + 1]))
                                                    : (float)(top[mt][i] * 65536 + mid[mt][i] * 256 + mid[mt][i + 1]);
                        }
                    } else
#pragma unroll
                    for (int w = 0; w < WK; w++) {
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            const uint32_t x = rows[mt][0][w], y = rows[mt][1][w];
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                if (w == 0) mma0(se[mt][nt], x & 0x000F000Fu, y & 0x000F000Fu, (x >> 8) & 0x000F000Fu, (y >> 8) & 0x000F000Fu, qb[w][nt][0], qb[w][nt][1]);
                                else mma(se[mt][nt], x & 0x000F000Fu, y & 0x000F000Fu, (x >> 8) & 0x000F000Fu, (y >> 8) & 0x000F000Fu, qb[w][nt][0], qb[w][nt][1]);
                            }
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            const uint32_t x = rows[mt][0][w], y = rows[mt][1][w];
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                mma(se[mt][nt], x & 0x00F000F0u, y & 0x00F000F0u, (x >> 8) & 0x00F000F0u, (y >> 8) & 0x00F000F0u, qb[w][nt][2], qb[w][nt][3]);
                        }
                    }
                }
                // ---- parameters of this lane's rows: token 8i + tokG ----
                const bool tail = tk + kStep > tokEnd;
                const uint32_t params = st + 2 * kStep * ROW;
                if (PAGED && tail) {  // whatever lies behind the sequence: step and least 0
                    for (int i = lane; i < kStep; i += 32) {
                        if (tk + i < tokEnd) continue;
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(params + i * 4), "r"(0) : "memory");
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(params + kStep * 4 + i * 4), "r"(0) : "memory");
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a later copy into this stage
                    }
                    __syncwarp();
                }
                float ks[2 * MT], kl[2 * MT], vs[2 * MT], vl[2 * MT], vSum = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * MT; i++) {
                    const uint32_t at = params + (8 * i + tokG) * 4;
                    unpack16_arith<DT>(lds32(at), ks[i], kl[i]);
                    unpack16_arith<DT>(lds32(at + kStep * 4), vs[i], vl[i]);
                    if (!QUAD) ks[i] *= 4096.f;  // (the other half of 2^24: see `up`)
                    vSum += vs[i];
                }
                // ---- scores in the log2 domain, relative to the reference, and their exponentials (sums times the query's scale first: that is
                // the size of q . n, while either factor alone may be far from 1) ----
                float x[NT][J][2 * MT], e[NT][J][2 * MT], eSum[NT][J], most = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int j = 0; j < J; j++) {
#pragma unroll
                        for (int i = 0; i < 2 * MT; i++)
                            x[nt][j][i] = fmaf(se[i >> 1][nt][2 * (i & 1) + j] * qScale[nt][j], ks[i], fmaf(kl[i], qSum[nt][j], -from[nt][j]));
                    }
                }
                if (tail) {
                    __syncwarp();  // (keeps this a branch: as selects it would cost every step)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < 2 * MT; i++)
                            if (tk + 8 * i + tokG >= tokEnd) x[nt][0][i] = x[nt][J - 1][i] = -INFINITY;
                }
                auto exponentials = [&]() {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < J; j++) {
                            eSum[nt][j] = 0.f;
#pragma unroll
                            for (int i = 0; i < 2 * MT; i++) {
                                e[nt][j][i] = ex2(x[nt][j][i]);
                                eSum[nt][j] += e[nt][j][i];
                            }
                        }
                };
                exponentials();
#pragma unroll
                for (int nt = 0; nt < NT; nt++) most += J == 2 ? eSum[nt][0] + eSum[nt][J - 1] : eSum[nt][0];
                // (sums in the place of maxima: they run on another pipe than the logic instructions and cover the maxima.  A sum over the heads of a
                // lane that is NaN says nothing of the others: it counts as too large)
                if (__any_sync(0xffffffffu, !(most <= limit) || vSum > 2 * MT * veUp)) {
                    float vTop = 0.f;
#pragma unroll
                    for (int i = 0; i < 2 * MT; i++) vTop = fmaxf(vTop, vs[i]);
                    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(vTop));
                    const int need = max(ve, min((int)((top + 0x7FFFFFu) >> 23) - 127, 110));
                    const float grow = ve - need < -126 ? 0.f : pow2(ve - need);
                    ve = need;
                    veUp = pow2(ve);
                    veInv = pow2(-ve);
                    limit = kMost;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float alpha[J];
#pragma unroll
                        for (int j = 0; j < J; j++) {
                            float mx = x[nt][j][0];
#pragma unroll
                            for (int i = 1; i < 2 * MT; i++) mx = fmaxf(mx, x[nt][j][i]);
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const float mNew = fmaxf(m[nt][j], mx + from[nt][j]);
                            const float a = mNew == -INFINITY ? 1.f : ex2(m[nt][j] - mNew), next = mNew == -INFINITY ? 0.f : mNew;
                            if (mNew == -INFINITY) limit = -INFINITY;  // still no reference: the next score makes one
#pragma unroll
                            for (int i = 0; i < 2 * MT; i++) x[nt][j][i] += from[nt][j] - next;
                            l[nt][j] *= a;
                            z[nt][j] *= a;
                            m[nt][j] = mNew;
                            from[nt][j] = next;
                            alpha[j] = a * grow;
                        }
#pragma unroll
                        for (int w = 0; w < WV; w++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                o[w][i][nt][0] *= alpha[0];
                                o[w][i][nt][2] *= alpha[0];
                                if (!QUAD || SPLIT) {
                                    o[w][i][nt][1] *= alpha[J - 1];
                                    o[w][i][nt][3] *= alpha[J - 1];
                                }
                            }
                    }
                    exponentials();
                }
#pragma unroll
                for (int i = 0; i < 2 * MT; i++) {
                    if (SPLIT) vl[i] = fmaf(8.f, vs[i], vl[i]);
                    vs[i] *= veInv;
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int j = 0; j < J; j++) {
                        l[nt][j] += eSum[nt][j];
#pragma unroll
                        for (int i = 0; i < 2 * MT; i++) {
                            z[nt][j] = fmaf(e[nt][j][i], vl[i], z[nt][j]);
                            se[i >> 1][nt][2 * (i & 1) + j] = e[nt][j][i] * vs[i];
                        }
                    }
                }
                // ---- O^T += V^T P^T ----
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    uint32_t pb[NT][2], pr[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float rest[4] = {0.f, 0.f, 0.f, 0.f};  // what the f16 weights leave
                        if (SPLIT) {
#pragma unroll
                            for (int i = 0; i < 4; i += QUAD ? 2 : 1) rest[i] = se[mt][nt][i] - __half2float(__float2half_rn(se[mt][nt][i]));
                        }
                        pb[nt][0] = transpose8(pack16_arith<DT_F16>(se[mt][nt][0], QUAD ? rest[0] : se[mt][nt][1]));
                        pb[nt][1] = transpose8(pack16_arith<DT_F16>(se[mt][nt][2], QUAD ? rest[2] : se[mt][nt][3]));
                        if (SPLIT && !QUAD) {
                            pr[nt][0] = transpose8(pack16_arith<DT_F16>(rest[0], rest[1]));
                            pr[nt][1] = transpose8(pack16_arith<DT_F16>(rest[2], rest[3]));
                        }
                    }
                    const uint32_t at = st + kStep * ROW + mt * 16 * ROW;
                    uint32_t va[2], vb[2], vc[2], vd[2];  // tokens of rows 2t, 2t + 1, 2t + 8, 2t + 9
                    if (WV == 2) {
                        lds64(at + vOffA, va); lds64(at + vOffB, vb); lds64(at + 8 * ROW + vOffA, vc); lds64(at + 8 * ROW + vOffB, vd);
                    } else {
                        va[0] = lds32(at + vOffA); vb[0] = lds32(at + vOffB); vc[0] = lds32(at + 8 * ROW + vOffA); vd[0] = lds32(at + 8 * ROW + vOffB);
                    }
#pragma unroll
                    for (int w = 0; w < WV; w++) {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const uint32_t x = __byte_perm(va[w], vb[w], half ? 0x7632 : 0x5410), y = __byte_perm(vc[w], vd[w], half ? 0x7632 : 0x5410);
                            const uint32_t x8 = __byte_perm(x, 0, 0x4341), y8 = __byte_perm(y, 0, 0x4341);
                            uint32_t a[2][4];  // dimensions 0 and 1, 2 and 3 of the word: even and whole byte, or even - 8 and odd - 8
                            if (SPLIT) {
                                a[0][0] = low8(x); a[0][1] = high8(x); a[0][2] = low8(y); a[0][3] = high8(y);
                                a[1][0] = low8(x8); a[1][1] = high8(x8); a[1][2] = low8(y8); a[1][3] = high8(y8);
                            } else {
                                a[0][0] = x & 0x000F000Fu; a[0][1] = x & 0x00FF00FFu; a[0][2] = y & 0x000F000Fu; a[0][3] = y & 0x00FF00FFu;
                                a[1][0] = x8 & 0x000F000Fu; a[1][1] = x8; a[1][2] = y8 & 0x000F000Fu; a[1][3] = y8;
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                                for (int i = 0; i < 2; i++) {
                                    mma(o[w][2 * half + i][nt], a[i][0], a[i][1], a[i][2], a[i][3], pb[nt][0], pb[nt][1]);
                                    if (SPLIT && !QUAD) mma(o[w][2 * half + i][nt], a[i][0], a[i][1], a[i][2], a[i][3], pr[nt][0], pr[nt][1]);
                                }
                            }
                        }
                    }
                }
            }

            // ---- end of this warp's part of the pair: the rows themselves, or a partial.  The last partial of a warp goes where its stages
            // were (every copy has landed and been read), an earlier one to the scratch. ----
            const bool begun = r > s0, whole = !begun && e == s1;
            const int which = begun ? 0 : 1;
            cur = (long long)cUnit * T + e;
            const bool near = cur >= hi;
            const long long slot = blockIdx.x * S::WARPS + warp;
            float* const acc = near ? (float*)mine : p.acc + slot * S::HEADS * D;
            float2* const ml = near ? (float2*)(mine + S::HEADS * D * 4) : p.ml + slot * S::HEADS;
            if (!whole) __syncwarp();  // every lane has read the stages
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int j = 0; j < J; j++) {
                    float sum = l[nt][j], least = z[nt][j];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) {
                        sum += __shfl_xor_sync(0xffffffffu, sum, off);
                        least += __shfl_xor_sync(0xffffffffu, least, off);
                    }
                    const int h = QUAD ? t : nt * 8 + 2 * t + j;
                    if (h >= heads) continue;
                    float x[8 * WV];
#pragma unroll
                    for (int w = 0; w < WV; w++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float even = o[w][i][nt][j], both = o[w][i][nt][2 + j];
                            if (QUAD && SPLIT) {
                                even += o[w][i][nt][1];
                                both += o[w][i][nt][3];
                            }
                            x[8 * w + 2 * i] = fmaf(SPLIT ? even : even * 16777216.f, veUp, least);
                            x[8 * w + 2 * i + 1] = fmaf(SPLIT ? both : (both - even) * 1048576.f, veUp, least);
                        }
                    if (whole) {
                        uint16_t* dst = p.out + ((size_t)b * p.numHeads + head0 + h) * D + g * (D / 8);
#pragma unroll
                        for (int w = 0; w < WV; w++) {
                            uint4 v;
                            v.x = pack16_arith<DT>(x[8 * w] / sum, x[8 * w + 1] / sum);
                            v.y = pack16_arith<DT>(x[8 * w + 2] / sum, x[8 * w + 3] / sum);
                            v.z = pack16_arith<DT>(x[8 * w + 4] / sum, x[8 * w + 5] / sum);
                            v.w = pack16_arith<DT>(x[8 * w + 6] / sum, x[8 * w + 7] / sum);
                            *(uint4*)(dst + 8 * w) = v;
                        }
                    } else {
                        float* dst = acc + h * D + g * (D / 8);
#pragma unroll
                        for (int i = 0; i < 2 * WV; i++) *(float4*)(dst + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                        if (g == 0) ml[h] = make_float2(m[nt][j], sum);
                    }
                }
            }
            if (!whole && lane == 0) {
                const int at = 2 * warp + which;
                const long long gs = (long long)cUnit * T + s0, ge = (long long)cUnit * T + s1;
                sSeg[at] = cUnit * p.batch + b;
                sB[at] = b;
                sUnit[at] = cUnit;
                sWhere[at] = gs >= clo && ge <= chi ? 2 : gs < clo ? 0 : 1;
                if (near) sNear[warp] = which;
            }
        }
        if (!PAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // ---- pairs that several warps of this CTA share: joined here, a warp per (pair, head), D / 32 dimensions a lane; written, or left as
    // the CTA's partial in the scratch.  (From here on every instruction runs once per launch and comes cold from the instruction
    // cache: short code before fast code.) ----
    __syncthreads();
    const long long ctaSlots = (long long)gridDim.x * S::WARPS;  // behind the warps' slots, two per CTA
    constexpr int E = D / 32;
    {
        const int seg = sSeg[lane];
        const uint32_t have = __ballot_sync(0xffffffffu, seg >= 0);
        const uint32_t below = have & ((1u << lane) - 1);
        const int before = __shfl_sync(0xffffffffu, seg, below ? 31 - __clz(below) : lane);
        const uint32_t starts = __ballot_sync(0xffffffffu, seg >= 0 && (!below || before != seg));
        if (warp == 0 && (starts >> lane & 1) && sWhere[lane] < 2) sShared[sWhere[lane]] = lane;
        for (int item = warp; item < __popc(starts) * S::HEADS; item += S::WARPS) {
            const int h = item % S::HEADS;
            uint32_t left = starts;
            for (int i = item / S::HEADS; i > 0; i--) left &= left - 1;
            const int e0 = __ffs(left) - 1;
            left &= left - 1;
            const uint32_t members = have & (left ? (1u << (__ffs(left) - 1)) - 1 : 0xffffffffu) & ~((1u << e0) - 1);
            const int unit = sUnit[e0], where = sWhere[e0];
            const int kvh = unit / p.blocks, block = unit - kvh * p.blocks, head = block * S::HEADS + h;
            if (head >= p.group) continue;
            // (a warp has at most one entry in a pair: entry e is of warp e / 2; lane i looks at warp w0 + i)
            const int w0 = e0 >> 1, n = ((31 - __clz(members)) >> 1) - w0 + 1, w = w0 + lane;
            const uint32_t bits = lane < n ? (members >> (2 * w)) & 3 : 0;
            float2 ml = make_float2(-INFINITY, 0.f);
            const float* at = p.acc;  // (where there is no partial: not read)
            if (bits) {
                const unsigned char* own = smemRaw + w * (S::STAGES * S::STAGE);
                const long long far = (long long)blockIdx.x * S::WARPS + w;
                const bool near = sNear[w] == (bits & 1 ? 0 : 1);
                ml = near ? ((const float2*)(own + S::HEADS * D * 4))[h] : p.ml[far * S::HEADS + h];
                at = (near ? (const float*)own : p.acc + far * (S::HEADS * D)) + h * D;
            }
            float M = ml.x;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
            const float k = weight(ml, M);
            float den = ml.y * k, num[E] = {};
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) den += __shfl_xor_sync(0xffffffffu, den, off);
            for (int i0 = 0; i0 < n; i0 += 4) {  // four parts on their way at a time: some lie in the scratch
                float x[4][E], wt[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int i = i0 + u;
                    wt[u] = __shfl_sync(0xffffffffu, k, i & 31);
                    const float* from = (const float*)__shfl_sync(0xffffffffu, (unsigned long long)at, i & 31) + lane * E;
#pragma unroll
                    for (int d = 0; d < E; d++) x[u][d] = 0.f;
                    if (i < n && ((members >> (2 * (w0 + i))) & 3)) {  // uniform
                        if (E == 4) *(float4*)x[u] = *(const float4*)from;
                        else *(float2*)x[u] = *(const float2*)from;
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int d = 0; d < E; d++) num[d] = fmaf(x[u][d], wt[u], num[d]);
            }
            const long long slot = (ctaSlots + 2ll * blockIdx.x + where) * S::HEADS + h;
            if (where == 2) {
                uint32_t* dst = (uint32_t*)(p.out + ((size_t)sB[e0] * p.numHeads + kvh * p.group + head) * D + lane * E);
#pragma unroll
                for (int d = 0; d < E; d += 2) dst[d / 2] = pack16_arith<DT>(num[d] / den, num[d + 1] / den);
            } else {
#pragma unroll
                for (int d = 0; d < E; d += 2) *(float2*)(p.acc + slot * D + lane * E + d) = make_float2(num[d], num[d + 1]);
                if (lane == 0) p.ml[slot] = make_float2(M, den);
            }
        }
    }
    __syncthreads();
    if (sShared[0] < 0 && sShared[1] < 0) return;  // uniform over the CTA
    // ---- pairs that several CTAs share ----
    if (threadIdx.x < 2) {
        const int e = sShared[threadIdx.x];
        int go = 0;
        if (e >= 0) {
            const long long at = (long long)sUnit[e] * T;
            const long long begin = at + ts[sB[e]], end = at + ts[sB[e] + 1];
            const int first = owned ? owner(begin) : split.holding(begin + kStart), owners = (owned ? owner(end) : split.holding(end - 1) + 1) - first;
            int* const counter = p.counters + sSeg[e];
            sFirst[threadIdx.x] = first;
            sOwners[threadIdx.x] = owners;
            __threadfence();  // the CTA's partial (ordered before this thread by the barrier) before its arrival
            const int came = atomicAdd(counter, 1);
            if (p.together) {
                go = 1;
                int seen;
                for (unsigned spins = 0;; spins++) {
                    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
                    if (seen >= owners) break;
                    if (spins > (1u << 21)) {  // about a second: an owner never arrived
                        atomicExch(p.errorFlag, 4);
                        go = 0;
                        break;
                    }
                    __nanosleep(40);
                }
            } else {
                go = came == owners - 1;
                if (go) *counter = 0;  // nobody else comes in this launch
            }
            __threadfence();
        }
        sGo[threadIdx.x] = go;
    }
    __syncthreads();
    float* const sums = (float*)smemRaw;  // [warp][32] sums, then maximum and sum of weights
    for (int s = 0; s < 2; s++) {
        if (!sGo[s]) continue;
        const int e = sShared[s], n = sOwners[s], unit = sUnit[e], kvh = unit / p.blocks, block = unit - kvh * p.blocks;
        const int heads = min(p.group - block * S::HEADS, S::HEADS);
        // this CTA's slices (of 32 dimensions): rank, rank + of, ...; a warp per slice, or several that take every `ways`-th owner each
        const int rank = p.together ? blockIdx.x - sFirst[s] : 0, of = p.together ? n : 1;
        const int mine = rank < heads * E ? (heads * E - rank + of - 1) / of : 0, cols = min(mine, S::WARPS), ways = cols ? S::WARPS / cols : 1;
        // slot of owner i: the pair begins inside the first one's range and before the others'
        const long long slot0 = ctaSlots + 2ll * sFirst[s];
        for (int c0 = 0; c0 < mine; c0 += cols) {
            const int way = warp / cols, c = c0 + warp - way * cols, slice = rank + c * of, h = slice / E;
            const bool on = way < ways && c < mine;
            float M = -INFINITY, den = 0.f, num = 0.f;
            if (on) {
                for (int i0 = way; i0 < n; i0 += 8 * ways) {
                    float2 ml[8];
                    float a[8], Mn = M;
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const int i = i0 + u * ways;
                        const long long row = (slot0 + 2 * i + (i == 0 ? 1 : 0)) * S::HEADS + h;
                        ml[u] = make_float2(-INFINITY, 0.f);
                        a[u] = 0.f;
                        if (i < n) {
                            ml[u] = __ldcg(p.ml + row);
                            a[u] = __ldcg(p.acc + row * D + (slice % E) * 32 + lane);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 8; u++) Mn = fmaxf(Mn, ml[u].x);
                    const float old = weight(make_float2(M, den), Mn);
                    den *= old;
                    num *= old;
                    M = Mn;
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const float w = weight(ml[u], M);
                        den = fmaf(ml[u].y, w, den);
                        num = fmaf(a[u], w, num);
                    }
                }
            }
            if (ways > 1) {
                float* const mineAt = sums + warp * 34;
                __syncthreads();
                mineAt[lane] = num;
                if (lane == 0) {
                    mineAt[32] = M;
                    mineAt[33] = den;
                }
                __syncthreads();
                if (on && way == 0) {
                    float all = M;
                    for (int w = 1; w < ways; w++) all = fmaxf(all, mineAt[w * cols * 34 + 32]);
                    float total = 0.f, sum = 0.f;
                    for (int w = 0; w < ways; w++) {
                        const float* other = mineAt + w * cols * 34;
                        const float k = weight(make_float2(other[32], other[33]), all);
                        total = fmaf(other[33], k, total);
                        sum = fmaf(other[lane], k, sum);
                    }
                    den = total;
                    num = sum;
                }
            }
            if (on && way == 0)
                Storage<DT>::store(p.out, ((size_t)sB[e] * p.numHeads + kvh * p.group + block * S::HEADS + h) * D + (slice % E) * 32 + lane, num / den);
        }
    }
    if (!p.together) return;
    __syncthreads();
    if (threadIdx.x < 2 && sShared[threadIdx.x] >= 0) {  // the last owner to leave a pair returns its counter to zero
        int* const counter = p.counters + sSeg[sShared[threadIdx.x]];
        if (atomicAdd(counter, 1) == 2 * sOwners[threadIdx.x] - 1) *counter = 0;
    }
}

template <int DT, typename S>
static int launch(Context* ctx, Params& p, CUDAStatus* status) {
    static_assert(2 * S::STEP <= INT_MAX - kMostTokens, "places behind the context are counted in 31 bits");
    const char* what = "paged decode attention (4 bits)";
    const unsigned grid = (unsigned)ctx->smCount;
    p.blocks = (p.group + S::HEADS - 1) / S::HEADS;
    p.units = p.kvHeads * p.blocks;
    const size_t slots = (size_t)grid * (S::WARPS + 2);
    const size_t accBytes = slots * S::HEADS * S::D * 4, mlBytes = slots * S::HEADS * 8;
    const size_t prefixBytes = p.batch > kPrefixSmem ? ((size_t)p.batch + 3) * 4 : 0;
    const size_t counterBytes = (size_t)p.units * p.batch * 4;
    Scratch ws;
    int rc = call_scratch(ctx, accBytes + mlBytes + prefixBytes, counterBytes, &ws, status);
    if (rc != 0) return rc;
    p.acc = (float*)ws.base;
    p.ml = (float2*)(ws.base + accBytes);
    p.counters = ws.counters;
    if (ws.clearCounters && cudaMemsetAsync(ws.counters, 0, counterBytes, ctx->stream) != cudaSuccess)
        return fail(status, -7, "%s: clearing the arrival counters failed", what);
    if (prefixBytes) {
        int* prefix = (int*)(ws.base + accBytes + mlBytes);
        prefix_kernel<<<1, 1024, 0, ctx->stream>>>(p, S::START, prefix);
        rc = check_launch(ctx, status, "paged decode attention (4 bits): prefix");
        if (rc != 0) return rc;
        p.tileStart = prefix;
    }
    // PUTER_DECODE_NO_COOPERATIVE (any value) forces the plain launch: the path a refused cooperative launch takes, reachable for tests
    const bool cooperative = getenv("PUTER_DECODE_NO_COOPERATIVE") == nullptr;
    const bool paged = p.pageSize % kTile == 0;
    const auto kernel = paged ? decode_kernel<DT, S, true> : decode_kernel<DT, S, false>;
    if (paged) allow_smem<decode_kernel<DT, S, true>>(ctx->device, S::SMEM);
    else allow_smem<decode_kernel<DT, S, false>>(ctx->device, S::SMEM);
    p.together = 1;
    void* args[] = {&p};
    if (!cooperative || cudaLaunchCooperativeKernel((const void*)kernel, dim3(grid), dim3(S::WARPS * 32), args, S::SMEM, ctx->stream) != cudaSuccess) {
        cudaGetLastError();
        p.together = 0;
        kernel<<<grid, S::WARPS * 32, S::SMEM, ctx->stream>>>(p);
    }
    return check_launch(ctx, status, what);
}

}  // namespace q4d

}  // namespace puter

using namespace puter;

extern "C" int cuda_dispatch_paged_decode_attention_q4(CUDADeviceRef contextRef, int elementDType, CUDABufferRef queryRef,
                                                       CUDABufferRef kCodesRef, CUDABufferRef kParamsRef, CUDABufferRef vCodesRef,
                                                       CUDABufferRef vParamsRef, CUDABufferRef pageTableRef, CUDABufferRef ctxLensRef,
                                                       CUDABufferRef outRef, CUDABufferRef errorFlagRef, uint32_t batch,
                                                       uint32_t maxPagesPerSeq, uint32_t pageCount, uint32_t pageSize, uint32_t numHeads,
                                                       uint32_t kvHeads, uint32_t headDim, uint64_t completionToken, CUDAStatus* status) {
    (void)completionToken;
    PUTER_ENTER(ctx);
    const char* what = "paged decode attention (4 bits)";
    if (batch == 0 || numHeads == 0) return ok(status);
    if (kvHeads == 0) kvHeads = numHeads;
    if (numHeads % kvHeads != 0) return fail(status, -2, "%s: %u heads are not a multiple of %u KV heads", what, numHeads, kvHeads);
    if ((elementDType != DT_F16 && elementDType != DT_BF16) || (headDim != 64 && headDim != 128))
        return fail(status, -6, "%s: supported are bf16 / f16 queries and head dimensions 64 and 128 (got dtype %d, head dimension %u)", what,
                    elementDType, headDim);
    if (pageSize == 0 || pageCount == 0 || maxPagesPerSeq == 0) return fail(status, -2, "%s: empty page geometry", what);
    if ((size_t)batch * numHeads > 0x7FFFFFFFull) return fail(status, -2, "%s: %u sequences of %u heads exceed 31 bits", what, batch, numHeads);
    const size_t slots = pool_vectors(pageCount, pageSize, kvHeads);
    if (slots > 0xFFFFFFFFull || (size_t)maxPagesPerSeq * pageSize > (size_t)q4d::kMostTokens || batch > 0x7FFFFFFEu)
        return fail(status, -2, "%s: a pool of %zu vectors or a context of %zu tokens exceeds the index range", what, slots,
                    (size_t)maxPagesPerSeq * pageSize);
    if ((size_t)batch * ((size_t)maxPagesPerSeq * pageSize / q4d::kTile + 16) > 0x7FFFFFFFull)  // tiles are counted in 31 bits
        return fail(status, -2, "%s: %u contexts of up to %zu tokens exceed the index range", what, batch, (size_t)maxPagesPerSeq * pageSize);
    PUTER_REQUIRE(queryRef, "query", (size_t)batch * numHeads * headDim * 2);
    PUTER_REQUIRE(outRef, "out", (size_t)batch * numHeads * headDim * 2);
    PUTER_REQUIRE(kCodesRef, "kCodes", slots * (headDim / 2));
    PUTER_REQUIRE(vCodesRef, "vCodes", slots * (headDim / 2));
    PUTER_REQUIRE(kParamsRef, "kParams", slots * 4);
    PUTER_REQUIRE(vParamsRef, "vParams", slots * 4);
    PUTER_REQUIRE(pageTableRef, "pageTable", (size_t)batch * maxPagesPerSeq * 4);
    PUTER_REQUIRE(ctxLensRef, "ctxLens", (size_t)batch * 4);
    int* flag = ctx->errorFlag;
    if (errorFlagRef) {
        PUTER_REQUIRE(errorFlagRef, "errorFlag", 4);
        flag = (int*)dev_ptr(errorFlagRef);
    }
    if ((((uintptr_t)dev_ptr(kCodesRef) | (uintptr_t)dev_ptr(vCodesRef) | (uintptr_t)dev_ptr(kParamsRef) | (uintptr_t)dev_ptr(vParamsRef) |
          (uintptr_t)dev_ptr(queryRef) | (uintptr_t)dev_ptr(outRef)) & 15u) != 0)
        return fail(status, -2, "%s: pools, query and output must be 16-byte aligned", what);
    if ((((uintptr_t)dev_ptr(pageTableRef) | (uintptr_t)dev_ptr(ctxLensRef) | (uintptr_t)flag) & 3u) != 0)
        return fail(status, -2, "%s: pageTable, ctxLens and errorFlag must be 4-byte aligned", what);
    q4d::Params p{};
    p.q = (const uint16_t*)dev_ptr(queryRef);
    p.kCodes = (const uint8_t*)dev_ptr(kCodesRef);
    p.vCodes = (const uint8_t*)dev_ptr(vCodesRef);
    p.kParams = (const uint32_t*)dev_ptr(kParamsRef);
    p.vParams = (const uint32_t*)dev_ptr(vParamsRef);
    p.table = (const int32_t*)dev_ptr(pageTableRef);
    p.ctxLens = (const int32_t*)dev_ptr(ctxLensRef);
    p.out = (uint16_t*)dev_ptr(outRef);
    p.errorFlag = flag;
    p.batch = (int)batch; p.maxPages = (int)maxPagesPerSeq; p.pageCount = (int)pageCount; p.pageSize = (int)pageSize;
    p.numHeads = (int)numHeads; p.kvHeads = (int)kvHeads; p.group = (int)(numHeads / kvHeads);
    p.scaleLog2 = (float)(1.4426950408889634 / sqrt((double)headDim));
    p.pageShift = -1;
    for (int s = 0; s < 31; s++)
        if (pageSize == (1u << s)) p.pageShift = s;
    // query heads per KV head: up to 4, up to 8, more (in blocks of 16)
#define DECODE(DT, D)                                                                       \
    (p.group <= 4   ? q4d::launch<DT, q4d::Shape<D, 0, 16, 2>>(ctx, p, status)               \
     : p.group <= 8 ? q4d::launch<DT, q4d::Shape<D, 1, 8, 4>>(ctx, p, status)               \
                    : q4d::launch<DT, q4d::Shape<D, 2, 8, 2>>(ctx, p, status))
    if (headDim == 128) return elementDType == DT_BF16 ? DECODE(DT_BF16, 128) : DECODE(DT_F16, 128);
    return elementDType == DT_BF16 ? DECODE(DT_BF16, 64) : DECODE(DT_F16, 64);
#undef DECODE
}
