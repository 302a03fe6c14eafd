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
//   * A code becomes an f16 operand with ONE instruction per two elements and no arithmetic: the four bits, masked in place, ARE
//     the subnormal f16 n * 2^-24 (bits 0-3) or 16 n * 2^-24 (bits 4-7), exact.  The factors are powers of two and are put back
//     into the scores and the output.  Bits 4-7 go to products and accumulators of their own.
//   * K: a lane's 16-byte (D = 128) piece of a token holds its A fragments for all of the contraction, since the order of the contraction
//     is free: the query fragments are loaded in the order in which the masks deliver the elements.  V: two byte permutes pair the
//     words of two tokens, then the same masks.
//   * Queries enter as f16, scaled by a power of two per (sequence, head) so that a bf16 query of any size fits; the weights
//     p_t * step_t enter as f16 (half a step of 2^-11, an eighth of what the 16-bit output keeps), relative to a running power of two above
//     the largest step, which joins the running maximum of the softmax in rescaling the accumulator.
// Sums, maxima and accumulators are float32.
//
// Work: the tiles of 16 tokens of all (KV head, sequence) pairs in one list, cut into equal contiguous ranges, one per CTA, and each
// CTA's range into equal ranges, one per warp.  A warp owns its pipeline (cp.async into its own stages, copies running ahead across
// sequence boundaries; page entries one step further ahead), so there is no block-wide barrier before the end.  A pair that lies inside a
// warp's range is written by the warp.  Otherwise the warps of a CTA put their partial (maximum, sum, accumulator) together, and
// the CTA that arrives last at a pair joins those of all CTAs, in their order: the same bits whoever is last.
#include <math.h>

#include "common.cuh"

namespace puter {

namespace q4d {

constexpr int kTile = 16;             // tokens per tile
constexpr int kStep = 32;             // tokens per step of a warp
constexpr int kPrefixSmem = 2048;     // sequences whose tile prefix sums fit shared memory
constexpr int kWarpTiles = 2;         // tiles that a warp gets at least before another CTA takes part

struct Params {
    const uint16_t* q;
    const uint8_t *kCodes, *vCodes;
    const uint32_t *kParams, *vParams;
    const int32_t *table, *ctxLens;
    uint16_t* out;
    int* errorFlag;
    const int* tileStart;  // [batch + 1] exclusive prefix of tiles, or nullptr: scanned in shared memory
    float* acc;            // partial accumulators [slots, heads of a block, D]: two slots per warp, then two per CTA
    float2* ml;            // (maximum in the log2 domain, sum) [slots, heads of a block]
    int* counters;         // arrivals per (unit, sequence): zero on entry and on exit
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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// exclusive prefix sum of tiles per sequence: out[0 .. batch].  Every thread of the block calls it.
__device__ void block_prefix(const Params& p, int* out) {
    __shared__ int sums[32];
    __shared__ int carry;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int base = 0; base < p.batch; base += blockDim.x) {
        const int b = base + threadIdx.x;
        const int tiles = b < p.batch ? (int)(((long long)seq_ctx(p, b) + kTile - 1) / kTile) : 0;
        int incl = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += n;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < warp; w++) before += sums[w];
        if (b < p.batch) out[b] = before + incl - tiles;
        __syncthreads();
        if (threadIdx.x == blockDim.x - 1) carry = before + incl;
        __syncthreads();
    }
    if (threadIdx.x == 0) out[p.batch] = carry;
    __syncthreads();
}
__global__ void __launch_bounds__(1024) prefix_kernel(Params p, int* out) { block_prefix(p, out); }

// the part that holds tile g when `total` tiles are cut into `parts` ranges [i * total / parts, (i + 1) * total / parts)
__device__ __forceinline__ int part_of(long long g, long long total, long long parts) { return (int)(((g + 1) * parts - 1) / total); }

// NT: blocks of eight query heads that a warp serves with one pass over the codes
template <int DT, int D, int NT>
struct Shape {
    static constexpr int WARPS = NT == 1 ? 16 : 8;  // 8: the accumulators of 16 heads need more than 128 registers a thread
    static constexpr int ROW = D / 2;               // bytes of a token's codes
    static constexpr int STAGE = 2 * kStep * ROW + 2 * kStep * 4;
    static constexpr int STAGES = (NT == 1 ? 3 : 6) * (D == 128 ? 1 : 2);
    static constexpr int SMEM = WARPS * STAGES * STAGE;
    static constexpr int HEADS = 8 * NT;
};

// Columns (head, four dimensions) of a block of heads, dealt to the threads of the CTA: joins the partials that `slot_of` names for
// i in [0, n), in order, and hands on (maximum, sum, four sums).  The loads of eight partials are issued together.
template <int D, typename SlotOf, typename Put>
__device__ __forceinline__ void join(const Params& p, int heads, int stride, int n, SlotOf slot_of, Put put) {
    for (int col = threadIdx.x; col < heads * (D / 4); col += blockDim.x) {
        const int h = col / (D / 4), d = (col % (D / 4)) * 4;
        float M = -INFINITY, den = 0.f;
        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < n; i0 += 8) {
            float2 ml[8];
            float4 a[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const long long slot = i0 + i < n ? slot_of(i0 + i) : -1;
                if (slot >= 0) {
                    ml[i] = __ldcg(p.ml + slot * stride + h);
                    a[i] = __ldcg((const float4*)(p.acc + (slot * stride + h) * D + d));
                } else {
                    ml[i] = make_float2(-INFINITY, 0.f);
                    a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            float Mn = M;
#pragma unroll
            for (int i = 0; i < 8; i++) Mn = fmaxf(Mn, ml[i].x);
            const float old = M == -INFINITY ? 0.f : exp2f(M - Mn);
            den *= old;
            num.x *= old; num.y *= old; num.z *= old; num.w *= old;
            M = Mn;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // (a part without a finite score has sum 0, or NaN, which stays NaN)
                const float w = ml[i].x == -INFINITY ? (ml[i].y == 0.f ? 0.f : ml[i].y) : exp2f(ml[i].x - M);
                den += ml[i].y * w;
                num.x += a[i].x * w; num.y += a[i].y * w; num.z += a[i].z * w; num.w += a[i].w * w;
            }
        }
        put(h, d, M, den, num);
    }
}

template <int DT>
__device__ __forceinline__ void store4(uint16_t* dst, float den, float4 num) {
    *(uint2*)dst = make_uint2(pack16_arith<DT>(num.x / den, num.y / den), pack16_arith<DT>(num.z / den, num.w / den));
}

template <int DT, int D, int NT>
__global__ void __launch_bounds__(Shape<DT, D, NT>::WARPS * 32, 1) decode_kernel(Params p) {
    using S = Shape<DT, D, NT>;
    constexpr int WK = D / 32;   // words of a token's K codes in a lane
    constexpr int WV = D / 64;   // words of a token's V codes in a lane
    constexpr int ROW = S::ROW;
    extern __shared__ __align__(128) unsigned char smemRaw[];
    __shared__ int sStart[kPrefixSmem + 1];
    __shared__ int sSeg[2 * S::WARPS];
    __shared__ int sLast[2];
    const int* ts = p.tileStart;
    if (!ts) {
        block_prefix(p, sStart);
        ts = sStart;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long long T = ts[p.batch], total = T * p.units;
    if (total == 0) return;
    // CTAs that take part: every one of them has work
    const long long most = (total + S::WARPS * kWarpTiles - 1) / (S::WARPS * kWarpTiles);
    const int parts = most < (long long)gridDim.x ? (int)most : (int)gridDim.x;
    if ((int)blockIdx.x >= parts) return;
    const long long clo = blockIdx.x * total / parts, chi = (blockIdx.x + 1) * total / parts;
    const long long lo = clo + warp * (chi - clo) / S::WARPS, hi = clo + (warp + 1) * (chi - clo) / S::WARPS;
    if (lane < 2) sSeg[2 * warp + lane] = -1;
    __syncwarp();

    const uint32_t base = smem_u32(smemRaw) + warp * (S::STAGES * S::STAGE);
    uint64_t pol;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));

    if (lo < hi) {
        // ---- the copies' own place in the range, ahead of the computation's ----
        long long iNext = lo;     // first tile behind the segment that is being copied
        int iUnit = (int)(lo / T), ib = 0, iTok = 0, iEnd = 0, iStage = 0;
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
        int entryPage = 0;        // page of this lane's token of the step to be copied next
        uint32_t inPage = 0;      // and its place in that page
        // Moves to the next step and starts fetching its page entries.
        auto look_ahead = [&]() {
            if (iTok >= iEnd) {
                if (iNext >= hi) return;
                long long r = iNext - (long long)iUnit * T;
                if (r >= T) { iUnit++; ib = 0; r -= T; }
                while (ts[ib + 1] <= r) ib++;
                const long long s0 = ts[ib], s1 = ts[ib + 1], stop = hi - (long long)iUnit * T, e = s1 < stop ? s1 : stop;
                const int ctx = seq_ctx(p, ib);
                const long long end = (e - s0) * kTile;
                iTok = (int)((r - s0) * kTile);
                iEnd = (int)(end < ctx ? end : ctx);
                iNext = (long long)iUnit * T + e;
            }
            const int tok = iTok + lane;
            const int entry = p.pageShift >= 0 ? tok >> p.pageShift : tok / p.pageSize;
            inPage = (uint32_t)(tok - entry * p.pageSize);
            entryPage = tok < iEnd ? __ldg(p.table + (size_t)ib * p.maxPages + entry) : 0;
        };
        // Copies the step that look_ahead found (tokens past its end are zero-filled: step and least 0, codes 0) and looks for the next.
        auto issue = [&]() {
            if (iTok < iEnd) {
                const bool live = iTok + lane < iEnd;
                int page = entryPage;
                if (page < 0 || page >= p.pageCount) {
                    atomicExch(p.errorFlag, 1);
                    page = 0;  // never dereferenced
                }
                const uint32_t kvh = (uint32_t)iUnit / (uint32_t)p.blocks;
                const uint32_t slot = live ? ((uint32_t)page * (uint32_t)p.kvHeads + kvh) * (uint32_t)p.pageSize + inPage : 0u;
                const uint32_t st = base + iStage * S::STAGE;
                copy4(st + 2 * kStep * ROW + lane * 4, p.kParams + slot, live ? 4 : 0);
                copy4(st + 2 * kStep * ROW + kStep * 4 + lane * 4, p.vParams + slot, live ? 4 : 0);
                constexpr int PER = ROW / 16;  // 16-byte pieces of a token
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int token = (lane + 32 * i) / PER, piece = (lane + 32 * i) % PER;
                    const uint32_t src = __shfl_sync(0xffffffffu, slot, token);
                    const uint32_t bytes = iTok + token < iEnd ? 16u : 0u;
                    // pieces 2, 3 before 0, 1 in every second pair of tokens: four tokens' 32-byte halves then lie in different banks
                    const uint32_t dst = st + token * ROW + ((piece ^ (PER == 4 ? (token & 2) : 0)) * 16);
                    copy16(dst, p.kCodes + (size_t)src * ROW + piece * 16, bytes, pol);
                    copy16(dst + kStep * ROW, p.vCodes + (size_t)src * ROW + piece * 16, bytes, pol);
                }
                iTok += kStep;
                look_ahead();
            }
            if (++iStage == S::STAGES) iStage = 0;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        look_ahead();
#pragma unroll
        for (int s = 0; s < S::STAGES - 1; s++) issue();

        // rows of a tile: row r is token rowTok(r); pairs of rows differ in the lowest bit and even rows cover all four classes mod 4, so that
        // neither the K nor the V loads meet in a bank
        auto rowTok = [](int r) { return r < 4 ? r : r ^ 1; };
        const int tokG = rowTok(g), tokA = rowTok(2 * t), tokB = rowTok(2 * t + 1);
        const uint32_t kOff = ROW == 64 ? tokG * 64 + ((t ^ (tokG & 2)) * 16) : tokG * 32 + t * 8;
        auto v_off = [&](int token) { return ROW == 64 ? token * 64 + ((((uint32_t)g >> 1) ^ (token & 2)) * 16) + (g & 1) * 8 : token * 32 + g * 4; };
        const uint32_t vOffA = v_off(tokA), vOffB = v_off(tokB);

        int stage = 0;
        long long cur = lo;
        while (cur < hi) {
            long long r = cur - (long long)cUnit * T;
            if (r >= T) { cUnit++; cb = 0; r -= T; }
            while (ts[cb + 1] <= r) cb++;
            const int b = cb;
            const long long s0 = ts[b], s1 = ts[b + 1], stop = hi - (long long)cUnit * T, e = s1 < stop ? s1 : stop;
            const int ctx = seq_ctx(p, b);
            const int tok0 = (int)((r - s0) * kTile);
            const long long endTok = (e - s0) * kTile;
            const int tokEnd = (int)(endTok < ctx ? endTok : ctx);
            const int kvh = cUnit / p.blocks, block = cUnit % p.blocks;
            const int head0 = kvh * p.group + block * S::HEADS, heads = min(p.group - block * S::HEADS, S::HEADS);

            // ---- queries: f16 fragments in the order of the masks, scaled by 2^-qe; sums for the least terms ----
            uint32_t qb[WK][NT][4];  // [word][block of heads][dims (0,4), (2,6), (1,5), (3,7)]
            float qScale[NT][2], qSum[NT][2];
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
                // the largest element to [2^14, 2^15): elements down to 2^-21 of it keep all bits of bf16
                const int qe = big > 0.f ? min(max((int)(__float_as_uint(big) >> 23) - 141, -112), 112) : 0;
                const float down = pow2(-qe);
#pragma unroll
                for (int w = 0; w < WK; w++) {
                    qb[w][nt][0] = pack16_arith<DT_F16>(x[w][0] * down, x[w][4] * down);
                    qb[w][nt][1] = pack16_arith<DT_F16>(x[w][2] * down, x[w][6] * down);
                    qb[w][nt][2] = pack16_arith<DT_F16>(x[w][1] * down, x[w][5] * down);
                    qb[w][nt][3] = pack16_arith<DT_F16>(x[w][3] * down, x[w][7] * down);
                }
                const float up = pow2(qe) * p.scaleLog2, scaled = sum * p.scaleLog2;
#pragma unroll
                for (int j = 0; j < 2; j++) {  // this lane's score columns: heads 2t, 2t + 1
                    qScale[nt][j] = __shfl_sync(0xffffffffu, up, (2 * t + j) * 4);
                    qSum[nt][j] = __shfl_sync(0xffffffffu, scaled, (2 * t + j) * 4);
                }
            }

            // O^T in units of 2^-24 2^ve (odd dimensions: 16 times that): word w, pair i: [0], [1] = dim base + 8w + 2i of heads 2t, 2t + 1,
            // [2], [3] = the dim behind it; base = g * D / 8
            float o[WV][4][NT][4];
            float m[NT][2], l[NT][2], z[NT][2];
#pragma unroll
            for (int w = 0; w < WV; w++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) o[w][i][nt][0] = o[w][i][nt][1] = o[w][i][nt][2] = o[w][i][nt][3] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) { m[nt][j] = -INFINITY; l[nt][j] = 0.f; z[nt][j] = 0.f; }
            int ve = -110;  // exponent of the power of two that the weights are relative to

            for (int tk = tok0; tk < tokEnd; tk += kStep) {
                asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
                __syncwarp();
                issue();
                const uint32_t st = base + stage * S::STAGE;
                if (++stage == S::STAGES) stage = 0;
                // ---- scores ----
                float se[2][NT][4], so[2][NT][4];
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < 4; i++) se[mt][nt][i] = so[mt][nt][i] = 0.f;
                    uint32_t lowRow[4], highRow[4];
                    const uint32_t at = st + mt * 16 * ROW + kOff;
                    if (WK == 4) { lds128(at, lowRow); lds128(at + 8 * ROW, highRow); }
                    else { lds64(at, lowRow); lds64(at + 8 * ROW, highRow); }
#pragma unroll
                    for (int w = 0; w < WK; w++) {
                        const uint32_t x = lowRow[w], y = highRow[w], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma(se[mt][nt], x & 0x000F000Fu, y & 0x000F000Fu, x8 & 0x000F000Fu, y8 & 0x000F000Fu, qb[w][nt][0], qb[w][nt][1]);
                            mma(so[mt][nt], x & 0x00F000F0u, y & 0x00F000F0u, x8 & 0x00F000F0u, y8 & 0x00F000F0u, qb[w][nt][2], qb[w][nt][3]);
                        }
                    }
                }
                // ---- parameters of this lane's rows: token 8i + tokG ----
                float ks[4], kl[4], vs[4], vl[4];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t at = st + 2 * kStep * ROW + (8 * i + tokG) * 4;
                    unpack16_arith<DT>(lds32(at), ks[i], kl[i]);
                    unpack16_arith<DT>(lds32(at + kStep * 4), vs[i], vl[i]);
                    ks[i] *= 16777216.f;
                    top = max(top, __float_as_uint(vs[i]) & 0x7FFFFFFFu);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                const int need = min(max((int)((top + 0x7FFFFFu) >> 23) - 127, -110), 110);
                float grow = 1.f;
                if (need > ve) {  // uniform over the warp
                    grow = ve - need < -126 ? 0.f : pow2(ve - need);
                    ve = need;
                }
                const float veInv = pow2(-ve);
                // ---- online softmax in the log2 domain ----
                const bool tail = tk + kStep > tokEnd;
                bool rescale = grow != 1.f;
                float alpha[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float x[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float dot = fmaf(so[i >> 1][nt][2 * (i & 1) + j], 0.0625f, se[i >> 1][nt][2 * (i & 1) + j]);
                            x[i] = fmaf(dot * ks[i], qScale[nt][j], kl[i] * qSum[nt][j]);
                            if (tail && tk + 8 * i + tokG >= tokEnd) x[i] = -INFINITY;
                        }
                        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mNew = fmaxf(m[nt][j], mx);
                        const float from = mNew == -INFINITY ? 0.f : mNew;
                        const float a = ex2(m[nt][j] - from);
                        float sum = 0.f, least = 0.f;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float w = ex2(x[i] - from);
                            sum += w;
                            least = fmaf(w, vl[i], least);
                            se[i >> 1][nt][2 * (i & 1) + j] = w * (vs[i] * veInv);
                        }
                        l[nt][j] = fmaf(l[nt][j], a, sum);
                        z[nt][j] = fmaf(z[nt][j], a, least);
                        m[nt][j] = mNew;
                        alpha[nt][j] = a * grow;
                        rescale |= a != 1.f;
                    }
                }
                if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                    for (int w = 0; w < WV; w++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                o[w][i][nt][0] *= alpha[nt][0];
                                o[w][i][nt][1] *= alpha[nt][1];
                                o[w][i][nt][2] *= alpha[nt][0];
                                o[w][i][nt][3] *= alpha[nt][1];
                            }
                }
                // ---- O^T += V^T P^T ----
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    uint32_t pb[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        pb[nt][0] = transpose8(pack16_arith<DT_F16>(se[mt][nt][0], se[mt][nt][1]));
                        pb[nt][1] = transpose8(pack16_arith<DT_F16>(se[mt][nt][2], se[mt][nt][3]));
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
                            const uint32_t x8 = x >> 8, y8 = y >> 8;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma(o[w][2 * half][nt], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pb[nt][0], pb[nt][1]);
                                mma(o[w][2 * half + 1][nt], x8 & 0x000F000Fu, x8 & 0x00F000F0u, y8 & 0x000F000Fu, y8 & 0x00F000F0u, pb[nt][0], pb[nt][1]);
                            }
                        }
                    }
                }
            }

            // ---- end of this warp's part of the pair: the rows themselves, or a partial ----
            const bool begun = r > s0, whole = !begun && e == s1;
            const int which = begun ? 0 : 1;
            const long long slot = 2ll * (blockIdx.x * S::WARPS + warp) + which;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float sum = l[nt][j], least = z[nt][j];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) {
                        sum += __shfl_xor_sync(0xffffffffu, sum, off);
                        least += __shfl_xor_sync(0xffffffffu, least, off);
                    }
                    const int h = nt * 8 + 2 * t + j;
                    if (h >= heads) continue;
                    const float unit = pow2(ve);
                    float x[8 * WV];
#pragma unroll
                    for (int w = 0; w < WV; w++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[8 * w + 2 * i] = fmaf(o[w][i][nt][j] * 16777216.f, unit, least);
                            x[8 * w + 2 * i + 1] = fmaf(o[w][i][nt][2 + j] * 1048576.f, unit, least);
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
                        float* dst = p.acc + (slot * S::HEADS + h) * D + g * (D / 8);
#pragma unroll
                        for (int i = 0; i < 2 * WV; i++) *(float4*)(dst + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                        if (g == 0) p.ml[slot * S::HEADS + h] = make_float2(m[nt][j], sum);
                    }
                }
            }
            if (!whole && lane == 0) sSeg[2 * warp + which] = cUnit * p.batch + b;
            cur = (long long)cUnit * T + e;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // ---- pairs that several warps of this CTA share: joined here; written, or left as the CTA's partial ----
    __syncthreads();
    const long long ctaSlots = 2ll * gridDim.x * S::WARPS;  // behind the warps' slots
    int shared[2] = {-1, -1};  // pairs that this CTA shares with its neighbours: began before its range / goes on behind it
    for (int e0 = 0; e0 < 2 * S::WARPS;) {
        const int seg = sSeg[e0];
        if (seg < 0) { e0++; continue; }
        int e1 = e0 + 1;
        while (e1 < 2 * S::WARPS && (sSeg[e1] < 0 || sSeg[e1] == seg)) e1++;
        const int unit = seg / p.batch, b = seg % p.batch, block = unit % p.blocks;
        const int head0 = (unit / p.blocks) * p.group + block * S::HEADS, heads = min(p.group - block * S::HEADS, S::HEADS);
        const long long gs = (long long)unit * T + ts[b], ge = (long long)unit * T + ts[b + 1];
        const bool mine = gs >= clo && ge <= chi;
        const int which = gs < clo ? 0 : 1;
        const long long slot = ctaSlots + 2ll * blockIdx.x + which;
        if (!mine) shared[which] = seg;
        auto slot_of = [&](int i) -> long long { return sSeg[e0 + i] < 0 ? -1ll : 2ll * blockIdx.x * S::WARPS + e0 + i; };
        join<D>(p, heads, S::HEADS, e1 - e0, slot_of, [&](int h, int d, float M, float den, float4 num) {
            if (mine) {
                store4<DT>(p.out + ((size_t)b * p.numHeads + head0 + h) * D + d, den, num);
            } else {
                *(float4*)(p.acc + (slot * S::HEADS + h) * D + d) = num;
                if (d == 0) p.ml[slot * S::HEADS + h] = make_float2(M, den);
            }
        });
        e0 = e1;
    }
    if (shared[0] < 0 && shared[1] < 0) return;  // uniform over the CTA
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 2) {
        const int seg = threadIdx.x == 0 ? shared[0] : shared[1];
        int last = 0;
        if (seg >= 0) {
            const int unit = seg / p.batch, b = seg % p.batch;
            const long long gs = (long long)unit * T + ts[b], ge = (long long)unit * T + ts[b + 1];
            const int owners = part_of(ge - 1, total, parts) - part_of(gs, total, parts) + 1;
            last = atomicAdd(p.counters + seg, 1) == owners - 1;
            if (last) p.counters[seg] = 0;  // nobody else comes in this launch
        }
        sLast[threadIdx.x] = last;
        __threadfence();
    }
    __syncthreads();
    for (int s = 0; s < 2; s++) {
        if (!sLast[s]) continue;
        const int seg = shared[s], unit = seg / p.batch, b = seg % p.batch, block = unit % p.blocks;
        const int head0 = (unit / p.blocks) * p.group + block * S::HEADS, heads = min(p.group - block * S::HEADS, S::HEADS);
        const long long gs = (long long)unit * T + ts[b], ge = (long long)unit * T + ts[b + 1];
        const int c0 = part_of(gs, total, parts), c1 = part_of(ge - 1, total, parts);
        auto slot_of = [&](int i) -> long long { return ctaSlots + 2ll * (c0 + i) + (gs < (c0 + i) * total / parts ? 0 : 1); };
        join<D>(p, heads, S::HEADS, c1 - c0 + 1, slot_of, [&](int h, int d, float M, float den, float4 num) {
            store4<DT>(p.out + ((size_t)b * p.numHeads + head0 + h) * D + d, den, num);
        });
    }
}

template <int DT, int D, int NT>
static int launch(Context* ctx, Params& p, CUDAStatus* status) {
    using S = Shape<DT, D, NT>;
    const char* what = "paged decode attention (4 bits)";
    const unsigned grid = (unsigned)ctx->smCount;
    p.blocks = (p.group + S::HEADS - 1) / S::HEADS;
    p.units = p.kvHeads * p.blocks;
    if ((long long)p.units * p.batch > 0x7FFFFFFFll) return fail(status, -2, "%s: batch times heads exceeds 31 bits", what);
    const size_t slots = 2ull * grid * (S::WARPS + 1);
    const size_t accBytes = slots * S::HEADS * D * 4, mlBytes = slots * S::HEADS * 8;
    const size_t prefixBytes = p.batch > kPrefixSmem ? ((size_t)p.batch + 1) * 4 : 0;
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
        prefix_kernel<<<1, 1024, 0, ctx->stream>>>(p, prefix);
        rc = check_launch(ctx, status, "paged decode attention (4 bits): prefix");
        if (rc != 0) return rc;
        p.tileStart = prefix;
    }
    cudaFuncSetAttribute(decode_kernel<DT, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    decode_kernel<DT, D, NT><<<grid, S::WARPS * 32, S::SMEM, ctx->stream>>>(p);
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
    const size_t slots = (size_t)pageCount * pageSize * kvHeads;
    if (slots > 0xFFFFFFFFull || (size_t)maxPagesPerSeq * pageSize > 0x7FFFFFE0ull || batch > 0x7FFFFFFEu)
        return fail(status, -2, "%s: a pool of %zu vectors or a context of %zu tokens exceeds the index range", what, slots,
                    (size_t)maxPagesPerSeq * pageSize);
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
    const int two = p.group > 8;
#define DECODE(DT)                                                                                                                      \
    (headDim == 128 ? (two ? q4d::launch<DT, 128, 2>(ctx, p, status) : q4d::launch<DT, 128, 1>(ctx, p, status))                      \
                    : (two ? q4d::launch<DT, 64, 2>(ctx, p, status) : q4d::launch<DT, 64, 1>(ctx, p, status)))
    return elementDType == DT_BF16 ? DECODE(DT_BF16) : DECODE(DT_F16);
#undef DECODE
}
