// Attention over whole prompts of different lengths, packed one behind the other.
//
// q / out [totalTokens, numHeads, D], k / v [totalTokens, kvHeads, D]; sequence i holds rows seqStarts[i] .. seqStarts[i + 1] - 1
// (int32 on the device, so a serving loop never waits for lengths).  Per sequence: RoPE(q), RoPE(k) at positions that restart with
// every sequence (device/cpu/rope/compute.go:55-193, results rounded to the storage type), then MultiHeadAttention
// (device/cpu/attention/typed_compute.go:142-237): out_r = sum_{t <= r} p_t v_t, p = softmax(q_r . k_t / sqrt(D)).
// Rows that belong to no sequence (before the first start, behind the last) are neither read into a result nor written.
// A pair of starts that is not 0 <= start <= end <= totalTokens with at most maxSeqLen rows is skipped and raises the error flag.
//
// cuda_context_set_exact(1) rotates into scratch and attends with the kernel that keeps the CPU's order of operations (attention_exact.cu).
//
// Three kernels otherwise.  rows_kernel is a warp per (row, head) for any type and head dimension.  short_kernel is for calls without long sequences: a
// block per (sequence, KV head), see there.  tiles_kernel is the tensor-core form (bf16 / f16,
// head dimensions up to 128 that are multiples of 8), built like the prefill kernel for equal lengths: two tiles of 128 rows that take turns
// on the tensor core, softmax in registers with one row a thread, P handed back through TMEM, K and V through a TMA ring.  What the
// different lengths change:
//   * A tile's 128 rows are PACK query heads of one KV head (PACK = the largest power of two in the group, 128 at most) times 128 / PACK
//     positions: a group of 4 turns 33 tokens into 132 rows instead of 4 x 33 of 128, and short prompts are what packing is for.
//     A TMA box of 64 dimensions x PACK heads x 128 / PACK rows brings such a tile in; long prompts cost the same either way.
//   * The work list (sequence, block of 2 * 128 / PACK positions) is built on the device, longest key ranges first, by the first block of the
//     launch that also rotates K: the host never learns the lengths.  Q is rotated in its tile (head dimensions 64 and 128).
//   * Keys behind the end of a sequence and keys that a row may not see are masked by position; their weights are exactly zero.  A value row
//     that is not finite would still reach every row of the tile through 0 * NaN, so a warp looks through the value tiles that are not
//     seen by all rows, clears what is not finite, and the rows that do see it add it back at the end.
//   * The last rows of a sequence share their TMA box with the next sequence, so that box is written row by row.
// Roundings to 16 bits: rotated q and k, as the framework's RoPE stores them and its other prefill uses them; the weights before P V, because one
// tcgen05 product takes one type for both operands and V comes in 16 bits (the sum of the weights stays in float32 and is not rounded).  In
// bf16 the weights leave an error of 1.8 to 2.0e-3 of the output's norm and RoPE 2.1 to 2.8e-3 (33 to 1500 tokens), where rounding the output alone
// leaves 1.6e-3; in f16 2.2 to 2.6e-4 and 2.7 to 3.5e-4 of 2.0e-4.  Maxima, sums and accumulators are float32.
// Bound: the softmax of a tile between its two products (one row a thread, 128 exponentials; counters: tensor pipe 52 % of the cycles, exponentials
// 53 %, issue slots 38 %) and, in long calls, the power limit.  bf16, 32 heads on 8 KV heads of 128, RoPE included: eight prompts of 150 to 4096
// tokens 301 to 309 us, 1.04 to 1.07 PFLOP/s counting what the mask leaves (193 us at the dense rate; 12 us are the list and K's rotation, a pass over K in
// memory), one of 16384 tokens 1.65 to 1.8 ms, 1.2 to 1.35 PFLOP/s, and 1.87 ms when called again and again.
#include <math.h>

#include "common.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace puter {

int validate_rope(CUDAStatus* status, double base, uint32_t halfMode, uint32_t scaling, double factor, double low, double high,
                  uint32_t origCtx);
const float* cached_rope_table_at_least(Context* ctx, size_t positions, int headDim, double base, long long startPos, int scaling,
                                        double factor, double low, double high, int origCtx, const float** sinT, CUDAStatus* status);

int check_mha_exact_packed(CUDAStatus* status, int maxLen, uint32_t numHeads, uint32_t headDim);
int launch_mha_exact_packed(Context* ctx, int dt, const void* q, const void* k, const void* v, void* out, const pk::Seqs& seqs, uint32_t numHeads,
                            uint32_t kvHeads, uint32_t headDim, uint32_t causal, CUDAStatus* status);

namespace pk {

// x [total, heads, D] rotated at the positions of its rows within their sequences, any even D
template <int DT>
__global__ void __launch_bounds__(256) rotate_kernel(const void* __restrict__ in, void* __restrict__ out, Seqs s, const float* __restrict__ cosT,
                                                     const float* __restrict__ sinT, int heads, int dim, int halfMode) {
    using T = typename Storage<DT>::type;
    const size_t half = dim / 2, perRow = (size_t)heads * half, total = (size_t)s.total * perRow;
    const size_t stride = (size_t)gridDim.x * blockDim.x;
    for (size_t it = (size_t)blockIdx.x * blockDim.x + threadIdx.x; it < total; it += stride) {
        const int row = (int)(it / perRow);
        int s0, s1;
        if (!seq_rows(s, seq_of(s, row), s0, s1) || row < s0 || row >= s1) continue;
        const size_t j = it % perRow, h = j / half, i = j % half, base = ((size_t)row * heads + h) * dim;
        const size_t ei = halfMode ? base + i : base + 2 * i, oi = halfMode ? ei + half : ei + 1;
        const float e = Storage<DT>::load((const T*)in, ei), o = Storage<DT>::load((const T*)in, oi);
        const float c = cosT[(size_t)(row - s0) * half + i], sn = sinT[(size_t)(row - s0) * half + i];
        Storage<DT>::store((T*)out, ei, sub(mul(e, c), mul(o, sn)));
        Storage<DT>::store((T*)out, oi, add(mul(e, sn), mul(o, c)));
    }
}

// Any type and head dimension up to 256: one warp per (row, head), eight elements a lane at most, one pass over the keys with a running
// maximum and sum.  It runs what the tensor-core kernel does not take; its bound is the five shuffles per key
// (eight prompts of 512 tokens, 32 heads on 8 of 128, float32: 6.9 ms, 2.5 TFLOP/s).
template <int DT>
__global__ void __launch_bounds__(256) rows_kernel(const void* __restrict__ q, const void* __restrict__ k, const void* __restrict__ v,
                                                   void* __restrict__ out, Seqs s, int heads, int kvHeads, int dim, int causal, float scaleLog2) {
    using T = typename Storage<DT>::type;
    const int lane = threadIdx.x & 31;
    const size_t units = (size_t)s.total * heads, warps = (size_t)gridDim.x * 8;
    for (size_t u = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += warps) {
        const int row = (int)(u / heads), head = (int)(u % heads), kvh = head / (heads / kvHeads);
        int s0, s1;
        if (!seq_rows(s, seq_of(s, row), s0, s1) || row < s0 || row >= s1) continue;
        float qr[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            qr[i] = i * 32 + lane < dim ? Storage<DT>::load((const T*)q, u * dim + i * 32 + lane) : 0.f;
            acc[i] = 0.f;
        }
        const int end = causal ? row + 1 : s1;
        for (int t = s0; t < end; t++) {
            const size_t at = ((size_t)t * kvHeads + kvh) * dim;
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i * 32 + lane < dim) dot = fmaf(qr[i], Storage<DT>::load((const T*)k, at + i * 32 + lane), dot);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            const float x = dot * scaleLog2, mNew = fmaxf(m, x);
            const float base = mNew == -INFINITY ? 0.f : mNew;  // nothing but scores of -inf so far
            const float alpha = exp2f(m - base), e = exp2f(x - base);
            l = l * alpha + e;
            m = mNew;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i * 32 + lane < dim) acc[i] = acc[i] * alpha + e * Storage<DT>::load((const T*)v, at + i * 32 + lane);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i * 32 + lane < dim) Storage<DT>::store((T*)out, u * dim + i * 32 + lane, acc[i] / l);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// the launch before the attention: block 0 builds the work list, the others rotate q and k
// ---------------------------------------------------------------------------------------------------------------------------------
struct Entry { int row0, len, pos, pad; };  // a block of `span` positions from pos on, of the sequence of `len` rows at row0

struct Lists {
    int* count;      // entries
    Entry* entries;
    int* above;      // [levels] scratch: sequences by number of blocks, then entries of higher levels
    int* cursor;     // [levels] scratch
    int span, levels, capacity;
};

// x[0 .. n) becomes its suffix sum (x[i] + x[i + 1] + ...), or the sum of what follows x[i] when `exclusive`.  The whole block calls it.
__device__ void suffix_sum(int* x, int n, bool exclusive) {
    __shared__ int sums[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    int carry = 0;
    for (int base = 0; base < n; base += blockDim.x) {
        const int i = n - 1 - (base + (int)threadIdx.x);
        const int v = i >= 0 ? x[i] : 0;
        int incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < warps; w++) {
            if (w < warp) before += sums[w];
            carry += sums[w];
        }
        if (i >= 0) x[i] = before + incl - (exclusive ? v : 0);
        __syncthreads();
    }
}

constexpr int kListLevels = 2048;  // whose counts fit shared memory

// Entries by level (block number within the sequence: what decides its number of keys), highest first; within a level in any order.
__device__ void build_list(const Seqs& s, Lists l) {
    __shared__ int levels[2][kListLevels];
    if (l.levels <= kListLevels) {  // the five passes then wait for the starts alone
        l.above = levels[0];
        l.cursor = levels[1];
    }
    for (int i = threadIdx.x; i < l.levels; i += blockDim.x) l.above[i] = l.cursor[i] = 0;
    __syncthreads();
    for (int b = threadIdx.x; b < s.batch; b += blockDim.x) {
        int s0, s1;
        if (seq_rows(s, b, s0, s1)) atomicAdd(l.above + (s1 - s0 - 1) / l.span, 1);  // by its last block
    }
    __syncthreads();
    suffix_sum(l.above, l.levels, false);  // entries per level: sequences with a block of that number
    __shared__ int total;
    if (threadIdx.x == 0) total = l.above[0];
    __syncthreads();
    suffix_sum(l.above, l.levels, true);   // entries of higher levels
    if (threadIdx.x == 0) *l.count = min(total + l.above[0], l.capacity);  // (starts that go back can count rows twice)
    const int lane = threadIdx.x & 31;
    for (int b = threadIdx.x >> 5; b < s.batch; b += blockDim.x >> 5) {
        int s0, s1;
        if (!seq_rows(s, b, s0, s1)) continue;
        const int blocks = (s1 - s0 + l.span - 1) / l.span;
        for (int i = lane; i < blocks; i += 32) {
            const int at = l.above[i] + atomicAdd(l.cursor + i, 1);
            if (at < l.capacity) l.entries[at] = Entry{s0, s1 - s0, i * l.span, 0};
        }
    }
}

// eight neighbouring elements rotated with their own pairs (interleaved) or with the eight `b` half a head further (halves)
template <bool BF16>
__device__ __forceinline__ void rotate8(Vec16& a, Vec16& b, const float* cosRow, const float* sinRow, bool halves) {
    constexpr int DT = BF16 ? DT_BF16 : DT_F16;
    if (halves) {
        float cs[8], sn[8];
        *(float4*)cs = __ldg((const float4*)cosRow);
        *(float4*)(cs + 4) = __ldg((const float4*)(cosRow + 4));
        *(float4*)sn = __ldg((const float4*)sinRow);
        *(float4*)(sn + 4) = __ldg((const float4*)(sinRow + 4));
#pragma unroll
        for (int w = 0; w < 4; w++) {
            float e0, e1, o0, o1;
            unpack16_arith<DT>(a.w[w], e0, e1);
            unpack16_arith<DT>(b.w[w], o0, o1);
            a.w[w] = pack16_arith<DT>(sub(mul(e0, cs[2 * w]), mul(o0, sn[2 * w])), sub(mul(e1, cs[2 * w + 1]), mul(o1, sn[2 * w + 1])));
            b.w[w] = pack16_arith<DT>(add(mul(e0, sn[2 * w]), mul(o0, cs[2 * w])), add(mul(e1, sn[2 * w + 1]), mul(o1, cs[2 * w + 1])));
        }
    } else {
        const float4 c = __ldg((const float4*)cosRow), n = __ldg((const float4*)sinRow);
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            float e, o;
            unpack16_arith<DT>(a.w[w], e, o);
            a.w[w] = pack16_arith<DT>(sub(mul(e, cs[w]), mul(o, sn[w])), add(mul(e, sn[w]), mul(o, cs[w])));
        }
    }
}

// Rotates [total, qHeads + kHeads, D] (two tensors, one row of both at a time, a warp per row) with 16-byte vectors.
template <int DT>
__global__ void __launch_bounds__(256) prologue_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ k, uint16_t* __restrict__ qOut,
                                                       uint16_t* __restrict__ kOut, Seqs s, Lists l, const float* __restrict__ cosT,
                                                       const float* __restrict__ sinT, int qHeads, int kHeads, int dim, int halfMode) {
    if (blockIdx.x == 0) {
        build_list(s, l);
        return;
    }
    const int lane = threadIdx.x & 31, half = dim / 2, perHead = halfMode ? half / 8 : dim / 8;  // vectors, or pairs of vectors
    const int items = (qHeads + kHeads) * perHead;
    for (int row = (blockIdx.x - 1) * 8 + (threadIdx.x >> 5); row < s.total; row += (gridDim.x - 1) * 8) {
        // two items of a lane are on their way before the search for the row's sequence, which is a chain of loads of its own
        constexpr int U = 2;
        int s0 = 0;
        for (int it0 = lane; it0 < items; it0 += 32 * U) {
            Vec16 a[U], b[U];
            uint16_t* dst[U];
            int j[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int it = min(it0 + 32 * u, items - 1), head = it / perHead;
                j[u] = it - head * perHead;
                const bool ofQ = head < qHeads;
                const size_t at = ofQ ? ((size_t)row * qHeads + head) * dim : ((size_t)row * kHeads + head - qHeads) * dim;
                const uint16_t* src = (ofQ ? q : k) + at;
                dst[u] = (ofQ ? qOut : kOut) + at;
                a[u] = ld_stream(src + 8 * j[u]);
                if (halfMode) b[u] = ld_stream(src + half + 8 * j[u]);
            }
            if (it0 == lane) {
                int s1;
                if (!seq_rows(s, seq_of(s, row), s0, s1) || row < s0 || row >= s1) break;  // uniform over the warp
            }
            const float* cr = cosT + (size_t)(row - s0) * half;
            const float* sr = sinT + (size_t)(row - s0) * half;
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (it0 + 32 * u >= items) break;
                const int c = (halfMode ? 8 : 4) * j[u];
                rotate8<DT == DT_BF16>(a[u], b[u], cr + c, sr + c, halfMode != 0);
                *(Vec16*)(dst[u] + 8 * j[u]) = a[u];
                if (halfMode) *(Vec16*)(dst[u] + half + 8 * j[u]) = b[u];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// tensor-core kernel
// ---------------------------------------------------------------------------------------------------------------------------------
using namespace pf;

constexpr int kThreads = 384;  // warps 0-3 / 4-7 softmax of tile 0 / 1, 8 MMA, 9 TMA loads, 10 output, 11 value tiles that not all rows see
constexpr int kRows = 128;     // rows (head, position) of a tile
constexpr int kKeys = 128;     // keys of a tile
constexpr uint32_t kBlock = 128 * 128;  // bytes of 128 rows x 64 dimensions

// NB: blocks of 64 dimensions
template <int NB>
struct Smem {
    static constexpr int STAGES = NB == 2 ? 2 : 4;
    static constexpr uint32_t TILE = NB * kBlock;
    static constexpr uint32_t Q = 0, K = 2 * TILE, V = K + STAGES * TILE, STAGING = V + STAGES * TILE, BARS = STAGING + TILE, TOTAL = BARS + 512 + 1024;
};

struct TileParams {
    CUtensorMap tmQ, tmK, tmV, tmO;
    const Entry* entries;
    const int* count;
    const uint16_t* v;  // values, for the rows that see one that is not finite
    uint16_t* out;
    int* errorFlag;
    int heads, kvHeads, dim, causal;
    const float *cosT, *sinT;  // nullptr: q comes rotated (or no rotation)
    int halves, posLast;       // last position of the tables
    int packLog, headGroups;  // PACK = 1 << packLog heads per tile, heads / PACK tiles per block of positions
    float scaleLog2;
};

// bounded wait for the count at `at`
__device__ __forceinline__ bool turn_wait(uint32_t at, int need, volatile int* abortFlag) {
    for (long long i = 0; i < kSpinLimit; i++) {
        int now;
        asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(now) : "r"(at) : "memory");
        if (now >= need) return true;
        if ((i & 1023) == 1023 && *abortFlag) return false;
    }
    return false;
}

template <int STAGES>
struct Bar {
    // VRAW: a value tile that not all rows see has landed (VFULL follows once it has been looked through)
    enum : uint32_t { Q = 0, QREADY = 2, S = 4, P = 6, P2 = 8, O = 10, QFREE = 12, STAGED = 14, KFULL = 16, KEMPTY = KFULL + STAGES,
                      VFULL = KEMPTY + STAGES, VEMPTY = VFULL + STAGES, VRAW = VEMPTY + STAGES, COUNT = VRAW + STAGES };
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(tm), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* tm, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(tm), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

// which halves of a word are not finite (their sign bits)
template <bool BF16> __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t E = BF16 ? 0x7F807F80u : 0x7C007C00u, ONE = BF16 ? 0x00800080u : 0x04000400u;
    return ((w & E) + ONE) & 0x80008000u;
}

// Adds to 32 normalised outputs of a row what is not finite among the values it sees in keys [k0, k1): any weight leaves an infinity
// or a NaN as it is.  Runs only where the value warp has met one.
template <bool BF16>
__device__ __noinline__ void add_not_finite(float* o, const uint16_t* v, size_t stride, int k0, int k1, int cols) {
    for (int key = k0; key < k1; key++)
        for (int i = 0; i < cols; i++) {
            const uint32_t bits = v[(size_t)key * stride + i];
            if (not_finite<BF16>(bits)) o[i] += widen16<BF16>(bits);
        }
}

// Rotates the 32 rows of a warp in a Q tile once it has landed: the lanes of a row own eight pairs each (halves: a 16-byte piece and its
// partner half a head further) or four (neighbouring pairs: one piece).  The cos / sin values are fetched before the wait.  Not inlined: its
// 128 table registers are apart from the scores of the caller.
template <bool BF16, int NB>
__device__ __noinline__ bool rotate_q_when_loaded(unsigned char* tile, int row0, int lane, bool halves, const float* cosT, const float* sinT, int pos0,
                                                   int posLast, int packLog, uint32_t bar, uint32_t parity, volatile int* abortFlag) {
    constexpr int HALF = 32 * NB;  // pairs of a head
    float4 tab[16 * NB];
    if (halves) {
        const int c = lane % (4 * NB);
#pragma unroll
        for (int it = 0; it < 4 * NB; it++) {
            const size_t at = (size_t)min(pos0 + ((row0 + it * (8 / NB) + lane / (4 * NB)) >> packLog), posLast) * HALF + 8 * c;
            tab[4 * it] = __ldg((const float4*)(cosT + at));
            tab[4 * it + 1] = __ldg((const float4*)(cosT + at + 4));
            tab[4 * it + 2] = __ldg((const float4*)(sinT + at));
            tab[4 * it + 3] = __ldg((const float4*)(sinT + at + 4));
        }
    } else {
        const int c = lane % (8 * NB);
#pragma unroll
        for (int it = 0; it < 8 * NB; it++) {
            const size_t at = (size_t)min(pos0 + ((row0 + it * (4 / NB) + lane / (8 * NB)) >> packLog), posLast) * HALF + 4 * c;
            tab[2 * it] = __ldg((const float4*)(cosT + at));
            tab[2 * it + 1] = __ldg((const float4*)(sinT + at));
        }
    }
    if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abortFlag))) return false;
    if (halves) {
        const int c = lane % (4 * NB);
#pragma unroll
        for (int it = 0; it < 4 * NB; it++) {
            const int row = row0 + it * (8 / NB) + lane / (4 * NB);
            unsigned char* const line = tile + row * 128;
            Vec16* const pa = (Vec16*)(line + ((c ^ (row & 7)) * 16));
            Vec16* const pb = NB == 2 ? (Vec16*)((unsigned char*)pa + kBlock) : (Vec16*)(line + (((c + 4) ^ (row & 7)) * 16));
            Vec16 a = *pa, b = *pb;
            const float4 c0 = tab[4 * it], c1 = tab[4 * it + 1], n0 = tab[4 * it + 2], n1 = tab[4 * it + 3];
            const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, sn[8] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint64_t E = pk2(widen16<BF16>(a.w[w] & 0xFFFFu), widen16<BF16>(a.w[w] >> 16)), O = pk2(widen16<BF16>(b.w[w] & 0xFFFFu), widen16<BF16>(b.w[w] >> 16));
                const uint64_t C = pk2(cs[2 * w], cs[2 * w + 1]), S = pk2(sn[2 * w], sn[2 * w + 1]), NS = pk2(-sn[2 * w], -sn[2 * w + 1]);
                float x0, x1, y0, y1;
                un2(fma2(O, NS, mul2(E, C)), x0, x1);  // e c - o s
                un2(fma2(E, S, mul2(O, C)), y0, y1);   // e s + o c
                a.w[w] = pack2<BF16>(x0, x1);
                b.w[w] = pack2<BF16>(y0, y1);
            }
            *pa = a;
            *pb = b;
        }
    } else {
        const int c = lane % (8 * NB);
#pragma unroll
        for (int it = 0; it < 8 * NB; it++) {
            const int row = row0 + it * (4 / NB) + lane / (8 * NB);
            Vec16* const pa = (Vec16*)(tile + (c >> 3) * kBlock + row * 128 + (((c & 7) ^ (row & 7)) * 16));
            Vec16 a = *pa;
            const float cs[4] = {tab[2 * it].x, tab[2 * it].y, tab[2 * it].z, tab[2 * it].w}, sn[4] = {tab[2 * it + 1].x, tab[2 * it + 1].y, tab[2 * it + 1].z, tab[2 * it + 1].w};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float e = widen16<BF16>(a.w[w] & 0xFFFFu), o = widen16<BF16>(a.w[w] >> 16);
                a.w[w] = pack2<BF16>(sub(mul(e, cs[w]), mul(o, sn[w])), add(mul(e, sn[w]), mul(o, cs[w])));
            }
            *pa = a;
        }
    }
    __syncwarp();
    return true;
}

template <bool BF16, int NB>
__global__ void __launch_bounds__(kThreads, 1) tiles_kernel(const __grid_constant__ TileParams p) {
    using M = Smem<NB>;
    using B = Bar<M::STAGES>;
    constexpr uint32_t kColS = 0, kColO = 256;  // TMEM columns: S0 S1 (P over their first halves), O0 O1
    extern __shared__ unsigned char smemRaw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);  // swizzled boxes: 1024-byte aligned
    const uint32_t sBase = smem_u32(smem);
    auto bar = [&](uint32_t i) { return sBase + M::BARS + i * 8; };
    __shared__ uint32_t tmemBaseShared;
    __shared__ int abortShared;
    __shared__ int turn;       // output tiles that have left the staging tile: item it's tile 0 is number 2 it, its tile 1 (or none) 2 it + 1
    __shared__ int notFinite;  // set once a value that is not finite has been cleared anywhere in this CTA's work
    volatile int* abortFlag = &abortShared;

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int posTile = kRows >> p.packLog;  // positions of a tile
    // A work item: one block of two tiles' positions of one sequence for PACK heads.  Dealt in serpentine order, heavy items first.
    struct Item { int row0, len, pos, head, kvHead, nMax, nT0, nT1, firstPartial; };  // nT: key tiles of a tile; firstPartial: first key tile not seen by all rows
    auto get_item = [&](int it, Item& w) -> bool {
        asm volatile("" : "+r"(it));  // decoded anew by every role: kept values would cost the softmax threads registers
        const int G = (int)gridDim.x;
        const int idx = it * G + ((it & 1) ? G - 1 - (int)blockIdx.x : (int)blockIdx.x);
        const int e = idx / p.headGroups;
        if (e >= __ldg(p.count)) return false;
        const int4 raw = __ldg((const int4*)(p.entries + e));
        w.row0 = raw.x;
        w.len = raw.y;
        w.pos = raw.z;
        w.head = (idx - e * p.headGroups) << p.packLog;
        w.kvHead = w.head / (p.heads / p.kvHeads);
        auto tiles_for = [&](int from) {
            const int last = p.causal ? min(w.len, from + posTile) : w.len;
            return from < w.len ? (last + kKeys - 1) / kKeys : 0;
        };
        w.nT0 = tiles_for(w.pos);
        w.nT1 = tiles_for(w.pos + posTile);
        w.nMax = max(w.nT0, w.nT1);
        w.firstPartial = p.causal ? (w.pos + 1) / kKeys : w.len / kKeys;  // tile j is seen by all rows if its keys end at pos + 1 / at len or before
        return true;
    };

    if (threadIdx.x == 0) {
        abortShared = 0;
        notFinite = 0;
        turn = 0;
        for (int t = 0; t < 2; t++) {
            mbar_init(bar(B::Q + t), 1);
            mbar_init(bar(B::QREADY + t), 128);
            mbar_init(bar(B::S + t), 1);
            mbar_init(bar(B::P + t), 128);
            mbar_init(bar(B::P2 + t), 128);
            mbar_init(bar(B::O + t), 1);
            mbar_init(bar(B::QFREE + t), 1);
            mbar_init(bar(B::STAGED + t), 128);
        }
        for (int s = 0; s < M::STAGES; s++) {
            mbar_init(bar(B::KFULL + s), 1);
            mbar_init(bar(B::KEMPTY + s), 1);
            mbar_init(bar(B::VFULL + s), 1);
            mbar_init(bar(B::VEMPTY + s), 1);
            mbar_init(bar(B::VRAW + s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmemBaseShared)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmemBaseShared, 0);

    // registers: 384 x 168 at launch; 256 x 200 + 128 x 96 afterwards
    if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 11) {
        // ------------------------------------------------ value tiles that not all rows see ------------------------------------
        uint32_t lc = 0;   // ring position of the item's first key tile
        uint32_t raw = 0;  // per stage: parity of its VRAW phases
        bool okay = true;
        Item w = {};
        for (int it = 0; okay && get_item(it, w); it++) {
            for (int j = w.firstPartial; j < w.nMax && okay; j++) {
                const uint32_t ring = lc + (uint32_t)j;
                const int st = ring % M::STAGES;
                okay = __all_sync(0xffffffffu, mbar_wait(bar(B::VRAW + st), (raw >> st) & 1, abortFlag));
                if (!okay) break;
                raw ^= 1u << st;
                Vec16* tile = (Vec16*)(smem + M::V + st * M::TILE);
                uint32_t found = 0;
#pragma unroll 8
                for (int i = lane; i < (int)(M::TILE / 16); i += 32) {
                    const Vec16 x = tile[i];
                    found |= not_finite<BF16>(x.w[0]) | not_finite<BF16>(x.w[1]) | not_finite<BF16>(x.w[2]) | not_finite<BF16>(x.w[3]);
                }
                if (__any_sync(0xffffffffu, found != 0)) {
                    for (int i = lane; i < (int)(M::TILE / 16); i += 32) {
                        Vec16 x = tile[i];
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const uint32_t bad = not_finite<BF16>(x.w[c]);
                            x.w[c] &= ~((bad >> 15) * 0xFFFFu);  // 0x8000 -> all ones of that half
                        }
                        tile[i] = x;
                    }
                    *(volatile int*)&notFinite = 1;
                    __threadfence_block();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B::VFULL + st));
            }
            lc += (uint32_t)w.nMax;
        }
        if (!okay && lane == 0) *abortFlag = 1;
    } else if (warp == 10) {
        // ------------------------------------------------ output: tile 0, tile 1, next item ... ---------------------------------
        uint32_t uc[2] = {};  // items each tile took part in so far
        bool okay = true;
        Item w = {};
        for (int it = 0; okay && get_item(it, w); it++) {
            for (int t = 0; t < 2; t++) {
                if ((t == 0 ? w.nT0 : w.nT1) == 0) continue;
                okay = __all_sync(0xffffffffu, mbar_wait(bar(B::STAGED + t), uc[t] & 1, abortFlag));  // every row staged
                if (!okay) break;
                uc[t]++;
                const int pos = w.pos + t * posTile;
                if (pos + posTile <= w.len) {
                    if (lane == 0) {
#pragma unroll
                        for (int n = 0; n < NB; n++) tma_store_3d(&p.tmO, sBase + M::STAGING + n * kBlock, 64 * n, w.head, w.row0 + pos);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // shared memory must outlive the read
                    }
                } else {
                    // rows behind the sequence belong to the next one: the live rows one by one, 16-byte pieces across the lanes
                    const int live = (w.len - pos) << p.packLog, perRow = p.dim / 8;
                    for (int i = lane; i < live * perRow; i += 32) {
                        const int row = i / perRow, c = i - row * perRow;
                        const Vec16 x = *(const Vec16*)(smem + M::STAGING + (c >> 3) * kBlock + row * 128 + (((c & 7) ^ (row & 7)) * 16));
                        const size_t at = ((size_t)(w.row0 + pos + (row >> p.packLog)) * p.heads + w.head + (row & ((1 << p.packLog) - 1))) * p.dim;
                        *(Vec16*)(p.out + at + c * 8) = x;
                    }
                }
                __syncwarp();
                if (lane == 0) asm volatile("st.release.cta.shared::cta.s32 [%0], %1;" ::"r"(smem_u32(&turn)), "r"(2 * it + (w.nT1 == 0 ? 2 : t + 1)) : "memory");
            }
        }
        if (!okay && lane == 0) *abortFlag = 1;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else if (warp == 9) {
        // ------------------------------------------------ TMA loads --------------------------------------------------------------
        if (lane == 0) {
            uint32_t lc = 0;
            uint32_t uc[2] = {};
            bool okay = true;
            Item w = {};
            auto load_kv = [&](const CUtensorMap* tm, uint32_t at, uint32_t full, uint32_t empty, int j) {  // `full`, `empty`: barriers of stage 0
                const uint32_t ring = lc + (uint32_t)j;
                const int st = ring % M::STAGES;
                if (ring >= M::STAGES && !mbar_wait(bar(empty + st), ((ring / M::STAGES) - 1) & 1, abortFlag)) return false;
                mbar_expect_tx(bar(full + st), M::TILE);
#pragma unroll
                for (int n = 0; n < NB; n++) tma_load_3d(sBase + at + st * M::TILE + n * kBlock, tm, bar(full + st), 64 * n, w.kvHead, w.row0 + j * kKeys);
                return true;
            };
            auto load_k = [&](int j) { return load_kv(&p.tmK, M::K, B::KFULL, B::KEMPTY, j); };
            auto load_v = [&](int j) { return load_kv(&p.tmV, M::V, j >= w.firstPartial ? B::VRAW : B::VFULL, B::VEMPTY, j); };
            auto load_q = [&](int t) {
                if ((t == 0 ? w.nT0 : w.nT1) == 0) return true;
                // the buffer is free once the last score product of the tile's previous item has run
                if (uc[t] > 0 && !mbar_wait(bar(B::QFREE + t), (uc[t] - 1) & 1, abortFlag)) return false;
                uc[t]++;
                mbar_expect_tx(bar(B::Q + t), M::TILE);
#pragma unroll
                for (int n = 0; n < NB; n++)
                    tma_load_3d(sBase + M::Q + t * M::TILE + n * kBlock, &p.tmQ, bar(B::Q + t), 64 * n, w.head, w.row0 + w.pos + t * posTile);
                return true;
            };
            // one thread issues every load, in the order in which the buffers come free at the end of the item before
            for (int it = 0; okay && get_item(it, w); it++) {
                if (it == 0) okay = load_q(0) && load_k(0) && load_q(1) && load_v(0);
                else okay = load_k(0) && load_q(0) && load_v(0) && load_q(1);
                for (int j = 1; j < w.nMax && okay; j++) okay = load_k(j) && load_v(j);
                lc += (uint32_t)w.nMax;
            }
            if (!okay) *abortFlag = 1;
        }
    } else if (warp == 8) {
        // ------------------------------------------------ MMA issue: the turns of the equal-length kernel --------------------------
        const bool leader = elect_one();
        const uint32_t idescQK = make_idesc(BF16, false), idescPV = make_idesc(BF16, true, 64 * NB);
        bool okay = true;
        const uint64_t kmajorHi = make_desc(0, 16, 1024) >> 32, vHi = make_desc(0, kBlock, 1024) >> 32;
        const uint32_t qLo = (uint32_t)make_desc(sBase + M::Q, 16, 1024), kLo = (uint32_t)make_desc(sBase + M::K, 16, 1024);
        const uint32_t vLo = (uint32_t)make_desc(sBase + M::V, kBlock, 1024);
        auto desc = [](uint64_t hi, uint32_t lo) { return (hi << 32) | (uint64_t)lo; };
        uint32_t lc = 0;        // ring position of key tile 0 of the current item
        uint32_t sc[2] = {}, uc[2] = {};  // key-tile steps / items each tile has run so far (parities of its barriers)
        int nT[2] = {};
        auto issue_qk = [&](int t, int j) {
            const uint32_t kS = kLo + ((lc + (uint32_t)j) % M::STAGES) * (M::TILE >> 4);
            const uint32_t qS = qLo + (uint32_t)t * (M::TILE >> 4);
            const uint32_t dS = tmem + kColS + t * 128;
#pragma unroll
            for (int kk = 0; kk < 4 * NB; kk++) {
                const uint32_t off = ((kk >> 2) * kBlock + (kk & 3) * 32) >> 4;
                if (leader) mma_ss(dS, desc(kmajorHi, qS + off), desc(kmajorHi, kS + off), idescQK, kk > 0);
            }
            if (leader) {
                mma_commit(bar(B::S + t));
                if (j + 1 == nT[t]) mma_commit(bar(B::QFREE + t));  // the Q tile is no longer read
                // last score product that reads this K stage (tile 1 while it is still running, else tile 0)
                if (t == 1 || j >= nT[1]) mma_commit(bar(B::KEMPTY + (lc + (uint32_t)j) % M::STAGES));
            }
            __syncwarp();
        };
        auto issue_pv = [&](int t, int j) {
            const uint32_t vS = vLo + ((lc + (uint32_t)j) % M::STAGES) * (M::TILE >> 4);
            const uint32_t dO = tmem + kColO + t * 128, aP = tmem + kColS + t * 128;
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
                if (leader) mma_ts(dO, aP + kk * 8, desc(vHi, vS + ((kk * 16 * 128) >> 4)), idescPV, j > 0 || kk > 0);
            if (!mbar_wait(bar(B::P2 + t), (sc[t] + (uint32_t)j) & 1, abortFlag)) return false;  // second half of P (keys 64..127)
            fence_after();
#pragma unroll
            for (int kk = 4; kk < 8; kk++)
                if (leader) mma_ts(dO, aP + kk * 8, desc(vHi, vS + ((kk * 16 * 128) >> 4)), idescPV, 1);
            __syncwarp();
            return true;
        };
        Item w = {};
        for (int it = 0; okay && get_item(it, w); it++) {
            nT[0] = w.nT0;
            nT[1] = w.nT1;
            for (int t = 0; t < 2 && okay; t++) {
                if (nT[t] == 0) continue;
                okay = mbar_wait(bar(B::QREADY + t), uc[t] & 1, abortFlag);
                if (okay) okay = mbar_wait(bar(B::KFULL + lc % M::STAGES), (lc / M::STAGES) & 1, abortFlag);
                if (!okay) break;
                fence_after();
                issue_qk(t, 0);
            }
            for (int j = 0; j < w.nMax && okay; j++) {
                const uint32_t ring = lc + (uint32_t)j;
                const int st = ring % M::STAGES;
                for (int t = 0; t < 2 && okay; t++) {
                    if (j >= nT[t]) continue;
                    if (t == 0 || j >= nT[0]) {  // (tile 1 finds the stages its neighbour has already waited for)
                        okay = mbar_wait(bar(B::VFULL + st), (ring / M::STAGES) & 1, abortFlag);
                        if (okay && j + 1 < w.nMax) okay = mbar_wait(bar(B::KFULL + (ring + 1) % M::STAGES), ((ring + 1) / M::STAGES) & 1, abortFlag);
                    }
                    if (okay) okay = mbar_wait(bar(B::P + t), (sc[t] + (uint32_t)j) & 1, abortFlag);
                    if (!okay) break;
                    fence_after();
                    okay = issue_pv(t, j);
                    if (!okay) break;
                    if (j + 1 < nT[t]) issue_qk(t, j + 1);
                    else if (leader) mma_commit(bar(B::O + t));
                    // last product that reads this V stage (tile 1 while it is still running, else tile 0)
                    if (leader && (t == 1 || j >= nT[1])) mma_commit(bar(B::VEMPTY + st));
                    __syncwarp();
                }
            }
            lc += (uint32_t)w.nMax;
            for (int t = 0; t < 2; t++) {
                sc[t] += (uint32_t)nT[t];
                uc[t] += nT[t] > 0 ? 1u : 0u;
            }
        }
        if (!okay) *abortFlag = 1;
    } else {
        // ------------------------------------------------ softmax / epilogue -------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int t = warp >> 2;
        const int row = threadIdx.x & 127;  // TMEM lane = row of the tile: head (row % PACK), position (row / PACK)
        const uint32_t laneBase = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t colS = kColS + t * 128, colO = kColO + t * 128;
        const float scale = p.scaleLog2;
        bool okay = true;
        uint32_t sc = 0, uc = 0;  // parities of the key-tile steps / items this group has run so far
#pragma unroll 1
        for (int it = 0; okay; it++) {
            int n, pos, len, row0, kvHead, partial;
            {
                Item w;
                if (!get_item(it, w)) break;
                n = t == 0 ? w.nT0 : w.nT1;
                pos = w.pos + t * posTile;
                len = w.len;
                row0 = w.row0;
                kvHead = w.kvHead;
                partial = w.firstPartial;
            }
            if (n == 0) continue;
            const int seen = p.causal ? min(pos + (row >> p.packLog) + 1, len) : len;  // keys this row sees
            if (p.cosT) {
                okay = rotate_q_when_loaded<BF16, NB>(smem + M::Q + t * M::TILE, (warp & 3) * 32, lane, p.halves != 0, p.cosT, p.sinT, pos, p.posLast, p.packLog,
                                                      bar(B::Q + t), uc & 1, abortFlag);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // generic writes -> visible to the tensor core
            } else {
                okay = __all_sync(0xffffffffu, mbar_wait(bar(B::Q + t), uc & 1, abortFlag));
            }
            mbar_arrive(bar(B::QREADY + t));
            float mUsed = -INFINITY;  // the maximum the stored P and O are relative to (scaled, log2 domain)
            float lsum = 0.f;
            for (int j = 0; j < n && okay; j++) {
                okay = __all_sync(0xffffffffu, mbar_wait(bar(B::S + t), (sc ^ (uint32_t)j) & 1, abortFlag));
                if (!okay) break;
                fence_after();
                uint32_t sreg[128];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld32(laneBase + colS + c * 32, sreg + c * 32);
                tmem_wait_ld();
                if (j >= partial) {
                    const int left = seen - j * kKeys;  // keys of this tile that the row sees
#pragma unroll
                    for (int i = 0; i < 128; i++)
                        if (i >= left) sreg[i] = 0xFF800000u;  // -inf
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 128; i += 8) {
#pragma unroll
                    for (int u = 0; u < 4; u++) mx4[u] = fmax3(mx4[u], __uint_as_float(sreg[i + 2 * u]), __uint_as_float(sreg[i + 2 * u + 1]));
                }
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale;  // scale > 0
                // keep the old reference maximum unless the row maximum grew by more than 8 (a factor 256)
                const bool first = mUsed == -INFINITY;
                const bool grow = first ? (mx > -INFINITY) : (mx > mUsed + 8.0f);
                const float mNew = grow ? mx : mUsed;
                const float alpha = (grow && !first) ? ex2_approx(mUsed - mNew) : 1.0f;
                if (j > 0 && __any_sync(0xffffffffu, grow && !first)) {
#pragma unroll 1
                    for (int c = 0; c < 2 * NB; c++) {
                        uint32_t oreg[32];
                        tmem_ld32(laneBase + colO + c * 32, oreg);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) oreg[i] = __float_as_uint(__uint_as_float(oreg[i]) * alpha);
                        tmem_st32(laneBase + colO + c * 32, oreg);
                    }
                }
                lsum *= alpha;
                mUsed = mNew;
                const float negM = first && !grow ? 0.f : -mUsed;  // no score above -inf so far: every exponential is 0
                const uint64_t SC = pk2(scale, scale), NM = pk2(negM, negM);
                uint64_t sumA = pk2(0.f, 0.f), sumB = pk2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const uint64_t X01 = fma2(pk2(__uint_as_float(sreg[2 * i]), __uint_as_float(sreg[2 * i + 1])), SC, NM);
                    const uint64_t X23 = fma2(pk2(__uint_as_float(sreg[2 * i + 2]), __uint_as_float(sreg[2 * i + 3])), SC, NM);
                    float x0, x1, x2, x3;
                    un2(X01, x0, x1);
                    un2(X23, x2, x3);
                    const uint64_t E01 = pk2(ex2_approx(x0), ex2_approx(x1)), E23 = pk2(ex2_approx(x2), ex2_approx(x3));
                    sumA = add2(sumA, E01);
                    sumB = add2(sumB, E23);
                    float e0, e1, e2, e3;
                    un2(E01, e0, e1);
                    un2(E23, e2, e3);
                    sreg[i] = pack2<BF16>(e0, e1);
                    sreg[i + 1] = pack2<BF16>(e2, e3);
                    if (i == 30) {
                        tmem_st32(laneBase + colS, sreg);
                        tmem_wait_st();
                        fence_before();
                        mbar_arrive(bar(B::P + t));
                    }
                }
                tmem_st32(laneBase + colS + 32, sreg + 32);
                tmem_wait_st();
                fence_before();
                mbar_arrive(bar(B::P2 + t));
                float a0, a1, b0, b1;
                un2(sumA, a0, a1);
                un2(sumB, b0, b1);
                lsum += (a0 + a1) + (b0 + b1);
            }
            // wait for the last P V product, normalise, stage in the swizzled box layout.  The staging tile is shared by the groups in turn
            // (tile 0, tile 1, tile 0 of the next item, ...).  A count, not a barrier's parity: a group that had no tile in some items may
            // be several turns ahead.
            if (okay) okay = __all_sync(0xffffffffu, mbar_wait(bar(B::O + t), uc & 1, abortFlag));
            if (okay) okay = __all_sync(0xffffffffu, turn_wait(smem_u32(&turn), 2 * it + t, abortFlag));
            if (okay) {
                fence_after();
                const float inv = 1.0f / lsum;
                unsigned char* stage = smem + M::STAGING + row * 128;
#pragma unroll 1
                for (int c = 0; c < 2 * NB; c++) {
                    uint32_t oreg[32];
                    tmem_ld32(laneBase + colO + c * 32, oreg);
                    tmem_wait_ld();
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = __uint_as_float(oreg[i]) * inv;
                    if (*(volatile int*)&notFinite && c * 32 < p.dim) {
                        float x[32];  // (memory of its own: o stays in registers)
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i] = o[i];
                        add_not_finite<BF16>(x, p.v + ((size_t)row0 * p.kvHeads + kvHead) * p.dim + c * 32, (size_t)p.kvHeads * p.dim, partial * kKeys, seen,
                                             min(32, p.dim - c * 32));
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = x[i];
                    }
#pragma unroll
                    for (int v4 = 0; v4 < 4; v4++) {
                        Vec16 x;
#pragma unroll
                        for (int w = 0; w < 4; w++) x.w[w] = pack2<BF16>(o[v4 * 8 + 2 * w], o[v4 * 8 + 2 * w + 1]);
                        const int chunk = c * 4 + v4;  // 16-byte chunk of the row
                        *(Vec16*)(stage + (chunk >> 3) * kBlock + (((chunk & 7) ^ (row & 7)) * 16)) = x;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(bar(B::STAGED + t));
            } else {
                *abortFlag = 1;
            }
            sc ^= (uint32_t)n;
            uc ^= 1u;
        }
    }
    // ---------------------------------------------------- teardown ----------------------------------------------------
    fence_before();
    __syncthreads();
    if (abortShared && threadIdx.x == 0) atomicExch(p.errorFlag, 2);
    if (warp == 8) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// short sequences (no longer than kShortMax): a block per (sequence, KV head)
// ---------------------------------------------------------------------------------------------------------------------------------
// The tensor-core kernel spends a pipeline of five barriers and a 128 x 128 tile on a sequence of a few tokens, ~5 us per (sequence, head)
// and SM.  Here a block brings K (rotated once) and V of its sequence into shared memory and its warps take 16 rows each, the row being
// (position, query head of the group) so that all heads of the group share them: warp-level products (mma.sync), one launch, no list,
// no scratch.  Q is rotated in registers.  Elements that are not finite are taken out of V and added back as in the tile kernel.
// Shared-memory order: K in 16-byte pieces, the upper half of eight exchanged in odd rows (the eight lanes of a load read two rows);
// V with the dimensions of 32 reordered so that a lane's accumulators are eight neighbouring dimensions, piece ^ (row & 7) for the
// transposing loads.
constexpr int kShortMax = 160;
// Warps of a block.  The registers of 128 dimensions leave room for twelve warps on an SM: two blocks of six share K and V more often than three
// of four (30 sequences of up to 160 tokens, 16 heads 52 -> 42 us, one of 33 tokens 7.4 -> 7.1, 64 of up to 32 14.3 -> 14.7; eight: 53, 6.9, 19.3).
// With 64 dimensions four: 200 sequences of up to 96 tokens 21.2 us, 64 of 128 26.5 (three: 20.2 and 32.8, six: 24.7 and 28).
template <int D> constexpr int kShortWarps = D == 128 ? 6 : 4;

__device__ __forceinline__ void mma16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t at, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}

// sum + 0 * v for two elements: 0 while all are finite, NaN from the first that is not
template <bool BF16> __device__ __forceinline__ uint32_t times0(uint32_t v, uint32_t sum) {
    uint32_t d;
    if (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v), "r"(0u), "r"(sum));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v), "r"(0u), "r"(sum));
    return d;
}

struct ShortParams {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    Seqs seqs;
    const float *cosT, *sinT;
    int heads, kvHeads, dim, causal, ropeMode, rows;  // rows of shared memory: the longest sequence, a multiple of 32
    float scaleLog2;
};

template <bool BF16, int D>
__global__ void __launch_bounds__(kShortWarps<D> * 32) short_kernel(ShortParams p) {
    constexpr int PIECES = D / 8;  // 16-byte pieces of a row
    constexpr int WARPS = kShortWarps<D>;
    extern __shared__ __align__(128) unsigned char smemShort[];
    __shared__ int notFinite;
    int row0, end;
    if (!seq_rows(p.seqs, blockIdx.x, row0, end)) return;
    const int len = end - row0, group = p.heads / p.kvHeads, kvh = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int blocks = (len * group + 15) / 16;  // of 16 rows
    const int firstBlock = blockIdx.z * WARPS;
    if (firstBlock >= blocks) return;
    // keys that this block's rows see
    const int stride = gridDim.z * WARPS;
    const int lastBlock = firstBlock + (blocks - 1 - firstBlock) / stride * stride + WARPS - 1;
    const int keys = p.causal ? min(len, (min(lastBlock * 16 + 15, len * group - 1)) / group + 1) : len;
    const int padded = (keys + 31) & ~31;
    unsigned char* const kTile = smemShort;
    unsigned char* const vTile = smemShort + (size_t)p.rows * D * 2;
    if (threadIdx.x == 0) notFinite = 0;
    __syncthreads();
    const int half = p.dim / 2;
    const bool halves = p.ropeMode == 1;
    {
        // (four pieces of a thread are on their way before the first is used: the loop waits for memory once, not per piece)
        constexpr int KP = PIECES / 2, THREADS = WARPS * 32, U = 4;  // a thread takes pieces c and c + KP of a K row: partners in half mode
        for (int i0 = threadIdx.x; i0 < padded * KP; i0 += U * THREADS) {
            Vec16 a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + u * THREADS, r = i / KP, c = i % KP;
                a[u] = b[u] = Vec16{};
                if (r < keys) {
                    const uint16_t* src = p.k + ((size_t)(row0 + r) * p.kvHeads + kvh) * p.dim;
                    if (c * 8 < p.dim) a[u] = *(const Vec16*)(src + c * 8);
                    if ((c + KP) * 8 < p.dim) b[u] = *(const Vec16*)(src + (c + KP) * 8);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + u * THREADS, r = i / KP, c = i % KP;
                if (r >= padded) break;
                if (p.ropeMode != 2 && r < keys) {  // (dim == D)
                    const float* cr = p.cosT + (size_t)r * half;
                    const float* sr = p.sinT + (size_t)r * half;
                    if (halves) {
                        rotate8<BF16>(a[u], b[u], cr + 8 * c, sr + 8 * c, true);
                    } else {
                        rotate8<BF16>(a[u], a[u], cr + 4 * c, sr + 4 * c, false);
                        rotate8<BF16>(b[u], b[u], cr + 4 * (c + KP), sr + 4 * (c + KP), false);
                    }
                }
                const int x = (r & 1) << 2;
                *(Vec16*)(kTile + ((size_t)r * PIECES + (c ^ x)) * 16) = a[u];
                *(Vec16*)(kTile + ((size_t)r * PIECES + ((c + KP) ^ x)) * 16) = b[u];
            }
        }
        uint32_t found = 0;
        for (int i0 = threadIdx.x; i0 < padded * PIECES; i0 += 2 * U * THREADS) {
            Vec16 a[2 * U];
#pragma unroll
            for (int u = 0; u < 2 * U; u++) {
                const int i = i0 + u * THREADS, r = i / PIECES, c = i % PIECES;
                a[u] = Vec16{};
                if (r < keys && c * 8 < p.dim) a[u] = *(const Vec16*)(p.v + ((size_t)(row0 + r) * p.kvHeads + kvh) * p.dim + c * 8);
            }
#pragma unroll
            for (int u = 0; u < 2 * U; u++) {
                const int i = i0 + u * THREADS, r = i / PIECES, c = i % PIECES;
                if (r >= padded) break;
                // dimension 32G + 8a + 2q + e goes to place 32G + 8q + 2a + e
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    found = times0<BF16>(a[u].w[q], found);
                    *(uint32_t*)(vTile + ((size_t)r * PIECES + (((c & ~3) + q) ^ (r & 7))) * 16 + (c & 3) * 4) = a[u].w[q];
                }
            }
        }
        if (found & 0x7FFF7FFFu) notFinite = 1;
    }
    __syncthreads();
    if (notFinite) {
        for (int i = threadIdx.x; i < padded * PIECES * 4; i += WARPS * 32) {
            uint32_t* const w = (uint32_t*)vTile + i;
            const uint32_t bad = not_finite<BF16>(*w);
            *w &= ~((bad >> 15) * 0xFFFFu);
        }
        __syncthreads();
    }
    for (int blk = firstBlock + warp; blk < blocks; blk += stride) {
        const int rA = blk * 16 + g, rB = rA + 8, rows = len * group;
        const int posA = min(rA, rows - 1) / group, posB = min(rB, rows - 1) / group;
        const size_t atA = ((size_t)(row0 + posA) * p.heads + kvh * group + min(rA, rows - 1) - posA * group) * p.dim;
        const size_t atB = ((size_t)(row0 + posB) * p.heads + kvh * group + min(rB, rows - 1) - posB * group) * p.dim;
        // lane t holds dimensions 32m + 8t .. + 7 of rows g and g + 8; K is read in the same order, so the order of the products is free
        Vec16 qa[D / 32], qb[D / 32];
#pragma unroll
        for (int m = 0; m < D / 32; m++) {
            const int d = 32 * m + 8 * t;
            qa[m] = qb[m] = Vec16{};
            if (d < p.dim) {
                qa[m] = *(const Vec16*)(p.q + atA + d);
                qb[m] = *(const Vec16*)(p.q + atB + d);
            }
        }
        if (p.ropeMode != 2) {
#pragma unroll
            for (int m = 0; m < D / 64; m++) {
                const int c = halves ? 32 * m + 8 * t : 16 * m + 4 * t;
                rotate8<BF16>(qa[m], qa[m + D / 64], p.cosT + (size_t)posA * half + c, p.sinT + (size_t)posA * half + c, halves);
                rotate8<BF16>(qb[m], qb[m + D / 64], p.cosT + (size_t)posB * half + c, p.sinT + (size_t)posB * half + c, halves);
                if (!halves) {
                    const int c2 = c + D / 4;
                    rotate8<BF16>(qa[m + D / 64], qa[m], p.cosT + (size_t)posA * half + c2, p.sinT + (size_t)posA * half + c2, false);
                    rotate8<BF16>(qb[m + D / 64], qb[m], p.cosT + (size_t)posB * half + c2, p.sinT + (size_t)posB * half + c2, false);
                }
            }
        }
        const int seenA = p.causal ? posA + 1 : len, seenB = p.causal ? posB + 1 : len;
        const int last = p.causal ? min(blk * 16 + 15, rows - 1) / group + 1 : len;  // keys that any of the rows sees
        const int allSee = p.causal ? blk * 16 / group + 1 : len;                    // and that all of them see
        float o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
        for (int key0 = 0; key0 < last; key0 += 32) {
            float s[4][4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                const int key = key0 + 8 * n + g;
#pragma unroll
                for (int m = 0; m < D / 32; m++) {
                    const Vec16 b = *(const Vec16*)(kTile + ((size_t)key * PIECES + ((4 * m + t) ^ ((key & 1) << 2))) * 16);
                    mma16(s[n], qa[m].w[0], qb[m].w[0], qa[m].w[1], qb[m].w[1], b.w[0], b.w[1], BF16);
                    mma16(s[n], qa[m].w[2], qb[m].w[2], qa[m].w[3], qb[m].w[3], b.w[2], b.w[3], BF16);
                }
            }
            if (key0 + 32 > allSee) {
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int key = key0 + 8 * n + 2 * t + e;
                        if (key >= seenA) s[n][e] = -INFINITY;
                        if (key >= seenB) s[n][2 + e] = -INFINITY;
                    }
            }
            float topA = fmaxf(s[0][0], s[0][1]), topB = fmaxf(s[0][2], s[0][3]);
#pragma unroll
            for (int n = 1; n < 4; n++) {
                topA = fmax3(topA, s[n][0], s[n][1]);
                topB = fmax3(topB, s[n][2], s[n][3]);
            }
            topA = fmaxf(topA, __shfl_xor_sync(0xffffffffu, topA, 1));
            topB = fmaxf(topB, __shfl_xor_sync(0xffffffffu, topB, 1));
            topA = fmaxf(topA, __shfl_xor_sync(0xffffffffu, topA, 2));
            topB = fmaxf(topB, __shfl_xor_sync(0xffffffffu, topB, 2));
            const float nA = fmaxf(mA, topA * p.scaleLog2), nB = fmaxf(mB, topB * p.scaleLog2);
            const float fromA = nA == -INFINITY ? 0.f : nA, fromB = nB == -INFINITY ? 0.f : nB;  // nothing but scores of -inf so far
            const float aA = ex2_approx(mA - fromA), aB = ex2_approx(mB - fromB);
            mA = nA;
            mB = nB;
            if (key0 > 0 && __any_sync(0xffffffffu, aA != 1.f || aB != 1.f)) {
                lA *= aA;
                lB *= aB;
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    o[n][0] *= aA;
                    o[n][1] *= aA;
                    o[n][2] *= aB;
                    o[n][3] *= aB;
                }
            }
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    s[n][e] = ex2_approx(fmaf(s[n][e], p.scaleLog2, -fromA));
                    s[n][2 + e] = ex2_approx(fmaf(s[n][2 + e], p.scaleLog2, -fromB));
                    lA += s[n][e];
                    lB += s[n][2 + e];
                }
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                if (ks == 1 && key0 + 16 >= last) break;
                const uint32_t p0 = pack2<BF16>(s[2 * ks][0], s[2 * ks][1]), p1 = pack2<BF16>(s[2 * ks][2], s[2 * ks][3]);
                const uint32_t p2 = pack2<BF16>(s[2 * ks + 1][0], s[2 * ks + 1][1]), p3 = pack2<BF16>(s[2 * ks + 1][2], s[2 * ks + 1][3]);
                const int key = key0 + 16 * ks + (lane & 15);
#pragma unroll
                for (int n = 0; n < D / 8; n += 2) {
                    uint32_t b[4];  // dimensions 8n .. + 7 of keys 0 - 7 and 8 - 15, then the next eight dimensions
                    ldmatrix_trans(smem_u32(vTile + ((size_t)key * PIECES + ((n + (lane >> 4)) ^ (key & 7))) * 16), b);
                    mma16(o[n], p0, p1, p2, p3, b[0], b[1], BF16);
                    mma16(o[n + 1], p0, p1, p2, p3, b[2], b[3], BF16);
                }
            }
        }
        lA += __shfl_xor_sync(0xffffffffu, lA, 1);
        lB += __shfl_xor_sync(0xffffffffu, lB, 1);
        lA += __shfl_xor_sync(0xffffffffu, lA, 2);
        lB += __shfl_xor_sync(0xffffffffu, lB, 2);
        const float iA = 1.0f / lA, iB = 1.0f / lB;
#pragma unroll
        for (int m = 0; m < D / 32; m++) {
            const int d = 32 * m + 8 * t;
            if (d >= p.dim) continue;
            float x[8], y[8];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                x[2 * q] = o[4 * m + q][0] * iA;
                x[2 * q + 1] = o[4 * m + q][1] * iA;
                y[2 * q] = o[4 * m + q][2] * iB;
                y[2 * q + 1] = o[4 * m + q][3] * iB;
            }
            if (notFinite) {
                const uint16_t* v = p.v + ((size_t)row0 * p.kvHeads + kvh) * p.dim + d;
                float xs[8], ys[8];  // (memory of their own: x and y stay in registers)
#pragma unroll
                for (int i = 0; i < 8; i++) { xs[i] = x[i]; ys[i] = y[i]; }
                add_not_finite<BF16>(xs, v, (size_t)p.kvHeads * p.dim, 0, seenA, 8);
                add_not_finite<BF16>(ys, v, (size_t)p.kvHeads * p.dim, 0, seenB, 8);
#pragma unroll
                for (int i = 0; i < 8; i++) { x[i] = xs[i]; y[i] = ys[i]; }
            }
            if (rA < rows) *(Vec16*)(p.out + atA + d) = Vec16{{pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7])}};
            if (rB < rows) *(Vec16*)(p.out + atB + d) = Vec16{{pack2<BF16>(y[0], y[1]), pack2<BF16>(y[2], y[3]), pack2<BF16>(y[4], y[5]), pack2<BF16>(y[6], y[7])}};
        }
    }
}

// [total, heads, dim] 16-bit -> 3-D map (dim, head, row) with a box of 64 x boxHeads x boxRows and 128-byte swizzle
static bool make_map(CUtensorMap* tm, const void* base, bool bf16, uint32_t total, uint32_t heads, uint32_t dim, uint32_t boxHeads, uint32_t boxRows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {dim, heads, total};
    cuuint64_t strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)heads * dim * 2};
    cuuint32_t box[3] = {64, boxHeads, boxRows};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)base, dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Call {
    int dt;
    const void *q, *k, *v;
    void* out;
    Seqs seqs;
    uint32_t heads, kvHeads, dim, causal, ropeMode;
    const float *cosT, *sinT;
};

// the tensor-core path; false where it does not take the shape
static bool tiles_take(const Call& c) {
    if (c.dt != DT_BF16 && c.dt != DT_F16) return false;
    if (c.dim > 128 || c.dim % 8 != 0) return false;                       // TMA: rows and row pitches of 16-byte multiples
    if (c.ropeMode != 2 && c.dim % 16 != 0) return false;                  // the rotation's vectors
    const uintptr_t all = (uintptr_t)c.q | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.out;
    return (all & 15u) == 0 && encode_fn() != nullptr;
}

// heads of a group that share a tile: the largest power of two in the group
static int pack_log(uint32_t group) {
    int log = 0;
    while (log < 7 && group % (2u << log) == 0) log++;
    return log;
}

// Measured on both sides (us, short against tiles), calls of up to 160 tokens per sequence.
// 64 dimensions: short wins (64 sequences of 160, 4 heads per KV head 33 : 42, 28 heads on 4 46 : 77; 300 of 64, 12 KV heads 50 : 130, 8 heads per KV
// head 35 : 53; 64 of 128, 16 heads per KV head 23 : 26, of 160 33 : 30) except where the group fills the tiles to four fifths, the keys most of a key
// tile, and there are more than 2^18 rows in all: 300 of 96 with 8 heads per KV head 67 : 69, 32 134 : 120; 300 of 112 with 8 83 : 83, 16 87 : 78; 300 of
// 128 with 8 98 : 85, 12 80 : 69, 32 203 : 158; 300 of 160 with 12 112 : 95, 16 147 : 107; 64 of 128 with 32 40 : 39, of 160 63 : 50.
// 128 dimensions, by rows (tokens x heads of a group) per sequence and KV head: 160 7.9 : 15.2 and 23 : 42, 192 28 : 43, 36 : 46 and 20 : 23, 256 54 : 43 and
// 163 : 134, 384 59 : 56, so up to 192; more where a group that is no power of two fills the tiles to a third at most (7 heads, 252 rows 18 : 77), or
// where few blocks let the shorter latency decide: one sequence of 128 tokens (8 x 512 rows) 12.4 : 13.2, of 160 13.8 : 13.6.
static bool short_takes(const Call& c) {
    if (!tiles_take(c) || c.seqs.maxLen > kShortMax || c.kvHeads > 65535 || (c.ropeMode != 2 && c.dim != 64 && c.dim != 128)) return false;
    const size_t rows = (size_t)c.seqs.maxLen * (c.heads / c.kvHeads), pairs = (size_t)c.seqs.batch * c.kvHeads;
    if (rows > 1u << 30) return false;  // a block counts its rows in 31 bits
    const int pack = pack_log(c.heads / c.kvHeads), span = 2 * (kRows >> pack);
    const size_t tileRows = ((size_t)c.seqs.maxLen + span - 1) / span * (c.heads / c.kvHeads >> pack) * 2 * kRows;
    if (c.dim <= 64) return c.seqs.maxLen < 96 || 5 * rows <= 4 * tileRows || pairs * rows <= 1u << 18;
    return rows <= 192 || 3 * rows <= tileRows || pairs * rows <= 4096;
}

template <bool BF16>
static int short_launch(Context* ctx, const Call& c, CUDAStatus* status) {
    const uint32_t group = c.heads / c.kvHeads, D = c.dim > 64 ? 128 : 64;
    ShortParams p{(const uint16_t*)c.q, (const uint16_t*)c.k, (const uint16_t*)c.v, (uint16_t*)c.out, c.seqs, c.cosT, c.sinT, (int)c.heads, (int)c.kvHeads,
                  (int)c.dim, (int)c.causal, (int)c.ropeMode, (c.seqs.maxLen + 31) & ~31, (float)(1.4426950408889634 / sqrt((double)c.dim))};
    const size_t warps = D == 128 ? kShortWarps<128> : kShortWarps<64>;
    // several blocks per (sequence, KV head) while there are too few to fill the GPU twice; each has 16 rows per warp at least
    const size_t pairs = (size_t)c.seqs.batch * c.kvHeads, most = ((size_t)c.seqs.maxLen * group + 16 * warps - 1) / (16 * warps);
    size_t split = (2 * (size_t)ctx->smCount + pairs - 1) / pairs;
    if (split > most) split = most;
    if (split > 65535) split = 65535;
    const size_t smem = (size_t)p.rows * D * 4;
    const dim3 grid((unsigned)c.seqs.batch, c.kvHeads, (unsigned)split);
#define SHORT(D)                                                                                                                        \
    do {                                                                                                                                \
        allow_smem<short_kernel<BF16, D>>(ctx->device, kShortMax * D * 4);                                                              \
        short_kernel<BF16, D><<<grid, kShortWarps<D> * 32, smem, ctx->stream>>>(p);                                                        \
    } while (0)
    if (D == 128) SHORT(128);
    else SHORT(64);
#undef SHORT
    return check_launch(ctx, status, "packed prefill attention (short)");
}

template <bool BF16>
static int tiles_launch(Context* ctx, const Call& c, CUDAStatus* status) {
    constexpr int DT = BF16 ? DT_BF16 : DT_F16;
    const uint32_t group = c.heads / c.kvHeads;
    const int packLog = pack_log(group), span = 2 * (kRows >> packLog);
    const uint32_t total = (uint32_t)c.seqs.total;
    const size_t levels = ((size_t)c.seqs.maxLen + span - 1) / span, most = (size_t)total / span + c.seqs.batch;  // entries at most
    const bool fused = c.ropeMode != 2 && (c.dim == 64 || c.dim == 128);  // q is rotated in its tile: a pass over q would cost as much as reading it all
    const size_t qBytes = c.ropeMode != 2 && !fused ? (((size_t)total * c.heads * c.dim * 2) + 255) & ~(size_t)255 : 0;
    const size_t kBytes = c.ropeMode != 2 ? (((size_t)total * c.kvHeads * c.dim * 2) + 255) & ~(size_t)255 : 0;
    if (most * c.heads > 0x3FFFFFFFull) return fail(status, -2, "packed prefill attention: %zu blocks of %u heads exceed the index range", most, c.heads);
    const size_t entryBytes = (most * sizeof(Entry) + 255) & ~(size_t)255;
    Scratch ws;
    int rc = call_scratch(ctx, qBytes + kBytes + entryBytes + 256 + 2 * levels * 4, 0, &ws, status);
    if (rc != 0) return rc;
    uint16_t* qRot = (uint16_t*)ws.base;
    uint16_t* kRot = (uint16_t*)(ws.base + qBytes);
    Lists l;
    l.entries = (Entry*)(ws.base + qBytes + kBytes);
    l.count = (int*)(ws.base + qBytes + kBytes + entryBytes);
    l.above = l.count + 64;
    l.cursor = l.above + levels;
    l.span = span;
    l.levels = (int)levels;
    l.capacity = (int)most;
    unsigned blocks = 1;
    if (c.ropeMode != 2) {
        const size_t want = ((size_t)total + 7) / 8, cap = (size_t)ctx->smCount * 8;
        blocks += (unsigned)(want < cap ? want : cap);
    }
    prologue_kernel<DT><<<blocks, 256, 0, ctx->stream>>>((const uint16_t*)c.q, (const uint16_t*)c.k, qRot, kRot, c.seqs, l, c.cosT, c.sinT, fused ? 0 : (int)c.heads,
                                                         (int)c.kvHeads, (int)c.dim, c.ropeMode == 1);
    rc = check_launch(ctx, status, "packed prefill attention: work list and RoPE");
    if (rc != 0) return rc;
    TileParams p;
    memset(&p, 0, sizeof(p));
    const void* q = c.ropeMode != 2 && !fused ? qRot : c.q;
    const void* k = c.ropeMode != 2 ? kRot : c.k;
    const uint32_t pack = 1u << packLog;
    if (!make_map(&p.tmQ, q, BF16, total, c.heads, c.dim, pack, kRows >> packLog) || !make_map(&p.tmK, k, BF16, total, c.kvHeads, c.dim, 1, kKeys) ||
        !make_map(&p.tmV, c.v, BF16, total, c.kvHeads, c.dim, 1, kKeys) || !make_map(&p.tmO, c.out, BF16, total, c.heads, c.dim, pack, kRows >> packLog))
        return fail(status, -7, "packed prefill attention: tensor map encoding failed");
    p.entries = l.entries;
    p.count = l.count;
    p.v = (const uint16_t*)c.v;
    p.out = (uint16_t*)c.out;
    p.errorFlag = ctx->errorFlag;
    p.heads = (int)c.heads; p.kvHeads = (int)c.kvHeads; p.dim = (int)c.dim; p.causal = (int)c.causal;
    p.cosT = fused ? c.cosT : nullptr;
    p.sinT = c.sinT;
    p.halves = c.ropeMode == 1;
    p.posLast = c.seqs.maxLen - 1;
    p.packLog = packLog;
    p.headGroups = (int)(c.heads >> packLog);
    p.scaleLog2 = (float)(1.4426950408889634 / sqrt((double)c.dim));
    const size_t items = most * p.headGroups;
    const unsigned grid = items < (size_t)ctx->smCount ? (unsigned)items : (unsigned)ctx->smCount;  // persistent: one CTA per SM
    // (started early, beside the launch before it, this kernel cost 10 of 305 us: its blocks need an SM each and wait for the other's to drain)
#define TILES(NB)                                                                                                                      \
    do {                                                                                                                               \
        allow_smem<tiles_kernel<BF16, NB>>(ctx->device, (int)Smem<NB>::TOTAL);                                                         \
        tiles_kernel<BF16, NB><<<grid, kThreads, Smem<NB>::TOTAL, ctx->stream>>>(p);                                                   \
    } while (0)
    if (c.dim > 64) TILES(2);
    else TILES(1);
#undef TILES
    return check_launch(ctx, status, "packed prefill attention");
}

}  // namespace pk

}  // namespace puter

using namespace puter;

extern "C" int cuda_dispatch_rope_packed_attention_prefill(CUDADeviceRef contextRef, int elementDType, CUDABufferRef queryRef,
                                                           CUDABufferRef keyRef, CUDABufferRef valueRef, CUDABufferRef seqStartsRef,
                                                           CUDABufferRef outRef, uint32_t batch, uint32_t totalTokens, uint32_t maxSeqLen,
                                                           uint32_t numHeads, uint32_t kvHeads, uint32_t headDim, uint32_t causal,
                                                           uint32_t ropeMode, double baseFreq, int64_t startPosition, uint32_t scaling,
                                                           double scalingFactor, double lowFreqFactor, double highFreqFactor,
                                                           uint32_t originalContext, uint64_t completionToken, CUDAStatus* status) {
    (void)completionToken;
    PUTER_ENTER(ctx);
    const char* what = "packed prefill attention";
    if (batch == 0 || totalTokens == 0 || maxSeqLen == 0 || numHeads == 0 || headDim == 0) return ok(status);
    if (kvHeads == 0) kvHeads = numHeads;
    if (numHeads % kvHeads != 0) return fail(status, -2, "%s: %u heads are not a multiple of %u KV heads", what, numHeads, kvHeads);
    if (elementDType != DT_F32 && elementDType != DT_F16 && elementDType != DT_BF16)
        return fail(status, -6, "%s: supported dtypes are float32, f16 and bf16 (got %d)", what, elementDType);
    if (headDim > 256) return fail(status, -6, "%s: head dimension %u exceeds 256", what, headDim);
    if (batch > 0x7FFFFFFEu || totalTokens > 0x7FFFFFFFu)
        return fail(status, -2, "%s: %u sequences of %u tokens in all exceed 31 bits", what, batch, totalTokens);
    if (ropeMode > 2) return fail(status, -2, "rope: unsupported mode %u", ropeMode);
    if (ropeMode != 2) {
        int rc = validate_rope(status, baseFreq, ropeMode, scaling, scalingFactor, lowFreqFactor, highFreqFactor, originalContext);
        if (rc != 0) return rc;
        if (headDim % 2 != 0) return fail(status, -2, "rope: head dimension must be even");
    }
    if (maxSeqLen > totalTokens) maxSeqLen = totalTokens;
    if ((size_t)numHeads * headDim > 0x7FFFFFFFull)  // the kernels count within a row in 31 bits
        return fail(status, -2, "%s: rows of %u heads of %u exceed 31 bits", what, numHeads, headDim);
    if ((size_t)totalTokens * numHeads > (size_t)1 << 48) return fail(status, -2, "%s: %u tokens of %u heads", what, totalTokens, numHeads);
    const size_t es = dtype_size(elementDType), qBytes = (size_t)totalTokens * numHeads * headDim * es,
                 kvBytes = (size_t)totalTokens * kvHeads * headDim * es;
    PUTER_REQUIRE(queryRef, "query", qBytes);
    PUTER_REQUIRE(keyRef, "key", kvBytes);
    PUTER_REQUIRE(valueRef, "value", kvBytes);
    PUTER_REQUIRE(seqStartsRef, "seqStarts", ((size_t)batch + 1) * 4);
    PUTER_REQUIRE(outRef, "out", qBytes);
    const void* q = dev_ptr(queryRef);
    const void* k = dev_ptr(keyRef);
    const void* v = dev_ptr(valueRef);
    void* out = dev_ptr(outRef);
    if (overlap(out, qBytes, q, qBytes) || overlap(out, qBytes, k, kvBytes) || overlap(out, qBytes, v, kvBytes))
        return fail(status, -2, "%s: out may not overlap an input", what);
    if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & (es - 1)) != 0 || ((uintptr_t)dev_ptr(seqStartsRef) & 3u) != 0)
        return fail(status, -2, "%s: a buffer is not aligned to its elements", what);
    if (ctx->exact) {
        int rc = check_mha_exact_packed(status, (int)maxSeqLen, numHeads, headDim);
        if (rc != 0) return rc;
    }
    const pk::Seqs seqs{(const int32_t*)dev_ptr(seqStartsRef), (int)batch, (int)totalTokens, (int)maxSeqLen, ctx->errorFlag};
    const float *table = nullptr, *sinT = nullptr;
    if (ropeMode != 2) {
        table = cached_rope_table_at_least(ctx, maxSeqLen, (int)headDim, baseFreq, (long long)startPosition, (int)scaling, scalingFactor,
                                           lowFreqFactor, highFreqFactor, (int)originalContext, &sinT, status);
        if (!table) return status ? status->code : -7;
    }
    const pk::Call c{elementDType, q, k, v, out, seqs, numHeads, kvHeads, headDim, causal ? 1u : 0u, ropeMode, table, sinT};
    if (!ctx->exact && pk::short_takes(c)) return elementDType == DT_BF16 ? pk::short_launch<true>(ctx, c, status) : pk::short_launch<false>(ctx, c, status);
    if (!ctx->exact && pk::tiles_take(c)) return elementDType == DT_BF16 ? pk::tiles_launch<true>(ctx, c, status) : pk::tiles_launch<false>(ctx, c, status);
    const int cap = ctx->smCount * 8;
    if (ropeMode != 2) {
        const size_t qAt = 0, kAt = (qBytes + 255) & ~(size_t)255;
        Scratch ws;
        int rc = call_scratch(ctx, kAt + kvBytes, 0, &ws, status);
        if (rc != 0) return rc;
#define ROTATE(DT, IN, AT, HEADS) \
    pk::rotate_kernel<DT><<<cap, 256, 0, ctx->stream>>>(IN, ws.base + AT, seqs, table, sinT, (int)(HEADS), (int)headDim, (int)ropeMode)
#define ROTATE_BOTH(DT)                                                   \
    do {                                                                  \
        ROTATE(DT, q, qAt, numHeads);                                     \
        rc = check_launch(ctx, status, "packed prefill attention: RoPE"); \
        if (rc != 0) return rc;                                           \
        ROTATE(DT, k, kAt, kvHeads);                                      \
    } while (0)
        if (elementDType == DT_F32) ROTATE_BOTH(DT_F32);
        else if (elementDType == DT_BF16) ROTATE_BOTH(DT_BF16);
        else ROTATE_BOTH(DT_F16);
#undef ROTATE_BOTH
#undef ROTATE
        rc = check_launch(ctx, status, "packed prefill attention: RoPE");
        if (rc != 0) return rc;
        q = ws.base + qAt;
        k = ws.base + kAt;
    }
    if (ctx->exact) return launch_mha_exact_packed(ctx, elementDType, q, k, v, out, seqs, numHeads, kvHeads, headDim, causal ? 1u : 0u, status);
    const size_t blocks = ((size_t)totalTokens * numHeads + 7) / 8;
    const int grid = blocks < (size_t)cap ? (int)blocks : cap;
    const float scaleLog2 = (float)(1.4426950408889634 / sqrt((double)headDim));
#define ROWS(DT) pk::rows_kernel<DT><<<grid, 256, 0, ctx->stream>>>(q, k, v, out, seqs, (int)numHeads, (int)kvHeads, (int)headDim, (int)causal, scaleLog2)
    if (elementDType == DT_F32) ROWS(DT_F32);
    else if (elementDType == DT_BF16) ROWS(DT_BF16);
    else ROWS(DT_F16);
#undef ROWS
    return check_launch(ctx, status, what);
}
