// The paged KV cache in 4 bits: its producer and the way back to 16 bits.
//
// A vector x of one (token, KV head) is held as 16 levels between its own extremes (no counterpart in the reference, whose cache is
// kept in the tensors' type):
//     least = rn16(min x),  step = rn16((max x - min x) * (1 / 15)),  code_d = clamp(rint((x_d - least) / step), 0, 15),
//     value_d = least + step * code_d,
// rn16 = rounding to the 16-bit type of the tensors (their range: a bf16 vector may hold 1e30).  The codes are chosen against the
// rounded step and least, so that rounding costs no accuracy but the cover of the extremes: in bf16 up to 15 / 256 of a step for the step's and
// 2^-8 of least for its own (0.4 of a step where least is a hundred steps), in f16 an eighth of both.
// A vector that holds a NaN or an infinity gets a step that is one of them: it reads back as NaN, never as finite numbers.  So does a finite one
// whose extremes lie further apart than float32 reaches (3.4e38, bf16).  K is rotated in float32 and not rounded before: a rotation that leaves f16
// (by a factor of 1.41 at most) gives an infinite least, as it gives an infinite element where K is kept in 16 bits.
//
// Layout: codes [page, kvHead, token, D / 2] bytes, byte j = element 2j in the low and 2j + 1 in the high four bits; params
// [page, kvHead, token, 2] = (step, least).  The head comes before the token so that the 16 tokens that a warp of the decode kernel
// takes of its head are one run of 16 * D / 2 bytes (and 64 of parameters) instead of 16 pieces.
//
// Both kernels stream: a group of D / 16 lanes holds a vector, sixteen elements a lane, so the extremes of a vector cost log2(D / 16)
// shuffles per bound and nothing goes through shared memory.  What bounds them and what was done about it is said at each.
#include <math.h>

#include "common.cuh"

namespace puter {

int validate_rope(CUDAStatus* status, double base, uint32_t halfMode, uint32_t scaling, double factor, double low, double high,
                  uint32_t origCtx);
const float* cached_rope_table_at_least(Context* ctx, size_t positions, int headDim, double base, long long startPos, int scaling,
                                        double factor, double low, double high, int origCtx, const float** sinT, CUDAStatus* status);

namespace q4 {

__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// of three
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// nearest level of t >= 0 (up to rounding) in units of s: rint(t / s) with the quotient's own rounding.  The product with the
// reciprocal is off by less than 4e-6 on 0 .. 15, so only a quotient that close to a tie is divided out: ties are common among
// 16-bit values, and they go to the even level as the division says.
__device__ __forceinline__ uint32_t level(float t, float s, float inv) {
    float y = t * inv;
    if (fabsf(fabsf(y - rintf(y)) - 0.5f) < 1e-5f || !(inv < 1e30f)) y = s > 0.f ? __fdiv_rn(t, s) : 0.f;
    return (uint32_t)__float2int_rn(fminf(fmaxf(y, 0.f), 15.f));
}

// Eight levels, packed: element i in bits 4i .. 4i + 3.  Where no clamp can act (see quantise) the quotient is a product with the
// reciprocal and one correction, which makes quotients that are ties exact; adding 1.5 * 2^23 rounds to nearest even and leaves the
// level in the lowest bits, and since shifting and adding is linear the constant above them comes off once at the end.
__device__ __forceinline__ uint32_t levels8(const float* x, float step, float least, float inv) {
    constexpr float kMagic = 12582912.f;  // 0x4B400000
    const uint64_t S = pk2(-step, -step), L = pk2(-least, -least), I = pk2(inv, inv), MAGIC = pk2(kMagic, kMagic);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t t = add2(pk2(x[i], x[i + 1]), L), q0 = mul2(t, I);
        const uint64_t q1 = fma2(fma2(q0, S, t), I, q0);
        un2(add2(q1, MAGIC), y[i], y[i + 1]);
    }
    uint32_t codes = __float_as_uint(y[7]);
#pragma unroll
    for (int i = 6; i >= 0; i--) codes = codes * 16u + __float_as_uint(y[i]);
    constexpr uint32_t kTop = 0x4B400000u * 0x11111111u;  // the constant in all eight places
    return codes - kTop;
}

// The sixteen elements of this lane, one vector per group of LANES lanes: packed codes of elements 0 - 7 and 8 - 15; params = step in the
// low, least in the high half.
template <int DT, int LANES>
__device__ __forceinline__ void quantise(const float* x, uint32_t& c0, uint32_t& c1, uint32_t& params) {
    float lo = min_nan(x[0], x[1]), hi = max_nan(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) {
        lo = min3_nan(lo, x[i], x[i + 1]);
        hi = max3_nan(hi, x[i], x[i + 1]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float step = __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f), least = lo;
    params = round_pair_arith<DT>(step, least);
    const float inv = 1.0f / step;
    // no element falls below level -0.4 or above 15.46 while the rounding of least (2^-8 of it at most) stays below 0.4 of a step and the
    // step is a normal number of its type (2^-8 off at most): then rounding alone keeps 0 .. 15
    const bool plain = fabsf(least) <= 100.f * step && step >= (DT == DT_F16 ? 6.103515625e-5f : 1e-30f) && step < INFINITY;
    if (__all_sync(0xffffffffu, plain)) {
        c0 = levels8(x, step, least, inv);
        c1 = levels8(x + 8, step, least, inv);
    } else {
        c0 = c1 = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            c0 |= level(__fsub_rn(x[i], least), step, inv) << (4 * i);
            c1 |= level(__fsub_rn(x[i + 8], least), step, inv) << (4 * i);
        }
    }
}

template <int DT> __device__ __forceinline__ void widen8(const Vec16& v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; i++) unpack16_arith<DT>(v.w[i], x[2 * i], x[2 * i + 1]);
}

// MODE 0: neighbouring pairs, 1: halves, 2: K comes rotated.
// Bound: no pipe is full (~10 instructions per element against the 14 that the memory system leaves time for; issue slots 65 %, logic pipe 49 %): a
// warp waits for its loads, and 60 registers leave four blocks on an SM.  Every lane has 64 bytes of K and V in flight before it looks at its
// indices.  59748 rows of 8 KV heads of 128 in bf16, rotated: 70 us for 310 MB, 4.5 TB/s (47 us at the copy rate); 64 rows 2.7 us.  The next
// vectors fetched a round ahead made it slower (78 us in registers, 74 through shared memory).
template <int DT, int D, int MODE>
__global__ void __launch_bounds__(256) append_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                     const int32_t* __restrict__ positions, const int32_t* __restrict__ pageIDs,
                                                     const int32_t* __restrict__ offsets, uint8_t* __restrict__ kCodes,
                                                     uint32_t* __restrict__ kParams, uint8_t* __restrict__ vCodes,
                                                     uint32_t* __restrict__ vParams, const float* __restrict__ cosT,
                                                     const float* __restrict__ sinT, uint32_t vectors, uint32_t kvHeads, uint32_t pageCount,
                                                     uint32_t pageSize, uint32_t maxPositions, int* __restrict__ errorFlag) {
    constexpr uint32_t LANES = D / 16, PER = 32 / LANES;  // lanes per vector, vectors of a warp
    const uint32_t lane = threadIdx.x & 31, j = lane % LANES;
    const size_t stride = (size_t)gridDim.x * (blockDim.x >> 5) * PER;
    for (size_t first = ((size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * PER; first < vectors; first += stride) {
        const bool have = first + lane / LANES < vectors;
        const uint32_t vec = have ? (uint32_t)first + lane / LANES : vectors - 1;
        const uint32_t row = vec / kvHeads, head = vec - row * kvHeads;
        const size_t src = (size_t)vec * D;
        const uint32_t at0 = MODE == 1 ? 8 * j : 16 * j, at1 = MODE == 1 ? D / 2 + 8 * j : 16 * j + 8;
        const Vec16 k0 = ld_stream(k + src + at0), k1 = ld_stream(k + src + at1);
        const Vec16 v0 = ld_stream(v + src + 16 * j), v1 = ld_stream(v + src + 16 * j + 8);
        const int page = pageIDs[row], off = offsets[row], pos = MODE == 2 ? 0 : positions[row];
        const bool good = page >= 0 && (uint32_t)page < pageCount && off >= 0 && (uint32_t)off < pageSize && pos >= 0 &&
                          (MODE == 2 || (uint32_t)pos < maxPositions);
        if (!good) atomicExch(errorFlag, 1);
        float x[16], y[16];
        widen8<DT>(k0, x);
        widen8<DT>(k1, x + 8);
        if (MODE != 2) {
            const size_t turn = (size_t)(good ? pos : 0) * (D / 2) + 8 * j;
            float cs[8], sn[8];
            *(float4*)cs = __ldg((const float4*)(cosT + turn));
            *(float4*)(cs + 4) = __ldg((const float4*)(cosT + turn + 4));
            *(float4*)sn = __ldg((const float4*)(sinT + turn));
            *(float4*)(sn + 4) = __ldg((const float4*)(sinT + turn + 4));
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int a = MODE == 1 ? i : 2 * i, b = MODE == 1 ? i + 8 : 2 * i + 1;
                const float e = x[a], o = x[b];
                x[a] = sub(mul(e, cs[i]), mul(o, sn[i]));
                x[b] = add(mul(e, sn[i]), mul(o, cs[i]));
            }
        }
        uint32_t kc0, kc1, kp, vc0, vc1, vp;
        quantise<DT, (int)LANES>(x, kc0, kc1, kp);
        widen8<DT>(v0, y);
        widen8<DT>(v1, y + 8);
        quantise<DT, (int)LANES>(y, vc0, vc1, vp);
        if (have && good) {
            const size_t slot = ((size_t)page * kvHeads + head) * pageSize + (uint32_t)off;
            if (MODE == 1) {
                *(uint32_t*)(kCodes + slot * (D / 2) + 4 * j) = kc0;
                *(uint32_t*)(kCodes + slot * (D / 2) + D / 4 + 4 * j) = kc1;
            } else {
                *(uint2*)(kCodes + slot * (D / 2) + 8 * j) = make_uint2(kc0, kc1);
            }
            *(uint2*)(vCodes + slot * (D / 2) + 8 * j) = make_uint2(vc0, vc1);
            if (j == 0) {
                kParams[slot] = kp;
                vParams[slot] = vp;
            }
        }
    }
}

// two elements: rn16(least + step * code) by one fused multiply-add of the 16-bit type, which rounds the exact sum once
template <int DT> __device__ __forceinline__ uint32_t value2(uint32_t byte, uint32_t step2, uint32_t least2) {
    constexpr uint32_t kOne = DT == DT_BF16 ? 0x3F803F80u : 0x3C003C00u;
    constexpr uint32_t kBase = DT == DT_BF16 ? 0x43004300u : 0x64006400u;   // 128 / 1024: a unit in the last place is 1
    uint32_t n = ((byte * 0x1001u) & 0x000F000Fu) | kBase, r;               // low four bits in the low half, high four in the high half
    if (DT == DT_BF16) {
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(n) : "r"(n), "r"(kOne), "r"(kBase | 0x80008000u));
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(n), "r"(step2), "r"(least2));
    } else {
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(n) : "r"(n), "r"(kOne), "r"(kBase | 0x80008000u));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(n), "r"(step2), "r"(least2));
    }
    return r;
}

// out[row] = rn16(least + step * code), row r from page table[r / pageSize], slot r % pageSize.
// Bound: the copies in flight (8 bytes of codes a lane turn into 32 bytes of output), so a lane starts UNROLL vectors before it finishes
// the first, and stores whole 32-byte sectors.  131072 rows of 8 heads of 128 in bf16: 57 us for 340 MB, 5.9 TB/s (52 us at the copy rate);
// four vectors ahead 73 us, eight 70.  1000 rows 2.6 us.
template <int DT, int D, bool WIDE>
__global__ void __launch_bounds__(256) gather_kernel(const uint8_t* __restrict__ codes, const uint32_t* __restrict__ params,
                                                     const int32_t* __restrict__ table, uint16_t* __restrict__ out, uint32_t vectors,
                                                     uint32_t kvHeads, uint32_t pageCount, uint32_t pageSize, int* __restrict__ errorFlag) {
    constexpr uint32_t LANES = D / 16, PER = 32 / LANES;
    constexpr int UNROLL = 2;
    const uint32_t lane = threadIdx.x & 31, j = lane % LANES;
    const size_t stride = (size_t)gridDim.x * (blockDim.x >> 5) * PER;
    for (size_t first = ((size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * PER + lane / LANES; first < vectors; first += UNROLL * stride) {
        uint2 c[UNROLL];
        uint32_t par[UNROLL];
        bool good[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const size_t vec = first + u * stride;
            good[u] = false;
            if (vec < vectors) {
                const uint32_t row = (uint32_t)vec / kvHeads, head = (uint32_t)vec - row * kvHeads, entry = row / pageSize;
                const int page = __ldg(table + entry);
                good[u] = page >= 0 && (uint32_t)page < pageCount;
                if (!good[u]) atomicExch(errorFlag, 1);
                const size_t slot = good[u] ? ((size_t)page * kvHeads + head) * pageSize + (row - entry * pageSize) : 0;
                c[u] = __ldcs((const uint2*)(codes + slot * (D / 2) + 8 * j));
                par[u] = __ldg(params + slot);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            if (!good[u]) continue;
            const uint32_t step2 = __byte_perm(par[u], 0, 0x1010), least2 = __byte_perm(par[u], 0, 0x3232);
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                o[i] = value2<DT>((c[u].x >> (8 * i)) & 255u, step2, least2);
                o[4 + i] = value2<DT>((c[u].y >> (8 * i)) & 255u, step2, least2);
            }
            uint16_t* dst = out + (first + u * stride) * D + 16 * j;
            if (WIDE) {
                asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                             ::"l"(dst), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
            } else {
                st_stream(dst, Vec16{{o[0], o[1], o[2], o[3]}});
                st_stream(dst + 8, Vec16{{o[4], o[5], o[6], o[7]}});
            }
        }
    }
}

static int grid_of(Context* ctx, size_t warps) {
    // 8 blocks of 256 threads fill an SM in the gather; the producer's registers leave room for 4, and 4, 8 and 16 times the SMs take it equally long
    const size_t blocks = (warps + 8) / 8, cap = (size_t)ctx->smCount * 8;
    return (int)(blocks < cap ? (blocks ? blocks : 1) : cap);
}

}  // namespace q4

}  // namespace puter

using namespace puter;

extern "C" int cuda_dispatch_rope_kv_page_write_q4(CUDADeviceRef contextRef, int elementDType, CUDABufferRef kRef, CUDABufferRef vRef,
                                                   CUDABufferRef positionsRef, CUDABufferRef pageIDsRef, CUDABufferRef offsetsRef,
                                                   CUDABufferRef kCodesRef, CUDABufferRef kParamsRef, CUDABufferRef vCodesRef,
                                                   CUDABufferRef vParamsRef, uint32_t rows, uint32_t kvHeads, uint32_t headDim,
                                                   uint32_t pageCount, uint32_t pageSize, uint32_t maxPositions, uint32_t ropeMode,
                                                   double baseFreq, uint32_t scaling, double scalingFactor, double lowFreqFactor,
                                                   double highFreqFactor, uint32_t originalContext, uint64_t completionToken,
                                                   CUDAStatus* status) {
    (void)completionToken;
    PUTER_ENTER(ctx);
    if (rows == 0 || kvHeads == 0 || pageCount == 0 || pageSize == 0) return ok(status);
    if (elementDType != DT_F16 && elementDType != DT_BF16) return fail(status, -6, "rope kv page write (4 bits): unsupported dtype %d", elementDType);
    if (headDim != 64 && headDim != 128)
        return fail(status, -6, "rope kv page write (4 bits): head dimension %u is not 64 or 128", headDim);
    if (ropeMode > 2) return fail(status, -2, "rope: unsupported mode %u", ropeMode);
    if (ropeMode != 2) {
        int rc = validate_rope(status, baseFreq, ropeMode, scaling, scalingFactor, lowFreqFactor, highFreqFactor, originalContext);
        if (rc != 0) return rc;
        if (maxPositions == 0) return fail(status, -2, "rope kv page write (4 bits): maxPositions must be positive");
        PUTER_REQUIRE(positionsRef, "positions", (size_t)rows * 4);
    }
    if ((size_t)rows * kvHeads > 0xFFFFFFFFull) return fail(status, -2, "rope kv page write (4 bits): %u rows of %u heads exceed 32 bits", rows, kvHeads);
    const size_t inner = (size_t)kvHeads * headDim, slots = pool_vectors(pageCount, pageSize, kvHeads);
    if (slots > kMostVectors) return fail(status, -2, "rope kv page write (4 bits): %u pages of %u tokens and %u heads", pageCount, pageSize, kvHeads);
    PUTER_REQUIRE(kRef, "k", (size_t)rows * inner * 2);
    PUTER_REQUIRE(vRef, "v", (size_t)rows * inner * 2);
    PUTER_REQUIRE(pageIDsRef, "pageIDs", (size_t)rows * 4);
    PUTER_REQUIRE(offsetsRef, "offsets", (size_t)rows * 4);
    PUTER_REQUIRE(kCodesRef, "kCodes", slots * (headDim / 2));
    PUTER_REQUIRE(vCodesRef, "vCodes", slots * (headDim / 2));
    PUTER_REQUIRE(kParamsRef, "kParams", slots * 4);
    PUTER_REQUIRE(vParamsRef, "vParams", slots * 4);
    if ((((uintptr_t)dev_ptr(kRef) | (uintptr_t)dev_ptr(vRef) | (uintptr_t)dev_ptr(kCodesRef) | (uintptr_t)dev_ptr(vCodesRef) |
          (uintptr_t)dev_ptr(kParamsRef) | (uintptr_t)dev_ptr(vParamsRef)) & 15u) != 0)
        return fail(status, -2, "rope kv page write (4 bits): buffers must be 16-byte aligned");
    if ((((uintptr_t)(ropeMode == 2 ? nullptr : dev_ptr(positionsRef)) | (uintptr_t)dev_ptr(pageIDsRef) | (uintptr_t)dev_ptr(offsetsRef)) & 3u) != 0)
        return fail(status, -2, "rope kv page write (4 bits): positions, pageIDs and offsets must be 4-byte aligned");
    const float *table = nullptr, *sinT = nullptr;
    if (ropeMode != 2) {
        table = cached_rope_table_at_least(ctx, maxPositions, (int)headDim, baseFreq, 0, (int)scaling, scalingFactor, lowFreqFactor, highFreqFactor,
                                           (int)originalContext, &sinT, status);
        if (!table) return status ? status->code : -7;
    }
    const uint32_t vectors = rows * kvHeads;
    const int grid = q4::grid_of(ctx, (size_t)vectors * headDim / 512);
#define APPEND_LAUNCH(DT, D, MODE)                                                                                                  \
    q4::append_kernel<DT, D, MODE><<<grid, 256, 0, ctx->stream>>>(                                                                  \
        (const uint16_t*)dev_ptr(kRef), (const uint16_t*)dev_ptr(vRef), MODE == 2 ? nullptr : (const int32_t*)dev_ptr(positionsRef), \
        (const int32_t*)dev_ptr(pageIDsRef), (const int32_t*)dev_ptr(offsetsRef), (uint8_t*)dev_ptr(kCodesRef),                     \
        (uint32_t*)dev_ptr(kParamsRef), (uint8_t*)dev_ptr(vCodesRef), (uint32_t*)dev_ptr(vParamsRef), table, sinT, vectors, kvHeads, \
        pageCount, pageSize, maxPositions, ctx->errorFlag)
#define APPEND_PICK(DT, D)                                 \
    do {                                                   \
        if (ropeMode == 0) APPEND_LAUNCH(DT, D, 0);        \
        else if (ropeMode == 1) APPEND_LAUNCH(DT, D, 1);   \
        else APPEND_LAUNCH(DT, D, 2);                      \
    } while (0)
    if (elementDType == DT_BF16) {
        if (headDim == 128) APPEND_PICK(DT_BF16, 128);
        else APPEND_PICK(DT_BF16, 64);
    } else {
        if (headDim == 128) APPEND_PICK(DT_F16, 128);
        else APPEND_PICK(DT_F16, 64);
    }
#undef APPEND_PICK
#undef APPEND_LAUNCH
    return check_launch(ctx, status, "rope kv page write (4 bits)");
}

extern "C" int cuda_dispatch_kv_page_gather_q4(CUDADeviceRef contextRef, int elementDType, CUDABufferRef codesRef, CUDABufferRef paramsRef,
                                               CUDABufferRef pageTableRef, CUDABufferRef outputRef, uint32_t pageCount, uint32_t pageSize,
                                               uint32_t kvHeads, uint32_t headDim, uint32_t outRows, uint64_t completionToken,
                                               CUDAStatus* status) {
    (void)completionToken;
    PUTER_ENTER(ctx);
    if (pageCount == 0 || pageSize == 0 || kvHeads == 0 || outRows == 0) return ok(status);
    if (elementDType != DT_F16 && elementDType != DT_BF16) return fail(status, -6, "page gather (4 bits): unsupported dtype %d", elementDType);
    if (headDim != 64 && headDim != 128) return fail(status, -6, "page gather (4 bits): head dimension %u is not 64 or 128", headDim);
    if ((size_t)outRows * kvHeads > 0xFFFFFFFFull) return fail(status, -2, "page gather (4 bits): %u rows of %u heads exceed 32 bits", outRows, kvHeads);
    const size_t slots = pool_vectors(pageCount, pageSize, kvHeads);
    if (slots > kMostVectors) return fail(status, -2, "page gather (4 bits): %u pages of %u tokens and %u heads", pageCount, pageSize, kvHeads);
    PUTER_REQUIRE(codesRef, "codes", slots * (headDim / 2));
    PUTER_REQUIRE(paramsRef, "params", slots * 4);
    PUTER_REQUIRE(pageTableRef, "pageTable", (((size_t)outRows + pageSize - 1) / pageSize) * 4);
    PUTER_REQUIRE(outputRef, "output", (size_t)outRows * kvHeads * headDim * 2);
    if ((((uintptr_t)dev_ptr(codesRef) | (uintptr_t)dev_ptr(paramsRef) | (uintptr_t)dev_ptr(outputRef)) & 15u) != 0)
        return fail(status, -2, "page gather (4 bits): buffers must be 16-byte aligned");
    if (((uintptr_t)dev_ptr(pageTableRef) & 3u) != 0) return fail(status, -2, "page gather (4 bits): pageTable must be 4-byte aligned");
    const uint32_t vectors = outRows * kvHeads;
    const int grid = q4::grid_of(ctx, (size_t)vectors * headDim / 512);
    const bool wide = ((uintptr_t)dev_ptr(outputRef) & 31u) == 0;
#define GATHER_KERNEL(DT, D, WIDE)                                                                                                    \
    q4::gather_kernel<DT, D, WIDE><<<grid, 256, 0, ctx->stream>>>((const uint8_t*)dev_ptr(codesRef), (const uint32_t*)dev_ptr(paramsRef), \
                                                                  (const int32_t*)dev_ptr(pageTableRef), (uint16_t*)dev_ptr(outputRef), \
                                                                  vectors, kvHeads, pageCount, pageSize, ctx->errorFlag)
#define GATHER_LAUNCH(DT, D)                          \
    do {                                              \
        if (wide) GATHER_KERNEL(DT, D, true);         \
        else GATHER_KERNEL(DT, D, false);             \
    } while (0)
    if (elementDType == DT_BF16) {
        if (headDim == 128) GATHER_LAUNCH(DT_BF16, 128);
        else GATHER_LAUNCH(DT_BF16, 64);
    } else {
        if (headDim == 128) GATHER_LAUNCH(DT_F16, 128);
        else GATHER_LAUNCH(DT_F16, 64);
    }
#undef GATHER_LAUNCH
#undef GATHER_KERNEL
    return check_launch(ctx, status, "page gather (4 bits)");
}
