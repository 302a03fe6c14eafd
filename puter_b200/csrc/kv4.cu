// The paged KV cache in 4 bits: its producer and the way back to 16 bits.
//
// A vector x of one (token, KV head) is held as 16 levels between its own extremes (no counterpart in the reference, whose cache is
// kept in the tensors' type):
//     least = rn16(min x),  step = rn16((max x - min x) / 15),  code_d = clamp(rint((x_d - least) / step), 0, 15),
//     value_d = least + step * code_d,
// rn16 = rounding to the 16-bit type of the tensors (their range: a bf16 vector may hold 1e30).  The codes are chosen against the
// rounded step and least, so that rounding costs no accuracy but the cover of the extremes (at most 15 / 512 of a step in bf16).
// A vector that holds a NaN or an infinity gets a NaN step: it reads back as NaN, never as finite numbers.
//
// Layout: codes [page, kvHead, token, D / 2] bytes, byte j = element 2j in the low and 2j + 1 in the high four bits; params
// [page, kvHead, token, 2] = (step, least).  The head comes before the token so that the 16 tokens that a warp of the decode kernel
// takes of its head are one run of 16 * D / 2 bytes (and 64 of parameters) instead of 16 pieces.
//
// Both kernels stream: a group of D / 8 lanes holds a vector, eight elements a lane, so the extremes of a vector cost log2(D / 8)
// shuffles and nothing goes through shared memory.
#include <math.h>

#include "common.cuh"

namespace puter {

int validate_rope(CUDAStatus* status, double base, uint32_t halfMode, uint32_t scaling, double factor, double low, double high,
                  uint32_t origCtx);
const float* cached_rope_table(Context* ctx, size_t seqLen, int headDim, double base, long long startPos, int scaling, double factor,
                               double low, double high, int origCtx, CUDAStatus* status);

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

// nearest level of t >= 0 (up to rounding) in units of s: rint(t / s) with the quotient's own rounding.  The product with the
// reciprocal is off by less than 4e-6 on 0 .. 15, so only a quotient that close to a tie is divided out: ties are common among
// 16-bit values, and they go to the even level as the division says.
__device__ __forceinline__ uint32_t level(float t, float s, float inv) {
    float y = t * inv;
    if (fabsf(fabsf(y - rintf(y)) - 0.5f) < 1e-5f || !(inv < 1e30f)) y = s > 0.f ? __fdiv_rn(t, s) : 0.f;
    return (uint32_t)__float2int_rn(fminf(fmaxf(y, 0.f), 15.f));
}

// The eight elements of this lane, one vector per group of LANES lanes: packed codes (element i in bits 4i .. 4i + 3); params = step
// in the low, least in the high half.
template <int DT, int LANES>
__device__ __forceinline__ uint32_t quantise(const float* x, uint32_t& params) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        lo = min_nan(lo, x[i]);
        hi = max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float step = __fdiv_rn(__fsub_rn(hi, lo), 15.f), least = lo;
    params = round_pair_arith<DT>(step, least);
    const float inv = 1.0f / step;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) codes |= level(__fsub_rn(x[i], least), step, inv) << (4 * i);
    return codes;
}

template <int DT> __device__ __forceinline__ void widen8(const Vec16& v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; i++) unpack16_arith<DT>(v.w[i], x[2 * i], x[2 * i + 1]);
}

// MODE 0: neighbouring pairs, 1: halves, 2: K comes rotated
template <int DT, int D, int MODE>
__global__ void __launch_bounds__(256) append_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                     const int32_t* __restrict__ positions, const int32_t* __restrict__ pageIDs,
                                                     const int32_t* __restrict__ offsets, uint8_t* __restrict__ kCodes,
                                                     uint32_t* __restrict__ kParams, uint8_t* __restrict__ vCodes,
                                                     uint32_t* __restrict__ vParams, const float* __restrict__ cosT,
                                                     const float* __restrict__ sinT, uint32_t rows, uint32_t kvHeads, uint32_t pageCount,
                                                     uint32_t pageSize, uint32_t maxPositions, int* __restrict__ errorFlag) {
    constexpr int LANES = D / 8, HEADS = 32 / LANES;  // lanes per vector, heads per pass of a warp
    const uint32_t lane = threadIdx.x & 31, j = lane % LANES;
    const uint32_t passes = (kvHeads + HEADS - 1) / HEADS;
    const size_t units = (size_t)rows * passes, warps = (size_t)gridDim.x * (blockDim.x >> 5);
    for (size_t u = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        const size_t row = u / passes;
        const uint32_t pass = (uint32_t)(u - row * passes), head = pass * HEADS + lane / LANES;
        const bool live = head < kvHeads;
        const size_t src = (row * kvHeads + (live ? head : 0)) * D;
        const int page = pageIDs[row], off = offsets[row], pos = MODE == 2 ? 0 : positions[row];
        // (fetched before the indices are looked at: they are one more round trip away)
        uint2 ka, kb;
        if (MODE == 1) {
            ka = __ldcs((const uint2*)(k + src + 4 * j));
            kb = __ldcs((const uint2*)(k + src + D / 2 + 4 * j));
        } else {
            const Vec16 t = ld_stream(k + src + 8 * j);
            ka = make_uint2(t.w[0], t.w[1]);
            kb = make_uint2(t.w[2], t.w[3]);
        }
        const Vec16 vr = ld_stream(v + src + 8 * j);
        if (page < 0 || (uint32_t)page >= pageCount || off < 0 || (uint32_t)off >= pageSize ||
            (MODE != 2 && (pos < 0 || (uint32_t)pos >= maxPositions))) {
            if (lane == 0) atomicExch(errorFlag, 1);
            continue;
        }
        float x[8], y[8];
        unpack16_arith<DT>(ka.x, x[0], x[1]);
        unpack16_arith<DT>(ka.y, x[2], x[3]);
        unpack16_arith<DT>(kb.x, x[4], x[5]);
        unpack16_arith<DT>(kb.y, x[6], x[7]);
        if (MODE != 2) {
            const float4 c = __ldg((const float4*)(cosT + (size_t)pos * (D / 2) + 4 * j));
            const float4 s = __ldg((const float4*)(sinT + (size_t)pos * (D / 2) + 4 * j));
            const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int a = MODE == 1 ? i : 2 * i, b = MODE == 1 ? i + 4 : 2 * i + 1;
                const float e = x[a], o = x[b];
                x[a] = sub(mul(e, cs[i]), mul(o, sn[i]));
                x[b] = add(mul(e, sn[i]), mul(o, cs[i]));
            }
        }
        uint32_t kp, vp;
        const uint32_t kc = quantise<DT, LANES>(x, kp);
        widen8<DT>(vr, y);
        const uint32_t vc = quantise<DT, LANES>(y, vp);
        // halves: this lane holds two bytes of either half; neighbours trade so that each stores one word
        uint32_t kw = kc, kAt = 4 * j;
        if (MODE == 1) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, (j & 1) ? (kc & 0xFFFFu) : (kc >> 16), 1);
            kw = (j & 1) ? (got | (kc & 0xFFFF0000u)) : ((kc & 0xFFFFu) | (got << 16));
            kAt = (j & 1) ? D / 4 + 2 * (j - 1) : 2 * j;
        }
        if (live) {
            const size_t slot = ((size_t)page * kvHeads + head) * pageSize + (uint32_t)off;
            *(uint32_t*)(kCodes + slot * (D / 2) + kAt) = kw;
            *(uint32_t*)(vCodes + slot * (D / 2) + 4 * j) = vc;
            if (j == 0) {
                kParams[slot] = kp;
                vParams[slot] = vp;
            }
        }
    }
}

// out[row] = rn16(least + step * code), row r from page table[r / pageSize], slot r % pageSize
template <int DT, int D>
__global__ void __launch_bounds__(256) gather_kernel(const uint8_t* __restrict__ codes, const uint32_t* __restrict__ params,
                                                     const int32_t* __restrict__ table, uint16_t* __restrict__ out, uint32_t rows,
                                                     uint32_t kvHeads, uint32_t pageCount, uint32_t pageSize, int* __restrict__ errorFlag) {
    constexpr int LANES = D / 8, HEADS = 32 / LANES;
    const uint32_t lane = threadIdx.x & 31, j = lane % LANES;
    const uint32_t passes = (kvHeads + HEADS - 1) / HEADS;
    const size_t units = (size_t)rows * passes, warps = (size_t)gridDim.x * (blockDim.x >> 5);
    for (size_t u = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        const size_t row = u / passes;
        const uint32_t pass = (uint32_t)(u - row * passes), head = pass * HEADS + lane / LANES;
        const size_t entry = row / pageSize;
        const int page = table[entry];
        if (page < 0 || (uint32_t)page >= pageCount) {
            if (lane == 0) atomicExch(errorFlag, 1);
            continue;
        }
        if (head >= kvHeads) continue;
        const size_t slot = ((size_t)page * kvHeads + head) * pageSize + (row - entry * pageSize);
        const uint32_t c = __ldcs((const uint32_t*)(codes + slot * (D / 2) + 4 * j));
        float step, least;
        unpack16_arith<DT>(__ldg(params + slot), step, least);
        Vec16 o;
#pragma unroll
        for (int i = 0; i < 4; i++)
            o.w[i] = pack16_arith<DT>(fmaf(step, (float)((c >> (8 * i)) & 15u), least), fmaf(step, (float)((c >> (8 * i + 4)) & 15u), least));
        st_stream(out + (row * kvHeads + head) * D + 8 * j, o);
    }
}

static int grid_of(Context* ctx, size_t warps) {
    const size_t blocks = (warps + 7) / 8, cap = (size_t)ctx->smCount * 8;  // 8 blocks of 256 threads fill an SM
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
    const size_t inner = (size_t)kvHeads * headDim, slots = (size_t)pageCount * pageSize * kvHeads;
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
    const float* table = nullptr;
    if (ropeMode != 2) {
        table = cached_rope_table(ctx, maxPositions, (int)headDim, baseFreq, 0, (int)scaling, scalingFactor, lowFreqFactor, highFreqFactor,
                                  (int)originalContext, status);
        if (!table) return status ? status->code : -7;
    }
    const float* sinT = table ? table + (size_t)maxPositions * (headDim / 2) : nullptr;
    const uint32_t heads = 256 / headDim;  // per pass of a warp
    const int grid = q4::grid_of(ctx, (size_t)rows * ((kvHeads + heads - 1) / heads));
#define APPEND_LAUNCH(DT, D, MODE)                                                                                                  \
    q4::append_kernel<DT, D, MODE><<<grid, 256, 0, ctx->stream>>>(                                                                  \
        (const uint16_t*)dev_ptr(kRef), (const uint16_t*)dev_ptr(vRef), MODE == 2 ? nullptr : (const int32_t*)dev_ptr(positionsRef), \
        (const int32_t*)dev_ptr(pageIDsRef), (const int32_t*)dev_ptr(offsetsRef), (uint8_t*)dev_ptr(kCodesRef),                     \
        (uint32_t*)dev_ptr(kParamsRef), (uint8_t*)dev_ptr(vCodesRef), (uint32_t*)dev_ptr(vParamsRef), table, sinT, rows, kvHeads,   \
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
    const size_t slots = (size_t)pageCount * pageSize * kvHeads;
    PUTER_REQUIRE(codesRef, "codes", slots * (headDim / 2));
    PUTER_REQUIRE(paramsRef, "params", slots * 4);
    PUTER_REQUIRE(pageTableRef, "pageTable", (((size_t)outRows + pageSize - 1) / pageSize) * 4);
    PUTER_REQUIRE(outputRef, "output", (size_t)outRows * kvHeads * headDim * 2);
    if ((((uintptr_t)dev_ptr(codesRef) | (uintptr_t)dev_ptr(paramsRef) | (uintptr_t)dev_ptr(outputRef)) & 15u) != 0)
        return fail(status, -2, "page gather (4 bits): buffers must be 16-byte aligned");
    const uint32_t heads = 256 / headDim;
    const int grid = q4::grid_of(ctx, (size_t)outRows * ((kvHeads + heads - 1) / heads));
#define GATHER_LAUNCH(DT, D)                                                                                                          \
    q4::gather_kernel<DT, D><<<grid, 256, 0, ctx->stream>>>((const uint8_t*)dev_ptr(codesRef), (const uint32_t*)dev_ptr(paramsRef),   \
                                                            (const int32_t*)dev_ptr(pageTableRef), (uint16_t*)dev_ptr(outputRef), outRows, \
                                                            kvHeads, pageCount, pageSize, ctx->errorFlag)
    if (elementDType == DT_BF16) {
        if (headDim == 128) GATHER_LAUNCH(DT_BF16, 128);
        else GATHER_LAUNCH(DT_BF16, 64);
    } else {
        if (headDim == 128) GATHER_LAUNCH(DT_F16, 128);
        else GATHER_LAUNCH(DT_F16, 64);
    }
#undef GATHER_LAUNCH
    return check_launch(ctx, status, "page gather (4 bits)");
}
