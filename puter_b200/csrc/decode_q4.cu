// Paged decode attention over the cache in 4 bits (layout and meaning of codes and params: kv4.cu).
//
// One new token per sequence:  score_t = (q . k_t) / sqrt(D),  k_t = least_t + step_t * code_t,  p = softmax(score) over the
// sequence's tokens,  out = sum_t p_t (least_t + step_t * code_t).  The dequantised values are never rounded to 16 bits.
#include <math.h>

#include "common.cuh"

namespace puter {

namespace q4d {

struct Params {
    const uint16_t* q;
    const uint8_t *kCodes, *vCodes;
    const uint32_t *kParams, *vParams;
    const int32_t *table, *ctxLens;
    uint16_t* out;
    int* errorFlag;
    int batch, maxPages, pageCount, pageSize, numHeads, kvHeads, group;
    float scaleLog2;
};

// tokens of sequence b: negative or over-long contexts are cut and flagged
__device__ __forceinline__ long long seq_ctx(const Params& p, int b) {
    long long ctx = p.ctxLens[b];
    const long long cap = (long long)p.maxPages * p.pageSize;
    if (ctx < 0 || ctx > cap) {
        atomicExch(p.errorFlag, 1);
        ctx = ctx < 0 ? 0 : cap;
    }
    return ctx;
}

// One warp per (sequence, query head), D / 32 elements a lane, one pass over the tokens with a running maximum and sum.
template <int DT, int D>
__global__ void __launch_bounds__(128) decode_kernel(Params p) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (long long)p.batch * p.numHeads) return;
    const int b = (int)(w / p.numHeads), head = (int)(w % p.numHeads), kvh = head / p.group;
    const long long ctx = seq_ctx(p, b);
    if (ctx == 0) return;
    float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        q[i] = Storage<DT>::widen(p.q[((size_t)b * p.numHeads + head) * D + lane * E + i]);
        acc[i] = 0.f;
    }
    for (long long t = 0; t < ctx; t++) {
        int page = p.table[(size_t)b * p.maxPages + t / p.pageSize];
        if (page < 0 || page >= p.pageCount) {
            if (lane == 0) atomicExch(p.errorFlag, 1);
            page = 0;
        }
        const size_t slot = ((size_t)page * p.kvHeads + kvh) * p.pageSize + t % p.pageSize;
        float ks, kl, vs, vl, dot = 0.f;
        unpack16_arith<DT>(p.kParams[slot], ks, kl);
        unpack16_arith<DT>(p.vParams[slot], vs, vl);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int d = lane * E + i;
            dot += q[i] * fmaf(ks, (float)((p.kCodes[slot * (D / 2) + d / 2] >> (4 * (d & 1))) & 15), kl);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float s = dot * p.scaleLog2, mNew = fmaxf(m, s);
        const float alpha = exp2f(m - mNew), e = exp2f(s - mNew);
        l = l * alpha + e;
        m = mNew;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int d = lane * E + i;
            acc[i] = acc[i] * alpha + e * fmaf(vs, (float)((p.vCodes[slot * (D / 2) + d / 2] >> (4 * (d & 1))) & 15), vl);
        }
    }
#pragma unroll
    for (int i = 0; i < E; i++) Storage<DT>::store(p.out, ((size_t)b * p.numHeads + head) * D + lane * E + i, acc[i] / l);
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
    const unsigned grid = (unsigned)(((size_t)batch * numHeads + 3) / 4);
    if (elementDType == DT_BF16) {
        if (headDim == 128) q4d::decode_kernel<DT_BF16, 128><<<grid, 128, 0, ctx->stream>>>(p);
        else q4d::decode_kernel<DT_BF16, 64><<<grid, 128, 0, ctx->stream>>>(p);
    } else {
        if (headDim == 128) q4d::decode_kernel<DT_F16, 128><<<grid, 128, 0, ctx->stream>>>(p);
        else q4d::decode_kernel<DT_F16, 64><<<grid, 128, 0, ctx->stream>>>(p);
    }
    return check_launch(ctx, status, "paged decode attention (4 bits)");
}
