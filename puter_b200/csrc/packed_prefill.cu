// Attention over whole prompts of different lengths, packed one behind the other.
//
// q / out [totalTokens, numHeads, D], k / v [totalTokens, kvHeads, D]; sequence i holds rows seqStarts[i] .. seqStarts[i + 1] - 1
// (int32 on the device, so a serving loop never waits for lengths).  Per sequence: RoPE(q), RoPE(k) at positions that restart with
// every sequence (device/cpu/rope/compute.go:55-193, results rounded to the storage type), then MultiHeadAttention
// (device/cpu/attention/typed_compute.go:142-237): out_r = sum_{t <= r} p_t v_t, p = softmax(q_r . k_t / sqrt(D)).
// Rows that belong to no sequence (before the first start, behind the last) are neither read into a result nor written.
// A pair of starts that is not 0 <= start <= end <= totalTokens with at most maxSeqLen rows is skipped and raises the error flag.
#include <math.h>

#include "common.cuh"

namespace puter {

int validate_rope(CUDAStatus* status, double base, uint32_t halfMode, uint32_t scaling, double factor, double low, double high,
                  uint32_t origCtx);
const float* cached_rope_table(Context* ctx, size_t seqLen, int headDim, double base, long long startPos, int scaling, double factor,
                               double low, double high, int origCtx, CUDAStatus* status);

namespace pk {

struct Seqs {
    const int32_t* starts;
    int batch, total, maxLen;
    int* errorFlag;
};

// rows [s0, s1) of sequence b; false (and the flag) where the starts make none
__device__ __forceinline__ bool seq_rows(const Seqs& s, int b, int& s0, int& s1) {
    s0 = s.starts[b];
    s1 = s.starts[b + 1];
    if (s0 < 0 || s1 < s0 || s1 > s.total || s1 - s0 > s.maxLen) {
        atomicExch(s.errorFlag, 1);
        s1 = s0;
        return false;
    }
    return s1 > s0;
}

// the sequence that holds `row`: the last one that starts at or before it
__device__ __forceinline__ int seq_of(const Seqs& s, int row) {
    int a = 0, z = s.batch;
    while (z - a > 1) {
        const int m = (a + z) >> 1;
        if (s.starts[m] <= row) a = m;
        else z = m;
    }
    return a;
}

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
// maximum and sum.  It runs what the tensor-core kernel does not take; its bound is the five shuffles per key.
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
    if (out == q || out == k || out == v) return fail(status, -2, "%s: out may not be an input", what);
    const pk::Seqs seqs{(const int32_t*)dev_ptr(seqStartsRef), (int)batch, (int)totalTokens, (int)maxSeqLen, ctx->errorFlag};
    const int cap = ctx->smCount * 8;
    if (ropeMode != 2) {
        const float* table = cached_rope_table(ctx, maxSeqLen, (int)headDim, baseFreq, (long long)startPosition, (int)scaling, scalingFactor,
                                               lowFreqFactor, highFreqFactor, (int)originalContext, status);
        if (!table) return status ? status->code : -7;
        const size_t qAt = 0, kAt = (qBytes + 255) & ~(size_t)255;
        Scratch ws;
        int rc = call_scratch(ctx, kAt + kvBytes, 0, &ws, status);
        if (rc != 0) return rc;
        const float* sinT = table + (size_t)maxSeqLen * (headDim / 2);
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
