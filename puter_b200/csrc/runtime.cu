// Runtime half of the C ABI: contexts (one per GPU ordinal), buffer handles, streams, status.
// Mirrors the conventions of the reference bridge (device/cuda/internal/bridge/runtime.c,
// status.c) with precompiled sm_100a kernels in place of the NVRTC module cache.
#include <stdarg.h>
#include <mutex>

#include "common.cuh"

namespace puter {

int fail(CUDAStatus* status, int code, const char* fmt, ...) {
    if (status) {
        status->code = code;
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(status->message, CUDA_STATUS_MESSAGE_BYTES, fmt, ap);
        va_end(ap);
    }
    return code;
}

int ok(CUDAStatus* status) {
    if (status) {
        status->code = 0;
        status->message[0] = 0;
    }
    return 0;
}

Context* ctx_of(CUDADeviceRef ref, CUDAStatus* status) {
    if (!ref) {
        fail(status, -1, "cuda: nil device context");
        return nullptr;
    }
    return (Context*)ref;
}

void* dev_ptr(CUDABufferRef ref) { return ref ? ((Buffer*)ref)->ptr : nullptr; }

int check_buffer(CUDAStatus* status, CUDABufferRef ref, const char* name, size_t needBytes) {
    if (!ref || !((Buffer*)ref)->ptr) return fail(status, -2, "cuda: nil buffer '%s'", name);
    Buffer* b = (Buffer*)ref;
    if (b->bytes >= 0 && (size_t)b->bytes < needBytes)
        return fail(status, -2, "cuda: buffer '%s' holds %lld bytes, call needs %zu", name, b->bytes, needBytes);
    return 0;
}

int check_launch(Context* ctx, CUDAStatus* status, const char* what) {
    ctx->launches++;
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return fail(status, -7, "cuda: launch of %s failed: %s", what, cudaGetErrorString(err));
    return ok(status);
}

void* ensure_workspace(Context* ctx, size_t bytes, CUDAStatus* status) {
    ctx->scratchUsed = 1;
    if (bytes <= ctx->workspaceBytes) return ctx->workspace;
    RelaxedCapture relaxed;  // (another stream may be under capture)
    // grow-only; the old block may still be in use by work queued on the stream
    if (ctx->workspace) {
        cudaStreamSynchronize(ctx->stream);
        cudaFree(ctx->workspace);
        ctx->workspace = nullptr;
        ctx->workspaceBytes = 0;
    }
    size_t want = bytes + (bytes >> 2);
    if (cudaMalloc(&ctx->workspace, want) != cudaSuccess) {
        cudaGetLastError();
        fail(status, -7, "cuda: workspace allocation of %zu bytes failed", want);
        return nullptr;
    }
    ctx->workspaceBytes = want;
    return ctx->workspace;
}

enum Capture { kNotCaptured, kCaptured, kUntouchable };  // kUntouchable: the legacy stream while a blocking stream is under capture

static Capture capture_of(cudaStream_t stream, unsigned long long* id) {
    cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
    unsigned long long name = 0;
    if (cudaStreamGetCaptureInfo(stream, &state, &name) != cudaSuccess) {
        cudaGetLastError();
        return kUntouchable;
    }
    if (id) *id = name;
    return state == cudaStreamCaptureStatusActive ? kCaptured : state == cudaStreamCaptureStatusNone ? kNotCaptured : kUntouchable;
}

bool stream_capturing(Context* ctx, unsigned long long* id) { return capture_of(ctx->stream, id) == kCaptured; }

// Goes over to another stream.  Two eager streams are ordered by an event, two streams of one capture by an edge of its graph (they share its
// scratch).  An event may not tie a stream under capture to work outside the capture, and such a stream runs nothing now: the wait stays
// outstanding until the context launches eagerly again, on whichever stream that is.
static void adopt_stream(Context* ctx, cudaStream_t next) {
    cudaSetDevice(ctx->device);
    cudaStream_t last = ctx->stream;
    unsigned long long idFrom = 0, idTo = 0;
    const Capture from = capture_of(last, &idFrom), to = capture_of(next, &idTo);
    bool covered = false;  // an event stands behind the eager work of `last`
    if (from == kNotCaptured) {
        if (ctx->switchWaits) cudaStreamWaitEvent(last, ctx->streamSwitchEvent, 0);  // the event moves on, and what it stood for with it
        covered = cudaEventRecord(ctx->streamSwitchEvent, last) == cudaSuccess;
        if (covered) ctx->switchWaits = 1;
    } else if (from == kCaptured && to == kCaptured && idFrom == idTo) {
        if (cudaEventRecord(ctx->captureEvent, last) == cudaSuccess) cudaStreamWaitEvent(next, ctx->captureEvent, 0);
    }
    if (ctx->scratchUsed && !covered) {
        ctx->switchLost = 1;
        ctx->lostStream = last;
    } else if (covered && ctx->switchLost && ctx->lostStream == last) {
        ctx->switchLost = 0;
    }
    ctx->stream = next;
    ctx->scratchUsed = 0;
    if (ctx->switchWaits && to == kNotCaptured && cudaStreamWaitEvent(next, ctx->streamSwitchEvent, 0) == cudaSuccess) ctx->switchWaits = 0;
    cudaGetLastError();
}

int settle_stream(Context* ctx, CUDAStatus* status) {
    if (capture_of(ctx->stream, nullptr) != kNotCaptured) return 0;
    if (ctx->switchWaits) {
        cudaError_t err = cudaStreamWaitEvent(ctx->stream, ctx->streamSwitchEvent, 0);
        if (err != cudaSuccess) return fail(status, -7, "cuda: ordering two streams failed: %s", cudaGetErrorString(cudaGetLastError()));
        ctx->switchWaits = 0;
    }
    if (ctx->lostStream == ctx->stream) ctx->switchLost = 0;  // back on the stream itself
    if (!ctx->switchLost) return 0;
    // nothing can wait for that work: it keeps the scratch and the tables, and this stream gets others
    RelaxedCapture relaxed;
    int* counters = nullptr;
    cudaError_t err = cudaMalloc((void**)&counters, ctx->decodeCounterBytes);
    if (err == cudaSuccess) err = cudaMemsetAsync(counters, 0, ctx->decodeCounterBytes, ctx->uploadStream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(ctx->uploadStream);
    if (err != cudaSuccess) {
        cudaGetLastError();
        if (counters) cudaFree(counters);
        return fail(status, -7, "cuda: scratch for another stream failed: %s", cudaGetErrorString(err));
    }
    ctx->setAside = new SetAside{ctx->workspace, ctx->decodeCounters, ctx->setAside};
    ctx->workspace = nullptr;
    ctx->workspaceBytes = 0;
    ctx->decodeCounters = counters;
    for (RopeTable* t = ctx->ropeTables; t; t = t->next) {
        if (t->valid && !t->finished) cudaStreamWaitEvent(ctx->stream, t->built, 0);
        t->held = 1;
    }
    ctx->switchLost = 0;
    return 0;
}

int call_scratch(Context* ctx, size_t bytes, size_t counterBytes, Scratch* out, CUDAStatus* status) {
    const bool own = counterBytes <= ctx->decodeCounterBytes;  // the kept, always-zero counters hold this call's
    const size_t body = (bytes + 255) & ~(size_t)255;
    const size_t need = body + (own ? 0 : counterBytes) + 512;
    unsigned long long id = 0;
    if (!stream_capturing(ctx, &id)) {
        char* ws = (char*)ensure_workspace(ctx, need, status);
        if (!ws) return status ? status->code : -7;
        out->base = ws;
        out->counters = own ? ctx->decodeCounters : (int*)(ws + body);
        out->clearCounters = !own;
        return 0;
    }
    GraphScratch* g = ctx->graphScratch;
    while (g && (g->id != id || g->bytes < need)) g = g->next;
    if (!g) {
        // allocating is not part of the captured work, and neither is clearing, on a stream of the context's own
        RelaxedCapture relaxed;
        void* p = nullptr;
        const size_t total = ctx->decodeCounterBytes + need;
        cudaError_t err = cudaMalloc(&p, total);
        if (err == cudaSuccess) err = cudaMemsetAsync(p, 0, ctx->decodeCounterBytes, ctx->uploadStream);
        if (err == cudaSuccess) err = cudaStreamSynchronize(ctx->uploadStream);
        if (err != cudaSuccess) {
            cudaGetLastError();
            if (p) cudaFree(p);
            return fail(status, -7, "cuda: scratch of %zu bytes for a captured call failed: %s", total, cudaGetErrorString(err));
        }
        g = new GraphScratch{id, (char*)p + ctx->decodeCounterBytes, need, (int*)p, ctx->graphScratch};
        ctx->graphScratch = g;
    }
    out->base = g->base;
    out->counters = own ? g->counters : (int*)(g->base + body);
    out->clearCounters = !own;
    return 0;
}

// Frees what captured calls and work set aside have used; none of it is in use any more.
static void free_held_scratch(Context* ctx) {
    while (GraphScratch* g = ctx->graphScratch) {
        ctx->graphScratch = g->next;
        cudaFree(g->counters);
        delete g;
    }
    while (SetAside* a = ctx->setAside) {
        ctx->setAside = a->next;
        cudaFree(a->workspace);
        cudaFree(a->counters);
        delete a;
    }
}

static std::mutex g_mu;
static Context* g_default = nullptr;

}  // namespace puter

using namespace puter;

extern "C" {

void cuda_status_clear(CUDAStatus* status) {
    if (!status) return;
    status->code = 0;
    status->message[0] = 0;
}

void cuda_status_set(CUDAStatus* status, int code, const char* message) {
    if (!status) return;
    status->code = code;
    snprintf(status->message, CUDA_STATUS_MESSAGE_BYTES, "%s", message ? message : "");
}

int cuda_open_device_index(int ordinal, CUDADeviceRef* outDevice, CUDAStatus* status) {
    cuda_status_clear(status);
    if (!outDevice) return fail(status, -2, "cuda: nil outDevice");
    *outDevice = nullptr;
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count <= 0) {
        cudaGetLastError();
        return fail(status, -1, "cuda: no CUDA device available (this library has no CPU fallback)");
    }
    if (ordinal < 0 || ordinal >= count) return fail(status, -1, "cuda: device ordinal %d out of range (%d devices)", ordinal, count);
    if (cudaSetDevice(ordinal) != cudaSuccess) return fail(status, -1, "cuda: cudaSetDevice(%d) failed", ordinal);
    cudaDeviceProp prop;
    if (cudaGetDeviceProperties(&prop, ordinal) != cudaSuccess) return fail(status, -1, "cuda: device properties unavailable");
    if (prop.major < 10)
        return fail(status, -1, "cuda: device %d is sm_%d%d; this library ships sm_100a code only", ordinal, prop.major, prop.minor);
    Context* ctx = new Context();
    memset(ctx, 0, sizeof(*ctx));
    ctx->device = ordinal;
    ctx->ccMajor = prop.major;
    ctx->smCount = prop.multiProcessorCount;
    ctx->totalMem = (long long)prop.totalGlobalMem;
    if (cudaStreamCreateWithFlags(&ctx->ownStream, cudaStreamNonBlocking) != cudaSuccess ||
        cudaStreamCreateWithFlags(&ctx->uploadStream, cudaStreamNonBlocking) != cudaSuccess) {
        delete ctx;
        return fail(status, -7, "cuda: stream creation failed");
    }
    ctx->stream = ctx->ownStream;
    for (int i = 0; i < 4; i++) cudaEventCreateWithFlags(&ctx->stageEvents[i], cudaEventDisableTiming);
    cudaEventCreateWithFlags(&ctx->streamSwitchEvent, cudaEventDisableTiming);
    cudaEventCreateWithFlags(&ctx->captureEvent, cudaEventDisableTiming);
    if (cudaMalloc((void**)&ctx->errorFlag, 256) != cudaSuccess) {
        delete ctx;
        return fail(status, -7, "cuda: context allocation failed");
    }
    cudaMemset(ctx->errorFlag, 0, 256);
    ctx->decodeCounterBytes = 64 << 10;
    if (cudaMalloc((void**)&ctx->decodeCounters, ctx->decodeCounterBytes) != cudaSuccess) {
        cudaFree(ctx->errorFlag);
        delete ctx;
        return fail(status, -7, "cuda: context allocation failed");
    }
    cudaMemset(ctx->decodeCounters, 0, ctx->decodeCounterBytes);
    *outDevice = ctx;
    std::lock_guard<std::mutex> lock(g_mu);
    if (!g_default) g_default = ctx;
    return ok(status);
}

int cuda_open_device(CUDADeviceRef* outDevice, CUDAStatus* status) { return cuda_open_device_index(0, outDevice, status); }

void cuda_close_device(CUDADeviceRef device) {
    if (!device) return;
    Context* ctx = (Context*)device;
    cudaSetDevice(ctx->device);
    cudaStreamSynchronize(ctx->stream);
    cudaStreamSynchronize(ctx->uploadStream);
    if (ctx->workspace) cudaFree(ctx->workspace);
    for (int i = 0; i < 2; i++)
        if (ctx->pinned[i]) cudaFreeHost(ctx->pinned[i]);
    if (ctx->errorFlag) cudaFree(ctx->errorFlag);
    if (ctx->decodeCounters) cudaFree(ctx->decodeCounters);
    for (RopeTable* t = ctx->ropeTables; t;) {
        RopeTable* next = t->next;
        cudaFree(t->data);
        cudaEventDestroy(t->built);
        delete t;
        t = next;
    }
    free_held_scratch(ctx);
    for (int i = 0; i < 4; i++)
        if (ctx->stageEvents[i]) cudaEventDestroy(ctx->stageEvents[i]);
    if (ctx->streamSwitchEvent) cudaEventDestroy(ctx->streamSwitchEvent);
    if (ctx->captureEvent) cudaEventDestroy(ctx->captureEvent);
    cudaStreamDestroy(ctx->ownStream);
    cudaStreamDestroy(ctx->uploadStream);
    {
        std::lock_guard<std::mutex> lock(g_mu);
        if (g_default == ctx) g_default = nullptr;
    }
    delete ctx;
}

long long cuda_device_total_memory(CUDADeviceRef device) { return device ? ((Context*)device)->totalMem : 0; }
int cuda_device_capability_major(CUDADeviceRef device) { return device ? ((Context*)device)->ccMajor : 0; }

CUDABufferRef cuda_buffer_alloc(CUDADeviceRef device, long long bytes) {
    if (!device || bytes <= 0) return nullptr;
    Context* ctx = (Context*)device;
    cudaSetDevice(ctx->device);
    void* p = nullptr;
    if (cudaMalloc(&p, (size_t)bytes) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    Buffer* b = new Buffer{p, bytes, 1, ctx->device};
    return b;
}

CUDABufferRef cuda_buffer_wrap(CUDADeviceRef device, void* devicePtr, long long bytes) {
    if (!device || !devicePtr) return nullptr;
    return new Buffer{devicePtr, bytes, 0, ((Context*)device)->device};
}

void cuda_buffer_release(CUDABufferRef buffer) {
    if (!buffer) return;
    Buffer* b = (Buffer*)buffer;
    if (b->owned == 1 && b->ptr) {
        cudaSetDevice(b->device);
        cudaFree(b->ptr);
    } else if (b->owned == 2 && b->ptr) {  // a peer's allocation mapped by cuda_buffer_ipc_import
        cudaSetDevice(b->device);
        cudaIpcCloseMemHandle(b->ptr);
    }
    delete b;
}

int cuda_buffer_ipc_export(CUDABufferRef buffer, void* outHandle64, CUDAStatus* status) {
    cuda_status_clear(status);
    if (!buffer || !outHandle64) return fail(status, -2, "cuda: nil argument in ipc export");
    Buffer* b = (Buffer*)buffer;
    if (b->owned != 1) return fail(status, -2, "cuda: only buffers allocated by cuda_buffer_alloc can be exported");
    static_assert(sizeof(cudaIpcMemHandle_t) == 64, "the C ABI fixes the handle at 64 bytes");
    cudaSetDevice(b->device);
    cudaIpcMemHandle_t h;
    cudaError_t err = cudaIpcGetMemHandle(&h, b->ptr);
    if (err != cudaSuccess) return fail(status, -7, "cuda: cudaIpcGetMemHandle failed: %s", cudaGetErrorString(err));
    memcpy(outHandle64, &h, 64);
    return ok(status);
}

CUDABufferRef cuda_buffer_ipc_import(CUDADeviceRef device, const void* handle64, long long bytes, CUDAStatus* status) {
    cuda_status_clear(status);
    Context* ctx = ctx_of(device, status);
    if (!ctx) return nullptr;
    if (!handle64 || bytes <= 0) { fail(status, -2, "cuda: nil handle in ipc import"); return nullptr; }
    cudaSetDevice(ctx->device);
    cudaIpcMemHandle_t h;
    memcpy(&h, handle64, 64);
    void* p = nullptr;
    cudaError_t err = cudaIpcOpenMemHandle(&p, h, cudaIpcMemLazyEnablePeerAccess);
    if (err != cudaSuccess || !p) {
        cudaGetLastError();
        fail(status, -7, "cuda: cudaIpcOpenMemHandle failed: %s", cudaGetErrorString(err));
        return nullptr;
    }
    ok(status);
    return new Buffer{p, bytes, 2, ctx->device};
}

void* cuda_buffer_device_ptr(CUDABufferRef buffer) { return dev_ptr(buffer); }

int cuda_memcpy_async_h2d(CUDABufferRef dst, const void* src, long long bytes, CUDAStreamRef stream, CUDAStatus* status) {
    cuda_status_clear(status);
    if (bytes == 0) return ok(status);
    if (!dst || !src) return fail(status, -2, "cuda: nil buffer in h2d copy");
    Buffer* b = (Buffer*)dst;
    if (b->bytes >= 0 && bytes > b->bytes) return fail(status, -2, "cuda: h2d copy of %lld bytes exceeds buffer (%lld)", bytes, b->bytes);
    cudaSetDevice(b->device);
    cudaError_t err = cudaMemcpyAsync(b->ptr, src, (size_t)bytes, cudaMemcpyHostToDevice, (cudaStream_t)stream);
    if (err != cudaSuccess) return fail(status, -7, "cuda: h2d copy failed: %s", cudaGetErrorString(err));
    return ok(status);
}

int cuda_memcpy_async_d2h(void* dst, CUDABufferRef src, long long bytes, CUDAStreamRef stream, CUDAStatus* status) {
    cuda_status_clear(status);
    if (bytes == 0) return ok(status);
    if (!dst || !src) return fail(status, -2, "cuda: nil buffer in d2h copy");
    Buffer* b = (Buffer*)src;
    if (b->bytes >= 0 && bytes > b->bytes) return fail(status, -2, "cuda: d2h copy of %lld bytes exceeds buffer (%lld)", bytes, b->bytes);
    cudaSetDevice(b->device);
    cudaError_t err = cudaMemcpyAsync(dst, b->ptr, (size_t)bytes, cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (err != cudaSuccess) return fail(status, -7, "cuda: d2h copy failed: %s", cudaGetErrorString(err));
    return ok(status);
}

int cuda_memcpy_async_d2d(CUDABufferRef dst, CUDABufferRef src, long long bytes, CUDAStreamRef stream, CUDAStatus* status) {
    cuda_status_clear(status);
    if (bytes == 0) return ok(status);
    if (!dst || !src) return fail(status, -2, "cuda: nil buffer in d2d copy");
    Buffer* d = (Buffer*)dst;
    Buffer* s = (Buffer*)src;
    if (d->bytes >= 0 && bytes > d->bytes) return fail(status, -2, "cuda: d2d copy of %lld bytes exceeds the destination (%lld)", bytes, d->bytes);
    if (s->bytes >= 0 && bytes > s->bytes) return fail(status, -2, "cuda: d2d copy of %lld bytes exceeds the source (%lld)", bytes, s->bytes);
    cudaSetDevice(d->device);
    cudaError_t err = cudaMemcpyAsync(d->ptr, s->ptr, (size_t)bytes, cudaMemcpyDeviceToDevice, (cudaStream_t)stream);
    if (err != cudaSuccess) return fail(status, -7, "cuda: d2d copy failed: %s", cudaGetErrorString(err));
    return ok(status);
}

int cuda_stream_synchronize(CUDAStreamRef stream, CUDAStatus* status) {
    cuda_status_clear(status);
    cudaError_t err = cudaStreamSynchronize((cudaStream_t)stream);
    if (err != cudaSuccess) return fail(status, -7, "cuda: stream synchronize failed: %s", cudaGetErrorString(err));
    return ok(status);
}

CUDADeviceRef cuda_default_context(void) {
    std::lock_guard<std::mutex> lock(g_mu);
    return g_default;
}

CUDAStreamRef cuda_context_upload_stream(CUDADeviceRef device) { return device ? (CUDAStreamRef)((Context*)device)->uploadStream : nullptr; }
CUDAStreamRef cuda_context_default_stream(CUDADeviceRef device) { return device ? (CUDAStreamRef)((Context*)device)->stream : nullptr; }

int cuda_context_set_stream(CUDADeviceRef device, void* cudaStream, CUDAStatus* status) {
    cuda_status_clear(status);
    Context* ctx = ctx_of(device, status);
    if (!ctx) return -1;
    cudaStream_t next = (cudaStream_t)cudaStream;  // NULL = the legacy default stream
    if (next != ctx->stream) adopt_stream(ctx, next);
    return ok(status);
}

int cuda_context_reset_stream(CUDADeviceRef device, CUDAStatus* status) {
    cuda_status_clear(status);
    Context* ctx = ctx_of(device, status);
    if (!ctx) return -1;
    if (ctx->stream != ctx->ownStream) adopt_stream(ctx, ctx->ownStream);
    return ok(status);
}

int cuda_context_release_captures(CUDADeviceRef device, CUDAStatus* status) {
    cuda_status_clear(status);
    Context* ctx = ctx_of(device, status);
    if (!ctx) return -1;
    cudaSetDevice(ctx->device);
    if (capture_of(ctx->stream, nullptr) != kNotCaptured) return fail(status, -2, "cuda: captures cannot be released while the context's stream is part of one");
    cudaError_t err = cudaDeviceSynchronize();  // replays may be in flight on any stream
    if (err != cudaSuccess) return fail(status, -7, "cuda: waiting for the device failed: %s", cudaGetErrorString(err));
    free_held_scratch(ctx);
    for (RopeTable** at = &ctx->ropeTables; *at;) {
        RopeTable* t = *at;
        if (!t->held) {
            at = &t->next;
            continue;
        }
        *at = t->next;
        cudaFree(t->data);
        cudaEventDestroy(t->built);
        delete t;
    }
    return ok(status);
}

int cuda_context_set_exact(CUDADeviceRef device, int exact, CUDAStatus* status) {
    cuda_status_clear(status);
    Context* ctx = ctx_of(device, status);
    if (!ctx) return -1;
    ctx->exact = exact ? 1 : 0;
    return ok(status);
}

int cuda_context_take_error(CUDADeviceRef device, int* outFlag, CUDAStatus* status) {
    cuda_status_clear(status);
    Context* ctx = ctx_of(device, status);
    if (!ctx) return -1;
    if (!outFlag) return fail(status, -2, "cuda: nil outFlag");
    cudaSetDevice(ctx->device);
    if (ctx->switchWaits | ctx->switchLost) {  // calls on the streams before may still raise it
        int rc = settle_stream(ctx, status);
        if (rc != 0) return rc;
    }
    int flag = 0;
    cudaError_t err = cudaMemcpyAsync(&flag, ctx->errorFlag, sizeof(int), cudaMemcpyDeviceToHost, ctx->stream);
    if (err == cudaSuccess) err = cudaMemsetAsync(ctx->errorFlag, 0, sizeof(int), ctx->stream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(ctx->stream);
    if (err != cudaSuccess) return fail(status, -7, "cuda: reading the error flag failed: %s", cudaGetErrorString(err));
    *outFlag = flag;
    return ok(status);
}

unsigned long long cuda_context_launch_count(CUDADeviceRef device) { return device ? ((Context*)device)->launches : 0ull; }

void* cuda_host_alloc(long long bytes) {
    void* p = nullptr;
    if (bytes <= 0 || cudaMallocHost(&p, (size_t)bytes) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    return p;
}

void cuda_host_free(void* ptr) {
    if (ptr) cudaFreeHost(ptr);
}

}  // extern "C"
