"""Argument order of the packed-prompt and 4-bit-cache methods in both mirrors, without a GPU: the Python one against a library that
records its calls, the C++ one linked with entry points that print theirs."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# method -> (entry point, tensors, sizes and settings in the order of the declaration, as the calls below give them)
WANT = {
    "RoPEPackedAttentionPrefill": ("rope_packed_attention_prefill", 5, [3, 40, 20, 8, 2, 64, 1, 1, 500.0, 7, 1, 8.0, 1.5, 4.5, 8192]),
    "RoPEKVPageWriteQ4": ("rope_kv_page_write_q4", 9, [4, 2, 64, 6, 16, 100, 1, 500.0, 1, 8.0, 1.5, 4.5, 8192]),
    "KVPageGatherQ4": ("kv_page_gather_q4", 4, [6, 16, 2, 64, 33]),
    "PagedDecodeAttentionQ4": ("paged_decode_attention_q4", 8, [3, 5, 6, 16, 8, 2, 64]),
}


class FakeTensor:
    is_cuda = True

    def __init__(self, addr):
        self.addr, self.nbytes = addr, 1 << 20

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.addr


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def fn(*args):
            if name == "cuda_buffer_wrap":
                return args[1].value
            self.calls.append((name, [getattr(a, "value", a) for a in args[1:-1]]))
            return 0
        return fn


@pytest.fixture()
def dev():
    from puter_b200 import _lib, device as D

    dev = D.Device.__new__(D.Device)
    dev.lib, dev.ref, dev._refs, dev._status, dev.follow_torch_stream = Recorder(), None, {}, _lib.CUDAStatus(), False
    return dev


def tensors(n):
    return [FakeTensor(0x1000 * (i + 1)) for i in range(n)]


def python_calls(dev):
    from puter_b200 import device as D

    rope = D.RoPEConfig(Mode=1, BaseFreq=500.0, StartPosition=7, Scaling=1, ScalingFactor=8.0, LowFreqFactor=1.5, HighFreqFactor=4.5, OriginalContext=8192)
    attn = D.MultiHeadAttentionConfig(NumHeads=8, HeadDim=64, Causal=True, KVHeadCount=2)
    dev.RoPEPackedAttentionPrefill(rope, attn, *tensors(5), 3, 40, 20, 2)
    dev.RoPEKVPageWriteQ4(rope, *tensors(9), 4, 2, 64, 6, 16, 100, 2)
    dev.KVPageGatherQ4(*tensors(4), 6, 16, 2, 64, 33, 2)
    dev.PagedDecodeAttentionQ4(attn, *tensors(8), 3, 5, 6, 16, 2)


def test_python(dev):
    python_calls(dev)
    assert [c[0] for c in dev.lib.calls] == ["cuda_dispatch_" + w[0] for w in WANT.values()]
    for (name, args), (entry, n, rest) in zip(dev.lib.calls, WANT.values()):
        refs = [0x1000 * (i + 1) for i in range(n)] + ([None] if entry.startswith("paged_decode") else [])
        assert args == [2, *refs, *rest, 0], entry


def test_python_inputs_that_come_rotated(dev):
    from puter_b200 import device as D

    attn = D.MultiHeadAttentionConfig(NumHeads=8, HeadDim=64, Causal=False)
    dev.RoPEPackedAttentionPrefill(None, attn, *tensors(5), 3, 40, 20, 2)
    dev.RoPEKVPageWriteQ4(None, *tensors(2), None, *tensors(6), 4, 2, 64, 6, 16, 100, 1)
    prompt, append = (c[1] for c in dev.lib.calls)
    assert prompt[6:14] == [3, 40, 20, 8, 8, 64, 0, 2] and append[0] == 1 and append[3] is None and append[16] == 2


SOURCE = r"""
#include <cstdio>
#include <initializer_list>
#include "%s/puter_b200/host/backend.hpp"
static int number = 0;
static void say(const char* name, std::initializer_list<const void*> bufs, std::initializer_list<double> rest) {
    std::printf("%%s", name);
    for (const void* b : bufs) std::printf(" %%lld", (long long)b);
    for (double x : rest) std::printf(" %%g", x);
    std::printf("\n");
}
extern "C" {
int cuda_open_device_index(int, CUDADeviceRef* out, CUDAStatus*) { *out = (CUDADeviceRef)&number; return 0; }
void cuda_close_device(CUDADeviceRef) {}
CUDABufferRef cuda_buffer_wrap(CUDADeviceRef, void* p, long long) { return (CUDABufferRef)p; }
void cuda_buffer_release(CUDABufferRef) {}
int cuda_dispatch_rope_packed_attention_prefill(CUDADeviceRef, int t, CUDABufferRef a, CUDABufferRef b, CUDABufferRef c, CUDABufferRef d, CUDABufferRef e,
        uint32_t batch, uint32_t total, uint32_t longest, uint32_t heads, uint32_t kv, uint32_t dim, uint32_t causal, uint32_t mode, double base, int64_t start,
        uint32_t scaling, double f, double l, double h, uint32_t ctx, uint64_t, CUDAStatus*) {
    say("prompt", {a, b, c, d, e}, {(double)t, (double)batch, (double)total, (double)longest, (double)heads, (double)kv, (double)dim, (double)causal, (double)mode, base, (double)start, (double)scaling, f, l, h, (double)ctx});
    return 0;
}
int cuda_dispatch_rope_kv_page_write_q4(CUDADeviceRef, int t, CUDABufferRef a, CUDABufferRef b, CUDABufferRef c, CUDABufferRef d, CUDABufferRef e, CUDABufferRef f,
        CUDABufferRef g, CUDABufferRef h, CUDABufferRef i, uint32_t rows, uint32_t kv, uint32_t dim, uint32_t pages, uint32_t page, uint32_t longest, uint32_t mode,
        double base, uint32_t scaling, double sf, double l, double hf, uint32_t ctx, uint64_t, CUDAStatus*) {
    say("append", {a, b, c, d, e, f, g, h, i}, {(double)t, (double)rows, (double)kv, (double)dim, (double)pages, (double)page, (double)longest, (double)mode, base, (double)scaling, sf, l, hf, (double)ctx});
    return 0;
}
int cuda_dispatch_kv_page_gather_q4(CUDADeviceRef, int t, CUDABufferRef a, CUDABufferRef b, CUDABufferRef c, CUDABufferRef d, uint32_t pages, uint32_t page, uint32_t kv,
        uint32_t dim, uint32_t rows, uint64_t, CUDAStatus*) {
    say("gather", {a, b, c, d}, {(double)t, (double)pages, (double)page, (double)kv, (double)dim, (double)rows});
    return 0;
}
int cuda_dispatch_paged_decode_attention_q4(CUDADeviceRef, int t, CUDABufferRef a, CUDABufferRef b, CUDABufferRef c, CUDABufferRef d, CUDABufferRef e, CUDABufferRef f,
        CUDABufferRef g, CUDABufferRef h, CUDABufferRef flag, uint32_t batch, uint32_t most, uint32_t pages, uint32_t page, uint32_t heads, uint32_t kv, uint32_t dim,
        uint64_t, CUDAStatus* st) {
    say("decode", {a, b, c, d, e, f, g, h, flag}, {(double)t, (double)batch, (double)most, (double)pages, (double)page, (double)heads, (double)kv, (double)dim});
    st->code = -6;
    st->message[0] = 0;
    return dim == 96 ? -6 : 0;
}
}
int main() {
    using namespace puter;
    Backend b(0);
    DeviceTensor t1(b.Context(), (void*)1, 4), t2(b.Context(), (void*)2, 4), t3(b.Context(), (void*)3, 4), t4(b.Context(), (void*)4, 4), t5(b.Context(), (void*)5, 4),
        t6(b.Context(), (void*)6, 4), t7(b.Context(), (void*)7, 4), t8(b.Context(), (void*)8, 4), t9(b.Context(), (void*)9, 4);
    RoPEConfig r{500.0, 7, RoPEMode::Half, RoPEScaling::Llama3, 8.0, 1.5, 4.5, 8192};
    MultiHeadAttentionConfig a{8, 64, true, 0, 0.f, 2};
    b.RoPEPackedAttentionPrefill(&r, a, &t1, &t2, &t3, &t4, &t5, 3, 40, 20, DType::BFloat16);
    b.RoPEKVPageWriteQ4(&r, &t1, &t2, &t3, &t4, &t5, &t6, &t7, &t8, &t9, 4, 2, 64, 6, 16, 100, DType::BFloat16);
    b.KVPageGatherQ4(&t1, &t2, &t3, &t4, 6, 16, 2, 64, 33, DType::BFloat16);
    b.PagedDecodeAttentionQ4(a, &t1, &t2, &t3, &t4, &t5, &t6, &t7, &t8, 3, 5, 6, 16, DType::BFloat16);
    b.RoPEKVPageWriteQ4(nullptr, &t1, &t2, nullptr, &t4, &t5, &t6, &t7, &t8, &t9, 4, 2, 64, 6, 16, 100, DType::Float16);
    int refused = 0;
    a.HeadDim = 96;
    try { b.PagedDecodeAttentionQ4(a, &t1, &t2, &t3, &t4, &t5, &t6, &t7, &t8, 3, 5, 6, 16, DType::BFloat16); } catch (const DeviceError& e) { refused += e.code == -6; }
    a.WindowSize = 4;
    try { b.PagedDecodeAttentionQ4(a, &t1, &t2, &t3, &t4, &t5, &t6, &t7, &t8, 3, 5, 6, 16, DType::BFloat16); } catch (const DeviceError& e) { refused += e.code == -6; }
    try { b.RoPEPackedAttentionPrefill(&r, a, &t1, &t2, &t3, &t4, &t5, 3, 40, 20, DType::BFloat16); } catch (const DeviceError& e) { refused += e.code == -6; }
    return refused == 3 ? 0 : 1;
}
"""


def test_cpp(tmp_path):
    src, exe = tmp_path / "use.cpp", tmp_path / "use"
    src.write_text(SOURCE % ROOT)
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", str(src), "-o", str(exe)])
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    got = [[float(x) for x in line.split()[1:]] for line in res.stdout.splitlines()]
    for line, (entry, n, rest) in zip(got, WANT.values()):
        refs = [*range(1, n + 1)] + ([0] if entry.startswith("paged_decode") else [])
        assert line == [*refs, 2, *rest], entry
    assert got[4][:9] == [1, 2, 0, 4, 5, 6, 7, 8, 9] and got[4][9] == 1 and got[4][16] == 2
