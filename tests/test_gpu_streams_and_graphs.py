"""What calls of one context share (scratch, arrival counters, RoPE tables) across CUDA graphs and streams: every output has the bits of the same
call made alone."""
import pytest
import torch

from test_gpu_kv4 import decode as decode4, make as make4
from test_gpu_packed_prefill import call as prompt, make as make_prompt

pytestmark = pytest.mark.gpu


@pytest.fixture()
def d():
    """A context of the test's own: nothing allocated yet."""
    import puter_b200

    return puter_b200.Device()


def decode16_inputs(lens, kv, group, fp8=False, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = [-(-n // 16) for n in lens]
    pages = sum(per) + 1
    k, v = (torch.randn(pages, 16, kv * 128, device="cuda", generator=g).to(torch.float8_e4m3fn if fp8 else torch.bfloat16) for _ in range(2))
    table = torch.zeros(len(lens), max(per), dtype=torch.int32, device="cuda")
    order, at = torch.randperm(pages, device="cuda", generator=g).to(torch.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(len(lens), kv * group * 128, device="cuda", generator=g).bfloat16()
    scale = torch.full((kv,), 0.5, device="cuda") if fp8 else None
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale


def decode16(d, t, kv, group, out):
    import puter_b200

    q, k, v, table, ctx, scale = t
    cfg = puter_b200.MultiHeadAttentionConfig(NumHeads=kv * group, HeadDim=128, Causal=True, KVHeadCount=kv)
    d.PagedDecodeAttention(cfg, q, k, v, table, ctx, out, q.shape[0], table.shape[1], k.shape[0], 16, 2, kvFormat=4 if scale is not None else 2,
                           kScale=scale, vScale=scale)
    return out


def prefill(d, x, heads, kv, batch, out, rope):
    import puter_b200

    cfg = puter_b200.MultiHeadAttentionConfig(NumHeads=heads, HeadDim=128, Causal=True, KVHeadCount=kv)
    d.RoPEAttentionPrefill(rope, cfg, *x, out, batch, x[0].shape[0] // batch, 2)
    return out


def capture(fn):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fn()
    return graph


@pytest.mark.parametrize("kind", ["bf16", "fp8", "one query", "prefill"])
def test_graphs_of_the_16_bit_steps_keep_their_scratch(d, kind):
    """Captured as the first call of the context; then packed prompts grow the workspace several times and run beside the replays."""
    import puter_b200

    rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=500000.0)
    if kind == "prefill":
        x = make_prompt(2, [600] * 2, 8, 2, 128, 5)[:3]
        run = lambda dev, out: prefill(dev, x, 8, 2, 2, out, rope)  # noqa: E731
        shape = x[0]
    elif kind == "one query":
        q, k, v = (torch.randn(n, h * 128, device="cuda").bfloat16() for n, h in ((1, 16), (5000, 4), (5000, 4)))
        cfg = puter_b200.MultiHeadAttentionConfig(NumHeads=16, HeadDim=128, Causal=True, KVHeadCount=4)
        run = lambda dev, out: dev.MultiHeadAttention(cfg, q, k, v, out, 1, 5000, 2)  # noqa: E731
        shape = q
    else:
        t = decode16_inputs([3000, 17, 900] if kind == "bf16" else [7000] + [40] * 1500, 8, 4, kind == "fp8")
        run = lambda dev, out: decode16(dev, t, 8, 4, out)  # noqa: E731
        shape = t[0]
    out, want = torch.full_like(shape, 7.0), torch.full_like(shape, 7.0)
    graph = capture(lambda: run(d, out))
    run(puter_b200.Device(), want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for n in (500, 2000, 8000):
        big = make_prompt(2, [n] * 2, 32, 8, 128, n)
        alone = prompt(puter_b200.Device(), *big, 32, 8, 128, 2, rope=rope)
        torch.cuda.synchronize()
        got = [torch.full_like(alone, 7.0) for _ in range(3)]
        for o in got:
            prompt(d, *big, 32, 8, 128, 2, rope=rope, out=o)
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(o, alone) for o in got)
        out.fill_(7)
        torch.cuda.synchronize()
    assert d.take_error() == 0


def busy(ms):
    """The current stream is occupied for longer than the host needs for what follows."""
    torch.cuda._sleep(int(ms * 1.8e6))


def raw_capture(graph, stream, fn):
    """What torch.cuda.graph does, without its synchronisation of the device."""
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="thread_local")
        try:
            fn()
        finally:
            graph.capture_end()


def warm(d, run, outs):
    """Scratch of its final size and the tables: growing frees memory, which waits for the device."""
    for i in range(len(outs)):
        run(d, i)
    torch.cuda.synchronize()
    for o in outs:
        o.fill_(7)
    torch.cuda.synchronize()


ROPE = dict(Mode=1, BaseFreq=500000.0)


def prompts(number, d=None):
    """Inputs, outputs and what each call gives alone: different sizes, so that scratch grows and tables differ."""
    import puter_b200

    rope = puter_b200.RoPEConfig(**ROPE)
    ts = [make_prompt(2, [300 + 200 * i, 150], 8, 2, 128, i) for i in range(number)]
    outs = [torch.full_like(t[0], 7.0) for t in ts]
    wants = [prompt(puter_b200.Device(), *t, 8, 2, 128, 2, rope=rope) for t in ts]
    run = lambda dev, i: prompt(dev, *ts[i], 8, 2, 128, 2, rope=rope, out=outs[i])  # noqa: E731
    torch.cuda.synchronize()
    return run, outs, wants


@pytest.mark.parametrize("after", ["the captured stream", "a third stream", "the default stream", "by way of a capture more"])
def test_eager_calls_after_a_capture_follow_those_before_it(d, after):
    """Eager on A, a capture on B that waits for nothing, eager again: the last call uses the scratch of the first, so it comes behind it."""
    run, outs, wants = prompts(4)
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    done = [torch.cuda.Event() for _ in range(2)]
    with torch.cuda.stream(a):
        warm(d, run, outs)
        busy(300)
        run(d, 0)
        done[0].record()
    raw_capture(graph, b, lambda: run(d, 1))
    if after == "by way of a capture more":
        raw_capture(other, c, lambda: run(d, 3))
    last = {"the captured stream": b, "a third stream": c, "the default stream": torch.cuda.default_stream(), "by way of a capture more": b}[after]
    with torch.cuda.stream(last):
        run(d, 2)
        done[1].record()
    done[1].synchronize()
    assert done[0].query()
    graph.replay()
    if after == "by way of a capture more":
        other.replay()
    else:
        run(d, 3)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants)) and d.take_error() == 0


def test_the_error_flag_of_calls_before_a_capture_is_seen(d):
    """take_error waits for the calls on the streams before, too."""
    run, outs, wants = prompts(2)
    t = make4(2, [40], 2, 64, 16, 2, 1)
    t[5][0, 0] = t[1].shape[0]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    graph, out = torch.cuda.CUDAGraph(), torch.full_like(t[0], 7.0)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        busy(300)
        decode4(d, t, 2, 64, 16, 2, 2, out=out)
    raw_capture(graph, b, lambda: run(d, 1))
    with torch.cuda.stream(b):
        assert d.take_error() == 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1], wants[1])


@pytest.mark.parametrize("way", ["plain", "through a fork of the capture"])
def test_eager_calls_beside_a_capture_whose_stream_has_work_queued(d, way):
    """Work queued on B in front of its capture cannot be waited for while the capture is open: a call on C gets scratch of its own."""
    run, outs, wants = prompts(5)
    steps = make4(2, [3000, 17, 900], 8, 128, 16, 4, 1)
    step = [torch.full_like(steps[0], 7.0) for _ in range(2)]
    b, c, side = (torch.cuda.Stream() for _ in range(3))
    want = decode4(d, steps, 8, 128, 16, 4, 2)
    graph = torch.cuda.CUDAGraph()
    fork, join = torch.cuda.Event(), torch.cuda.Event()
    with torch.cuda.stream(b):
        warm(d, run, outs)
        busy(300)
        run(d, 0)
        decode4(d, steps, 8, 128, 16, 4, 2, out=step[0])
        graph.capture_begin(capture_error_mode="relaxed")
        run(d, 1)
        if way != "plain":
            fork.record()
            with torch.cuda.stream(side):
                side.wait_event(fork)
                run(d, 4)
                join.record()
        with torch.cuda.stream(c):
            for _ in range(3):
                run(d, 2)
                decode4(d, steps, 8, 128, 16, 4, 2, out=step[1])
        if way != "plain":
            b.wait_event(join)
        run(d, 3)
        graph.capture_end()
    graph.replay()
    torch.cuda.synchronize()
    if way == "plain":
        run(d, 4)
        torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    assert torch.equal(step[0], want) and torch.equal(step[1], want) and d.take_error() == 0


def test_back_to_the_own_stream_in_the_middle_of_a_capture():
    """cuda_context_reset_stream neither joins its stream to the capture nor forgets the stream before."""
    import ctypes

    import puter_b200

    d = puter_b200.Device(follow_torch_stream=False)
    run, outs, wants = prompts(3)
    adopt = lambda s: d._check(d.lib.cuda_context_set_stream(d.ref, ctypes.c_void_p(s.cuda_stream), ctypes.byref(d._status)))  # noqa: E731
    back = lambda: d._check(d.lib.cuda_context_reset_stream(d.ref, ctypes.byref(d._status)))  # noqa: E731
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    done = torch.cuda.Event()
    graph = torch.cuda.CUDAGraph()
    adopt(a)
    warm(d, run, outs)
    with torch.cuda.stream(a):
        busy(300)
    run(d, 0)
    done.record(a)

    def middle():
        adopt(b)
        run(d, 1)
        back()
        run(d, 2)

    raw_capture(graph, b, middle)
    assert d.take_error() == 0  # (synchronises the own stream, which waits for a)
    assert done.query()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants))


def free_memory():
    import gc

    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("eager", [False, True])
def test_what_captured_calls_hold_is_freed_on_request(d, eager):
    """A program that captures again and again: 4- and 16-bit steps and prompts, each time with another RoPE setting."""
    import puter_b200

    steps = make4(2, [3000, 17, 900], 8, 128, 16, 4, 1)
    step16 = decode16_inputs([3000, 17, 900], 8, 4)
    big = make_prompt(2, [4000, 3000], 8, 2, 128, 1)
    outs = [torch.full_like(x[0], 7.0) for x in (steps, step16, big)]
    wants = [decode4(d, steps, 8, 128, 16, 4, 2), decode16(d, step16, 8, 4, torch.full_like(step16[0], 7.0))]
    free = []
    for i in range(24):
        rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=10000.0 + i)

        def fn():
            decode4(d, steps, 8, 128, 16, 4, 2, out=outs[0])
            decode16(d, step16, 8, 4, outs[1])
            prompt(d, *big, 8, 2, 128, 2, rope=rope, out=outs[2])

        graph = capture(fn)
        for o in outs:
            o.fill_(7)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1])
        if i in (0, 23):
            assert torch.equal(outs[2], prompt(puter_b200.Device(), *big, 8, 2, 128, 2, rope=rope))
        if eager:
            other = puter_b200.RoPEConfig(Mode=1, BaseFreq=20000.0 + i // 2)
            prompt(d, *big, 8, 2, 128, 2, rope=other, out=outs[2])
        graph.reset()
        del graph
        d.release_captures()
        free.append(free_memory())
    assert free[8] - free[23] < 4 << 20, free  # a graph's scratch and table are 25 MB
    assert d.take_error() == 0


def test_release_waits_for_replays_and_is_refused_in_a_capture(d):
    import puter_b200

    run, outs, wants = prompts(2)
    graph, a = capture(lambda: run(d, 0)), torch.cuda.Stream()
    with torch.cuda.stream(a):
        busy(100)
        graph.replay()
    d.release_captures()
    assert torch.equal(outs[0], wants[0])
    graph.reset()

    def refused():
        with pytest.raises(puter_b200.DeviceError) as e:
            d.release_captures()
        assert e.value.code == -2
        run(d, 1)

    again = capture(refused)
    run(d, 0)
    again.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants)) and d.take_error() == 0


@pytest.mark.parametrize("positions", [(1 << 20) + 1, 1 << 20, 1500001])
def test_tables_are_little_larger_than_asked_for(d, positions):
    """maxPositions is a bound that a program may set generously: 512 bytes a position with 128 dimensions, an eighth more at most."""
    import puter_b200

    x = torch.randn(3, 256, device="cuda").bfloat16()
    codes, params = torch.zeros(1, 2, 16, 64, dtype=torch.uint8, device="cuda"), torch.zeros(1, 2, 16, 2, dtype=torch.bfloat16, device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    pos, ids, off = i32([0, 5, positions - 1]), i32([0, 0, 0]), i32([0, 1, 2])
    free = free_memory()
    d.RoPEKVPageWriteQ4(puter_b200.RoPEConfig(Mode=1), x, x, pos, ids, off, codes, params, codes.clone(), params.clone(), 3, 2, 128, 1, 16, positions, 2)
    torch.cuda.synchronize()
    assert 0 <= free - torch.cuda.mem_get_info()[0] <= positions * 512 * 9 // 8 + (16 << 20)
    assert d.take_error() == 0
    pos[2] = positions
    d.RoPEKVPageWriteQ4(puter_b200.RoPEConfig(Mode=1), x, x, pos, ids, off, codes, params, codes.clone(), params.clone(), 3, 2, 128, 1, 16, positions, 2)
    assert d.take_error() == 1
