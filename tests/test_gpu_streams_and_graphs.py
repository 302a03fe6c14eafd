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
