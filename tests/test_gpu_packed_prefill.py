"""Packed prompts of different lengths: causal grouped attention (RoPE included) against a plain implementation in 64 bits.

Tolerances, with u = eps / 2 of the storage type (half a step of its rounding, relative) and V = max |v|:
  out is rounded once                                                  u |out|
  the weights enter the product rounded to the type, sum of them = 1   u V      (16-bit types; nothing for float32)
  float32 sums over at most 4096 keys, exp2 good to 2^-22              1e-4 V   (scores below 40 in magnitude: 2 * 40 * 2^-20)
  with RoPE, rotated q and k are rounded to the type in both; the float32 rotation may land on the other side of a tie in a few
  elements, each moving a score by at most 2 u |q_d| |k_d| / sqrt(D)   4 u 16 V / sqrt(D)   (|q_d| |k_d| < 16, a move counted twice)
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {1: torch.float16, 2: torch.bfloat16, 0: torch.float32}


@pytest.fixture(scope="module")
def d():
    import puter_b200

    return puter_b200.Device()


def rope64(x, dt, base, mode, start):
    """x [n, heads, dim] rotated at positions start.., angles in 64 bits, rounded to the storage type."""
    n, _, dim = x.shape
    rate = base ** (-torch.arange(0, dim, 2, device=x.device, dtype=torch.float64) / dim)
    angle = (torch.arange(n, device=x.device, dtype=torch.float64) + start)[:, None] * rate
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    a, b = (x[..., :dim // 2], x[..., dim // 2:]) if mode == 1 else (x[..., 0::2], x[..., 1::2])
    lo, hi = a * c - b * s, a * s + b * c
    y = torch.cat([lo, hi], -1) if mode == 1 else torch.stack([lo, hi], -1).flatten(-2)
    return y.to(dt).double()


def attend64(q, k, v, causal):
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.empty(n, heads, dim, dtype=torch.float64, device=q.device)
    hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if causal else None
    for h in range(heads):
        s = q[:, h] @ k[:, h // group].t() / dim ** 0.5
        if causal:
            s = s.masked_fill(hidden, -torch.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, h // group]
    return out


def make(fmt, lens, heads, kv, dim, seed, lead=0, tail=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = lead + sum(lens) + tail
    q, k, v = (torch.randn(total, h * dim, device="cuda", generator=g).to(TYPES[fmt]) for h in (heads, kv, kv))
    starts = torch.tensor(np.cumsum([lead] + list(lens)), dtype=torch.int32, device="cuda")
    return q, k, v, starts


def call(d, q, k, v, starts, heads, kv, dim, fmt, causal=True, rope=None, longest=None, out=None):
    import puter_b200

    attn = puter_b200.MultiHeadAttentionConfig(NumHeads=heads, HeadDim=dim, Causal=causal, KVHeadCount=kv)
    if out is None:
        out = torch.full_like(q, 7.0)
    n = starts.numel() - 1
    d.RoPEPackedAttentionPrefill(rope, attn, q, k, v, starts, out, n, q.shape[0], q.shape[0] if longest is None else longest, fmt)
    return out


def check(got, q, k, v, starts, heads, kv, dim, fmt, causal, rope):
    """Compares every sequence's rows; rows of no sequence must still hold 7."""
    dt = TYPES[fmt]
    u = torch.finfo(dt).eps / 2
    at = starts.tolist()
    seen = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for a, b in zip(at, at[1:]):
        if b <= a:
            continue
        seen[a:b] = True
        x, y, z = (t[a:b].view(b - a, -1, dim) for t in (q, k, v))
        if rope is not None:
            x, y = (rope64(t, dt, rope.BaseFreq, int(rope.Mode), rope.StartPosition) for t in (x, y))
        want = attend64(x.double(), y.double(), z.double(), causal)
        big = z.double().abs().max()
        tol = u * want.abs() + (u * big if fmt else 0) + 1e-4 * big + (4 * u * 16 * big / dim ** 0.5 if rope is not None else 0)
        err = (got[a:b].view(b - a, heads, dim).double() - want).abs()
        assert bool((err <= tol).all()), f"rows {a}..{b}: {float((err / tol).max()):.2f} of the tolerance"
        norm = float(want.norm())
        assert float(err.norm()) <= (3 * u if fmt else 1e-5) * norm + 1e-12
    assert bool((got[~seen] == 7).all())


RAGGED = [1, 0, 2, 31, 32, 33, 127, 128, 129, 0, 255, 256, 257, 300, 5]


SHORT = [1, 0, 2, 31, 32, 33, 127, 128, 129, 0, 255, 256, 7, 15, 16, 17]


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("longest", [17, 40, 128, 160])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (8, 8, 64), (6, 2, 128), (16, 1, 64), (10, 2, 96), (28, 4, 128), (15, 5, 64), (2, 1, 8)])
def test_calls_without_long_sequences(d, fmt, longest, heads, kv, dim):
    """Few rows per KV head take the kernel for short sequences."""
    lens = [n for n in SHORT if n <= longest]
    q, k, v, starts = make(fmt, lens, heads, kv, dim, 7 * heads + dim, lead=3, tail=5)
    for causal in (True, False):
        got = call(d, q, k, v, starts, heads, kv, dim, fmt, causal=causal, longest=longest)
        check(got, q, k, v, starts, heads, kv, dim, fmt, causal, None)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("dim", [128, 64])
def test_rope_of_short_sequences(d, fmt, mode, dim):
    import puter_b200

    rope = puter_b200.RoPEConfig(BaseFreq=500000.0, Mode=mode, StartPosition=70)
    q, k, v, starts = make(fmt, [1, 65, 0, 128, 33], 12, 4, dim, 5 + mode)
    got = call(d, q, k, v, starts, 12, 4, dim, fmt, rope=rope, longest=128)
    check(got, q, k, v, starts, 12, 4, dim, fmt, True, rope)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (8, 8, 128), (6, 2, 128), (16, 1, 128), (12, 12, 64), (28, 4, 64), (10, 2, 96), (4, 2, 80), (2, 1, 8)])
def test_ragged_lengths_and_head_layouts(d, fmt, heads, kv, dim):
    q, k, v, starts = make(fmt, RAGGED, heads, kv, dim, 11 * heads + dim)
    got = call(d, q, k, v, starts, heads, kv, dim, fmt)
    check(got, q, k, v, starts, heads, kv, dim, fmt, True, None)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("dim", [128, 64, 96])
@pytest.mark.parametrize("start", [0, 70])
def test_rope_restarts_with_every_sequence(d, fmt, mode, dim, start):
    import puter_b200

    rope = puter_b200.RoPEConfig(BaseFreq=500000.0, Mode=mode, StartPosition=start)
    q, k, v, starts = make(fmt, [200, 1, 65, 128, 0, 260], 8, 2, dim, 5 + mode)
    got = call(d, q, k, v, starts, 8, 2, dim, fmt, rope=rope, longest=260)
    check(got, q, k, v, starts, 8, 2, dim, fmt, True, rope)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt,dim", [(2, 128), (1, 64), (2, 72)])
def test_not_causal(d, fmt, dim):
    q, k, v, starts = make(fmt, RAGGED, 8, 2, dim, 3)
    check(call(d, q, k, v, starts, 8, 2, dim, fmt, causal=False), q, k, v, starts, 8, 2, dim, fmt, False, None)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt,heads,kv,dim", [(0, 4, 2, 64), (0, 3, 3, 33), (2, 4, 2, 20), (1, 2, 1, 256), (2, 3, 1, 129)])
def test_types_and_head_dimensions_without_tensor_cores(d, fmt, heads, kv, dim):
    import puter_b200

    q, k, v, starts = make(fmt, [1, 17, 130, 0, 64], heads, kv, dim, dim)
    check(call(d, q, k, v, starts, heads, kv, dim, fmt), q, k, v, starts, heads, kv, dim, fmt, True, None)
    if dim % 2 == 0:
        rope = puter_b200.RoPEConfig(Mode=1)
        got = call(d, q, k, v, starts, heads, kv, dim, fmt, rope=rope)
        if fmt == 0:  # the float32 table and rotation against 64 bits: 2^-22 of a score per element
            check(got, q, k, v, starts, heads, kv, dim, fmt, True, rope)
        else:
            check(got, q, k, v, starts, heads, kv, dim, fmt, True, rope)
    assert d.take_error() == 0


def test_long_sequences(d):
    q, k, v, starts = make(2, [4096, 1500], 8, 2, 128, 9)
    check(call(d, q, k, v, starts, 8, 2, 128, 2), q, k, v, starts, 8, 2, 128, 2, True, None)
    assert d.take_error() == 0


def test_many_sequences(d):
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 40, 3000).tolist()
    q, k, v, starts = make(2, lens, 4, 1, 64, 2)
    check(call(d, q, k, v, starts, 4, 1, 64, 2), q, k, v, starts, 4, 1, 64, 2, True, None)
    assert d.take_error() == 0


@pytest.mark.parametrize("longest", [None, 130])
@pytest.mark.parametrize("dim", [128, 64])
def test_rows_outside_every_sequence_stay_and_do_not_leak(d, dim, longest):
    """NaN and infinities before the first, behind the last and in the neighbouring sequence change nothing."""
    lens = [130, 7, 64, 129]
    q, k, v, starts = make(2, lens, 8, 2, dim, 21, lead=9, tail=200)
    clean = call(d, q, k, v, starts, 8, 2, dim, 2, longest=longest)
    check(clean, q, k, v, starts, 8, 2, dim, 2, True, None)
    for t in (q, k, v):
        t[:9] = float("nan")
        t[9 + sum(lens):] = float("inf")
        t[9 + 130:9 + 137] = float("nan")  # the whole second sequence
    got = call(d, q, k, v, starts, 8, 2, dim, 2, longest=longest)
    keep = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    keep[139:146] = False
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[139:146].isnan().all())
    assert d.take_error() == 0


@pytest.mark.parametrize("length", [290, 128])  # the tile kernel, the kernel for short sequences
@pytest.mark.parametrize("at", [0, 60, 127, 128, 200])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(d, at, length):
    """A NaN key or value at position `at` leaves every earlier row of its own sequence as it was."""
    q, k, v, starts = make(2, [length], 8, 2, 128, 31)
    at = min(at, length - 1)
    clean = call(d, q, k, v, starts, 8, 2, 128, 2)
    for t, x in ((k, float("nan")), (v, float("nan")), (v, float("inf"))):
        old = t[at].clone()
        t[at] = x
        got = call(d, q, k, v, starts, 8, 2, 128, 2)
        assert torch.equal(got[:at], clean[:at])
        assert not bool(got[at:].isfinite().any())
        t[at] = old
    assert d.take_error() == 0


def test_scores_of_minus_infinity_and_extreme_scores(d):
    """Keys whose score is -inf drop out; scores of +-1e4 neither overflow nor make the row NaN."""
    q, k, v, starts = make(2, [200, 40], 4, 2, 128, 8)
    q *= 50
    k *= 50
    got = call(d, q, k, v, starts, 4, 2, 128, 2)
    # such rows are one-hot up to the rounding of scores: 2^-20 of 2e5 in magnitude, so compare where the best key leads by 8
    for a, b in ((0, 200), (200, 240)):
        s = torch.einsum("nhd,mhd->hnm", q[a:b].view(-1, 4, 128).double(), k[a:b].view(-1, 2, 128).repeat_interleave(2, 1).double()) / 128 ** 0.5
        s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
        top = s.topk(min(2, b - a), -1)
        lead = top.values[..., 0] - (top.values[..., 1] if b - a > 1 else 0)
        want = v[a:b].view(-1, 2, 128).repeat_interleave(2, 1).transpose(0, 1).gather(1, top.indices[..., :1].expand(-1, -1, 128))
        sure = (lead > 12) | (torch.arange(b - a, device="cuda") == 0)
        err = (got[a:b].view(-1, 4, 128).transpose(0, 1).double() - want.double()).abs()
        assert bool(sure.any()) and float(err[sure].max()) <= 0.02  # e^-12 * 8 and a rounding of 2^-8 * 4
    k2 = k.clone()
    k2[10] = -torch.inf
    q2 = q.abs()
    got = call(d, q2, k2, v, starts, 4, 2, 128, 2)
    assert bool(got[:10].isfinite().all()) and bool(got[11:].isfinite().all())
    assert d.take_error() == 0


def test_bad_starts_are_skipped_and_flagged(d):
    q, k, v, _ = make(2, [100], 4, 2, 128, 1)
    good = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    want = call(d, q, k, v, good, 4, 2, 128, 2)
    assert d.take_error() == 0
    for starts, longest in (([0, 40, 101], 100), ([0, 40, -3], 100), ([0, 40, 100], 50)):
        got = call(d, q, k, v, torch.tensor(starts, dtype=torch.int32, device="cuda"), 4, 2, 128, 2, longest=longest)
        assert torch.equal(got[:40], want[:40])
        assert bool((got[40:] == 7).all())
        assert d.take_error() == 1


def test_refusals(d):
    import puter_b200

    q, k, v, starts = make(2, [10], 4, 2, 64, 1)
    ok = puter_b200.MultiHeadAttentionConfig(NumHeads=4, HeadDim=64, Causal=True, KVHeadCount=2)
    out = torch.empty_like(q)

    def go(attn=ok, rope=None, out=out, fmt=2, total=10, **kw):
        d.RoPEPackedAttentionPrefill(rope, attn, q, k, v, starts, out, 1, total, 10, fmt)

    go()
    cases = [(-2, dict(attn=puter_b200.MultiHeadAttentionConfig(NumHeads=5, HeadDim=64, Causal=True, KVHeadCount=2))),
             (-6, dict(attn=puter_b200.MultiHeadAttentionConfig(NumHeads=4, HeadDim=64, Causal=True, KVHeadCount=2, WindowSize=3))),
             (-6, dict(attn=puter_b200.MultiHeadAttentionConfig(NumHeads=4, HeadDim=64, Causal=True, KVHeadCount=2, ALiBiSlope=1.0))),
             (-6, dict(fmt=4)), (-2, dict(total=11)), (-2, dict(out=q)), (-2, dict(rope=puter_b200.RoPEConfig(BaseFreq=0.0))),
             (-2, dict(rope=puter_b200.RoPEConfig(Mode=5)))]
    for code, kw in cases:
        with pytest.raises(puter_b200.DeviceError) as e:
            go(**kw)
        assert e.value.code == code
    go(total=0)  # nothing to do is not an error
    assert d.take_error() == 0


def test_two_captured_graphs_and_eager_calls_do_not_share_scratch(d):
    """Two captured calls of different sizes and RoPE settings, replayed at the same time on two streams while eager calls grow the
    context's own workspace and bring other tables."""
    import puter_b200

    first = make(2, [300, 20], 8, 2, 128, 1)
    second = make(1, [90, 1, 400], 4, 4, 64, 2)
    ropes = [puter_b200.RoPEConfig(Mode=1, BaseFreq=500000.0), puter_b200.RoPEConfig(Mode=0)]
    shapes = [(8, 2, 128, 2), (4, 4, 64, 1)]
    wants, outs, graphs = [], [], []
    for t, rope, (h, kv, dim, fmt) in zip((first, second), ropes, shapes):
        wants.append(call(d, *t, h, kv, dim, fmt, rope=rope))
        out = torch.full_like(t[0], 7.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(d, *t, h, kv, dim, fmt, rope=rope, out=out)
        outs.append(out)
        graphs.append(graph)
    big = make(2, [2000] * 4, 16, 4, 128, 3)
    for base in (1e4, 2e4, 3e4, 4e4, 5e4):  # more tables than are kept
        call(d, *big, 16, 4, 128, 2, rope=puter_b200.RoPEConfig(Mode=1, BaseFreq=base))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        assert torch.equal(out, want)
    assert d.take_error() == 0


def test_capture_makes_the_rope_table_that_is_missing(d):
    """A first call with a RoPE setting may be a captured one: the table is there before any replay, and stays while others come and go."""
    import puter_b200

    t = make(2, [30, 200], 4, 2, 128, 1)
    rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=777.0)
    out, graph = torch.full_like(t[0], 7.0), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(d, *t, 4, 2, 128, 2, rope=rope, out=out)
    for base in (11.0, 12.0, 13.0, 14.0, 15.0, 16.0):
        other = puter_b200.RoPEConfig(Mode=1, BaseFreq=base)
        check(call(d, *t, 4, 2, 128, 2, rope=other), *t, 4, 2, 128, 2, True, other)
    graph.replay()
    torch.cuda.synchronize()
    check(out, *t, 4, 2, 128, 2, True, rope)
    assert d.take_error() == 0


@pytest.mark.parametrize("length", [300, 60])  # the tile kernel, the kernel for short sequences
def test_rows_behind_2_to_the_31_elements(d, length):
    import puter_b200

    heads, kv, dim, total = 32, 8, 128, 530000  # 2.17e9 elements of q
    rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=10000.0)
    q, k, v = (torch.zeros(total, h * dim, dtype=torch.bfloat16, device="cuda") for h in (heads, kv, kv))
    live = 3 * length
    for t in (q, k, v):
        t[-live:].normal_()
    starts = torch.tensor([total - live, total - 2 * length - 7, total - length, total], dtype=torch.int32, device="cuda")
    out = call(d, q, k, v, starts, heads, kv, dim, 2, rope=rope, longest=length + 7)
    tail = [t[-live:].clone() for t in (q, k, v)]
    check(out[-live:], *tail, starts - (total - live), heads, kv, dim, 2, True, rope)
    assert bool((out[:4096] == 7).all()) and bool((out[-live - 4096:-live] == 7).all()) and d.take_error() == 0


@pytest.mark.parametrize("longest", [600, 128])  # the tile kernel, the kernel for short sequences
def test_a_replay_follows_other_lengths(d, longest):
    """Lengths come from memory: a captured call of up to `longest` tokens per sequence serves other batches of its size, empty ones too."""
    import puter_b200

    rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=10000.0)
    total = 700
    q, k, v, _ = make(2, [total], 8, 2, 128, 9)
    starts = torch.zeros(7, dtype=torch.int32, device="cuda")
    out, graph = torch.full_like(q, 7.0), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(d, q, k, v, starts, 8, 2, 128, 2, rope=rope, longest=longest, out=out)
    for at in ([0, 100, 100, 228, 230, 231, 300], [5, 5, 5, 5, 5, 5, 5], [0, 1, 2, 3, 131, 259, 259 + min(longest, 441)], [700 - longest, 700, 700, 700, 700, 700, 700]):
        out.fill_(7)
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(out, q, k, v, starts, 8, 2, 128, 2, True, rope)
    assert d.take_error() == 0


def test_two_streams_of_one_capture(d):
    """Both calls use the scratch of the capture: the graph orders them, whatever the program's own streams leave open."""
    ts = [make(2, [300, 20], 8, 2, 128, 1), make(2, [250, 90], 8, 2, 128, 2)]
    import puter_b200

    rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=10000.0)
    wants = [call(d, *t, 8, 2, 128, 2, rope=rope) for t in ts]
    outs, graph, side = [torch.full_like(t[0], 7.0) for t in ts], torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        call(d, *ts[0], 8, 2, 128, 2, rope=rope, out=outs[0])
        with torch.cuda.stream(side):
            call(d, *ts[1], 8, 2, 128, 2, rope=rope, out=outs[1])
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(5):
        for o in outs:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))


def test_lengths_and_settings_of_rope_from_call_to_call(d):
    """Tables are shared by calls of different lengths and told apart by every setting."""
    import puter_b200

    for lens in ([40, 300], [17], [700], [300, 1], [1500, 40], [64], [65]):
        for rope in (puter_b200.RoPEConfig(Mode=1, BaseFreq=10000.0), puter_b200.RoPEConfig(Mode=0, BaseFreq=10000.0),
                     puter_b200.RoPEConfig(Mode=1, BaseFreq=10000.0, StartPosition=9), puter_b200.RoPEConfig(Mode=1, BaseFreq=300.0)):
            for dim in (128, 64):
                t = make(2, lens, 4, 2, dim, len(lens))
                check(call(d, *t, 4, 2, dim, 2, rope=rope, longest=max(lens)), *t, 4, 2, dim, 2, True, rope)


def test_calls_on_other_streams_follow_one_another(d):
    t = make(2, [700, 300], 8, 2, 128, 6)
    want = call(d, *t, 8, 2, 128, 2)
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs.append(call(d, *t, 8, 2, 128, 2, out=torch.full_like(t[0], 7.0)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
