"""Packed prompts with cuda_context_set_exact(1): per sequence the bits of the calls that it stands for, with the same setting."""
import pytest
import torch

from test_gpu_packed_prefill import RAGGED, call, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    import puter_b200

    dev = puter_b200.Device()
    dev.set_exact(True)
    return dev


def one_by_one(d, q, k, v, starts, heads, kv, dim, fmt, causal, rope):
    import dataclasses

    import puter_b200

    out = torch.full_like(q, 7.0)
    cfg = puter_b200.MultiHeadAttentionConfig(NumHeads=heads, HeadDim=dim, Causal=causal, KVHeadCount=kv)
    at = starts.tolist()
    for a, b in zip(at, at[1:]):
        if a == b:
            continue
        x, y, z, o = (t[a:b].clone() for t in (q, k, v, out))
        if rope is not None:
            for t, h in ((x, heads), (y, kv)):
                turned = torch.empty_like(t)
                d.RoPE(dataclasses.replace(rope), t, turned, b - a, h, dim, fmt)
                t.copy_(turned)
        d.MultiHeadAttention(cfg, x, y, z, o, b - a, b - a, fmt)
        out[a:b] = o
    return out


@pytest.mark.parametrize("fmt", [2, 1, 0])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim,mode", [(8, 2, 128, 1), (6, 3, 64, 0), (4, 2, 96, 1), (4, 4, 40, 2), (2, 1, 256, 1), (1, 1, 30, 0)])
def test_exact_mode(d, fmt, causal, heads, kv, dim, mode):
    import puter_b200

    rope = None if mode == 2 else puter_b200.RoPEConfig(BaseFreq=500000.0, Mode=mode, StartPosition=70)
    t = make(fmt, RAGGED, heads, kv, dim, 31 * heads + dim, lead=3, tail=5)
    got = call(d, *t, heads, kv, dim, fmt, causal=causal, rope=rope)
    want = one_by_one(d, *t, heads, kv, dim, fmt, causal, rope)
    assert torch.equal(got, want) and d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
def test_exact_mode_is_the_prefill_of_each_sequence(d, fmt):
    import puter_b200

    rope = puter_b200.RoPEConfig(BaseFreq=500000.0, Mode=1)
    cfg = puter_b200.MultiHeadAttentionConfig(NumHeads=8, HeadDim=128, Causal=True, KVHeadCount=2)
    q, k, v, starts = make(fmt, [130, 1, 200], 8, 2, 128, 3)
    got = call(d, q, k, v, starts, 8, 2, 128, fmt, rope=rope)
    for a, b in zip(starts.tolist(), starts.tolist()[1:]):
        x, y, z, o = (t[a:b].clone() for t in (q, k, v, got))
        o.fill_(7)
        d.RoPEAttentionPrefill(rope, cfg, x, y, z, o, 1, b - a, fmt)
        assert torch.equal(got[a:b], o)
    assert d.take_error() == 0


def test_exact_mode_flags_bad_starts_and_refuses_long_rows(d):
    import puter_b200

    q, k, v, starts = make(2, [40, 30, 20], 4, 2, 64, 1)
    want = call(d, q, k, v, starts, 4, 2, 64, 2)
    assert d.take_error() == 0
    got = call(d, q, k, v, starts, 4, 2, 64, 2, longest=35)
    assert d.take_error() == 1
    assert bool((got[:40] == 7).all()) and torch.equal(got[40:], want[40:])
    long = torch.zeros(60000, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    with pytest.raises(puter_b200.DeviceError) as e:
        call(d, long, long, long, at, 1, 1, 64, 2)
    assert e.value.code == -6
    assert torch.equal(call(d, long, long, long, at, 1, 1, 64, 2, longest=100)[:100], long[:100])
    d.set_exact(False)
    try:
        call(d, long, long, long, at, 1, 1, 64, 2)
    finally:
        d.set_exact(True)
    assert d.take_error() == 0
