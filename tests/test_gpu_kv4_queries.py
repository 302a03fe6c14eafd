"""Decode attention over the 4-bit cache with queries that are not finite or very far from 1.  Tolerances as in test_gpu_kv4.py: they scale with
the values and the scores."""
import pytest
import torch

from test_gpu_kv4 import check_decode, decode, make, values64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    import puter_b200

    return puter_b200.Device()


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("kv,group,dim", [(2, 8, 128), (3, 5, 64), (2, 16, 128), (2, 16, 64), (1, 32, 128), (2, 4, 128)])
def test_a_query_that_is_not_finite_spoils_its_own_head_only(d, fmt, bad, kv, group, dim):
    """The first head of every group of eight holds one value that is not finite; the one beside it has scores that rise by 20 and fall again
    every 64 tokens, the others scores near zero.  An output is NaN in the first and within tolerance in the rest."""
    page = 16
    t = make(fmt, [2000] * 24 + [50, 1], kv, dim, page, group, 17 + group)
    q, kc, kp, vc, vp, table, ctx = t
    heads = q.view(-1, kv, group, dim)
    heads.mul_(0.01)
    step, least = 0.02, 20 * dim ** 0.5 / (0.8 * dim)
    kp[..., 0], kp[..., 1] = step, 0
    for b, n in enumerate(ctx.tolist()):
        pages = table[b, :-(-n // page)].long()
        high = (torch.arange(pages.numel(), device="cuda") * page // 64 % 2).to(kp.dtype)
        kp[pages, :, :, 1] = (high * least)[:, None, None]
    first = torch.arange(group, device="cuda") % 8 == 0
    beside = torch.arange(group, device="cuda") % 8 == 1
    heads[:, :, beside] = (heads[:, :, beside] * 100).abs()
    heads[:, :, first] = 0
    clean = decode(d, t, kv, dim, page, group, fmt)
    check_decode(clean, t, kv, dim, page, group, fmt)
    spoilt = q.clone()
    spoilt.view(-1, kv, group, dim)[:, :, first, 3] = bad
    got = decode(d, (spoilt, *t[1:]), kv, dim, page, group, fmt).view(-1, kv, group, dim)
    assert bool(got[:, :, first].isnan().all())
    got[:, :, first] = clean.view(-1, kv, group, dim)[:, :, first]
    check_decode(got.view(q.shape), t, kv, dim, page, group, fmt)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("kv,group,dim", [(8, 4, 128), (4, 1, 64), (2, 8, 128)])
@pytest.mark.parametrize("strong", [1, 50, 200, 1000])
def test_a_strong_channel_in_the_query(d, fmt, kv, group, dim, strong):
    """One channel far larger than the others leaves the output as near as its rounding, half a step of the type (2^-11, 2^-8), in the norm over a
    sequence's heads; float32 scores of magnitude S and their exponentials: 2^-22 S of the values."""
    t = make(fmt, [3000, 700, 40, 1], kv, dim, 16, group, 3)
    q, kc, kp, vc, vp, table, ctx = t
    q.view(4, -1, dim)[:, :, 7] *= strong
    got = decode(d, t, kv, dim, 16, group, fmt)
    u = float(torch.finfo(q.dtype).eps) / 2
    for b, n in enumerate(ctx.tolist()):
        pages = table[b, :-(-n // 16)].long()
        k, v = values64(kc, kp, pages, n), values64(vc, vp, pages, n)
        s = torch.einsum("hgd,nhd->hgn", q[b].double().view(kv, group, dim), k) / dim ** 0.5
        want = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(-1)
        assert float((got[b].double() - want).norm()) <= u * float(want.norm()) + 2.0 ** -22 * float(s.abs().max()) * float(v.abs().max()) * want.numel() ** 0.5
    assert d.take_error() == 0


@pytest.mark.parametrize("kv,group,dim", [(2, 4, 128), (3, 1, 64), (2, 8, 128), (1, 16, 64)])
@pytest.mark.parametrize("power", [121, 60, -60, -110])
def test_queries_keys_and_values_of_any_size_in_bf16(d, power, kv, group, dim):
    """Queries times 2^power, keys times 2^-power: the scores are those of ordinary numbers.  Values times 2^power then."""
    t = make(2, [300, 20, 1], kv, dim, 16, group, 6)
    t[0].mul_(2.0 ** power)
    t[2].mul_(2.0 ** -power)
    check_decode(decode(d, t, kv, dim, 16, group, 2), t, kv, dim, 16, group, 2)
    if power > -100:  # (a value of 2^-110 takes part as a subnormal weight: not this format's business)
        t[4].mul_(2.0 ** min(power, 100))
        check_decode(decode(d, t, kv, dim, 16, group, 2), t, kv, dim, 16, group, 2)
    assert d.take_error() == 0
