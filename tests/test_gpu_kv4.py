"""The paged cache in 4 bits: producer, page gather and decode attention against plain implementations.

Quantisation is defined operation by operation in float32, so codes and params are compared bit for bit (numpy float32 rounds like the
kernel: separate products and sums; the span times float32(1 / 15), the levels by IEEE division).  K goes through a cos / sin table: a table entry may differ from numpy's in the last
bit of float32 on a rare tie of float64, so up to 1 in 10^4 codes may be another one, never by more than one level.

Decode, with u = eps / 2 of the storage type, S = max over tokens of 15 * step (the span of a value's levels), V = max |value|:
  out is rounded once: u |out|;  p * step enters the product in f16: 2^-11 S;  float32 sums and exp2: scores up to 40, 2e-5 V."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {1: torch.float16, 2: torch.bfloat16}


@pytest.fixture(scope="module")
def d():
    import puter_b200

    return puter_b200.Device()


def round16(x, fmt):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TYPES[fmt]).float().numpy()


def quantise(x, fmt):
    """(levels uint8 [..., dim], step, least) of float32 vectors."""
    x = np.asarray(x, np.float32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    step, least = round16((hi - lo) * np.float32(1 / 15), fmt), round16(lo, fmt)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(step > 0, (x - least) / step, np.float32(0))
    return np.clip(np.rint(y), 0, 15).astype(np.uint8), step, least


def rotate(x, pos, base, mode):
    dim = x.shape[-1]
    rate = np.power(base, -np.arange(0, dim, 2) / dim)
    angle = pos.astype(np.float64)[:, None] * rate
    c, s = np.cos(angle).astype(np.float32)[:, None], np.sin(angle).astype(np.float32)[:, None]
    a, b = (x[..., :dim // 2], x[..., dim // 2:]) if mode == 1 else (x[..., 0::2], x[..., 1::2])
    lo, hi = a * c - b * s, a * s + b * c
    return np.concatenate([lo, hi], -1) if mode == 1 else np.stack([lo, hi], -1).reshape(x.shape)


def pool(pages, kv, page, dim, fmt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (pages, kv, page, dim // 2), dtype=torch.uint8, device="cuda", generator=g)
    params = torch.rand(pages, kv, page, 2, device="cuda", generator=g).to(TYPES[fmt])
    return codes, params


def levels(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def append(d, rope, k, v, pos, ids, off, kc, kp, vc, vp, fmt, max_pos=40000):
    rows, kv, dim = k.shape[0], kc.shape[1], 2 * kc.shape[3]
    i32 = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    d.RoPEKVPageWriteQ4(rope, k, v, i32(pos), i32(ids), i32(off), kc, kp, vc, vp, rows, kv, dim, kc.shape[0], kc.shape[2], max_pos, fmt)


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kv,dim,page", [(8, 128, 16), (1, 128, 1), (3, 64, 20), (5, 128, 24), (4, 64, 64)])
def test_producer(d, fmt, mode, kv, dim, page):
    import puter_b200

    rng = np.random.default_rng(kv * dim + mode)
    rows, pages = 45, 50
    k, v = (torch.from_numpy(rng.standard_normal((rows, kv * dim)).astype(np.float32)).to(TYPES[fmt]).cuda() for _ in range(2))
    pos = rng.integers(0, 40000, rows)
    slots = rng.permutation(pages * page)[:rows]
    ids, off = slots // page, slots % page
    (kc, kp), (vc, vp) = pool(pages, kv, page, dim, fmt, 1), pool(pages, kv, page, dim, fmt, 2)
    before = [t.clone() for t in (kc, kp, vc, vp)]
    rope = None if mode == 2 else puter_b200.RoPEConfig(BaseFreq=500000.0, Mode=mode)
    append(d, rope, k, v, None if mode == 2 else pos, ids, off, kc, kp, vc, vp, fmt)
    assert d.take_error() == 0
    kx, vx = (t.float().cpu().numpy().reshape(rows, kv, dim) for t in (k, v))
    if mode != 2:
        kx = rotate(kx, pos, 500000.0, mode)
    for x, c, p, loose in ((kx, kc, kp, mode != 2), (vx, vc, vp, False)):
        lev, step, least = quantise(x, fmt)
        got = levels(c)[ids, :, off].cpu().numpy()
        gp = p[ids, :, off].float().cpu().numpy()
        if loose:
            assert (got != lev).mean() <= 1e-4 and np.abs(got.astype(int) - lev).max() <= 1
            assert (gp != np.concatenate([step, least], -1)).mean() <= 1e-2
        else:
            assert np.array_equal(got, lev) and np.array_equal(gp, np.concatenate([step, least], -1))
        # what comes back is within half a level, and the rounding of step and least at the ends
        u = float(torch.finfo(TYPES[fmt]).eps) / 2
        assert (np.abs(gp[..., 1:] + gp[..., :1].astype(np.float64) * got - x) <= step * (0.5 + 1e-4) + u * (np.abs(least) + 15 * step)).all()
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[ids, off] = False
    rest = rest.cuda()
    for t, old in zip((kc, kp, vc, vp), before):
        assert torch.equal(t.transpose(1, 2)[rest], old.transpose(1, 2)[rest])


@pytest.mark.parametrize("fmt", [2, 1])
def test_producer_ties_constants_and_values_that_are_not_finite(d, fmt):
    dim, kv = 128, 2
    x = torch.zeros(12, kv, dim)
    ramp = torch.arange(dim) % 31
    x[0] = ramp * 0.5                       # step 1: every second element sits on a tie
    x[1] = -3.25                            # constant: step 0
    x[2] = torch.linspace(-1, 1, dim)
    x[3, :, 5] = float("nan")
    x[4, :, 7] = float("inf")
    x[5, :, 0] = float("-inf")
    x[6] = ramp * 1e-7                      # f16: subnormal elements, a step of a few units of the last place
    x[7] = (ramp - 15) * 4000.0             # f16: a span of 120000
    x[8] = 1000 + ramp * 2 ** -4            # least is far larger than the step
    x[9, :, :64] = 1
    x[10] = -ramp * 0.5
    if fmt == 2:
        x[11] = (ramp - 15) * 1e36
    k = x.to(TYPES[fmt]).cuda().reshape(12, -1)
    (kc, kp), (vc, vp) = pool(2, kv, 16, dim, fmt, 1), pool(2, kv, 16, dim, fmt, 2)
    append(d, None, k, k, None, np.ones(12), np.arange(12), kc, kp, vc, vp, fmt)
    assert torch.equal(kc, vc) is False and torch.equal(kc[1, :, :12], vc[1, :, :12]) and torch.equal(kp[1, :, :12].view(torch.int16), vp[1, :, :12].view(torch.int16))
    good = [0, 1, 2, 6, 7, 8, 9, 10, 11]
    lev, step, least = quantise(k.float().cpu().numpy().reshape(12, kv, dim)[good], fmt)
    got = levels(vc[1].transpose(0, 1))[good].cpu().numpy()
    gp = vp[1].transpose(0, 1)[good].float().cpu().numpy()
    assert np.array_equal(gp, np.concatenate([step, least], -1))
    assert np.array_equal(got, lev)
    table = torch.tensor([1], dtype=torch.int32, device="cuda")
    out = torch.zeros(16, kv * dim, dtype=TYPES[fmt], device="cuda")
    d.KVPageGatherQ4(vc, vp, table, out, 2, 16, kv, dim, 16, fmt)
    assert bool(out[3:6].isnan().all()) and bool(out[good].isfinite().all())
    assert torch.equal(out[1], k[1])
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("kv,dim,page,rows", [(8, 128, 16, 1000), (1, 64, 1, 7), (3, 128, 20, 41), (7, 64, 24, 1), (2, 128, 256, 700)])
def test_gather(d, fmt, kv, dim, page, rows):
    entries = -(-rows // page)
    codes, params = pool(entries + 5, kv, page, dim, fmt, rows)
    table = torch.randperm(entries + 5, device="cuda")[:entries].to(torch.int32)
    out = torch.full((rows + 3, kv * dim), 7.0, dtype=TYPES[fmt], device="cuda")
    d.KVPageGatherQ4(codes, params, table, out, entries + 5, page, kv, dim, rows, fmt)
    t = table.long()
    x = params[t][..., 1:].double() + params[t][..., :1].double() * levels(codes[t]).double()
    want = x.transpose(1, 2).reshape(-1, kv * dim)[:rows]
    u = float(torch.finfo(TYPES[fmt]).eps) / 2
    assert bool(((out[:rows].double() - want).abs() <= u * (1 + 1e-5) * want.abs() + 1e-7).all())  # one rounding of a float32 result
    assert bool((out[rows:] == 7).all())
    assert d.take_error() == 0


def test_bad_rows_and_pages_are_skipped_and_flagged(d):
    import puter_b200

    kv, dim, page, pages, fmt = 2, 64, 16, 3, 2
    x = torch.randn(6, kv * dim, device="cuda").bfloat16()
    (kc, kp), (vc, vp) = pool(pages, kv, page, dim, fmt, 1), pool(pages, kv, page, dim, fmt, 2)
    old = [t.clone() for t in (kc, kp, vc, vp)]
    rope = puter_b200.RoPEConfig()
    append(d, rope, x, x, [0, 0, 0, 100, -1, 5], [3, -1, 0, 0, 0, 1], [0, 0, 16, 0, 0, 4], kc, kp, vc, vp, fmt, max_pos=100)
    assert d.take_error() == 1
    keep = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    keep[1, 4] = False
    for t, o in zip((kc, kp, vc, vp), old):
        assert torch.equal(t.transpose(1, 2)[keep], o.transpose(1, 2)[keep])
        assert not torch.equal(t.transpose(1, 2)[1, 4], o.transpose(1, 2)[1, 4])
    out = torch.full((40, kv * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    d.KVPageGatherQ4(kc, kp, torch.tensor([1, 9, 2], dtype=torch.int32, device="cuda"), out, pages, page, kv, dim, 40, fmt)
    assert d.take_error() == 1
    assert bool((out[16:32] == 7).all()) and not bool((out[:16] == 7).all()) and not bool((out[32:] == 7).all())


def test_offsets_behind_4_gigabytes(d):
    """Producer, gather and decode attention in the last pages of pools whose byte offsets pass 32 bits."""
    kv, dim, page, group, fmt, pages = 8, 128, 16, 4, 2, 560000  # 4.6 GB of codes a side
    g = torch.Generator(device="cuda").manual_seed(61)
    pools = [torch.empty(pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    params = [torch.zeros(pages, kv, page, 2, dtype=TYPES[fmt], device="cuda") for _ in range(2)]
    rows = 40
    k, v = (torch.randn(rows, kv * dim, device="cuda", generator=g).to(TYPES[fmt]) for _ in range(2))
    where = [pages - 1, 7, pages - 3]
    append(d, None, k, v, None, [where[r // page] for r in range(rows)], [r % page for r in range(rows)], pools[0], params[0], pools[1], params[1], fmt)
    table = torch.tensor([where], dtype=torch.int32, device="cuda")
    outs = []
    for codes, par, x in zip(pools, params, (k, v)):
        out = torch.full((rows, kv * dim), 7.0, dtype=TYPES[fmt], device="cuda")
        d.KVPageGatherQ4(codes, par, table.view(-1), out, pages, page, kv, dim, rows, fmt)
        n, step, least = quantise(x.float().cpu().numpy().reshape(rows, kv, dim), fmt)
        want = torch.from_numpy(least.astype(np.float64) + step.astype(np.float64) * n).to(TYPES[fmt]).reshape(rows, -1)
        assert torch.equal(out.cpu(), want)
        outs.append(out)
    t = (torch.randn(1, kv * group * dim, device="cuda", generator=g).to(TYPES[fmt]), pools[0], params[0], pools[1], params[1], table,
         torch.tensor([rows], dtype=torch.int32, device="cuda"))
    check_decode(decode(d, t, kv, dim, page, group, fmt), t, kv, dim, page, group, fmt)
    assert d.take_error() == 0


# ---------------------------------------------------------------------------------------------------------------------- decode
def make(fmt, lens, kv, dim, page, group, seed, sharp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lens), max(per + [1]) + 1), 0, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    made = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pages, kv, page, dim // 2), dtype=torch.uint8, device="cuda", generator=g)
        step = torch.rand(pages, kv, page, 1, device="cuda", generator=g) * 0.4 + 0.1
        least = -7.5 * step + torch.randn(pages, kv, page, 1, device="cuda", generator=g) * 0.2
        made.append((codes, torch.cat([step, least], -1).to(TYPES[fmt])))
    q = (torch.randn(len(lens), kv * group * dim, device="cuda", generator=g) * sharp).to(TYPES[fmt])
    return q, *made[0], *made[1], table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def decode(d, t, kv, dim, page, group, fmt, out=None, flag=None):
    import puter_b200

    q, kc, kp, vc, vp, table, ctx = t
    cfg = puter_b200.MultiHeadAttentionConfig(NumHeads=kv * group, HeadDim=dim, Causal=True, KVHeadCount=kv)
    if out is None:
        out = torch.full_like(q, 7.0)
    d.PagedDecodeAttentionQ4(cfg, q, kc, kp, vc, vp, table, ctx, out, q.shape[0], table.shape[1], kc.shape[0], page, fmt, errorFlag=flag)
    return out


def values64(codes, params, pages, n):
    x = params[pages][..., 1:].double() + params[pages][..., :1].double() * levels(codes[pages]).double()
    return x.transpose(1, 2).flatten(0, 1)[:n]


def check_decode(got, t, kv, dim, page, group, fmt):
    q, kc, kp, vc, vp, table, ctx = t
    u = float(torch.finfo(TYPES[fmt]).eps) / 2
    for b, n in enumerate(ctx.tolist()):
        if n == 0:
            assert bool((got[b] == 7).all())
            continue
        pages = table[b, :-(-n // page)].long()
        k, v = values64(kc, kp, pages, n), values64(vc, vp, pages, n)
        s = torch.einsum("hgd,nhd->hgn", q[b].double().view(kv, group, dim), k) / dim ** 0.5
        want = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(-1)
        span = 15 * float(vp[pages][..., 0].transpose(1, 2).flatten(0, 1)[:n].max())
        tol = u * want.abs() + 2.0 ** -11 * span + 2e-5 * float(v.abs().max()) * max(1.0, float(s.abs().max()) / 40)
        err = (got[b].double() - want).abs()
        assert bool((err <= tol).all()), f"sequence {b} of {n}: {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("kv,group,dim,page", [(8, 4, 128, 16), (2, 16, 128, 64), (12, 1, 64, 20), (1, 32, 128, 16), (5, 3, 128, 24), (8, 8, 64, 16), (1, 1, 64, 1),
                                               (16, 2, 128, 32), (3, 9, 64, 128), (9, 5, 128, 8)])
def test_decode_layouts_and_lengths(d, fmt, kv, group, dim, page):
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 64, 100, 513, 1500, 0, 7]
    t = make(fmt, lens, kv, dim, page, group, kv * 100 + group)
    check_decode(decode(d, t, kv, dim, page, group, fmt), t, kv, dim, page, group, fmt)
    assert d.take_error() == 0


@pytest.mark.parametrize("lens", [[1], [40000], [20000, 3], [5] * 700, [1] * 1100 + [300], [16 * 148, 16 * 148 * 2 + 1]])
def test_decode_batches(d, lens):
    t = make(2, lens, 8, 128, 16, 4, len(lens))
    check_decode(decode(d, t, 8, 128, 16, 4, 2), t, 8, 128, 16, 4, 2)
    t = make(1, lens, 2, 64, 16, 2, len(lens))
    check_decode(decode(d, t, 2, 64, 16, 2, 1), t, 2, 64, 16, 2, 1)
    assert d.take_error() == 0


@pytest.mark.parametrize("kv,group", [(2, 16), (8, 4), (4, 8), (1, 3)])
@pytest.mark.parametrize("lens", [[9000], [30000, 28000], [20000, 0, 17000, 0], [7000, 6900, 5000], [1, 40, 2, 3, 17, 1, 1, 90, 2000] * 12, [3000] + [1] * 60])
def test_decode_where_blocks_divide_pairs(d, kv, group, lens):
    """Whole blocks per pair, blocks that end one pair and begin another, blocks of many pairs; starts that cost more than their pair."""
    t = make(2, lens, kv, 128, 16, group, 13)
    check_decode(decode(d, t, kv, 128, 16, group, 2), t, kv, 128, 16, group, 2)
    assert d.take_error() == 0


@pytest.mark.parametrize("fmt", [2, 1])
def test_decode_peaked_scores_and_steps_of_very_different_size(d, fmt):
    kv, group, dim, page = 4, 4, 128, 16
    t = make(fmt, [700, 33], kv, dim, page, group, 3, sharp=6.0)
    check_decode(decode(d, t, kv, dim, page, group, fmt), t, kv, dim, page, group, fmt)
    # value steps over a factor of 1000, growing along the sequence and shrinking: the weights are scaled as they go
    for order in (1, -1):
        t = make(fmt, [700, 33], kv, dim, page, group, 4)
        vp, table = t[4], t[5]
        for b, n in enumerate((700, 33)):
            f = torch.logspace(-1.5 * order, 1.5 * order, -(-n // page), device="cuda").to(vp.dtype)
            vp[table[b, :f.numel()].long()] *= f[:, None, None, None]
        check_decode(decode(d, t, kv, dim, page, group, fmt), t, kv, dim, page, group, fmt)
    assert d.take_error() == 0


def test_decode_large_queries_in_bf16(d):
    """bf16 queries far outside the range of f16, with keys small enough for ordinary scores."""
    kv, group, dim, page = 2, 4, 128, 16
    t = make(2, [300, 20], kv, dim, page, group, 6)
    t[0].mul_(1e6)
    t[2].mul_(1e-6)
    check_decode(decode(d, t, kv, dim, page, group, 2), t, kv, dim, page, group, 2)
    assert d.take_error() == 0


@pytest.mark.parametrize("page", [16, 20])
def test_decode_does_not_read_behind_the_context(d, page):
    """NaN parameters behind the last token and in unused pages change nothing; a zero query gives the mean of the values."""
    kv, group, dim = 3, 4, 128
    t = make(2, [37, 1, 160], kv, dim, page, group, 5)
    want = decode(d, t, kv, dim, page, group, 2)
    q, kc, kp, vc, vp, table, ctx = t
    live = torch.zeros(kc.shape[0], page, dtype=torch.bool, device="cuda")
    for b, n in enumerate((37, 1, 160)):
        at = torch.arange(n, device="cuda")
        live[table[b, at // page].long(), at % page] = True
    for p in (kp, vp):
        p.transpose(1, 2)[~live] = float("nan")
    assert torch.equal(decode(d, t, kv, dim, page, group, 2), want)
    q.zero_()
    check_decode(decode(d, t, kv, dim, page, group, 2), t, kv, dim, page, group, 2)
    assert d.take_error() == 0


def test_decode_flags(d):
    kv, group, dim, page = 2, 4, 128, 16
    t = make(2, [100, 40], kv, dim, page, group, 2)
    want = decode(d, t, kv, dim, page, group, 2)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    for change in ("page", "negative page", "long", "negative"):
        q, kc, kp, vc, vp, table, ctx = (x.clone() for x in t)
        if change == "page":
            table[0, 2] = kc.shape[0]
        elif change == "negative page":
            table[0, 0] = -1
        else:
            ctx[0] = 10 ** 6 if change == "long" else -5
        got = decode(d, (q, kc, kp, vc, vp, table, ctx), kv, dim, page, group, 2)
        assert d.take_error() == 1
        if "page" in change:
            assert torch.equal(got[1], want[1])
        else:  # another length of sequence 0 divides the work at other tokens of sequence 1: other sums, the same tolerance
            ctx[0] = 0
            got[0] = 7
            check_decode(got, (q, kc, kp, vc, vp, table, ctx), kv, dim, page, group, 2)
            ctx[0] = 10 ** 6 if change == "long" else -5
        decode(d, (q, kc, kp, vc, vp, table, ctx), kv, dim, page, group, 2, flag=flag)
        assert int(flag) == 1 and d.take_error() == 0
        flag.zero_()


def test_decode_repeats_its_bits_and_replays_from_graphs(d):
    a, b = make(2, [3000, 17, 900], 8, 128, 16, 4, 1), make(1, [5000], 2, 64, 16, 8, 2)
    shapes = [(8, 128, 16, 4, 2), (2, 64, 16, 8, 1)]
    wants = [decode(d, t, *s) for t, s in zip((a, b), shapes)]
    for t, s, w in zip((a, b), shapes, wants):
        assert all(torch.equal(decode(d, t, *s), w) for _ in range(5))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t, s in zip((a, b), shapes):
        out, graph = torch.full_like(t[0], 7.0), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            decode(d, t, *s, out=out)
        graphs.append(graph)
        outs.append(out)
    big = make(2, [50] * 900, 8, 128, 16, 4, 7)
    check_decode(decode(d, big, 8, 128, 16, 4, 2), big, 8, 128, 16, 4, 2)
    torch.cuda.synchronize()
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    assert d.take_error() == 0


def test_two_graphs_of_decode_steps_replayed_at_the_same_time(d):
    """Each graph has its own scratch; a launch that waits for its other blocks has all of them on the GPU."""
    shapes = [(8, 128, 16, 4, 2), (2, 128, 16, 16, 1)]
    ts = [make(2, [3000, 17, 900, 12000], 8, 128, 16, 4, 41), make(1, [5000, 8000], 2, 128, 16, 16, 42)]
    wants = [decode(d, t, *s) for t, s in zip(ts, shapes)]
    outs, graphs = [torch.full_like(t[0], 7.0) for t in ts], []
    torch.cuda.synchronize()
    for t, s, o in zip(ts, shapes, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(10):
                decode(d, t, *s, out=o)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants)) and d.take_error() == 0


def test_a_decode_replay_follows_its_lengths_and_pages(d):
    """Lengths, page table and queries come from memory: the step grows from token to token, one sequence ends, another is added."""
    kv, dim, page, group, fmt = 4, 128, 16, 4, 2
    q, kc, kp, vc, vp, table, ctx = make(fmt, [900, 40, 2000, 16], kv, dim, page, group, 51)
    table = torch.cat([table, table[:, -1:].repeat(1, 3)], 1)
    out, graph = torch.full_like(q, 7.0), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        decode(d, (q, kc, kp, vc, vp, table, ctx), kv, dim, page, group, fmt, out=out)
    for lens in ([900, 40, 2000, 16], [901, 41, 2001, 17], [0, 42, 2002, 0], [1, 2000, 0, 2000], [0, 0, 0, 0]):
        out.fill_(7)
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(torch.randint(0, kc.shape[0], table.shape, device="cuda").to(torch.int32))
        q.copy_(torch.randn(q.shape, device="cuda").to(q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        check_decode(out, (q, kc, kp, vc, vp, table, ctx), kv, dim, page, group, fmt)
    assert d.take_error() == 0


@pytest.mark.parametrize("group,kv", [(16, 2), (2, 4), (7, 1)])
def test_decode_of_long_contexts_in_f16(d, group, kv):
    """What many tokens leave of values that nearly cancel is small: the error stays that of the output's rounding, 2^-11 of it.
    The weights (two f16 parts, 2^-22) and float32 sums of codes less 8 (a few hundred terms per warp, 2^-24 each, of sums no larger
    than the square root of their number) together stay below another 2^-11."""
    t = make(1, [60001], kv, 128, 16, group, 11)
    got = decode(d, t, kv, 128, 16, group, 1)
    q, kc, kp, vc, vp, table, ctx = t
    pages = table[0, :-(-60001 // 16)].long()
    k, v = values64(kc, kp, pages, 60001), values64(vc, vp, pages, 60001)
    s = torch.einsum("hgd,nhd->hgn", q[0].double().view(kv, group, 128), k) / 128 ** 0.5
    want = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(-1)
    assert float((got[0].double() - want).norm()) <= 2.0 ** -10 * float(want.norm())


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("kv,group,dim,page", [(8, 4, 128, 16), (2, 16, 64, 20), (4, 7, 128, 64)])
def test_decode_with_a_plain_launch(d, monkeypatch, fmt, kv, group, dim, page):
    """Where a cooperative launch is refused, the last block to arrive joins a pair's parts."""
    t = make(fmt, [9000, 1, 700, 33, 0, 2500], kv, dim, page, group, 21)
    monkeypatch.setenv("PUTER_DECODE_NO_COOPERATIVE", "1")
    first = decode(d, t, kv, dim, page, group, fmt)
    check_decode(first, t, kv, dim, page, group, fmt)
    assert torch.equal(decode(d, t, kv, dim, page, group, fmt), first)
    monkeypatch.delenv("PUTER_DECODE_NO_COOPERATIVE")
    check_decode(decode(d, t, kv, dim, page, group, fmt), t, kv, dim, page, group, fmt)
    assert d.take_error() == 0


def test_decode_where_the_output_is_the_query(d):
    """Every part of a pair has read the query before its output is written."""
    t = make(2, [5000, 3, 800] * 20, 8, 128, 16, 4, 31)
    want = decode(d, t, 8, 128, 16, 4, 2)
    for _ in range(3):
        q = t[0].clone()
        decode(d, (q, *t[1:]), 8, 128, 16, 4, 2, out=q)
        assert torch.equal(q, want)


@pytest.mark.parametrize("fmt", [2, 1])
def test_gather_to_an_odd_address(d, fmt):
    """16 but not 32 bytes aligned: the narrower stores."""
    codes, params = pool(5, 3, 16, 128, fmt, 4)
    table = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    n = 40 * 3 * 128
    room = torch.full((n + 16,), 7.0, dtype=TYPES[fmt], device="cuda")
    assert room.data_ptr() % 32 == 0
    outs = [room[at:at + n] for at in (0, 8)]
    got = []
    for out in outs:
        d.KVPageGatherQ4(codes, params, table, out, 5, 16, 3, 128, 40, fmt)
        got.append(out.clone())
    assert torch.equal(got[0], got[1]) and bool((room[n + 8:] == 7).all())


def test_append_in_a_graph_follows_its_inputs(d):
    """A captured step of one token per sequence, replayed with other tokens at other places (slots, positions and values come from
    memory); the RoPE table is made during the capture."""
    import puter_b200

    kv, dim, page, pages, fmt = 2, 128, 16, 6, 2
    rope = puter_b200.RoPEConfig(Mode=1, BaseFreq=4321.0)
    g = torch.Generator(device="cuda").manual_seed(3)
    xs = [torch.randn(3, kv * dim, device="cuda", generator=g).bfloat16() for _ in range(4)]
    where = [([5, 0, 2], [0, 15, 7], [80, 15, 39]), ([1, 3, 4], [4, 5, 6], [4, 99, 0])]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = torch.zeros_like(xs[0]), torch.zeros_like(xs[0])
    ids, off, pos = i32([0, 0, 0]), i32([0, 1, 2]), i32([0, 0, 0])
    mine, plain = [[*pool(pages, kv, page, dim, fmt, 1), *pool(pages, kv, page, dim, fmt, 2)] for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        d.RoPEKVPageWriteQ4(rope, k, v, pos, ids, off, *mine, 3, kv, dim, pages, page, 100, fmt)
    for n, (p, o, at) in enumerate(where):
        k.copy_(xs[2 * n]), v.copy_(xs[2 * n + 1]), ids.copy_(i32(p)), off.copy_(i32(o)), pos.copy_(i32(at))
        graph.replay()
        append(d, rope, xs[2 * n], xs[2 * n + 1], at, p, o, *plain, fmt, max_pos=100)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(mine, plain)) and d.take_error() == 0


def test_refusals(d):
    import puter_b200

    kv, group, dim, page, fmt = 2, 2, 64, 16, 2
    q, kc, kp, vc, vp, table, ctx = make(fmt, [20], kv, dim, page, group, 1)
    x = torch.zeros(2, kv * dim, dtype=torch.bfloat16, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    cfg = lambda **k: puter_b200.MultiHeadAttentionConfig(**{**dict(NumHeads=4, HeadDim=64, Causal=True, KVHeadCount=2), **k})  # noqa: E731
    n = kc.shape[0]
    rope = puter_b200.RoPEConfig
    calls = [
        (-6, lambda: d.RoPEKVPageWriteQ4(None, x, x, None, i, i, kc, kp, vc, vp, 2, kv, 32, n, page, 9, fmt)),
        (-6, lambda: d.RoPEKVPageWriteQ4(None, x, x, None, i, i, kc, kp, vc, vp, 2, kv, dim, n, page, 9, 0)),
        (-2, lambda: d.RoPEKVPageWriteQ4(rope(), x, x, None, i, i, kc, kp, vc, vp, 2, kv, dim, n, page, 9, fmt)),
        (-2, lambda: d.RoPEKVPageWriteQ4(rope(), x, x, i, i, i, kc, kp, vc, vp, 2, kv, dim, n, page, 0, fmt)),
        (-2, lambda: d.RoPEKVPageWriteQ4(rope(BaseFreq=-1.0), x, x, i, i, i, kc, kp, vc, vp, 2, kv, dim, n, page, 9, fmt)),
        (-2, lambda: d.RoPEKVPageWriteQ4(None, x, x, None, i, i, kc, kp, vc, vp, 3, kv, dim, n, page, 9, fmt)),
        (-2, lambda: d.RoPEKVPageWriteQ4(None, x, x, None, i, i, kc, kp, vc, vp, 2, kv, dim, n + 1, page, 9, fmt)),
        (-6, lambda: d.KVPageGatherQ4(kc, kp, table, x, n, page, kv, 96, 2, fmt)),
        (-6, lambda: d.KVPageGatherQ4(kc, kp, table, x, n, page, kv, dim, 2, 5)),
        (-2, lambda: d.KVPageGatherQ4(kc, kp, table, x, n, page, kv, dim, 3, fmt)),
        (-2, lambda: d.KVPageGatherQ4(kc, None, table, x, n, page, kv, dim, 2, fmt)),
        (-6, lambda: d.PagedDecodeAttentionQ4(cfg(HeadDim=80), q, kc, kp, vc, vp, table, ctx, out, 1, table.shape[1], n, page, fmt)),
        (-2, lambda: d.PagedDecodeAttentionQ4(cfg(NumHeads=5), q, kc, kp, vc, vp, table, ctx, out, 1, table.shape[1], n, page, fmt)),
        (-6, lambda: d.PagedDecodeAttentionQ4(cfg(WindowSize=4), q, kc, kp, vc, vp, table, ctx, out, 1, table.shape[1], n, page, fmt)),
        (-6, lambda: d.PagedDecodeAttentionQ4(cfg(), q, kc, kp, vc, vp, table, ctx, out, 1, table.shape[1], n, page, 0)),
        (-2, lambda: d.PagedDecodeAttentionQ4(cfg(), q, kc, kp, vc, vp, table, ctx, out, 2, table.shape[1], n, page, fmt)),
        (-2, lambda: d.PagedDecodeAttentionQ4(cfg(), q, kc, kp, vc, vp, table, ctx, out, 1, 0, n, page, fmt)),
        (-2, lambda: d.PagedDecodeAttentionQ4(cfg(), q, kc.view(-1)[1:].contiguous().view(-1)[1:], kp, vc, vp, table, ctx, out, 1, table.shape[1], n - 1, page, fmt)),
    ]
    for number, (code, go) in enumerate(calls):
        with pytest.raises(puter_b200.DeviceError) as e:
            go()
        assert e.value.code == code, number
    d.RoPEKVPageWriteQ4(None, x, x, None, i, i, kc, kp, vc, vp, 0, kv, dim, n, page, 9, fmt)  # nothing to do is not an error
    d.KVPageGatherQ4(kc, kp, table, x, n, page, kv, dim, 0, fmt)
    d.PagedDecodeAttentionQ4(cfg(), q, kc, kp, vc, vp, table, ctx, out, 0, table.shape[1], n, page, fmt)
    assert d.take_error() == 0


# -------------------------------------------------------------------------------------------------------------- all of them together
@pytest.mark.parametrize("fmt,mode", [(2, 1), (1, 0)])
def test_prompt_then_cache_then_decode(d, fmt, mode):
    """A serving step over three prompts: attend, fill the 4-bit cache, decode two tokens, read a prefix back."""
    import puter_b200
    from test_gpu_packed_prefill import call as attend, check as check_prompt

    kv, group, dim, page, heads, dt = 2, 4, 128, 16, 8, TYPES[fmt]
    lens = [130, 1, 47]
    g = torch.Generator(device="cuda").manual_seed(5)
    normal = lambda n, h: torch.randn(n, h * dim, device="cuda", generator=g).to(dt)  # noqa: E731
    rope = puter_b200.RoPEConfig(Mode=mode, BaseFreq=500000.0)
    q, k, v = normal(sum(lens), heads), normal(sum(lens), kv), normal(sum(lens), kv)
    starts = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
    check_prompt(attend(d, q, k, v, starts, heads, kv, dim, fmt, rope=rope), q, k, v, starts, heads, kv, dim, fmt, True, rope)
    pages = 40
    (kc, kp), (vc, vp) = pool(pages, kv, page, dim, fmt, 1), pool(pages, kv, page, dim, fmt, 2)
    table = torch.randperm(pages, device="cuda", generator=g)[:36].view(3, 12).to(torch.int32)
    host = table.cpu().numpy()
    pos = np.concatenate([np.arange(n) for n in lens])
    seq = np.repeat(np.arange(3), lens)
    append(d, rope, k, v, pos, host[seq, pos // page], pos % page, kc, kp, vc, vp, fmt)
    kx = rotate(k.float().cpu().numpy().reshape(-1, kv, dim), pos, 500000.0, mode)
    vx = v.float().cpu().numpy().reshape(-1, kv, dim)
    now = list(lens)
    for _ in range(2):
        qn, kn, vn = normal(3, heads), normal(3, kv), normal(3, kv)
        at = np.array(now)
        append(d, rope, kn, vn, at, host[np.arange(3), at // page], at % page, kc, kp, vc, vp, fmt)
        now = [n + 1 for n in now]
        t = (qn, kc, kp, vc, vp, table, torch.tensor(now, dtype=torch.int32, device="cuda"))
        check_decode(decode(d, t, kv, dim, page, group, fmt), t, kv, dim, page, group, fmt)
    for b, n in enumerate(lens):  # the prefix read back is the prompt's K and V up to half a level
        for x, c, p in ((kx, kc, kp), (vx, vc, vp)):
            out = torch.empty(n, kv * dim, dtype=dt, device="cuda")
            d.KVPageGatherQ4(c, p, table[b].contiguous(), out, pages, page, kv, dim, n, fmt)
            mine = x[seq == b]
            step = (mine.max(-1, keepdims=True) - mine.min(-1, keepdims=True)) / 15
            u = float(torch.finfo(dt).eps) / 2  # roundings of step and least (both at most max |x|) and of the result
            assert (np.abs(out.float().cpu().numpy().reshape(n, kv, dim) - mine) <= 0.51 * step + u * 4 * np.abs(mine).max()).all()
    assert d.take_error() == 0
