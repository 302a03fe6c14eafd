"""Cases, plain forms and exact values of the prompt and 4-bit-cache operators.

Four operators, as a serving loop calls them:

  prompt   causal attention over packed prompts of different lengths, grouped heads, RoPE restarting with every prompt
  append   rotate K, quantise K and V to 4 bits and write them into a paged cache; read back as the next chunk of a prompt would (gather)
  gather   pages of the 4-bit cache back to 16 bits
  decode   attention of one new token per sequence over the 4-bit paged cache

The 4-bit cache: codes [pages, kvHeads, pageSize, dim / 2] (byte j of a row holds element 2j in its low and 2j + 1 in its high four
bits) and params [pages, kvHeads, pageSize, 2] = (step, least) in the 16-bit type of the inputs; an element is least + step * code.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_FORMATS = {"f16": 1, "bf16": 2}  # element codes of the C ABI
_BASE = 500000.0


# ---------------------------------------------------------------------------------------------------------------------- cases
def _case(name, op, dtype, heads, kv, dim, batch, shortest, longest, mix, **more):
    return dict(name=name, op=op, dtype=dtype, heads=heads, kv=kv, dim=dim, batch=batch, shortest=shortest, longest=longest, mix=mix, **more)


def listed():
    return [
        # one short prompt: what a chat turn costs before its first token, bound by launches
        _case("prompt_one_short", "prompt", "bf16", 32, 8, 128, 1, 33, 33, 1, rope=1),
        # a serving step's mix of prompts
        _case("prompt_mixed", "prompt", "bf16", 32, 8, 128, 8, 150, 4096, 2, rope=1),
        # one long document
        _case("prompt_long", "prompt", "bf16", 32, 8, 128, 1, 16384, 16384, 3, rope=1),
        # many short inputs of a small model, each head with a cache of its own, rotated beforehand
        _case("prompt_many_short", "prompt", "f16", 12, 12, 64, 200, 1, 96, 4, rope=2),
        # one new token of each of 64 sequences
        _case("append_step", "append", "bf16", 32, 8, 128, 64, 512, 32768, 5, rope=1, page=16, rows=1),
        # the prompts of a prefill step go into the cache
        _case("append_prompts", "append", "bf16", 32, 8, 128, 16, 1000, 8192, 6, rope=1, page=16, rows=0),
        # a cached prefix of one sequence, read back for the next chunk of its prompt
        _case("gather_prefix", "gather", "f16", 32, 8, 128, 1, 1000, 1000, 7, page=64),
        # a long prefix
        _case("gather_long", "gather", "bf16", 32, 8, 128, 1, 131072, 131072, 8, page=16),
        # a single short conversation: bound by latency
        _case("decode_one", "decode", "bf16", 32, 8, 128, 1, 1024, 1024, 9, page=16),
        # the batch that the framework's own decode benchmark runs: 64 sequences of 512 to 32768 tokens
        _case("decode_batch", "decode", "bf16", 32, 8, 128, 64, 512, 32768, 10, page=16),
        # two very long contexts, large pages, many query heads on one KV head
        _case("decode_long", "decode", "f16", 32, 2, 128, 2, 100001, 131072, 11, page=64),
        # a small model with a page size that no tile divides
        _case("decode_small_model", "decode", "f16", 12, 12, 64, 48, 1, 3000, 12, page=20),
    ]


def _log_between(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(["prompt", "append", "gather", "decode", "prompt", "decode"])
    kv, group = rng.choice([(8, 4), (8, 4), (4, 7), (2, 8), (1, 16), (12, 1), (5, 3), (8, 2)])
    dim = rng.choice([128, 128, 64])
    page = rng.choice([16, 16, 32, 64, 128, 1, 20, 24])
    mix = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    batch = _log_between(rng, 1, 64)
    if op == "prompt":
        longest = _log_between(rng, 1, min(8192, 16384 // batch))
        dim = rng.choice([128, 128, 64, 96, 80])
        case = _case("", op, dtype, kv * group, kv, dim, batch, max(1, longest // rng.choice([1, 3, 20])), longest, mix, rope=rng.choice([0, 1, 1, 2]))
    elif op == "append":
        longest = _log_between(rng, 1, min(8192, 40000 // batch))
        case = _case("", op, dtype, kv * group, kv, dim, batch, max(1, longest // 8), longest, mix, rope=rng.choice([0, 1, 1, 2]), page=page, rows=rng.choice([0, 0, 1]))
    elif op == "gather":
        longest = _log_between(rng, 1, 80000)
        case = _case("", op, dtype, kv * group, kv, dim, 1, longest, longest, mix, page=page)
    else:
        longest = _log_between(rng, 1, min(131072, 300000 // batch))
        case = _case("", op, dtype, kv * group, kv, dim, batch, max(1, longest // rng.choice([1, 5, 50])), longest, mix, page=page)
    del case["name"]
    return case


def _lengths(case):
    """The sequence lengths of a case, spread over their logarithm; the first is the longest."""
    rng = random.Random(case["mix"])
    got = [_log_between(rng, case["shortest"], case["longest"]) for _ in range(case["batch"])]
    got[0] = case["longest"]
    return got


def _pages(case):
    """(tokens per sequence, pages per sequence, first page entry per sequence)."""
    n = _lengths(case)
    per = [-(-x // case["page"]) for x in n]
    first = [0]
    for p in per:
        first.append(first[-1] + p)
    return n, per, first


def work(case):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    n = _lengths(case)
    row4 = kv * (dim // 2 + 4)  # a token's codes and params in one pool
    if case["op"] == "prompt":
        return {"bytes": sum(n) * (2 * heads + 2 * kv) * dim * 2, "flops": 4 * dim * heads * sum(x * (x + 1) // 2 for x in n)}
    if case["op"] == "append":
        rows = case["batch"] if case["rows"] else sum(n)
        pages = case["batch"] if case["rows"] else _pages(case)[2][-1]
        back = pages * case["page"]
        return {"bytes": rows * (2 * kv * dim * 2 + 2 * row4 + 12) + back * 2 * (row4 + kv * dim * 2), "flops": rows * 2 * kv * dim * 8 + back * 2 * kv * dim * 2}
    if case["op"] == "gather":
        return {"bytes": sum(n) * (row4 + kv * dim * 2), "flops": sum(n) * kv * dim * 2}
    return {"bytes": sum(n) * 2 * row4 + case["batch"] * heads * dim * 4 + 4 * sum(_pages(case)[1]), "flops": 4 * dim * heads * sum(n)}


# --------------------------------------------------------------------------------------------------------------------- inputs
def _fill(pages, case, gen):
    """A pool of quantised normal values with a few strong channels, as keys have them: (codes, params)."""
    kv, page, dim, dt = case["kv"], case["page"], case["dim"], _TYPES[case["dtype"]]
    strong = 1 + 3 * (torch.rand(kv, 1, dim, device="cuda", generator=gen) > 0.95)
    codes = torch.empty(pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
    params = torch.empty(pages, kv, page, 2, dtype=dt, device="cuda")
    part = max(1, (1 << 27) // (kv * page * dim))
    for a in range(0, pages, part):
        x = torch.randn(min(part, pages - a), kv, page, dim, device="cuda", generator=gen) * strong
        c, p = _quantise(x, dt)
        codes[a:a + part], params[a:a + part] = c, p
    return codes, params


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    heads, kv, dim, dt = case["heads"], case["kv"], case["dim"], _TYPES[case["dtype"]]
    n = _lengths(case)
    st = {"case": case, "longest": max(n)}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dt)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["op"] == "prompt":
        st["q"], st["k"], st["v"] = normal(sum(n), heads * dim), normal(sum(n), kv * dim), normal(sum(n), kv * dim)
        starts = [0]
        for x in n:
            starts.append(starts[-1] + x)
        st["starts"] = ints(starts)
        return st
    n, per, first = _pages(case)
    count = first[-1] + 3  # a pool is never exactly full
    order = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)
    if case["op"] == "gather":
        st["codes"], st["params"] = _fill(count, case, gen)
        st["table"] = order[:per[0]].contiguous()
        return st
    st["kc"], st["kp"] = _fill(count, case, gen)
    st["vc"], st["vp"] = _fill(count, case, gen)
    if case["op"] == "decode":
        table = torch.zeros(case["batch"], max(per), dtype=torch.int32, device="cuda")
        for b in range(case["batch"]):
            table[b, :per[b]] = order[first[b]:first[b + 1]]
        st["table"], st["ctx"] = table, ints(n)
        st["q"] = normal(case["batch"], heads * dim)
        return st
    if case["rows"]:  # one new token at the end of each sequence
        at = torch.tensor([x - 1 for x in n], device="cuda")
        entry = torch.tensor(first[:-1], device="cuda") + at // case["page"]
        st["touched"] = order[entry].contiguous()
    else:  # whole prompts
        at = torch.cat([torch.arange(x, device="cuda") for x in n])
        entry = torch.cat([first[b] + torch.arange(x, device="cuda") // case["page"] for b, x in enumerate(n)])
        st["touched"] = order[:first[-1]].contiguous()
    st["positions"], st["ids"], st["offsets"] = at.to(torch.int32), order[entry].contiguous(), (at % case["page"]).to(torch.int32)
    st["k"], st["v"] = normal(at.numel(), kv * dim), normal(at.numel(), kv * dim)
    return st


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _quantise(x, dt):
    """(codes, params) of the rows of x: step and least in the 16-bit type, then the nearest of 16 levels."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step, least = ((high - low) / 15).to(dt), low.to(dt)
    s = step.to(x.dtype)
    level = torch.where(s > 0, (x - least.to(x.dtype)) / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15).to(torch.uint8)
    return level[..., 0::2] | (level[..., 1::2] << 4), torch.cat([step, least], -1)


def _values(codes, params):
    """What the codes stand for, in 32 bits."""
    level = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return params[..., 1:].float() + params[..., :1].float() * level


def _rotate(x, position, mode):
    """x [rows, heads, dim] rotated by its rows' positions (0: neighbouring pairs, 1: halves); angles in 64 bits."""
    if mode == 2:
        return x
    dim = x.shape[-1]
    rate = _BASE ** (-torch.arange(0, dim, 2, device=x.device, dtype=torch.float64) / dim)
    angle = position.double()[:, None] * rate
    c, s = angle.cos().to(x.dtype)[:, None, :], angle.sin().to(x.dtype)[:, None, :]
    if mode == 1:
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _plain_prompt(st):
    case = st["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    rows = st["q"].shape[0]
    index = torch.arange(rows, device="cuda", dtype=torch.int32)
    owner = torch.searchsorted(st["starts"], index, right=True) - 1
    position = index - st["starts"][owner]
    q = _rotate(st["q"].float().view(rows, heads, dim), position, case["rope"]).view(rows, kv, heads // kv, dim)
    k = _rotate(st["k"].float().view(rows, kv, dim), position, case["rope"])
    v = st["v"].float().view(rows, kv, dim)
    unseen = (owner[:, None] != owner[None, :]) | (index[None, :] > index[:, None])
    out = torch.empty(rows, kv, heads // kv, dim, device="cuda")
    for h in range(kv):  # the scores of all heads at once would not fit
        score = torch.matmul(q[:, h].transpose(0, 1), k[:, h].t()).mul_(1 / math.sqrt(dim)).masked_fill_(unseen, -math.inf)
        p = score.sub_(score.amax(-1, keepdim=True)).exp_()
        out[:, h] = (torch.matmul(p, v[:, h]) / p.sum(-1, keepdim=True)).transpose(0, 1)
    return out.view(rows, heads * dim).to(st["q"].dtype)


def _plain_append(st):
    case = st["case"]
    kv, dim, dt = case["kv"], case["dim"], st["k"].dtype
    k = _rotate(st["k"].float().view(-1, kv, dim), st["positions"], case["rope"])
    v = st["v"].float().view(-1, kv, dim)
    ids, offsets = st["ids"].long(), st["offsets"].long()
    st["kc"][ids, :, offsets], st["kp"][ids, :, offsets] = _quantise(k, dt)
    st["vc"][ids, :, offsets], st["vp"][ids, :, offsets] = _quantise(v, dt)
    t = st["touched"].long()
    return [_values(c[t], p[t]).to(dt).transpose(1, 2).reshape(-1, kv * dim) for c, p in ((st["kc"], st["kp"]), (st["vc"], st["vp"]))]


def _plain_gather(st):
    case, t = st["case"], st["table"].long()
    got = _values(st["codes"][t], st["params"][t]).to(st["params"].dtype).transpose(1, 2)
    return got.reshape(-1, case["kv"] * case["dim"])[:case["longest"]].contiguous()


def _plain_decode(st):
    case, t = st["case"], st["table"].long()
    batch, kv, dim = case["batch"], case["kv"], case["dim"]
    k = _values(st["kc"][t], st["kp"][t]).transpose(1, 2).reshape(batch, kv, -1, dim)
    q = st["q"].float().view(batch, kv, -1, dim)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim)
    del k
    unseen = torch.arange(score.shape[-1], device="cuda") >= st["ctx"][:, None]
    score = score.masked_fill(unseen[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    v = _values(st["vc"][t], st["vp"][t]).transpose(1, 2).reshape(batch, kv, -1, dim)
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(batch, -1).to(st["q"].dtype)


# ------------------------------------------------------------------------------------------------------ the framework's calls
_device = None


def _own(st):
    global _device
    import puter_b200

    if _device is None:
        _device = puter_b200.Device()
    d, case, fmt = _device, st["case"], _FORMATS[st["case"]["dtype"]]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    attn = puter_b200.MultiHeadAttentionConfig(NumHeads=heads, HeadDim=dim, Causal=True, KVHeadCount=kv)
    rope = None if case.get("rope", 2) == 2 else puter_b200.RoPEConfig(BaseFreq=_BASE, Mode=case["rope"])
    if case["op"] == "prompt":
        out = torch.empty_like(st["q"])
        d.RoPEPackedAttentionPrefill(rope, attn, st["q"], st["k"], st["v"], st["starts"], out, case["batch"], st["q"].shape[0], st["longest"], fmt)
        return out
    if case["op"] == "append":
        pages = st["kc"].shape[0]
        d.RoPEKVPageWriteQ4(rope, st["k"], st["v"], st["positions"], st["ids"], st["offsets"], st["kc"], st["kp"], st["vc"], st["vp"],
                            st["k"].shape[0], kv, dim, pages, case["page"], 32768, fmt)
        rows = st["touched"].numel() * case["page"]
        got = [torch.empty(rows, kv * dim, dtype=st["k"].dtype, device="cuda") for _ in range(2)]
        d.KVPageGatherQ4(st["kc"], st["kp"], st["touched"], got[0], pages, case["page"], kv, dim, rows, fmt)
        d.KVPageGatherQ4(st["vc"], st["vp"], st["touched"], got[1], pages, case["page"], kv, dim, rows, fmt)
        return got
    if case["op"] == "gather":
        out = torch.empty(case["longest"], kv * dim, dtype=st["params"].dtype, device="cuda")
        d.KVPageGatherQ4(st["codes"], st["params"], st["table"], out, st["codes"].shape[0], case["page"], kv, dim, case["longest"], fmt)
        return out
    out = torch.empty_like(st["q"])
    d.PagedDecodeAttentionQ4(attn, st["q"], st["kc"], st["kp"], st["vc"], st["vp"], st["table"], st["ctx"], out, case["batch"],
                             st["table"].shape[1], st["kc"].shape[0], case["page"], fmt)
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "prompt":
        return _plain_prompt(state)
    if op == "append":
        return _plain_append(state)
    return _plain_gather(state) if op == "gather" else _plain_decode(state)


# --------------------------------------------------------------------------------------------------------------- exact values
def _turn64(x, position, mode):
    """x [rows, heads, dim] in 64 bits as complex numbers times e^(i angle)."""
    if mode == 2:
        return x
    dim = x.shape[-1]
    j = torch.arange(dim // 2, device=x.device, dtype=torch.float64)
    angle = position.double()[:, None, None] * torch.pow(torch.tensor(_BASE, dtype=torch.float64, device=x.device), -2 * j / dim)
    pair = x.unflatten(-1, (2, dim // 2)).transpose(-1, -2) if mode == 1 else x.unflatten(-1, (dim // 2, 2))
    turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(angle), angle))
    return (turned.transpose(-1, -2) if mode == 1 else turned).flatten(-2)


def _levels64(x, dt):
    """The 4-bit values nearest to the rows of x, in 64 bits; step and least are held in the 16-bit type."""
    least = x.min(-1, keepdim=True).values.to(dt).double()
    step = ((x.max(-1, keepdim=True).values - x.min(-1, keepdim=True).values) / 15.0).to(dt).double()
    grid = torch.round((x - least) / step.clamp_min(1e-300)).clamp(0, 15)
    return least + step * torch.where(step > 0, grid, torch.zeros_like(grid))


def _read64(codes, params):
    c = codes.to(torch.int64)
    both = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=torch.float64, device=c.device)
    both[..., 0::2] = (c % 16).double()
    both[..., 1::2] = torch.div(c, 16, rounding_mode="floor").double()
    return both * params[..., 0].double()[..., None] + params[..., 1].double()[..., None]


def _attend64(q, k, v, first):
    """q [rows, heads, dim], k and v [keys, kv, dim]: row r sees keys 0 .. first + r."""
    rows, heads, dim = q.shape
    out = torch.empty_like(q)
    key = torch.arange(k.shape[0], device=q.device)
    group = heads // k.shape[1]
    part = max(1, (1 << 28) // k.shape[0])
    for h in range(heads):
        for a in range(0, rows, part):
            s = q[a:a + part, h] @ k[:, h // group].t() / math.sqrt(dim)
            seen = key[None, :] <= first + a + torch.arange(s.shape[0], device=q.device)[:, None]
            out[a:a + part, h] = torch.softmax(torch.where(seen, s, -math.inf), -1) @ v[:, h // group]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    heads, kv, dim, page, n = case["heads"], case["kv"], case["dim"], case.get("page"), _lengths(case)
    if case["op"] == "prompt":
        got, at = [], 0
        for x in n:
            part = slice(at, at + x)
            pos = torch.arange(x, device="cuda")
            q = _turn64(st["q"][part].double().view(x, heads, dim), pos, case["rope"])
            k = _turn64(st["k"][part].double().view(x, kv, dim), pos, case["rope"])
            got.append(_attend64(q, k, st["v"][part].double().view(x, kv, dim), 0).view(x, heads * dim))
            at += x
        return torch.cat(got)
    if case["op"] == "append":
        got = []
        slot = st["ids"].long() * page + st["offsets"].long()
        back = (st["touched"].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()
        place = torch.full((st["kc"].shape[0] * page,), -1, dtype=torch.int64, device="cuda")
        place[back] = torch.arange(back.numel(), device="cuda")
        for x, c, p, mode in ((st["k"], st["kc"], st["kp"], case["rope"]), (st["v"], st["vc"], st["vp"], 2)):
            t = st["touched"].long()
            old = _read64(c[t], p[t]).permute(0, 2, 1, 3).reshape(-1, kv, dim)
            old[place[slot]] = _levels64(_turn64(x.double().view(-1, kv, dim), st["positions"], mode), x.dtype)
            got.append(old.view(-1, kv * dim))
        return got
    if case["op"] == "gather":
        t = st["table"].long()
        return _read64(st["codes"][t], st["params"][t]).permute(0, 2, 1, 3).reshape(-1, kv * dim)[:case["longest"]].contiguous()
    got = []
    for b, x in enumerate(n):
        t = st["table"][b, :-(-x // page)].long()
        k = _read64(st["kc"][t], st["kp"][t]).permute(0, 2, 1, 3).reshape(-1, kv, dim)[:x]
        v = _read64(st["vc"][t], st["vp"][t]).permute(0, 2, 1, 3).reshape(-1, kv, dim)[:x]
        got.append(_attend64(st["q"][b].double().view(1, heads, dim), k, v, x - 1).view(1, heads * dim))
    return torch.cat(got)
