"""Refusals of the packed-prompt and 4-bit-cache entry points, without a GPU: a context that is zeroed memory serves, since arguments are
checked before anything is launched, and buffer handles are (address, size) records."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from puter_b200.csrc import build as b

    b.build()
    from puter_b200 import _lib

    return _lib.load()


@pytest.fixture()
def env(lib):
    from puter_b200 import _lib

    context = ctypes.create_string_buffer(4096)
    made = []

    def buf(nbytes, at=1 << 20):
        made.append(lib.cuda_buffer_wrap(ctypes.addressof(context), at, nbytes))
        return made[-1]

    status = _lib.CUDAStatus()

    def call(name, *args):
        return getattr(lib, "cuda_dispatch_" + name)(ctypes.addressof(context), *args, ctypes.byref(status)), status.message.decode()

    yield buf, call
    for m in made:
        lib.cuda_buffer_release(m)


BIG = 1 << 40


def test_packed_prefill(env):
    buf, call = env

    def go(fmt=2, q=None, out=None, starts=BIG, batch=2, total=100, longest=100, heads=8, kv=2, dim=128, mode=2, base=1e4, scaling=0):
        q = q or buf(BIG, 1 << 20)
        return call("rope_packed_attention_prefill", fmt, q, buf(BIG, 2 << 20), buf(BIG, 3 << 20), buf(starts), out or buf(BIG, 5 << 20), batch, total,
                    longest, heads, kv, dim, 1, mode, base, 0, scaling, 0.0, 0.0, 0.0, 0, 0)

    for code, kw in [(-6, dict(fmt=3)), (-6, dict(fmt=4)), (-6, dict(dim=257)), (-2, dict(heads=9)), (-2, dict(mode=3)), (-2, dict(mode=1, base=0.0)),
                     (-2, dict(mode=1, scaling=1)), (-2, dict(mode=0, dim=33)), (-2, dict(starts=8)), (-2, dict(q=buf(100 * 8 * 128 * 2 - 1))),
                     (-2, dict(out=buf(BIG, 2 << 20))), (-2, dict(total=1 << 31))]:
        assert go(**kw)[0] == code, kw
    for kw in (dict(batch=0), dict(total=0), dict(longest=0), dict(heads=0)):
        assert go(**kw)[0] == 0
    assert "seqStarts" in go(starts=8)[1]


def test_append(env):
    buf, call = env

    def go(fmt=2, rows=4, kv=2, dim=128, pages=3, page=16, longest=9, mode=2, base=1e4, pos=0, k=None, codes=3 * 16 * 2 * 64, params=3 * 16 * 2 * 4, at=1 << 20):
        return call("rope_kv_page_write_q4", fmt, k or buf(BIG), buf(BIG), pos, buf(16), buf(16), buf(codes, at), buf(params), buf(BIG), buf(BIG), rows, kv,
                    dim, pages, page, longest, mode, base, 0, 0.0, 0.0, 0.0, 0, 0)

    for code, kw in [(-6, dict(fmt=0)), (-6, dict(fmt=4)), (-6, dict(dim=32)), (-6, dict(dim=256)), (-2, dict(mode=3)), (-2, dict(mode=1)),
                     (-2, dict(mode=1, pos=buf(16), longest=0)), (-2, dict(mode=0, pos=buf(16), base=-1.0)), (-2, dict(mode=1, pos=buf(15))), (-2, dict(rows=5)),
                     (-2, dict(codes=3 * 16 * 2 * 64 - 1)), (-2, dict(params=3 * 16 * 2 * 4 - 1)), (-2, dict(at=(1 << 20) + 8)), (-2, dict(k=buf(4 * 2 * 128 * 2 - 1)))]:
        assert go(**kw)[0] == code, kw
    for kw in (dict(rows=0), dict(kv=0), dict(pages=0), dict(page=0)):
        assert go(**kw)[0] == 0


def test_gather_and_decode(env):
    buf, call = env

    def gather(fmt=2, codes=BIG, table=8, out=None, pages=3, page=16, kv=2, dim=64, rows=32):
        return call("kv_page_gather_q4", fmt, buf(codes), buf(BIG), buf(table), out or buf(rows * kv * dim * 2), pages, page, kv, dim, rows, 0)

    for code, kw in [(-6, dict(fmt=5)), (-6, dict(dim=96)), (-2, dict(codes=3 * 16 * 2 * 32 - 1)), (-2, dict(rows=33)), (-2, dict(out=buf(BIG, (1 << 20) + 2)))]:
        assert gather(**kw)[0] == code, kw
    assert gather(rows=0)[0] == 0

    def decode(fmt=2, q=BIG, codes=BIG, table=BIG, flag=0, batch=2, longest=4, pages=3, page=16, heads=8, kv=2, dim=128, at=1 << 20):
        return call("paged_decode_attention_q4", fmt, buf(q, at), buf(codes), buf(BIG), buf(BIG), buf(BIG), buf(table), buf(BIG), buf(BIG), flag, batch,
                    longest, pages, page, heads, kv, dim, 0)

    for code, kw in [(-6, dict(fmt=0)), (-6, dict(dim=96)), (-2, dict(heads=7)), (-2, dict(pages=0)), (-2, dict(page=0)), (-2, dict(longest=0)),
                     (-2, dict(q=2 * 8 * 128 * 2 - 1)), (-2, dict(codes=3 * 16 * 2 * 64 - 1)), (-2, dict(table=31)), (-2, dict(flag=buf(3))), (-2, dict(at=(1 << 20) + 4))]:
        assert decode(**kw)[0] == code, kw
    for kw in (dict(batch=0), dict(heads=0)):
        assert decode(**kw)[0] == 0


TOP = (1 << 32) - 1


def test_sizes_whose_products_leave_64_bits(env):
    """Never a small product of large sizes that a small buffer would satisfy."""
    buf, call = env
    big = [buf(BIG) for _ in range(9)]
    for pages, page, kv in [(1 << 31, 1 << 30, 8), (TOP, TOP, 2), (1 << 31, 1 << 31, 4), (1 << 31, TOP, 2)]:
        code, message = call("rope_kv_page_write_q4", 2, *big[:2], 0, *big[3:5], *big[5:], 1, kv, 128, pages, page, 9, 2, 1e4, 0, 0.0, 0.0, 0.0, 0, 0)
        assert code == -2, message
        assert call("kv_page_gather_q4", 2, *big[:4], pages, page, kv, 128, 1, 0)[0] == -2
        assert call("paged_decode_attention_q4", 2, *big[:8], 0, 1, 1, pages, page, kv, kv, 128, 0)[0] == -2
    assert call("rope_kv_page_write_q4", 2, *big[:2], 0, *big[3:5], *big[5:], TOP, TOP, 128, 1, 1, 9, 2, 1e4, 0, 0.0, 0.0, 0.0, 0, 0)[0] == -2
    assert call("kv_page_gather_q4", 2, *big[:4], 1, 1, TOP, 128, TOP, 0)[0] == -2
    assert call("paged_decode_attention_q4", 2, *big[:8], 0, 1 << 31, 1, 1, 1, TOP, 1, 128, 0)[0] == -2
    assert call("paged_decode_attention_q4", 2, *big[:8], 0, 1 << 16, 1 << 16, 100, 16, 8, 8, 128, 0)[0] == -2  # more tiles than 31 bits count
    assert call("rope_packed_attention_prefill", 2, *big[:4], big[4], 1, (1 << 31) - 1, 10, TOP, 1, 128, 1, 2, 1e4, 0, 0, 0.0, 0.0, 0.0, 0, 0)[0] == -2


def test_alignment_and_overlap(env):
    buf, call = env
    odd, big = buf(BIG, (1 << 20) + 2), buf(BIG)

    def append(positions=big, ids=big, offsets=big):
        return call("rope_kv_page_write_q4", 2, big, big, positions, ids, offsets, *[big] * 4, 1, 1, 64, 1, 1, 9, 1, 1e4, 0, 0.0, 0.0, 0.0, 0, 0)

    for kw in (dict(positions=odd), dict(ids=odd), dict(offsets=odd)):
        assert append(**kw)[0] == -2 and "aligned" in append(**kw)[1]
    assert "aligned" in call("kv_page_gather_q4", 2, big, big, odd, big, 1, 1, 1, 64, 1, 0)[1]
    for k in (6, 7, 9):
        args = [big] * 8 + [0]
        args[k - 1 if k < 9 else 8] = odd
        assert "aligned" in call("paged_decode_attention_q4", 2, *args, 1, 1, 1, 1, 1, 1, 64, 0)[1], k

    def prompt(q=buf(BIG, 1 << 20), k=buf(BIG, 2 << 20), v=buf(BIG, 3 << 20), starts=big, out=buf(BIG, 5 << 20), fmt=2):
        return call("rope_packed_attention_prefill", fmt, q, k, v, starts, out, 1, 16, 16, 4, 2, 64, 1, 2, 1e4, 0, 0, 0.0, 0.0, 0.0, 0, 0)

    for at in ((1 << 20) + 16, (1 << 20) - 16, (2 << 20) + 4080, (3 << 20) - 8176):
        assert prompt(out=buf(BIG, at))[0] == -2 and "overlap" in prompt(out=buf(BIG, at))[1], at
    assert "aligned" in prompt(starts=odd)[1] and "aligned" in prompt(out=buf(BIG, (5 << 20) + 1))[1] and "aligned" in prompt(k=odd, fmt=0)[1]


def test_python_refuses_windows_and_alibi():
    from puter_b200 import device as D

    dev = D.Device.__new__(D.Device)
    for kw in (dict(WindowSize=4), dict(ALiBiSlope=0.5)):
        cfg = D.MultiHeadAttentionConfig(NumHeads=4, HeadDim=64, KVHeadCount=2, **kw)
        with pytest.raises(D.DeviceError) as e:
            dev.RoPEPackedAttentionPrefill(None, cfg, *[None] * 5, 1, 1, 1, 2)
        assert e.value.code == -6
        with pytest.raises(D.DeviceError) as e:
            dev.PagedDecodeAttentionQ4(cfg, *[None] * 8, 1, 1, 1, 16, 2)
        assert e.value.code == -6
    dev.ref = None
