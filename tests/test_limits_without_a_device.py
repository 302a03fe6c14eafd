"""The largest sizes that the packed-prompt and 4-bit-cache entry points take, without a GPU (see test_refusals_without_a_device.py): what
is larger is refused before anything is allocated or launched."""
import pytest

from test_refusals_without_a_device import BIG, env, lib  # noqa: F401


@pytest.mark.parametrize("heads", [4, 8, 16])
def test_decode_contexts_end_before_their_steps_leave_31_bits(env, heads):  # noqa: F811
    """A warp's place runs up to two steps of 64 tokens beyond the end of a context.  The pool is small: page entries may repeat."""
    buf, call = env
    big = [buf(BIG) for _ in range(8)]

    def go(pages, page):
        return call("paged_decode_attention_q4", 2, *big, 0, 1, pages, 2, page, heads, 1, 128, 0)

    top = (1 << 31) - 256
    for pages, page in [(1, top + 1), (1, (1 << 31) - 32), (1, (1 << 31) - 1), ((top >> 4) + 1, 16), ((1 << 27) - 2, 16), (1 << 31, 1)]:
        code, message = go(pages, page)
        assert code == -2 and "index range" in message, (pages, page, message)


@pytest.mark.parametrize("fmt", [2, 0])
def test_rows_of_packed_prompts_are_counted_in_31_bits(env, fmt):  # noqa: F811
    """One token of 2^31 heads of one element takes 8 GB in 16 bits: the buffers alone do not refuse it."""
    buf, call = env
    big = [buf(BIG, (i + 1) << 42) for i in range(5)]
    for heads, kv, dim in [(1 << 31, 1, 1), ((1 << 32) - 1, 1, 1), (1 << 31, 1 << 31, 2), (1 << 24, 1 << 24, 128), (1 << 24, 1, 128), (1 << 23, 1 << 23, 256)]:
        code, message = call("rope_packed_attention_prefill", fmt, *big, 1, 1, 1, heads, kv, dim, 1, 2, 1e4, 0, 0, 0.0, 0.0, 0.0, 0, 0)
        assert code == -2 and "31 bits" in message, (heads, kv, dim, message)
