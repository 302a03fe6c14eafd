"""What the packed-prompt and 4-bit-cache methods take as sizes and tensors, without a GPU: the library's own argument types with a missing
context, which every call that passes the conversion reports."""
import numpy as np
import pytest
import torch

from test_packed_and_q4_bindings import FakeTensor, dev, tensors  # noqa: F401


@pytest.fixture()
def real():
    from puter_b200 import _lib, device as D
    from puter_b200.csrc import build as b

    b.build()
    d = D.Device.__new__(D.Device)
    d.lib, d.ref, d._refs, d._status, d.follow_torch_stream = _lib.load(), None, {}, _lib.CUDAStatus(), False
    return d


def calls(d, size, fmt=2):
    from puter_b200 import device as D

    attn = D.MultiHeadAttentionConfig(NumHeads=size, HeadDim=64, Causal=True, KVHeadCount=size)
    return [lambda: d.RoPEPackedAttentionPrefill(D.RoPEConfig(), attn, *tensors(5), 3, size, 20, fmt),
            lambda: d.RoPEKVPageWriteQ4(None, *tensors(2), None, *tensors(6), size, 2, 64, 6, 16, 100, fmt),
            lambda: d.KVPageGatherQ4(*tensors(4), 6, 16, size, 64, 33, fmt),
            lambda: d.PagedDecodeAttentionQ4(attn, *tensors(8), size, 5, 6, 16, fmt)]


@pytest.mark.parametrize("size", [4, np.int64(4), np.int32(4), np.uint8(4), torch.tensor(4)])
def test_integers_of_other_libraries(real, size):
    """As the methods beside them: what Python can index with is a size."""
    from puter_b200 import device as D

    for go in calls(real, size) + calls(real, 4, size):
        with pytest.raises(D.DeviceError) as e:
            go()
        assert e.value.code == -1 and "nil device context" in e.value.message


@pytest.mark.parametrize("size", [b"4", 4.0, "4", None])
def test_what_is_no_integer_is_refused(real, size):
    import ctypes

    for go in calls(real, size)[1:] + calls(real, 4, size):
        with pytest.raises((ctypes.ArgumentError, TypeError)):
            go()


def test_integers_arrive_as_they_are(dev):  # noqa: F811
    from puter_b200 import device as D

    for size in (4, np.int64(4)):
        dev.KVPageGatherQ4(*tensors(4), 6, 16, size, 64, 33, 2)
    assert [[int(x) for x in c[1][5:]] for c in dev.lib.calls] == [[6, 16, 4, 64, 33, 0]] * 2
    assert D._NO_TOKEN.value == 0


def test_a_known_address_does_not_make_memory_of_the_device(dev):  # noqa: F811
    """A handle is found by address and size: the tensor that brings them must still be CUDA memory."""
    dev.KVPageGatherQ4(*tensors(4), 6, 16, 2, 64, 33, 2)
    other = tensors(4)
    other[1].is_cuda = False
    with pytest.raises(AssertionError):
        dev.KVPageGatherQ4(*other, 6, 16, 2, 64, 33, 2)
    other[1].is_cuda = True
    other[1].is_contiguous = lambda: False
    with pytest.raises(AssertionError):
        dev.KVPageGatherQ4(*other, 6, 16, 2, 64, 33, 2)
    assert len(dev.lib.calls) == 1 and isinstance(other[0], FakeTensor)
