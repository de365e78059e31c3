"""The native module that checks tensors and calls entry points: what it passes on and what it refuses."""
import ctypes
import struct

import pytest
import torch

from xinfer_b200 import kernels as k
from xinfer_b200.native import wrap_module

ENTRY = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(ctypes.c_longlong), ctypes.c_int)


def test_words_of_a_call():
    got = []
    entry = ENTRY(lambda words, n: got.extend(words[i] for i in range(n)) or 7)
    t = torch.zeros(3)
    call = wrap_module().call
    assert call(ctypes.cast(entry, ctypes.c_void_p).value, t, None, -5, 2 ** 62, 0.375, True, t[1:]) == 7
    bits = struct.unpack("q", struct.pack("d", 0.375))[0]
    assert got == [t.data_ptr(), 0, -5, 2 ** 62, bits, 1, t.data_ptr() + 4]
    got.clear()
    assert call(ctypes.cast(entry, ctypes.c_void_p).value, *range(47)) == 7 and got == list(range(47))


def test_calls_that_are_refused():
    call, entry = wrap_module().call, ENTRY(lambda words, n: 0)
    at = ctypes.cast(entry, ctypes.c_void_p).value
    for args, why in (((at, 2 ** 70), OverflowError), ((at, "x"), TypeError), ((), TypeError), ((at, *range(48)), TypeError), ((0,), ValueError), (("x",), TypeError)):
        with pytest.raises(why):
            call(*args)


def test_tensors_that_are_refused():
    check, rows = k._check, wrap_module().rows
    for t in (torch.zeros(4, dtype=torch.int32), None, 3, [1]):
        with pytest.raises(k.KernelError):
            check(t, "x", torch.int32, (4,))
        assert rows(t, torch.int32, (4,)) is None
    with pytest.raises(TypeError):
        wrap_module().check(torch.zeros(4))


@pytest.mark.gpu
def test_tensors_on_the_device():
    check, rows = k._check, wrap_module().rows
    t = torch.zeros(6, 4, 8, device="cuda:0")
    for args in ((t, "t", torch.float32, (6, 4, 8)), (t, "t", None, (6, None, 8)), (t, "t", torch.float32, None), (t[:, 0, :0], "t", None, (6, 0))):
        assert check(*args) is None
    for args in ((t, "t", torch.int32, (6, 4, 8)), (t, "t", None, (6, 4)), (t, "t", None, (6, 5, None)), (t.transpose(0, 1), "t", None, None), (t, "t", None, ("a", 4, 8)),
                 (t[:, :2], "t", None, (6, 2, 8))):
        with pytest.raises(k.KernelError):
            check(*args)
    assert rows(t, torch.float32, (6, 4, 8)) == 32 and rows(t[:, 1:3], torch.float32, (6, 2, 8)) == 32 and rows(t[:1, 1:3], torch.float32, (1, 2, 8)) == 16
    assert rows(t[::2], torch.float32, (3, 4, 8)) == 64 and rows(t[:, :, :1], torch.float32, (6, 4, 1)) is None and rows(t[:, :1, :4], torch.float32, (6, 1, 4)) == 32
    assert rows(t[:1].expand(6, 4, 8), torch.float32, (6, 4, 8)) is None and rows(t[:0], torch.float32, (0, 4, 8)) == 32
    assert rows(t, torch.bfloat16, (6, 4, 8)) is None and rows(t[0, 0], torch.float32, (8,)) is None
