"""Weights in 4 bits: the packing, what it holds, and what it and the wrappers refuse."""
import numpy as np
import pytest
import torch

import fourbit
from xinfer_b200 import kernels as k
from xinfer_b200.native import wrap_module
from xinfer_b200.weights import pack4


@pytest.mark.parametrize("n,c,group", [(1, 1, 32), (16, 128, 32), (17, 129, 64), (5, 1000, 128), (40, 96, 32), (33, 300, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values(n, c, group, dtype):
    gen = torch.Generator().manual_seed(n * c)
    w = (torch.randn((n, c), generator=gen) * torch.exp(torch.randn((n, 1), generator=gen))).to(dtype)
    data = pack4(w, group)
    assert tuple(data.shape) == k.linear4_shape(n, c, group) and data.dtype == torch.uint8
    got = fourbit.weight_values(data.numpy(), group, n, c)
    full = np.zeros((n, -(-c // 128) * 128))
    full[:, :c] = w.double().numpy()
    for r in range(n):
        for j in range(0, full.shape[1], group):
            codes, s, m = fourbit.encode(full[r, j:j + group])
            want, many = (m + s * codes)[:max(0, c - j)], len(got[r, j:j + group])
            assert np.array_equal(got[r, j:j + many], want[:many])


def test_groups_of_one_number():
    w = torch.full((3, 64), 0.7109375)                 # (a bfloat16 number: the scale is zero, the least value holds it)
    assert np.array_equal(fourbit.weight_values(pack4(w, 64).numpy(), 64, 3, 64)[:, :64], np.full((3, 64), 0.7109375))
    assert np.all(fourbit.weight_values(pack4(torch.zeros(2, 32)).numpy(), 32, 2, 32) == 0)


def test_refusals():
    for bad in (torch.zeros(4), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(0, 4), torch.full((2, 2), float("nan")), torch.full((2, 2), float("inf")),
                torch.full((2, 2), -3.4e38), torch.tensor([[-3e38, 3e38]])):
        with pytest.raises(ValueError):
            pack4(bad)
    # (the columns behind a weight are zeros, so a short group of numbers above zero has the least value 0, and 3.4e38 / 15 is an ordinary scale)
    assert pack4(torch.full((2, 2), 3.4e38)).shape == (1, 1, 1280)
    for group in (0, 16, 48, 256):
        with pytest.raises(ValueError):
            pack4(torch.zeros(4, 4), group)
        with pytest.raises(k.KernelError):
            k.linear4_shape(4, 4, group)
    for ps, d in ((0, 64), (16, 0), (16, 257), (2 ** 27, 1), (2 ** 24, 256)):
        with pytest.raises(k.KernelError):
            k.cache4_page_bytes(ps, d)
    assert k.cache4_page_bytes(16, 128) == 1280 and k.cache4_page_bytes(8, 80) == 480


def test_tensors_on_the_host_are_refused():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    cache, x = torch.zeros((2, 2, 640), dtype=torch.uint8), torch.zeros(3, 4, 64)
    with pytest.raises(k.KernelError):
        k.cache4_write(x, cache, cache, torch.zeros(3, 512), i32(3), torch.zeros(3, dtype=torch.int64), 16, i32(1))
    with pytest.raises(k.KernelError):
        k.cache4_attention(x, x, cache, cache, i32(1), i32(2), i32(1, 2), 16, 1.0, i32(1))
    with pytest.raises(k.KernelError):
        k.linear4(torch.zeros(3, 8), torch.zeros(3, 64), pack4(torch.zeros(8, 64)))


def test_the_first_tensor_of_another_device():
    elsewhere = wrap_module().elsewhere
    assert elsewhere(0) is None and elsewhere(0, None, None) is None
    assert elsewhere(0, None, torch.zeros(1), torch.zeros(1)) == 1 and elsewhere(0, 3) == 0
    for args in ((), ("x",), (None, torch.zeros(1))):
        with pytest.raises(TypeError):
            elsewhere(*args)
