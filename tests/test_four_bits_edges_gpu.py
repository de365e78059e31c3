"""The 4-bit operators where calls meet, where numbers are very small or large, and at other edges of what their documentation allows."""
import math

import numpy as np
import pytest
import torch

import fourbit
from test_cache4_gpu import BF, DEV, F32, HALF, Attend, Write, i32
from test_linear4_gpu import case, check, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [20, 64])
def test_products_on_two_streams_whose_blocks_hold_tensor_memory(tokens):
    """Clusters of the 16-bit product for few rows and of the 4-bit one for many, at the same time again and again: both come to their end with their bits."""
    from xinfer_b200 import kernels as k
    x, w = case(tokens, 2048, 8192, 64, BF)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x16, w16 = (torch.randn(s, generator=gen, device=DEV).to(BF) for s in ((8, 4096), (4096, 4096)))
    err = i32([0])
    want, want16 = product(x, w, 2048), torch.zeros((8, 4096), dtype=BF, device=DEV)
    assert k.gemm_skinny_tc(want16, x16, w16, err)
    out, out16 = torch.zeros_like(want), torch.zeros_like(want16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(100):
        with torch.cuda.stream(streams[0]):
            k.linear4(out, x, w)
        with torch.cuda.stream(streams[1]):
            k.gemm_skinny_tc(out16, x16, w16, err)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(out16, want16) and int(err) == 0
