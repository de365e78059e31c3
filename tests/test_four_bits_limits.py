"""What the 4-bit operators' entry points refuse before they look at a GPU."""
import ctypes

import pytest

from xinfer_b200 import kernels as k
from xinfer_b200.native import kernels_lib

INVALID = 1                # cudaErrorInvalidValue


def attention_status(tokens=1, requests=1, table=1, nh=1, nkv=1, d=1, page_size=16, pages=1):
    words = [k.BF16] + [0] * 7 + [nh * d, nh * d, tokens, requests, table, nh, nkv, d, page_size, pages, 0, 1, 0, 0, 0, 0]
    array = (ctypes.c_longlong * len(words))(*words)
    entry = kernels_lib().xb_cache4_attention
    entry.restype, entry.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int]
    return entry(array, len(words))


def test_rows_that_32_bits_do_not_count():
    # (rows are rounded up to blocks of 256: 2^31 - 1 of them would be counted as fewer than none)
    assert attention_status(tokens=2 ** 31 - 1) == INVALID and attention_status(tokens=2 ** 29, nh=4) == INVALID
    assert attention_status(tokens=0) == 0 and attention_status(requests=0) == 0


@pytest.mark.parametrize("what", [dict(requests=8193), dict(d=257), dict(d=0), dict(nkv=0), dict(nh=3, nkv=2), dict(page_size=0), dict(table=2 ** 30, page_size=16), dict(page_size=2 ** 27)])
def test_other_sizes(what):
    assert attention_status(**what) == INVALID
