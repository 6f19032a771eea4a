"""Matrices whose strides PyTorch leaves as they are (a single row or column),
as the cross entropy hands them to the C entry, which checks them itself."""
import ctypes

import pytest
import torch

import rapidalign_b200 as ra
from rapidalign_b200 import _lib
from test_saved_tensors_host import recorder  # noqa: F401

ONE_ROW = {
    "column": lambda d, dt: torch.randn(d, 1, dtype=dt).t(),
    "view": lambda d, dt: torch.randn(40 * d, dtype=dt).as_strided((1, d), (0, 1)),
    "slice": lambda d, dt: torch.randn(3, 2 * d, dtype=dt)[1:2, :d],
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [1, 8, 13])
@pytest.mark.parametrize("make", ONE_ROW.values(), ids=ONE_ROW.keys())
def test_single_rows(make, d, dtype, recorder):  # noqa: F811
    from rapidalign_b200 import build as b
    b.build()
    lib = ctypes.CDLL(_lib.LIB_PATH)
    lib.ra_ce_state_bytes.restype = ctypes.c_size_t
    x, w = torch.randn(5, d, dtype=dtype), torch.randn(5, d, dtype=dtype)
    for a, t in ((x, make(d, dtype)), (make(d, dtype), w), (make(d, dtype), make(d, dtype))):
        ra.linear_cross_entropy(a, t, torch.zeros(a.shape[0], dtype=torch.long))
        got = recorder.last("ra_ce_forward")[0]
        assert got["ld_x"] >= d and got["ld_w"] >= d
        assert lib.ra_ce_state_bytes(ctypes.byref(_lib.RaCeDesc(**got))) > 0
