"""linear_cross_entropy: what it refuses, before anything reaches a device."""
import ctypes

import pytest
import torch

import rapidalign_b200 as ra
from rapidalign_b200 import _lib


def args(n=4, v=6, d=8, dtype=torch.float32):
    return torch.zeros(n, d, dtype=dtype), torch.zeros(v, d, dtype=dtype), torch.zeros(n).long()


@pytest.mark.parametrize("change, message", [
    (lambda x, w, t: ((x[0], w, t), {}), "x and weight must be"),
    (lambda x, w, t: ((x, w[:, :4], t), {}), "x and weight must be"),
    (lambda x, w, t: ((x, w, t[:3]), {}), "target length"),
    (lambda x, w, t: ((x, w, t.float()), {}), "integers"),
    (lambda x, w, t: ((x, w, t.bool()), {}), "integers"),
    (lambda x, w, t: ((x, w.half(), t), {}), "share dtype"),
    (lambda x, w, t: ((x.double(), w.double(), t), {}), "share dtype"),
    (lambda x, w, t: ((x, w[:0], t), {}), "at least one row"),
    (lambda x, w, t: ((x[:, :0], w[:, :0], t), {}), "at least one row"),
    (lambda x, w, t: ((x, w, t), {"scale": float("inf")}), "scale"),
    (lambda x, w, t: ((x, w, t), {"softcap": -1.0}), "softcap"),
    (lambda x, w, t: ((x, w, t), {"softcap": 1e-7}), "softcap"),
    (lambda x, w, t: ((x, w, t), {"softcap": float("nan")}), "softcap"),
    (lambda x, w, t: ((x, w, t), {"reduction": "max"}), "Unsupported reduction"),
])
def test_refuses(change, message):
    a, kw = change(*args())
    with pytest.raises(ValueError, match=message):
        ra.linear_cross_entropy(*a, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        ra.linear_cross_entropy(*args())


@pytest.fixture(scope="module")
def lib():
    from rapidalign_b200 import build as b
    b.build()
    return _lib.load()


def desc(**kw):
    word = ctypes.c_int32(0)
    d = _lib.RaCeDesc(rows=100, vocab=1000, ld_x=64, ld_w=64, ignore_index=-100, dim=64,
                      dtype=_lib.RA_BF16, reduction=_lib.RA_REDUCE_MEAN, scale=1.0, softcap=0.0,
                      status=ctypes.addressof(word))
    d.keep = word
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_c_sizes(lib):
    d = desc()
    state = lib.ra_ce_state_bytes(ctypes.byref(d))
    assert state >= 256 + 8 * 100 and state % 256 == 0
    assert lib.ra_ce_workspace_bytes(ctypes.byref(d), 0) > 0
    assert lib.ra_ce_workspace_bytes(ctypes.byref(d), 1) >= 2 * 128 * 1024
    # fp32 keeps both halves of both operands
    f = desc(dtype=_lib.RA_F32)
    assert lib.ra_ce_state_bytes(ctypes.byref(f)) >= state + 4 * 64 * 1100


@pytest.mark.parametrize("sizes", [dict(rows=0), dict(rows=1, vocab=1, dim=1, ld_x=8, ld_w=8),
                                   dict(vocab=2 ** 31 - 512), dict(rows=2 ** 31 - 256, vocab=1)])
def test_c_sizes_at_the_ends(lib, sizes):
    d = desc(**sizes)
    assert lib.ra_ce_workspace_bytes(ctypes.byref(d), 0) >= 256
    assert lib.ra_ce_workspace_bytes(ctypes.byref(d), 1) >= 256


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(vocab=0), dict(dim=0), dict(dim=65537), dict(dtype=3), dict(dtype=-1),
    dict(ld_x=63), dict(ld_w=60), dict(ld_x=65), dict(reduction=3), dict(softcap=-1.0),
    dict(softcap=float("inf")), dict(scale=float("nan")), dict(status=None), dict(rows=2 ** 31),
])
def test_c_refuses(lib, bad):
    d = desc(**bad)
    assert lib.ra_ce_state_bytes(ctypes.byref(d)) == 0
    assert lib.ra_ce_workspace_bytes(ctypes.byref(d), 0) == 0
    rc = lib.ra_ce_forward(ctypes.byref(d), None, None, None, None, None, None, 0, None, 0, None)
    assert rc == _lib.RA_ERR_INVALID_ARGUMENT


def test_c_refuses_buffers(lib):
    d = desc()
    base = 1 << 20  # never touched: the checks come first
    rc = lib.ra_ce_forward(ctypes.byref(d), base + 2, base, base, base, base, base, 1 << 30, base,
                           1 << 30, None)
    assert rc == _lib.RA_ERR_INVALID_ARGUMENT  # x not 16-byte aligned
    rc = lib.ra_ce_forward(ctypes.byref(d), base, base, base, base, base, base, 16, base, 1 << 30,
                           None)
    assert rc == _lib.RA_ERR_WORKSPACE
    rc = lib.ra_ce_backward(ctypes.byref(d), base, base, base, base, None, base, base + 8, base,
                            1 << 30, base, 1 << 30, None)
    assert rc == _lib.RA_ERR_INVALID_ARGUMENT  # dw not 16-byte aligned
