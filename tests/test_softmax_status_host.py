"""The status word of the softmax operators on the host: a wait that ran out is
raised by the next call of either, once; and the test hooks the C entries take."""
import ctypes

import pytest
import torch

import rapidalign_b200 as ra
from rapidalign_b200 import _lib
from test_attention_host import desc as attn_desc
from test_cross_entropy_host import desc as ce_desc
from test_saved_tensors_host import recorder  # noqa: F401


def calls():
    q, x = torch.randn(1, 5, 2, 8), torch.randn(9, 16)
    return {
        "kernel attention": lambda: ra.kernel_attention_dense(q, q, q),
        "linear cross entropy": lambda: ra.linear_cross_entropy(x, x, torch.zeros(9).long()),
    }


@pytest.mark.parametrize("name", ["kernel attention", "linear cross entropy"])
def test_raised_once_by_the_next_call(name, recorder, monkeypatch):  # noqa: F811
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(_lib, "_STATUS", word)
    monkeypatch.setattr(_lib, "check", lambda rc, what="": (_ for _ in ()).throw(
        RuntimeError(f"{what} {rc}")) if rc else None)
    call = calls()[name]
    call()
    word.fill_(1)
    with pytest.raises(RuntimeError, match=f"{name} .an earlier call. {_lib.RA_ERR_DEVICE_TIMEOUT}"):
        call()
    assert int(word) == 0
    call()


def test_hooks_are_validated():
    from rapidalign_b200 import build as b
    b.build()
    lib = _lib.load()
    for make, size in ((attn_desc, lib.ra_attn_workspace_bytes), (ce_desc, lib.ra_ce_workspace_bytes)):
        assert size(ctypes.byref(make(test_hooks=_lib.RA_TEST_NO_MMA)), 1) > 0
        for other in (_lib.RA_TEST_RING_IDLE, 4, -1):
            assert size(ctypes.byref(make(test_hooks=other)), 1) == 0
