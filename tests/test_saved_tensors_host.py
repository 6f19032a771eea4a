"""What the backward passes hand to the kernels when PyTorch gives back other
tensors than the forward saved (checkpoints, hooks on saved tensors): a library
that records its arguments stands in for the kernels, on CPU tensors."""
import contextlib
import ctypes

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import rapidalign_b200 as ra
from rapidalign_b200 import _lib


def fields(ref):
    s = ref._obj
    return {n: getattr(s, n) for n, _ in s._fields_}


class Recorder:
    """Size queries of 512 bytes; passes that only note what they were given."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *a: 512
        if not name.startswith(("ra_attn_", "ra_ce_")):
            raise AttributeError(name)

        def fn(*args):
            got = [fields(a) if hasattr(a, "_obj") else a for a in args]
            self.calls.append((name, got))
            return _lib.RA_OK
        return fn

    def last(self, name):
        return [got for n, got in self.calls if n == name][-1]


@pytest.fixture
def recorder(monkeypatch):
    rec, word = Recorder(), ctypes.c_int32(0)
    monkeypatch.setattr(_lib, "load", lambda path=None: rec)
    monkeypatch.setattr(_lib, "require_cuda",
                        lambda *t: next(x for x in t if x is not None).device)
    monkeypatch.setattr(_lib, "status_word", lambda: ctypes.addressof(word))
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 0)
    rec.word = word
    return rec


class Clones:
    """Hooks that give every saved tensor back as `again` makes it."""

    def __init__(self, again):
        self.again, self.given = again, []

    def __enter__(self):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), self.unpack)
        return self.hooks.__enter__()

    def __exit__(self, *exc):
        return self.hooks.__exit__(*exc)

    def unpack(self, t):
        self.given.append(self.again(t))
        return self.given[-1]

    def owner(self, address):
        return next(t for t in self.given if t.data_ptr() == address)


N, H, HK, D, C = 6, 4, 2, 8, 3


def attention(leaf, dtype=torch.float32, mask=True):
    """Operands made inside, as in a layer."""
    q = (leaf * 2).view(1, N, H, D).to(dtype)
    k, v = (leaf.view(1, N, H, D)[:, :, :HK] * c for c in (3, 4))
    k, v = k.to(dtype).contiguous(), v.to(dtype).contiguous()
    pos = (leaf.view(N, H * D)[:, :C] * 1).contiguous()[None]
    sigma = leaf.view(-1)[:H] * 0 + 1.0
    m = torch.ones(1, N, dtype=torch.bool) if mask else None
    return ra.kernel_attention_dense(q, k, v, m, m, q_pos=pos, sigma=sigma)


ATTN_INPUTS = ("q", "k", "v", "q_pos", "k_pos", "sigma", "q_mask", "k_mask")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_under_a_checkpoint(recorder, dtype):
    leaf = torch.randn(N * H * D, requires_grad=True)
    out = checkpoint(attention, leaf, dtype, use_reentrant=False)
    out.sum().backward()
    forwards = [got[1] for n, got in recorder.calls if n == "ra_attn_forward"]
    assert len(forwards) == 2
    backward = recorder.last("ra_attn_backward")[1]
    for name in ATTN_INPUTS:  # the second forward's tensors live, the first's do not
        assert backward[name] == forwards[1][name], name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_under_hooks(recorder, dtype):
    """Clones, each where it is given back."""
    leaf = torch.randn(N * H * D, requires_grad=True)
    hooks = Clones(lambda t: t.clone())
    with hooks:
        out = attention(leaf, dtype)
    out.sum().backward()
    backward = recorder.last("ra_attn_backward")
    for name in ATTN_INPUTS:
        assert any(t.data_ptr() == backward[1][name] for t in hooks.given), name
    assert any(t.data_ptr() == backward[3 if dtype == torch.float32 else 4] for t in hooks.given)


def test_attention_strides_of_what_is_given_back(recorder):
    """q as a slice of wider rows comes back contiguous, k and v the other way."""
    base = torch.randn(N, 2 * H, D, requires_grad=True)

    def again(t):
        if t.dtype == torch.float32 and t.shape == (N, HK, D):
            wide = torch.zeros(N, HK + 1, D + 8)
            wide[:, :HK, :D] = t
            return wide[:, :HK, :D]
        return t.contiguous() if t.is_contiguous() else t.clone(
            memory_format=torch.contiguous_format)

    hooks = Clones(again)
    seg = ra.AttentionSegments(*[torch.zeros(2, dtype=torch.long)] * 2,
                               *[torch.zeros(1, 4, dtype=torch.int32)] * 2, 1, N, N, N, N)
    with hooks:
        rows = base * 1
        out = ra.pyg_kernel_attention(rows[:, :H], rows[:, H:H + HK].contiguous(),
                                      rows[:, :HK].contiguous(), segments=seg)
    assert recorder.last("ra_attn_forward")[0]["q_row"] == 2 * H * D
    out.sum().backward()
    desc, inputs = recorder.last("ra_attn_backward")[:2]
    for n in "qkv":
        t = hooks.owner(inputs[n])
        assert (desc[n + "_row"], desc[n + "_head"]) == t.stride()[:2]
    assert desc["q_row"] == H * D and desc["k_row"] == (HK + 1) * (D + 8)


def cross_entropy(leaf, weight, target):
    return ra.linear_cross_entropy(leaf * 2, weight * 3, target)[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cross_entropy_under_a_checkpoint(recorder, dtype):
    x, w = (torch.randn(n, 16, dtype=dtype, requires_grad=True) for n in (9, 20))
    loss = checkpoint(cross_entropy, x, w, torch.zeros(9, dtype=torch.long), use_reentrant=False)
    loss.backward()
    forwards = [got for n, got in recorder.calls if n == "ra_ce_forward"]
    assert len(forwards) == 2
    assert recorder.last("ra_ce_backward")[:4] == forwards[1][:4]  # desc, x, w, target


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cross_entropy_strides_of_what_is_given_back(recorder, dtype):
    """Strided operands come back contiguous, and the other way round."""
    for wide_first in (True, False):
        def again(t, wide=not wide_first):
            if not wide or t.dim() < 2:
                return t.clone(memory_format=torch.contiguous_format)
            rows = torch.zeros(t.shape[0], 40, dtype=t.dtype)
            rows[:, :16] = t
            return rows[:, :16]

        hooks = Clones(again)
        leaves = [torch.randn(n, 40 if wide_first else 16, dtype=dtype, requires_grad=True)
                  for n in (9, 20)]
        with hooks:
            x, w = ((t * 2)[:, :16] for t in leaves)
            loss, _ = ra.linear_cross_entropy(x, w, torch.zeros(9, dtype=torch.long))
        before = recorder.last("ra_ce_forward")[0]
        assert before["ld_x"] == before["ld_w"] == (40 if wide_first else 16)
        loss.backward()
        desc, x, w, target = recorder.last("ra_ce_backward")[:4]
        assert desc["ld_x"] == hooks.owner(x).stride(0) == (16 if wide_first else 40)
        assert desc["ld_w"] == hooks.owner(w).stride(0) == (16 if wide_first else 40)
        assert hooks.owner(target).dtype == torch.long


def tensors_of(node):
    held = [v for v in vars(node).values()]
    return [v for h in held for v in (h if isinstance(h, (tuple, list)) else [h])
            if isinstance(v, torch.Tensor)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing_is_held_after_the_backward(recorder, dtype):
    """What the passes keep between them is saved, and freed with the rest."""
    leaf = torch.randn(N * H * D, requires_grad=True)
    x, w = (torch.randn(n, 16, dtype=dtype, requires_grad=True) for n in (9, 20))
    for out in (attention(leaf, dtype), cross_entropy(x, w, torch.zeros(9, dtype=torch.long))):
        assert not tensors_of(out.grad_fn)
        out.sum().backward()
        with pytest.raises(RuntimeError, match="already been freed"):
            out.grad_fn.saved_tensors


def test_state_is_aligned_again(recorder):
    def again(t):
        if t.dtype != torch.uint8:
            return t.clone()
        odd = torch.zeros(t.numel() + 264, dtype=torch.uint8)
        at = (-odd.data_ptr()) % 256 + 8
        return odd[at:at + t.numel()].copy_(t)

    leaf = torch.randn(N * H * D, requires_grad=True)
    x, w = (torch.randn(n, 16, requires_grad=True) for n in (9, 20))
    with Clones(again):
        outs = [attention(leaf, mask=False),
                cross_entropy(x, w, torch.zeros(9, dtype=torch.long))]
    for out in outs:
        out.sum().backward()
    got = recorder.last("ra_attn_backward")
    assert got[7] % 256 == 0 and got[8] > 0 and (got[5] - got[7]) % 256 == 0
    got = recorder.last("ra_ce_backward")
    assert got[8] % 256 == 0 and got[9] > 0
