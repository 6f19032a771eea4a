"""Forward-mode derivatives and function transforms of the softmax operators are
refused, not dropped (a recording library stands in for the kernels)."""
import pytest
import torch
from torch.autograd import forward_ad

import rapidalign_b200 as ra
from test_saved_tensors_host import recorder  # noqa: F401

Q, K = torch.randn(1, 5, 2, 8), torch.randn(1, 5, 2, 8)
X, W, T = torch.randn(9, 16), torch.randn(20, 16), torch.zeros(9, dtype=torch.long)


def attention(**kw):
    a = dict(q=Q, k=K, v=K, q_pos=torch.zeros(1, 5, 3), k_pos=torch.zeros(1, 5, 3),
             sigma=torch.ones(2))
    a.update(kw)
    return ra.kernel_attention_dense(a["q"], a["k"], a["v"], q_pos=a["q_pos"], k_pos=a["k_pos"],
                                     sigma=a["sigma"])


@pytest.mark.parametrize("name", ["q", "k", "v", "q_pos", "k_pos", "sigma"])
def test_attention_refuses_tangents(recorder, name):  # noqa: F811
    t = {"q": Q, "k": K, "v": K, "sigma": torch.ones(2)}.get(name, torch.zeros(1, 5, 3))
    for grad in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises(RuntimeError, match="forward"):
                attention(**{name: forward_ad.make_dual(t, torch.ones_like(t))})


@pytest.mark.parametrize("which", [0, 1])
def test_cross_entropy_refuses_tangents(recorder, which):  # noqa: F811
    for grad in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            a = [X, W]
            a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
            with pytest.raises(RuntimeError, match="forward"):
                ra.linear_cross_entropy(*a, T)


def test_plain_tensors_inside_a_level(recorder):  # noqa: F811
    with forward_ad.dual_level():
        attention()
        ra.linear_cross_entropy(X, W, T)
    assert [n for n, _ in recorder.calls] == ["ra_attn_forward", "ra_ce_forward"]


def test_transforms_are_refused(recorder):  # noqa: F811
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: attention(q=q))(Q[None])
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: attention(q=q), (Q,), (Q,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: ra.linear_cross_entropy(x, W, T))(X[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: ra.linear_cross_entropy(x, W, T)[0])(X)
