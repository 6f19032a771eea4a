"""Waits of the softmax operators that run out, without faulting the GPU: with
the test hook RA_TEST_NO_MMA the kernels issue no product, and the waits for
them run out after 4096 polls or sooner.  The call returns, the next one raises, and what runs after it is
what it was before (an aborted launch that kept tensor memory, or copies that
still land, would show there)."""
import pytest
import torch

import rapidalign_b200 as ra
from rapidalign_b200 import _lib

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def raises_once(again):
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="an earlier call.*status 22"):
        again()


def hooked(monkeypatch, name):
    """Descriptors made from here on ask for the hook."""
    plain = getattr(_lib, name)
    monkeypatch.setattr(_lib, name, lambda: plain(test_hooks=_lib.RA_TEST_NO_MMA))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("n", [[20], [300, 70, 640, 129, 1] * 40])
def test_attention(n, dim, dtype, monkeypatch, cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    q, k, v, g = (torch.randn(sum(n), 4, dim, generator=gen, device="cuda").to(dtype)
                  for _ in range(4))
    pos = torch.randn(sum(n), 3, generator=gen, device="cuda")
    seg = ra.attention_segments(torch.tensor([0, *n], device="cuda").cumsum(0))
    leaves = [t.requires_grad_(True) for t in (q, k, v, pos)]

    def forward():
        return ra.pyg_kernel_attention(q, k, v, segments=seg, q_pos=pos, sigma=0.7)

    def step():
        o = forward()
        return (o.detach(), *torch.autograd.grad(o, leaves, g))

    want = step()
    with monkeypatch.context() as m:
        hooked(m, "RaAttnDesc")
        forward()
    raises_once(forward)
    o = forward()
    o.grad_fn.desc.test_hooks = _lib.RA_TEST_NO_MMA
    torch.autograd.grad(o, leaves, g)
    raises_once(forward)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(20, 30, 16), (3000, 2500, 128), (700, 5000, 520)])
def test_cross_entropy(n, v, d, dtype, monkeypatch, cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(n)
    x, w = (torch.randn(m, d, generator=gen, device="cuda").to(dtype).requires_grad_(True)
            for m in (n, v))
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")

    def forward():
        return ra.linear_cross_entropy(x, w, t)[0]

    def step():
        loss = forward()
        return (loss.detach(), *torch.autograd.grad(loss, [x, w]))

    want = step()
    with monkeypatch.context() as m:
        hooked(m, "RaCeDesc")
        forward()
    raises_once(forward)
    loss = forward()
    loss.grad_fn.desc.test_hooks = _lib.RA_TEST_NO_MMA
    torch.autograd.grad(loss, [x, w])
    raises_once(forward)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
