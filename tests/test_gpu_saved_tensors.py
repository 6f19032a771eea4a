"""Gradients of the softmax operators where PyTorch gives the backward other
tensors than the forward saved: checkpoints and hooks.  Bitwise what they are
without, since the values are the same and the backward repeats bitwise."""
import contextlib

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import rapidalign_b200 as ra
from test_gpu_cross_entropy import close, exact

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def moved(t):
    """The same values elsewhere: in wider rows where it is a matrix or more."""
    if t.dim() < 2 or not t.is_floating_point():
        return t.clone()
    wide = torch.full((*t.shape[:-1], t.shape[-1] + 16), 7.0, dtype=t.dtype, device=t.device)
    out = wide[..., 8:8 + t.shape[-1]]
    out.copy_(t)
    return out


def hooks(unpack):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack)


CONTEXTS = {
    "clones": lambda: hooks(lambda t: t.clone()),
    "wider rows": lambda: hooks(moved),
    "dense": lambda: hooks(lambda t: t.clone(memory_format=torch.contiguous_format)),
    "on the host": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
}


def compare(step, leaves, up):
    def grads(context, fn):
        with context:
            out = fn(*leaves)
        # what the forward freed is written over
        torch.full((1 << 22,), float("nan"), device="cuda")
        return (out.detach(), *torch.autograd.grad(out, leaves, up))

    want = grads(contextlib.nullcontext(), step)
    for name, context in CONTEXTS.items():
        for a, b in zip(grads(context(), step), want):
            assert torch.equal(a, b), name
    again = grads(contextlib.nullcontext(),
                  lambda *a: checkpoint(step, *a, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 20])
@pytest.mark.parametrize("nq", [[70, 150], [2, 1]])
def test_attention(dtype, dim, nq, cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    H, HK, n = 4, 2, [90, 700]

    def rn(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    x = [rn(sum(nq), H, dim), rn(sum(n), 2 * HK, dim), rn(sum(nq), 3), rn(sum(n), 3),
         torch.rand(H, generator=gen, device="cuda") + 0.5]
    leaves = [t.requires_grad_(True) for t in x]
    mask = torch.rand(sum(n), generator=gen, device="cuda") > 0.2
    seg = ra.attention_segments(*(torch.tensor([0, *m], device="cuda").cumsum(0) for m in (nq, n)))

    def step(q, kv, q_pos, k_pos, sigma):  # operands made inside, k and v slices
        kv = (kv * 1.5).to(dtype)
        return ra.pyg_kernel_attention((q * 1.25).to(dtype), kv[:, :HK], kv[:, HK:], segments=seg,
                                       q_pos=q_pos * 1.0, k_pos=k_pos * 1.0, sigma=sigma * 1.0,
                                       k_mask=mask.clone())

    compare(step, leaves, rn(sum(nq), H, dim).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(3, 700, 64), (200, 500, 36), (150, 90, 72)])
def test_cross_entropy(dtype, n, v, d, cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(n)
    leaves = [torch.randn(m, 2 * d, generator=gen, device="cuda").requires_grad_(True)
              for m in (n, v)]
    target = torch.randint(0, v, (n,), generator=gen, device="cuda")

    def step(x, w):  # both are slices of wider rows
        x, w = ((t * 0.5).to(dtype)[:, :d] for t in (x, w))
        loss, lse = ra.linear_cross_entropy(x, w, target + 0, reduction="none")
        return loss + 0.1 * lse

    compare(step, leaves, torch.randn(n, generator=gen, device="cuda"))


@pytest.mark.parametrize("first", [0, 1])
def test_cross_entropy_alignment_changes(first, cuda_device):
    """fp32, few rows: the forward's choice of kernel is by the table's alignment,
    which the backward may not find again."""
    gen = torch.Generator(device="cuda").manual_seed(first)
    n, v, d = 3, 800, 64
    x, w = (torch.randn(m, d, generator=gen, device="cuda") for m in (n, v))
    target = torch.tensor([0, 5, v - 1], device="cuda")

    def placed(t, at):
        wide = torch.zeros(t.shape[0], d + 4, device="cuda")
        wide[:, at:at + d] = t
        return wide[:, at:at + d]

    def grads(start, end):
        a = x.clone().requires_grad_(True)
        b = placed(w, start).requires_grad_(True)
        with hooks(lambda t: placed(t, end) if t.shape == (v, d) else t):
            loss, _ = ra.linear_cross_entropy(a, b, target)
        return torch.autograd.grad(loss, [a, b])

    gl = torch.full((n,), 1 / n, device="cuda").double()
    (_, _, *want), (_, _, *bound) = exact(x, w, target, 1.0, 0.0, gl, torch.zeros_like(gl))
    for got, t, b in zip(grads(first, 1 - first), want, bound):
        close(got, t, b, "gradient")


def test_memory_after_the_backward(cuda_device):
    """With the results alive, nothing of a pass is left but results and gradients."""
    q = torch.randn(4096, 4, 64, device="cuda", requires_grad=True)
    x = torch.randn(2048, 256, device="cuda", requires_grad=True)
    w = torch.randn(8192, 256, device="cuda", requires_grad=True)
    t = torch.randint(0, 8192, (2048,), device="cuda")
    seg = ra.attention_segments(torch.tensor([0, 4096], device="cuda"))
    calls = (lambda: ra.pyg_kernel_attention(q, q, q, segments=seg),
             lambda: ra.linear_cross_entropy(x, w, t, reduction="sum")[0])
    for call, leaves in zip(calls, ([q], [x, w])):
        call().sum().backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = call()
        torch.autograd.backward(out.sum())  # into gradients that are there
        left = torch.cuda.memory_allocated() - before
        assert left <= out.numel() * out.element_size() + 8192
