"""Training steps of the softmax operators in captured graphs: every type, the
forms with scales of their own, and two graphs replayed in turn."""
import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_attention import make as make_attention
from test_gpu_attention import ptr
from test_gpu_cross_entropy import make as make_cross_entropy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def attention(dtype, nq, nk, seed, cap):
    d = make_attention(nq, nk, 4, 2, 32, dtype, 2, seed=seed)
    names = ("q", "k", "v", "q_pos", "k_pos", "sigma")
    x = [d[n].requires_grad_(True) for n in names]
    mask = torch.rand(sum(nk), device="cuda") > 0.2
    seg = ra.attention_segments(ptr(nq), ptr(nk))

    def step():
        o = ra.pyg_kernel_attention(*x[:3], segments=seg, q_pos=x[3], k_pos=x[4], sigma=x[5],
                                    k_mask=mask, softcap=cap)
        return (o.detach(), *torch.autograd.grad(o, x, d["g"]))

    def renew(seed):
        new = make_attention(nq, nk, 4, 2, 32, dtype, 2, seed=seed)
        with torch.no_grad():
            for n in names + ("g",):
                d[n].copy_(new[n])
            d["g"][::2] *= 2.0 ** -8
            mask.copy_(torch.rand(sum(nk), device="cuda") > 0.4)
    return step, renew


def cross_entropy(dtype, n, v, seed, lse):
    x, w, t = make_cross_entropy(n, v, 40, dtype, seed=seed)
    x.requires_grad_(True), w.requires_grad_(True)
    g = [torch.randn(n, device="cuda") for _ in range(1 + lse)]

    def step():
        outs = ra.linear_cross_entropy(x, w, t, reduction="none")[:1 + lse]
        return (outs[0].detach(), *torch.autograd.grad(outs, [x, w], g))

    def renew(seed):
        new = make_cross_entropy(n, v, 40, dtype, seed=seed)
        with torch.no_grad():
            for a, b in zip((x, w, t), new):
                a.copy_(b)
            g[0].copy_(torch.randn(n, device="cuda") * torch.logspace(0, -3, n, device="cuda"))
    return step, renew


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_replayed_in_turn(dtype, cuda_device):
    cases = [attention(dtype, [150, 40, 7], [90, 300, 1], 1, 0.0),
             attention(dtype, [1, 2, 1], [500, 33, 2000], 2, 4.0),
             cross_entropy(dtype, 150, 700, 3, True), cross_entropy(dtype, 5, 900, 4, False)]
    graphs = []
    for step, _ in cases:
        step()  # kernels' attributes, the status word
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for seed in (11, 12):
        for _, renew in cases:
            renew(seed)
        for _ in range(2):
            for graph, _ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for (step, _), (_, held) in zip(cases, graphs):
            for got, want in zip(held, step()):
                assert torch.isfinite(want).all()
                assert torch.equal(got, want)
