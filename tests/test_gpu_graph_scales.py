"""A graph's results are its own: graphs of one batch whose gradients or values
lie orders of magnitude apart, each against the bounds of that graph alone."""
import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_attention import close, exact, make, ptr

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("q", "k", "v", "q_pos", "k_pos")


def run(d, nq, nk, cap=0.0, mask=None):
    x = {n: d[n].detach().requires_grad_(True) for n in NAMES}
    seg = ra.attention_segments(ptr(nq), ptr(nk))
    o = ra.pyg_kernel_attention(x["q"], x["k"], x["v"], segments=seg, q_pos=x["q_pos"],
                                k_pos=x["k_pos"], sigma=d["sigma"], softcap=cap, k_mask=mask)
    return dict(zip(("out",) + NAMES, (o.detach(),
                                       *torch.autograd.grad(o, [x[n] for n in NAMES], d["g"]))))


def part(t, n, i, side):
    if not side:
        return t
    first = sum(n[:i])
    return t[first:first + n[i]]


def graph(d, nq, nk, i):
    """Graph i of the batch as a batch of its own."""
    of = dict(q=nq, g=nq, q_pos=nq, k=nk, v=nk, k_pos=nk)
    return {n: part(t, of.get(n), i, n in of) for n, t in d.items()}


def check_graphs(d, nq, nk, cap=0.0, mask=None):
    got = run(d, nq, nk, cap, mask)
    D = d["q"].shape[2]
    for i in range(len(nq)):
        km = None if mask is None else part(mask, nk, i, True)
        (o64, bo), g64 = exact(graph(d, nq, nk, i), [nq[i]], [nk[i]], D ** -0.5, cap, None, km)
        close(part(got["out"], nq, i, True), o64, bo, f"out of graph {i}")
        for n in NAMES:
            close(part(got[n], nq if n.startswith("q") else nk, i, True), *g64[n],
                  f"d{n} of graph {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv", [(32, 2, 2), (96, 2, 1), (64, 4, 2)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_gradients_apart(cap, dim, heads, kv, dtype, cuda_device):
    """Upstream gradients 1, 1e-3 and 1e-6 of each other (fp16: down to 1e-4, as far
    as its results reach)."""
    nq, nk = [150, 300, 40, 129], [150, 260, 70, 1]
    d = make(nq, nk, heads, kv, dim, dtype, 3, seed=dim)
    low = 1e-6 if dtype != torch.float16 else 1e-4
    for i, f in enumerate((1.0, 1e-3, low, low)):
        part(d["g"], nq, i, True).mul_(f)
    check_graphs(d, nq, nk, cap)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["v", "k", "q"])
def test_values_apart(which, dtype, cuda_device):
    """A graph whose v (k, q) is 1e4 of the others' costs those nothing."""
    nq, nk = [100, 200, 33], [120, 64, 190]
    d = make(nq, nk, 4, 2, 32, dtype, 3, seed=3)
    part(d[which], nk if which != "q" else nq, 1, True).mul_(2.0 ** 13 if which == "v" else 2.0 ** 6)
    if which != "v":  # scores of the usual size: only the operand is large
        part(d["q" if which == "k" else "k"], nq if which == "k" else nk, 1, True).mul_(2.0 ** -6)
    check_graphs(d, nq, nk)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_apart(dtype, cuda_device):
    """Query rows of one graph whose upstream gradients lie apart: dq of a row
    counts by the row's own (fp16: do itself keeps its 11 bits), dk and dv by
    the graph's."""
    nq = nk = [200]
    d = make(nq, nk, 2, 2, 64, dtype, 0, seed=5)
    d["sigma"], d["q_pos"], d["k_pos"] = torch.ones(2, device="cuda"), *torch.zeros(
        2, 200, 3, device="cuda")
    low = 2.0 ** -10
    d["g"][::2] *= low
    got = run(d, nq, nk)
    (o64, bo), g64 = exact(d, nq, nk, 0.125, 0.0)
    for n in NAMES[:3]:
        close(got[n], *g64[n], "d" + n)
    small = {n: t[::2] if n in ("q", "g", "q_pos") else t for n, t in d.items()}
    _, g64 = exact(small, [100], nk, 0.125, 0.0)
    dq, b = g64["q"]
    if dtype == torch.float32:  # halves of do count by the graph's largest: 2^-38 of it in dP
        P = torch.softmax(0.125 * torch.einsum("ihd,jhd->hij", small["q"].double(),
                                               d["k"].double()), -1)
        edp = 2.0 ** -38 * d["g"].abs().max().double() * d["v"].double().abs().sum(-1).T
        eS = P * (edp[:, None] + (P * edp[:, None]).sum(-1, keepdim=True))
        b = b + 0.125 * torch.einsum("hij,jhd->ihd", eS, d["k"].double().abs())
    close(got["q"][::2], dq, b, "dq of small rows")


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_values_count_for_nothing(dtype, cuda_device):
    nq, nk = [90, 140], [200, 77]
    d = make(nq, nk, 2, 2, 32, dtype, 2, seed=9)
    mask = torch.rand(sum(nk), device="cuda") > 0.3
    for n in ("k", "v"):
        d[n][~mask] = 3e4
    check_graphs(d, nq, nk, mask=mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
def test_bitwise_what_it_is_alone(heads, kv, dtype, cuda_device):
    """Graphs too short for key ranges: the same bits alone, in a batch with far
    larger neighbours, among empty graphs and in a long batch."""
    nq, nk = [0, 70, 140, 0, 300, 33] + [20] * 70, [0, 90, 200, 5, 300, 150] + [20] * 70
    d = make(nq, nk, heads, kv, 32, dtype, 3, seed=11)
    for i, f in ((1, 16.0), (2, 2.0 ** -9), (5, 64.0)):
        for n in "gvq":
            part(d[n], nk if n == "v" else nq, i, True).mul_(f)
    got = run(d, nq, nk)
    for i in (1, 2, 4, 5, 6, 75):
        one = run(graph(d, nq, nk, i), [nq[i]], [nk[i]])
        for n, t in one.items():
            assert torch.equal(part(got[n], nq if n in ("out", "q", "q_pos") else nk, i, True), t), \
                (n, i)


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_clouds_apart(dtype, cuda_device):
    B, N = 3, 130
    n = [N] * B
    d = make(n, n, 2, 2, 64, dtype, 3, seed=13)
    for i, f in enumerate((1.0, 1e-3, 1e-4)):
        part(d["g"], n, i, True).mul_(f)
    x = {k: d[k].view(B, N, *d[k].shape[1:]).detach().requires_grad_(True) for k in NAMES}
    o = ra.kernel_attention_dense(x["q"], x["k"], x["v"], q_pos=x["q_pos"], k_pos=x["k_pos"],
                                  sigma=d["sigma"])
    grads = torch.autograd.grad(o, [x[k] for k in NAMES], d["g"].view_as(o))
    for i in range(B):
        _, g64 = exact(graph(d, n, n, i), [N], [N], 0.125, 0.0)
        for k, g in zip(NAMES, grads):
            close(g[i], *g64[k], f"d{k} of cloud {i}")
