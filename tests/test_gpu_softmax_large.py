"""The softmax operators on tensors of more than 2^31 elements (the last rows by
the bounds, as a call of their own), empty sides, and backward passes run twice."""
import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_attention import close as close_attention
from test_gpu_attention import exact as exact_attention
from test_gpu_attention import make as make_attention
from test_gpu_attention import ptr
from test_gpu_cross_entropy import close, exact, make

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("q", "k", "v", "q_pos", "k_pos")


def test_attention_rows_past_32_bits(cuda_device):
    """2.15e9 elements a tensor, in graphs of 100 to 300 rows."""
    H, D = 8, 128
    n = [100, 300, 200] * 3500
    d = make_attention(n, n, H, H, D, torch.bfloat16, 2, seed=1)
    assert d["q"].numel() > 2 ** 31
    x = {k: d[k].requires_grad_(True) for k in NAMES}
    o = ra.pyg_kernel_attention(x["q"], x["k"], x["v"], segments=ra.attention_segments(ptr(n)),
                                q_pos=x["q_pos"], k_pos=x["k_pos"], sigma=d["sigma"])
    grads = torch.autograd.grad(o, [x[k] for k in NAMES], d["g"])
    for rows, m in ((slice(0, 400), [100, 300]), (slice(-500, None), [300, 200])):
        part = {k: t.detach()[rows] if k != "sigma" else t for k, t in d.items()}
        (o64, bo), g64 = exact_attention(part, m, m, D ** -0.5, 0.0)
        close_attention(o[rows], o64, bo, "out")
        for k, g in zip(NAMES, grads):
            close_attention(g[rows], *g64[k], "d" + k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_query_on_keys_past_32_bits(dtype, cuda_device):
    """The mask leaves the last keys only."""
    HK, D, n = 8, 128, 2_100_003
    gen = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.empty(n, HK, D, dtype=dtype, device="cuda").normal_(generator=gen)
            for _ in range(2))
    assert k.numel() > 2 ** 31
    q = torch.randn(1, HK, D, generator=gen, device="cuda").to(dtype)
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[-3000:] = True
    o = ra.pyg_kernel_attention(q, k, v, q_ptr=ptr([1]), k_ptr=ptr([n]), k_mask=mask)
    d = dict(q=q, k=k[-3000:], v=v[-3000:], g=q)
    (o64, bo), _ = exact_attention(d, [1], [3000], D ** -0.5, 0.0)
    close_attention(o, o64, bo, "out")


@pytest.mark.parametrize("n", [5, 40])
def test_a_table_past_32_bits(n, cuda_device):
    v, d = 2_100_003, 1024
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_(0, 2 / 32, generator=gen)
    assert w.numel() > 2 ** 31
    x = torch.randn(n, d, generator=gen, device="cuda").to(torch.bfloat16)
    t = torch.full((n,), v - 1, device="cuda")
    t[0], t[1] = 0, v - 7
    x.requires_grad_(True), w.requires_grad_(True)
    loss, lse = ra.linear_cross_entropy(x, w, t, reduction="none")
    g = torch.ones(n, device="cuda")
    dx, dw = torch.autograd.grad(loss, [x, w], g)
    x, w = x.detach(), w.detach()
    # the logsumexp in pieces of the table; the error of z as if all were there
    z = torch.cat([x.double() @ w[a:a + 100000].double().T for a in range(0, v, 100000)], 1)
    lse64 = torch.logsumexp(z, 1)
    (_, _, _, _), (_, bl, _, _) = exact(x, w[-100000:], torch.zeros_like(t), 1.0, 0.0, g.double(),
                                        torch.zeros(n, device="cuda").double())
    close(lse, lse64, 2 * bl, "lse")
    close(loss, lse64 - z.gather(1, t[:, None])[:, 0], 4 * bl, "loss")
    # the last rows' gradients: p - [v = target], rounded to bf16 (2^-8) as dw is
    rows = slice(v - 300, v)
    du = torch.exp(z[:, rows] - lse64[:, None])
    du[torch.arange(2, n), 299] -= 1.0
    du[1, 300 - 7] -= 1.0
    want = du.T @ x.double()
    bound = (2.0 ** -8 + 4 * bl.max()) * (du.abs().T @ x.double().abs()) + 2.0 ** -8 * want.abs()
    close(dw[rows], want, bound + 1e-30, "dw")
    sure = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(sure)
    for a in range(0, v, 100000):
        part = w[a:a + 100000].double()
        p = torch.exp(z[:, a:a + 100000] - lse64[:, None])
        inside = (t >= a) & (t < a + part.shape[0])
        p[inside, t[inside] - a] -= 1.0
        sure += p @ part
        size += p.abs() @ part.abs()
    close(dx, sure, (2.0 ** -8 + 4 * bl.max()) * size + 2.0 ** -8 * sure.abs() + 1e-30, "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 20])
def test_empty_sides_of_padded_clouds(dim, dtype, cuda_device):
    for N, M in ((0, 5), (5, 0), (0, 0)):
        q = torch.randn(2, N, 4, dim, device="cuda").to(dtype).requires_grad_(True)
        k = torch.randn(2, M, 2, dim, device="cuda").to(dtype).requires_grad_(True)
        p = [torch.randn(2, m, 3, device="cuda", requires_grad=True) for m in (N, M)]
        s = torch.ones(4, device="cuda", requires_grad=True)
        o = ra.kernel_attention_dense(q, k, k, q_pos=p[0], k_pos=p[1], sigma=s)
        assert o.shape == (2, N, 4, dim) and not o.any()
        for g in torch.autograd.grad(o.sum(), [q, k, *p, s]):
            assert not g.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_twice(dtype, cuda_device):
    """A kept graph gives the same again, and other gradients for other seeds."""
    n = [150, 70]
    d = make_attention(n, n, 4, 2, 32, dtype, 3, seed=4)
    leaves = [d[k].requires_grad_(True) for k in NAMES + ("sigma",)]
    o = ra.pyg_kernel_attention(*leaves[:3], q_ptr=ptr(n), q_pos=leaves[3], k_pos=leaves[4],
                                sigma=leaves[5])
    x, w, t = make(60, 300, 40, dtype, seed=4)
    x.requires_grad_(True), w.requires_grad_(True)
    few = x.detach()[:5].clone().requires_grad_(True)
    cases = [(o, leaves, d["g"])]
    for a in (x, few):
        loss, _ = ra.linear_cross_entropy(a, w, t[:a.shape[0]], reduction="none")
        cases.append((loss, [a, w], torch.randn(a.shape[0], device="cuda")))
    for out, ins, g in cases:
        first = torch.autograd.grad(out, ins, g, retain_graph=True)
        other = torch.autograd.grad(out, ins, g * 1e-4, retain_graph=True)
        again = torch.autograd.grad(out, ins, g)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert not any(torch.equal(a, b) for a, b in zip(first, other))
