"""fp32 attention over long sums: the tensor core's accumulators drop the bits below
their last one at each step of 16 rows, so a sum of n terms of one sign in one
accumulator is off by up to n / 16 steps of 2^-23.  The kernels add rounds of at
most 512 rows (dk and dv of heads wider than 64: 128 rows, three steps for 16 of
them) with rounding.  Where all terms have one sign each element's relative error
is then at most

    32 steps of 2^-23 in a round, n / 512 or n / 128 additions of 2^-24, the
    operands' pairs 2 x 2^-21, P and its sum 2^-19, the factors and dP 2^-20

9e-6 at n = 16384 in rounds of 512, 1.1e-5 at 8192 in rounds of 128, where one
accumulator loses 3e-5 to 7e-5.
"""
import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_attention import ptr

pytestmark = pytest.mark.gpu

N = 8192


def bound(n, rows=512):
    return 32 * 2.0 ** -23 + n / rows * 2.0 ** -24 + 2 * 2.0 ** -21 + 2.0 ** -19 + 2.0 ** -20


def positive(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(*shape, generator=g, device="cuda") + 0.5


def near(got, want, limit, what):
    off = ((got.double() - want).abs() / want.abs()).max()
    assert off <= limit, (what, float(off), limit)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("graphs", [1, 80])
def test_outputs(graphs, dim, cuda_device):
    """In one range of the keys (many graphs) and in several; scores up to 1/2, off
    by 2^-20 each, so that no weight is a power of two."""
    H, nq, n = 4, 16, 2 * N
    q = torch.zeros(graphs * nq, H, dim, device="cuda")
    k = torch.zeros(graphs * n, H, dim, device="cuda")
    score = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(9),
                       device="cuda") / 2
    q[..., 0], k[..., 0] = 1.0, score.repeat(graphs)[:, None]
    v = positive(graphs * n, H, dim)
    o = ra.pyg_kernel_attention(q, k, v, q_ptr=ptr([nq] * graphs), k_ptr=ptr([n] * graphs),
                                scale=1.0)
    p = torch.softmax(score.double(), 0)
    for g in (0, graphs - 1):
        want = torch.einsum("j,jhd->hd", p, v[g * n:(g + 1) * n].double())
        near(o[g * nq:(g + 1) * nq], want[None].expand(nq, H, dim), bound(n) + 2.0 ** -20, "out")


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_outputs_while_the_maximum_grows(dim, cuda_device):
    """Earlier rounds count by the references they were relative to."""
    graphs, H, nq, n = 80, 4, 16, 2048
    q = torch.zeros(graphs * nq, H, dim, device="cuda")
    k = torch.zeros(graphs * n, H, dim, device="cuda")
    q[..., 0], v = 1.0, positive(graphs * n, H, dim, seed=1)
    steps = torch.arange(n, device="cuda") // 256 * 6.0 + torch.rand(n, device="cuda")
    for order in (steps, steps.flip(0)):
        k[..., 0] = order.repeat(graphs)[:, None]
        o = ra.pyg_kernel_attention(q, k, v, q_ptr=ptr([nq] * graphs), k_ptr=ptr([n] * graphs),
                                    scale=1.0)
        p = torch.softmax(order.double(), 0)
        for g in (0, graphs - 1):
            want = torch.einsum("j,jhd->hd", p, v[g * n:(g + 1) * n].double())
            # a score of 48 carries the pairs' 2^-21 and a few steps: 5e-5 of P
            near(o[g * nq:(g + 1) * nq], want[None].expand(nq, H, dim),
                 bound(n) + 48 * 2.0 ** -20, "out")


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_gradients(masked, dim, cuda_device):
    """dk and dv over N queries; dq over N keys (its products have one sign: dP and
    k change theirs together, and D is 0)."""
    H, m = 2, 40
    sign = torch.ones(m, device="cuda")
    sign[::2] = -1.0

    # many queries, few keys: v = +-1 gives dP one size, D = 0
    q, g = positive(N, H, dim, seed=2), positive(N, H, dim, seed=3)
    k = torch.zeros(m, H, dim, device="cuda").requires_grad_(True)
    v = sign[:, None, None].expand(m, H, dim).clone().requires_grad_(True)
    mq = torch.ones(N, dtype=torch.bool, device="cuda")
    if masked:
        mq[::3] = False
    o = ra.pyg_kernel_attention(q, k, v, q_ptr=ptr([N]), k_ptr=ptr([m]), scale=1.0, q_mask=mq)
    dk, dv = torch.autograd.grad(o, [k, v], g)
    live = mq.double()[:, None, None]
    gs = (g.double() * live).sum(-1)  # (N, H)
    want = torch.einsum("ih,ihd->hd", gs, q.double()) / m
    limit = bound(N, 128 if dim > 64 else 512)
    near(dk, sign.double()[:, None, None] * want, limit, "dk")
    near(dv, ((g.double() * live).sum(0) / m)[None].expand(m, H, dim), limit, "dv")

    # few queries, many keys
    sign = torch.ones(N, device="cuda")
    sign[::2] = -1.0
    q = torch.zeros(m, H, dim, device="cuda").requires_grad_(True)
    size = positive(N // 2, H, dim, seed=4).repeat_interleave(2, 0)  # pairs of opposite keys
    k = size * sign[:, None, None]
    v = sign[:, None, None].expand(N, H, dim).clone()
    mk = torch.ones(N, dtype=torch.bool, device="cuda")
    if masked:
        mk[::6] = mk[1::6] = False
    g = positive(m, H, dim, seed=5)
    o = ra.pyg_kernel_attention(q, k, v, q_ptr=ptr([m]), k_ptr=ptr([N]), scale=1.0, k_mask=mk)
    dq, = torch.autograd.grad(o, [q], g)
    near(dq, g.double().sum(-1)[..., None] * size.double()[mk].mean(0),
         bound(N), "dq")


def test_long_sums_are_repeatable(cuda_device):
    n = [3000, 700]
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = [torch.randn(sum(n), 2, 64, generator=gen, device="cuda").requires_grad_(True)
         for _ in range(3)]
    g = torch.randn(sum(n), 2, 64, generator=gen, device="cuda")
    runs = []
    for _ in range(3):
        o = ra.pyg_kernel_attention(*x, q_ptr=ptr(n))
        runs.append((o.detach(), *torch.autograd.grad(o, x, g)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
