"""linear_cross_entropy against the formula in float64, element by element.

Error bounds, with u the half step of the gradients' 16-bit type (fp32
inputs: pairs of fp16 halves, 2^-21 for a product of two pairs without its
smallest term) and e = 2^-23 for each fp32 addition:
  z:   (D + 4) e' sum_d |x_d w_d| |s|, e' = e (+ 2^-21 / D for pairs), and a
       few steps of z itself (capped: of the cap, for tanh and its factors)
  lse: max_v err(z), a few steps of lse, and the exponentials' and sums' own
       relative error, 2^-20
  p:   relative 2 max err(z) + 2^-19
  dx:  s sum_v (|du| (u + rel p) + |gl| onehot parts) |w| + fp32 sums + half a
       step of dx; dw likewise.
An fp16 number below 2^-14 has an absolute half step of 2^-25, and a pair's low
half reaches there too.  Tensors held in fp16 are scaled by the power of two
that brings their largest magnitude to 2^13 or more, so such an element is off
by at most 2^-38 of the largest.
"""
import math

import pytest
import torch

import rapidalign_b200 as ra
from rapidalign_b200 import _lib

pytestmark = pytest.mark.gpu

IGN = -100
E = 2.0 ** -23


def make(n, v, d, dtype, seed=0, ignore=0.1, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, generator=g, device="cuda").to(dtype)
    w = (torch.randn(v, d, generator=g, device="cuda") * spread / math.sqrt(d)).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    if n > 2:
        t[torch.rand(n, generator=g, device="cuda") < ignore] = IGN
        t[0] = v - 1
    return x, w, t


def exact(x, w, t, scale, cap, gl, ge):
    """Float64 (loss rows, lse, dx, dw) for row gradients gl, ge, and bounds."""
    dtype = x.dtype
    u = torch.finfo(dtype).eps / 2
    pair = 2.0 ** -21 if dtype == torch.float32 else 0.0
    n, d = x.shape
    v = w.shape[0]
    x, w = x.double(), w.double()
    raw = scale * (x @ w.T)
    z = cap * torch.tanh(raw / cap) if cap else raw
    ax, aw = ((2.0 ** -38 * m.abs().max() if pair else 0.0) for m in (x, w))
    ez = abs(scale) * ((d + 4) * E + pair) * (x.abs() @ w.abs().T) + 8 * E * z.abs()
    ez = ez + abs(scale) * (ax * w.abs().sum(1)[None] + aw * x.abs().sum(1)[:, None])
    if cap:
        ez = ez + 8 * E * cap
    lse = torch.logsumexp(z, 1)
    valid = t != IGN
    at = torch.where(valid, t, 0)
    zt = z.gather(1, at[:, None])[:, 0]
    rows = torch.where(valid, lse - zt, torch.zeros_like(lse))
    ezm = ez.amax(1)
    b_lse = ezm + 2.0 ** -20 + 4 * E * lse.abs()
    b_row = torch.where(valid, b_lse + ezm + 4 * E * (rows.abs() + zt.abs()),
                        torch.zeros_like(lse))
    gl = torch.where(valid, gl, torch.zeros_like(gl))
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p)
    onehot[torch.arange(n, device=x.device), at] = valid.double()
    slope = 1 - (z / cap) ** 2 if cap else torch.ones_like(z)
    du = ((gl + ge)[:, None] * p - gl[:, None] * onehot) * slope
    eslope = 16 * E + 2 * ez / cap * (z.abs() / cap) if cap else torch.zeros_like(z)
    edu = ((gl + ge).abs()[:, None] * p * (2 * ezm[:, None] + 2.0 ** -19 + 4 * E)
           + gl.abs()[:, None] * onehot * 4 * E)
    edu = edu + eslope * ((gl + ge).abs()[:, None] * p + gl.abs()[:, None] * onehot)
    ru = pair if pair else u
    edu = edu + ru * du.abs()
    if dtype != torch.bfloat16:  # fp16 below its normal range: scaled to 2^13
        top = torch.stack([(gl + ge).abs().max(), gl.abs().max()]).max()
        edu = edu + top * 2.0 ** -38
    dx, dw = scale * (du @ w), scale * (du.T @ x)
    bx = abs(scale) * (edu @ w.abs() + ((v + 4) * E + pair) * (du.abs() @ w.abs())) + u * dx.abs()
    bw = abs(scale) * (edu.T @ x.abs() + ((n + 4) * E + pair) * (du.abs().T @ x.abs())) \
        + u * dw.abs()
    bx = bx + abs(scale) * aw * du.abs().sum(1)[:, None]
    bw = bw + abs(scale) * ax * du.abs().sum(0)[:, None]
    # results below the type's normal range
    tiny = torch.finfo(dtype).tiny
    return (rows, lse, dx, dw), (b_row, b_lse, bx + tiny, bw + tiny)


def close(got, want, bound, what):
    off = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    off = off.detach()
    assert float(off.max()) <= 0, (what, float(off.max()), float(bound.max()))


def check(x, w, t, scale=1.0, cap=0.0, reduction="mean", lse_weight=0.0, seed=7):
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, lse = ra.linear_cross_entropy(xl, wl, t, scale=scale, softcap=cap, reduction=reduction)
    n = x.shape[0]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    count = int((t != IGN).sum())
    if reduction == "none":
        up = torch.randn(n, generator=gen, device="cuda")
        gl = up.double()
    else:
        up = torch.full((), 1.5, device="cuda")
        gl = torch.full((n,), 1.5 / (count if reduction == "mean" else 1), device="cuda").double()
    ge = torch.randn(n, generator=gen, device="cuda") * lse_weight
    outs, ups = [loss], [up]
    if lse_weight:
        outs, ups = outs + [lse], ups + [ge]
    dx, dw = torch.autograd.grad(outs, [xl, wl], ups)
    (rows, l64, dx64, dw64), (b_row, b_lse, bx, bw) = exact(x, w, t, scale, cap, gl, ge.double())
    close(lse, l64, b_lse, "lse")
    if reduction == "none":
        close(loss, rows, b_row, "loss")
    else:
        div = count if reduction == "mean" else 1
        close(loss, rows.sum() / div, b_row.sum() / div + 2 * E * rows.sum().abs() / div, "loss")
    close(dx, dx64, bx, "dx")
    close(dw, dw64, bw, "dw")
    assert loss.dtype == lse.dtype == torch.float32
    assert dx.dtype == x.dtype and dw.dtype == w.dtype


SIZES = [(1, 1, 1), (1, 2, 3), (2, 33, 8), (5, 257, 100), (127, 128, 16), (128, 1000, 128),
         (129, 255, 65), (300, 513, 264), (2049, 3, 8), (7, 5000, 72), (1000, 1531, 130)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", SIZES)
def test_sizes(n, v, d, dtype, cuda_device):
    check(*make(n, v, d, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 8, 9])
@pytest.mark.parametrize("v,d", [(3, 8), (1000, 264), (2049, 1024), (70, 2048), (70, 2056)])
def test_few_rows(n, v, d, dtype, cuda_device):
    x, w, t = make(n, v, d, dtype, seed=n + d)
    check(x, w, t, lse_weight=0.5)
    if n > 2:
        t[1] = v  # outside the table
        t[2] = IGN
        loss, lse = ra.linear_cross_entropy(x, w, t, reduction="none", softcap=3.0)
        assert torch.isnan(loss[1]) and loss[2] == 0 and torch.isfinite(lse).all()
    t[:] = torch.arange(n, device="cuda") % v
    check(x, w, t, reduction="none", cap=4.0, scale=2.0)
    x[-1, 0] = math.nan
    loss, lse = ra.linear_cross_entropy(x, w, t, reduction="none")
    assert torch.isnan(loss[-1]) and torch.isfinite(loss[:-1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("cap,scale", [(0.0, 1.7), (5.0, 1.0), (30.0, -2.0)])
def test_cap_scale_reduction(dtype, reduction, cap, scale, cuda_device):
    check(*make(190, 700, 96, dtype, seed=3), scale=scale, cap=cap, reduction=reduction,
          lse_weight=0.3)


def test_several_pieces_and_passes(cuda_device):
    """du of more than one piece of the vocabulary; more rows than one
    forward pass takes."""
    check(*make(16500, 17000, 16, torch.bfloat16, seed=5))
    check(*make(33000, 300, 24, torch.float16, seed=6))


def test_long_table_few_rows(cuda_device):
    """dx of one tile over a long K: sliced and joined."""
    check(*make(3, 60001, 40, torch.float32, seed=8))
    check(*make(40000, 5, 40, torch.bfloat16, seed=9))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype, cuda_device):
    x, w, t = make(60, 90, 48, dtype, seed=11)
    big = torch.zeros(60, 101, dtype=dtype, device="cuda")
    odd = big[:, 3:51]
    odd.copy_(x)
    cols = w.t().contiguous().t()
    check(odd, cols, t)
    check(x[:1].expand(60, 48), w, t)  # one row for all: stride 0
    every_other = torch.zeros(180, 48, dtype=dtype, device="cuda")[::2]
    every_other.copy_(w)
    check(x, every_other, t[:60].to(torch.int32))


def test_scales_of_fp32(cuda_device):
    """Tensors far from 1, and rows far apart, keep the pairs' precision."""
    x, w, t = make(200, 400, 64, torch.float32, seed=12)
    check(x * 2.0 ** 60, w * 2.0 ** -60, t)
    check(x * 2.0 ** -60, w, t, scale=2.0 ** 60)


def test_large_logits(cuda_device):
    """Probabilities of 0 and 1: no overflow, the other rows untouched."""
    x, w, t = make(150, 300, 32, torch.bfloat16, seed=13, spread=60.0)
    check(x, w, t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_labels(dtype, cuda_device):
    x, w, t = make(20, 30, 16, dtype)
    t[:] = IGN
    loss, lse = ra.linear_cross_entropy(x.requires_grad_(True), w.requires_grad_(True), t)
    assert torch.isnan(loss)  # as a mean of nothing
    loss, lse = ra.linear_cross_entropy(x, w, t, reduction="sum")
    assert float(loss.detach()) == 0.0
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert not dx.any() and not dw.any()


def test_no_rows(cuda_device):
    w = torch.randn(9, 8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.long, device="cuda")
    for reduction, want in (("mean", math.nan), ("sum", 0.0)):
        loss, lse = ra.linear_cross_entropy(x, w, t, reduction=reduction)
        assert lse.shape == (0,)
        got = float(loss.detach())
        assert math.isnan(got) if math.isnan(want) else got == want
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert dx.shape == (0, 8) and not dw.any()
    loss, _ = ra.linear_cross_entropy(x, w, t, reduction="none")
    assert loss.shape == (0,)


def test_target_outside_the_table(cuda_device):
    x, w, t = make(40, 50, 24, torch.float32)
    t[3], t[17] = 50, -5
    loss, lse = ra.linear_cross_entropy(x, w, t, reduction="none")
    bad = torch.isnan(loss)
    assert bad[3] and bad[17] and int(bad.sum()) == 2
    assert torch.isfinite(lse).all()
    loss, _ = ra.linear_cross_entropy(x.requires_grad_(True), w, t)
    assert torch.isnan(loss)
    dx, = torch.autograd.grad(loss, [x])
    assert torch.isnan(dx[3]).all() and torch.isnan(dx[17]).all()


def test_not_a_number_stays_in_its_row(cuda_device):
    x, w, t = make(300, 200, 32, torch.float32, seed=4, ignore=0)
    clean, lse0 = ra.linear_cross_entropy(x, w, t, reduction="none")
    y = x.clone()
    y[5, 3] = math.nan
    y[140, 0] = math.inf
    loss, lse = ra.linear_cross_entropy(y, w, t, reduction="none")
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[5] = keep[140] = False
    assert torch.isnan(loss[5]) and torch.isnan(lse[5]) and not torch.isfinite(loss[140])
    assert torch.equal(loss[keep], clean[keep]) and torch.equal(lse[keep], lse0[keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_only_one_gradient(dtype, cuda_device):
    x, w, t = make(70, 80, 32, dtype)
    both = torch.autograd.grad(
        ra.linear_cross_entropy(x.requires_grad_(True), w.requires_grad_(True), t)[0], [x, w])
    x2, w2 = x.detach(), w.detach()
    dx, = torch.autograd.grad(ra.linear_cross_entropy(x, w2, t)[0], [x])
    dw, = torch.autograd.grad(ra.linear_cross_entropy(x2, w, t)[0], [w])
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeatable(dtype, cuda_device):
    x, w, t = make(3000, 2500, 128, dtype, seed=21)
    x.requires_grad_(True), w.requires_grad_(True)
    runs = []
    for _ in range(3):
        loss, lse = ra.linear_cross_entropy(x, w, t)
        runs.append((loss, lse, *torch.autograd.grad(loss, [x, w])))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_differences(cuda_device):
    """Directional derivatives against central differences of the loss: the
    loss is smooth on the scale of h |d|, so the difference is off by about
    h^2 of the third derivative (< 1e-3 of the slope here) and by the loss's
    own rounding, 2^-22 |loss| / h."""
    x, w, t = make(100, 220, 48, torch.float32, seed=30)
    x.requires_grad_(True), w.requires_grad_(True)

    def f(a, b):
        loss, lse = ra.linear_cross_entropy(a, b, t, softcap=8.0)
        return loss + 1e-2 * (lse ** 2).mean()

    loss = f(x, w)
    grads = torch.autograd.grad(loss, [x, w])
    g = torch.Generator(device="cuda").manual_seed(1)
    h = 2.0 ** -7
    for i, g64 in enumerate(grads):
        d = torch.randn(g64.shape, generator=g, device="cuda")
        d = d / d.norm()
        slope = float((g64.double() * d.double()).sum())
        move = [torch.zeros_like(x), torch.zeros_like(w)]
        move[i] = d * h
        with torch.no_grad():
            up = f(x + move[0], w + move[1])
            down = f(x - move[0], w - move[1])
        got = float((up.double() - down.double()) / (2 * h))
        assert abs(got - slope) <= 2e-3 * float(g64.norm()) + 2.0 ** -22 * abs(float(loss)) / h


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_other_stream_and_capture(dtype, cuda_device):
    x, w, t = make(500, 900, 64, dtype, seed=40)
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        loss, lse = ra.linear_cross_entropy(x, w, t)
        return (loss.detach(), lse.detach(), *torch.autograd.grad(loss, [x, w]))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():  # new values in the same places
        x2, w2, t2 = make(500, 900, 64, dtype, seed=41)
        x.copy_(x2), w.copy_(w2), t.copy_(t2)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(1, 1, 8), (3, 15, 24), (5, 17, 56), (8, 4097, 72),
                                   (6, 300, 128), (7, 129, 136), (8, 20000, 64)])
def test_few_rows_of_a_wider_table(n, v, d, dtype, cuda_device):
    """Tables and rows as slices, NaN in what lies between; every row's target
    in turn at the ends of the table; replayed from a graph."""
    x, w, t = make(n, v, d, dtype, seed=v, ignore=0)
    wide = torch.full((v, d + 8), math.nan, dtype=dtype, device="cuda")
    wide[:, :d] = w
    rows = torch.full((n, d + 16), math.nan, dtype=dtype, device="cuda")
    rows[:, 8:8 + d] = x
    t[-1], t[0] = 0, v - 1
    w, x = wide[:, :d], rows[:, 8:8 + d]
    check(x, w, t, reduction="none", lse_weight=0.3)
    step = lambda: ra.linear_cross_entropy(x, w, t, softcap=3.0, reduction="none")  # noqa: E731
    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.copy_(make(n, v, d, dtype, seed=v + 1)[0])
    graph.replay()
    torch.cuda.synchronize()
    got = step()
    assert all(torch.equal(a, b) for a, b in zip(held, got))
    assert not torch.equal(got[1], want[1]) or v == 1
    (r64, l64, _, _), (br, bl, _, _) = exact(x, w, t, 1.0, 3.0, torch.ones(n, device="cuda"),
                                             torch.zeros(n, device="cuda"))
    close(got[0], r64, br, "loss")
    close(got[1], l64, bl, "lse")


def test_launches_are_counted(cuda_device):
    x, w, t = make(50, 60, 32, torch.bfloat16)
    before = _lib.launch_count()
    ra.linear_cross_entropy(x, w, t)
    assert _lib.launch_count() == before + 2  # the product, the joined rows
