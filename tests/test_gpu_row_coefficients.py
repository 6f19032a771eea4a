"""linear_cross_entropy with upstream gradients of the rows orders of magnitude
apart: dx of a row counts by the row's own, dw by all."""
import math

import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_cross_entropy import IGN, close, exact, make

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def run(x, w, t, gl, ge, cap=0.0, scale=1.0):
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, lse = ra.linear_cross_entropy(xl, wl, t, reduction="none", softcap=cap, scale=scale)
    outs = [(o, g) for o, g in ((loss, gl), (lse, ge)) if g is not None]
    return torch.autograd.grad([o for o, _ in outs], [xl, wl], [g for _, g in outs])


def check(x, w, t, gl, ge, cap=0.0, groups=4, scale=1.0):
    """Rows r, r + groups, ... are of one size."""
    dx, dw = run(x, w, t, gl, ge, cap, scale)
    zero = torch.zeros(x.shape[0], device="cuda").double()
    a, b = (zero if g is None else g.double() for g in (gl, ge))
    for r in range(groups):
        s = slice(r, None, groups)
        (_, _, want, _), (_, _, bound, _) = exact(x[s], w, t[s], scale, cap, a[s], b[s])
        close(dx[s], want, bound, f"dx of rows of size {r}")
    (_, _, _, want), (_, _, _, bound) = exact(x, w, t, scale, cap, a, b)
    close(dw, want, bound, "dw")


def sizes(n, low):
    f = torch.tensor([1.0, low ** 0.5, low, 1.0], device="cuda")
    return f.repeat(n // 4 + 1)[:n]


# fp16: as far down as its results reach
LOW = {torch.float32: 1e-8, torch.bfloat16: 1e-8, torch.float16: 1e-4}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(200, 700, 96), (7, 900, 64), (130, 1000, 36), (600, 20000, 264)])
@pytest.mark.parametrize("cap", [0.0, 6.0])
def test_losses_weighted_apart(n, v, d, cap, dtype, cuda_device):
    x, w, t = make(n, v, d, dtype, seed=n)
    g = torch.randn(n, device="cuda") * sizes(n, LOW[dtype])
    check(x, w, t, g, None, cap, scale=1.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_rows_with_a_gradient_of_lse(dtype, cuda_device):
    n = 240
    x, w, t = make(n, 500, 64, dtype, seed=2, ignore=0.0)
    t[1::4] = IGN
    g = torch.randn(n, device="cuda")
    check(x, w, t, g, torch.randn(n, device="cuda") * sizes(n, LOW[dtype]))
    check(x, w, t, None, torch.randn(n, device="cuda") * sizes(n, LOW[dtype]))
    check(x, w, t, g * sizes(n, LOW[dtype]), torch.zeros(n, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_some_rows_without_any(dtype, cuda_device):
    """Coefficients of exactly 0; a mean with a z-loss of few rows."""
    x, w, t = make(100, 300, 40, dtype, seed=3)
    g = torch.zeros(100, device="cuda")
    g[7::9] = 1e-3
    check(x, w, t, g, None, groups=1)
    dx, dw = run(x, w, t, torch.zeros(100, device="cuda"), None)
    assert not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_a_number_stays_in_its_row(dtype, cuda_device):
    x, w, t = make(90, 200, 32, dtype, seed=4, ignore=0.0)
    g = torch.randn(90, device="cuda") * sizes(90, 1e-4)
    want, _ = run(x, w, t, g, None)
    t[5] = 200  # outside the table
    g[50] = math.inf
    dx, _ = run(x, w, t, g, None)
    keep = torch.ones(90, dtype=torch.bool, device="cuda")
    keep[5] = keep[50] = False
    assert not torch.isfinite(dx[5]).any() and not torch.isfinite(dx[50]).all()
    assert torch.equal(dx[keep], want[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_row_of_dx_is_its_own(dtype, cuda_device):
    """Bitwise the same next to rows of any size."""
    x, w, t = make(140, 800, 64, dtype, seed=5, ignore=0.0)
    g = torch.randn(140, device="cuda")
    a, _ = run(x, w, t, g, None)
    big = g.clone()
    big[1::2] *= 2.0 ** 12
    b, _ = run(x, w, t, big, None)
    assert torch.equal(a[::2], b[::2])
