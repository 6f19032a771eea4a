"""Memory of the softmax operators on the device, and the forward of the cross
entropy in several passes over the rows."""
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


def peak_of(call):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_scoring_a_few_rows(offset, dtype, cuda_device):
    n, v, d = 5, 20000, 512
    x, w, t = make(n, v, d, dtype, seed=1)
    wide = torch.zeros(v, d + 8, dtype=dtype, device="cuda")
    table = wide[:, offset:offset + d].copy_(w)
    with torch.no_grad():
        peak, (loss, lse) = peak_of(lambda: ra.linear_cross_entropy(x, table, t, reduction="none"))
    if offset == 0:  # (an unaligned table is copied)
        assert peak < 4 << 20
    zero = torch.zeros(n, device="cuda")
    (r64, l64, _, _), (br, bl, _, _) = exact(x, w, t, 1.0, 0.0, zero, zero)
    close(loss, r64, br, "loss")
    close(lse, l64, bl, "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_pooling(offset, dtype, cuda_device):
    nq, nk, H, D = [1, 1], [60000, 300], 2, 64
    d = make_attention(nq, nk, H, H, D, dtype, 2, seed=2)
    for n in "kv":
        wide = torch.zeros(sum(nk), H, D + 8, dtype=dtype, device="cuda")
        d[n] = wide[..., offset:offset + D].copy_(d[n])
    seg = ra.attention_segments(ptr(nq), ptr(nk))
    peak, o = peak_of(lambda: ra.pyg_kernel_attention(
        d["q"], d["k"], d["v"], segments=seg, q_pos=d["q_pos"], k_pos=d["k_pos"],
        sigma=d["sigma"]))
    if offset == 0:
        assert peak < 4 << 20
    (o64, bo), _ = exact_attention(d, nq, nk, D ** -0.5, 0.0)
    close_attention(o, o64, bo, "out")


@pytest.mark.parametrize("dtype", DTYPES)
def test_passes_over_the_rows(dtype, cuda_device):
    """A long table: the partials of all rows would pass their share of memory.
    Rows are what they are in calls of their own (both halves hold the largest
    element, which scales fp32 inputs; the tiles are as wide)."""
    n, v, d = 20480, 70001, 16
    x, w, t = make(n, v, d, dtype, seed=3)
    x[0, 0] = x[n // 2, 0] = 6.0
    peak, (loss, lse) = peak_of(lambda: ra.linear_cross_entropy(x, w, t, reduction="none"))
    assert peak < 200 << 20
    h = n // 2
    for s in (slice(None, h), slice(h, None)):
        a, b = ra.linear_cross_entropy(x[s], w, t[s], reduction="none")
        assert torch.equal(loss[s], a) and torch.equal(lse[s], b)
    mean, _ = ra.linear_cross_entropy(x, w, t)
    count = int((t != -100).sum())
    assert abs(float(mean) - float(loss.double().sum()) / count) <= 2.0 ** -22 * float(mean)
    rows = torch.tensor([0, 1, 8191, 8192, 15000, n - 1], device="cuda")
    zero = torch.zeros(6, device="cuda")
    (r64, l64, _, _), (br, bl, _, _) = exact(x[rows], w, t[rows], 1.0, 0.0, zero, zero)
    if dtype == torch.float32:  # the halves' scale is all rows'
        extra = 2.0 ** -38 * x.abs().max().double() * w.double().abs().sum(1).max()
        br, bl = br + 2 * extra, bl + extra
    close(loss[rows], r64, br, "loss")
    close(lse[rows], l64, bl, "lse")
