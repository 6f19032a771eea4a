"""Rows of small and of large capped scores side by side in one warp: the two
forms of tanh, whose choice is the warp's, give each row what it has alone."""
import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_attention import check as check_attention
from test_gpu_attention import make as make_attention
from test_gpu_cross_entropy import check as check_cross_entropy
from test_gpu_cross_entropy import make as make_cross_entropy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [24, 64, 128])
def test_attention(dim, dtype, cuda_device):
    nq, nk = [150, 40], [200, 70]
    d = make_attention(nq, nk, 2, 2, dim, dtype, 2, seed=dim)
    small = torch.arange(sum(nq), device="cuda") % 3 != 0
    d["q"][small] *= 2.0 ** -6
    o, grads = check_attention(d, nq, nk, cap=4.0)
    # alone: every row small, then every row large; q's rows are their own
    for part in (small, ~small):
        alone = {n: t.clone() for n, t in d.items()}
        other = torch.nonzero(part)[:, 0][0]
        alone["q"][~part] = d["q"][other]
        seg = ra.attention_segments(*(torch.tensor([0, *n], device="cuda").cumsum(0)
                                      for n in (nq, nk)))
        got = ra.pyg_kernel_attention(alone["q"], alone["k"], alone["v"], segments=seg,
                                      q_pos=alone["q_pos"], k_pos=alone["k_pos"],
                                      sigma=alone["sigma"], softcap=4.0)
        if dtype != torch.float32:  # (pairs: with a scale by the tensor's largest)
            with torch.no_grad():
                want = ra.pyg_kernel_attention(d["q"], d["k"], d["v"], segments=seg,
                                               q_pos=d["q_pos"], k_pos=d["k_pos"],
                                               sigma=d["sigma"], softcap=4.0)
            assert torch.equal(got[part], want[part])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(200, 700, 96), (5, 900, 64)])
def test_cross_entropy(n, v, d, dtype, cuda_device):
    x, w, t = make_cross_entropy(n, v, d, dtype, seed=n)
    x[::3] *= 2.0 ** -6
    check_cross_entropy(x, w, t, cap=3.0, reduction="none", lse_weight=0.5)
