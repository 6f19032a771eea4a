"""Operands of strides that the kernels do not read as they are."""
import pytest
import torch

import rapidalign_b200 as ra
from test_gpu_attention import check as check_attention
from test_gpu_attention import close, exact, make, ptr
from test_gpu_cross_entropy import check as check_cross_entropy

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 64])
def test_tables_and_inputs_of_one_row(d, dtype, cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(d)
    column = torch.randn(d, 1, generator=gen, device="cuda").to(dtype).t()  # (1, d)
    x = torch.randn(50, d, generator=gen, device="cuda").to(dtype)
    check_cross_entropy(x, column, torch.zeros(50, dtype=torch.long, device="cuda"))
    check_cross_entropy(column, x, torch.tensor([7], device="cuda"))
    check_cross_entropy(x[:3], column, torch.zeros(3, dtype=torch.long, device="cuda"),
                        reduction="none", lse_weight=0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 20])
def test_slices_of_a_projection(dim, dtype, cuda_device):
    """Unaligned slices of a fused projection, forward and backward, by the bounds."""
    n = [31, 140]
    rows, H = sum(n), 4
    d = make(n, n, H, H, dim, dtype, 2, seed=dim)
    fused = torch.zeros(rows, 3 * H * dim + 5, dtype=dtype, device="cuda")
    for i, name in enumerate("qkv"):
        view = fused[:, 2 + i * H * dim:2 + (i + 1) * H * dim].view(rows, H, dim)
        view.copy_(d[name])
        d[name] = view
    check_attention(d, n, n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_single_queries_and_heads_of_any_stride(dtype, cuda_device):
    nq, nk = [1], [700]
    d = make(nq, nk, 1, 1, 32, dtype, 2, seed=3)
    d["q"] = torch.randn(64, device="cuda").to(dtype).as_strided((1, 1, 32), (3, 5, 1))
    (o64, bo), _ = exact(d, nq, nk, 32 ** -0.5, 0.0)
    o = ra.pyg_kernel_attention(d["q"], d["k"], d["v"], q_ptr=ptr(nq), k_ptr=ptr(nk),
                                q_pos=d["q_pos"], k_pos=d["k_pos"], sigma=d["sigma"])
    close(o, o64, bo, "out")
