"""linear_cross_entropy with upstream gradients of each row: what fp16's smallest
step costs an element of dx or dw, at the sizes where nothing else hides it (few
rows, most probabilities far below fp16's range)."""
import pytest
import torch

from test_gpu_cross_entropy import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v,d", [(1, 71, 7), (2, 223, 22), (2, 2899, 49), (4, 136, 216),
                                   (4, 4353, 40), (2, 2670, 8), (3, 2446, 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_smallest_elements(n, v, d, dtype, cuda_device):
    for seed in range(12):
        x, w, t = make(n, v, d, dtype, seed=seed, ignore=0.0)
        for reduction, lse in (("none", 0.0), ("none", 0.5), ("sum", 0.5)):
            check(x, w, t, scale=-2.0, reduction=reduction, lse_weight=lse, seed=seed)
