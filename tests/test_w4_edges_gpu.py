"""4-bit products at the largest activations that their documentation allows."""
import pytest
import torch

from prism_infer_b200 import capi
from test_w4_gpu import DEV, check_linear, gen_of, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 3, 16, 40, 300])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_at_the_largest_activations(M, G, zeros):
    """2^113 in every place: a group's sum comes to 143 * 128 * 2^113 < 2^128 before its scale."""
    w = weights(M, (), 264, 1024, G, zeros)
    x = torch.full((M, 1024), 2.0 ** 113, device=DEV, dtype=torch.bfloat16)
    x[M // 2] *= torch.randint(0, 2, (1024,), generator=gen_of(M), device=DEV) * 2 - 1
    y = capi.linear_w4(x, w)
    assert y.isfinite().all()
    check_linear(x, w, y)
