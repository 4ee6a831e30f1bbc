"""What the block entry points refuse before anything is launched, without a GPU."""
import pytest
import torch

from prism_infer_b200 import capi
from prism_infer_b200.quant import quantize_w4

H, I, E, K, T = 64, 32, 4, 2, 5
BF16 = torch.bfloat16


def call_args(w4):
    ids = torch.zeros(T, K, dtype=torch.int64)
    if w4:
        weights = (quantize_w4(torch.randn(E, 2 * I, H), 32, gate_up=True),
                   quantize_w4(torch.randn(E, H, I), 32))
    else:
        weights = torch.randn(E, 2 * I, H).to(BF16), torch.randn(E, H, I).to(BF16)
    return torch.randn(T, H).to(BF16), ids, torch.ones(T, K, dtype=BF16), *weights


def epilogue_of(residual, weight=None):
    """What norm_epilogue gives for tensors on a GPU."""
    epi = capi.NormEpilogue(0, 0, 1e-6, 0)
    epi.held = (residual, torch.ones(H, dtype=BF16) if weight is None else weight, residual)
    return epi


WRONG = [torch.empty(T - 1, H, dtype=BF16), torch.empty(T, H // 2, dtype=BF16),
         torch.empty(T * H, dtype=BF16), torch.empty(T, H)]


@pytest.mark.parametrize("w4", [False, True])
@pytest.mark.parametrize("wrong", WRONG, ids=lambda t: f"{tuple(t.shape)}{t.dtype}")
def test_outputs_unlike_the_hidden_states(w4, wrong):
    with pytest.raises(RuntimeError, match="out must be"):
        capi.block_forward_routed(*call_args(w4), out=wrong)
    with pytest.raises(RuntimeError, match="epilogue's residual must be"):
        capi.block_forward_routed(*call_args(w4), epilogue=epilogue_of(wrong))


def test_norm_epilogue_of_tensors_that_do_not_match():
    res, w = torch.empty(T, H, dtype=BF16), torch.empty(H, dtype=BF16)
    for bad in ((res, w[:-1], res), (res, w, res[:-1]), (res[0], w, res[0]), (res, w[None], res),
                (res[:, :-1], w, res)):
        with pytest.raises(RuntimeError, match="must be"):
            capi.norm_epilogue(bad[0], bad[1], 1e-6, bad[2])
    for bad in ((res, w.float(), res), (res.float(), w, res), (res, w, res.float())):
        with pytest.raises(RuntimeError, match="dtype"):
            capi.norm_epilogue(bad[0], bad[1], 1e-6, bad[2])
    with pytest.raises(RuntimeError, match="CUDA"):
        capi.norm_epilogue(res, w, 1e-6, res)
