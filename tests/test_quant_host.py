"""4-bit weights: values that have no 4-bit form with a finite scale, without a GPU."""
import pytest
import torch

from prism_infer_b200.quant import dequantize_w4, pack_w4, quantize_w4

BIG = torch.finfo(torch.bfloat16).max


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_weights_that_are_not_finite_are_refused(symmetric, value):
    w = torch.randn(2, 16, 64)
    w[1, 5, 40] = value
    with pytest.raises(RuntimeError, match="finite"):
        quantize_w4(w, 32, symmetric=symmetric)


def test_scales_that_are_not_finite_in_bf16_are_refused():
    codes = torch.randint(0, 16, (16, 64))
    for value in (float("inf"), float("nan"), 3.4e38):      # the last rounds to infinity
        scales = torch.ones(16, 2)
        scales[7, 1] = value
        with pytest.raises(RuntimeError, match="finite"):
            pack_w4(codes, scales, group_size=32)
    w = torch.zeros(16, 64)
    w[0, 0], w[0, 1] = BIG, -BIG                            # their difference is past fp32
    with pytest.raises(RuntimeError, match="finite"):
        quantize_w4(w, 32, symmetric=False)
    back = dequantize_w4(quantize_w4(w, 32))                # 2 BIG / 14 is not
    assert ((back - w).abs() <= BIG * 2.0 ** -8).all()
