"""Where a failing kernel's status goes when the caller gives no error word, without a GPU."""
import ctypes

import pytest
import torch

from prism_infer_b200 import build, capi
from prism_infer_b200.quant import quantize_w4

BF16 = torch.bfloat16
WORD = 0x1230


@pytest.fixture
def calls(monkeypatch):
    """Arguments of every launch, on tensors that stand for a GPU's."""
    build.build()
    capi.load()
    made = []
    monkeypatch.setattr(capi, "_one_device", lambda first, *others: 0)
    monkeypatch.setattr(capi, "device_error_word", lambda index: WORD)
    monkeypatch.setattr(capi, "_launch", lambda index, what, fn, *args: made.append(args))
    return made


def test_products_without_a_word_use_the_devices(calls):
    x = torch.zeros(4, 64, dtype=BF16)
    capi.linear_w4(x, quantize_w4(torch.randn(16, 64), 32))
    gu = quantize_w4(torch.randn(2, 64, 64), 32, gate_up=True)
    dn = quantize_w4(torch.randn(2, 64, 32), 32)
    seg = torch.tensor([0, 1, 4], dtype=torch.int32)
    capi.expert_swiglu_w4(x, seg, gu, dn)
    assert [c[-1] for c in calls] == [WORD, WORD]
    own = torch.zeros(1, dtype=torch.int32)
    capi.expert_swiglu_w4(x, seg, gu, dn, device_error=own)
    assert calls[-1][-1] == own.data_ptr()


def test_word_of_a_device_is_looked_up_once_and_refuses_null():
    build.build()
    lib = capi.load()
    assert lib.prism_moe_device_error_word(None) == capi.ERR_ARG
    assert "prism_moe_device_error_word" in capi._SIGNATURES
    word = ctypes.c_void_p()
    if not torch.cuda.is_available():
        assert lib.prism_moe_device_error_word(ctypes.byref(word)) != capi.OK and not word.value
