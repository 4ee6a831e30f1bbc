"""What the block entry points refuse before anything is launched, without a GPU."""
import ctypes

import pytest
import torch

from prism_infer_b200 import build, capi
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


# ------------------------------------------------------------------------------ the C ABI

P = 1 << 20   # an aligned address that no refused call looks at


@pytest.fixture(scope="module")
def lib():
    build.build()
    return capi.load()


def block(lib, x=P, out=P, ws=P, res=3 * P, w=P, res_out=2 * P, dense=False, norm=True):
    q = ctypes.byref(capi.W4(P, P, None, 64))
    epi = capi.NormEpilogue(res, w, 1e-6, res_out)
    experts = (P, P, None, None) if dense else (None, None, q, q)
    return lib.prism_moe_block_forward_routed(x, P, P, capi.BF16, 2, 128, 64, 4, 2, *experts, out, ws,
                                              1 << 30, None, ctypes.byref(epi) if norm else None)


@pytest.mark.parametrize("dense", [False, True])
def test_buffers_that_are_not_16_byte_aligned(lib, dense):
    """A view that starts inside a row: the kernels read 16 bytes at a time."""
    for bad in (dict(x=P + 8), dict(x=P + 2), dict(out=P + 8), dict(ws=P + 4), dict(res=3 * P + 2),
                dict(w=P + 8), dict(res_out=2 * P + 4), dict(x=P + 8, norm=False)):
        assert block(lib, dense=dense, **bad) == capi.ERR_ARG, bad
        assert b"16-byte aligned" in lib.prism_moe_last_error()
    for bad in (dict(x=P + 8), dict(out=P + 2)):
        kw = dict(x=P, out=P) | bad
        assert lib.prism_moe_block_forward(kw["x"], P, capi.BF16, 2, 128, 64, 4, 2, 1, P, P, kw["out"],
                                           None, None, P, 1 << 30, None) == capi.ERR_ARG
        assert b"16-byte aligned" in lib.prism_moe_last_error()


@pytest.mark.parametrize("dense", [False, True])
def test_norm_epilogue_on_one_buffer_twice(lib, dense):
    """The residual is read again for the second pass, after the outputs have been written."""
    for bad in (dict(out=P, res=P), dict(res=P, res_out=P, out=3 * P), dict(out=P, res_out=P)):
        assert block(lib, dense=dense, **bad) == capi.ERR_ARG, bad
        assert b"three buffers" in lib.prism_moe_last_error()
