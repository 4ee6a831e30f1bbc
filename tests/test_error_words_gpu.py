"""Errors of calls that carry no error word of their own: captured steps, operators and modules."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from prism_infer_b200 import capi, ops  # noqa: F401
from prism_infer_b200.engine.parallel import set_expert_parallel_size
from prism_infer_b200.layers.mlp import Qwen3MLP
from prism_infer_b200.layers.moe import MoE
from prism_infer_b200.layers.w4 import W4Linear
from prism_infer_b200.quant import quantize_w4

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, I, E, K, T = 128, 64, 8, 2, 6


@pytest.fixture
def moe():
    set_expert_parallel_size(1)
    torch.manual_seed(0)
    moe = MoE(H, I, E, K, scoring="sigmoid")
    with torch.no_grad():
        for t in (moe.gate.weight, moe.w_gate_up, moe.w_down):
            t.normal_(std=0.1)
    return moe.to(DEV, torch.bfloat16).quantize_experts_(64)


def tokens():
    g = torch.Generator(device=DEV).manual_seed(1)
    return torch.randn(T, H, generator=g, device=DEV).to(torch.bfloat16)


def test_a_captured_block_reports_ids_of_no_expert(moe):
    x = tokens()
    _, ids, w = moe.route(x)
    gu, dn = moe.w4_gate_up.weight, moe.w4_down.weight
    want = capi.block_forward_routed(x, ids, w, gu, dn)
    static = ids.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = capi.block_forward_routed(x, static, w, gu, dn)
    graph.replay()
    moe.check_device_error()
    assert torch.equal(out, want)
    static[3, 1] = E
    graph.replay()
    with pytest.raises(RuntimeError):
        moe.check_device_error()
    moe.check_device_error()                 # reported once
    static[3, 1] = ids[3, 1]
    graph.replay()
    moe.check_device_error()
    assert torch.equal(out, want)


def test_operators_and_modules_report():
    x = tokens()
    gu = quantize_w4(torch.randn(2, 2 * I, H, device=DEV), 64, gate_up=True)
    dn = quantize_w4(torch.randn(2, H, I, device=DEV), 64)
    seg = torch.tensor([0, 2, T], dtype=torch.int32, device=DEV)
    lin = W4Linear.from_weight(torch.randn(16, H, device=DEV), 64)
    mlp = Qwen3MLP(H, I).to(DEV, torch.bfloat16)
    for p in mlp.parameters():
        p.data.normal_()
    for bad in ((0, 2), (-1, 1)):
        experts = torch.tensor(bad, dtype=torch.int32, device=DEV)
        torch.ops.prism_moe.expert_swiglu_w4(x, seg, gu.qweight, gu.scales, gu.zeros, dn.qweight,
                                             dn.scales, dn.zeros, I, 64, 64, experts)
        for module in (lin, mlp, mlp.quantize_(64) if bad[0] else mlp):
            with pytest.raises(RuntimeError):
                module.check_device_error()
            module.check_device_error()
            torch.ops.prism_moe.expert_swiglu_w4(x, seg, gu.qweight, gu.scales, gu.zeros,
                                                 dn.qweight, dn.scales, dn.zeros, I, 64, 64, experts)
        with pytest.raises(RuntimeError):
            capi.check_device_error()
    lin(x)
    lin.check_device_error()


FIRST = """
import sys
import torch
from prism_infer_b200 import capi
from prism_infer_b200.layers.w4 import W4Linear
from prism_infer_b200.layers.moe import MoE
x = torch.ones({T}, {H}, device="cuda", dtype=torch.bfloat16)
if {block}:
    step = MoE({H}, {I}, {E}, {K}, scoring="sigmoid")
    for t in (step.gate.weight, step.w_gate_up, step.w_down):
        t.data.normal_(std=0.1)
    step = step.to("cuda", torch.bfloat16).quantize_experts_(64)
    step.gate(x)
else:
    step = W4Linear.from_weight(torch.randn(16, {H}, device="cuda"), 64)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = step(x)
graph.replay()
step.check_device_error()
assert torch.equal(y, step(x)) and y.isfinite().all()
"""


@pytest.mark.parametrize("block", [False, True])
def test_a_processs_first_call_can_be_captured(block):
    """The word exists before any call: nothing is allocated for it while a graph is captured."""
    code = FIRST.format(T=T, H=H, I=I, E=E, K=K, block=block)
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parent.parent)
    assert run.returncode == 0, run.stderr[-2000:]
