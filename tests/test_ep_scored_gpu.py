"""The scored router's choice through the expert-parallel step as an operator, in a group of one."""
import pytest
import torch

from prism_infer_b200 import ops  # noqa: F401
from prism_infer_b200.engine.parallel import set_expert_parallel_size
from prism_infer_b200.engine.parallel.expert_parallel import ExpertParallelMoE
from prism_infer_b200.layers.layernorm import RMSNorm
from prism_infer_b200.layers.moe import MoE

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, I, E, K = 256, 128, 32, 4


@pytest.mark.parametrize("T", [1, 70, 300])
def test_the_module_takes_the_step_and_fuses_the_norm(T):
    set_expert_parallel_size(1)
    torch.manual_seed(T)
    moe = MoE(H, I, E, K, scoring="sigmoid", score_bias=True, num_groups=8, topk_groups=3,
              group_score="top2", routed_scale=2.5)
    bank = ExpertParallelMoE(H, I, E, 1, 0, transport="p2p")
    norm = RMSNorm(H)
    with torch.no_grad():
        moe.gate.weight.normal_(std=H ** -0.5)
        moe.gate.e_score_correction_bias.normal_(std=0.1)
        bank.w_gate_up.copy_(moe.w_gate_up.normal_(std=H ** -0.5))
        bank.w_down.copy_(moe.w_down.normal_(std=I ** -0.5))
        norm.weight.normal_()
    moe, bank, norm = (m.to(DEV, torch.bfloat16) for m in (moe, bank, norm))
    x, res = torch.randn(2, T, H, device=DEV).to(torch.bfloat16)
    want, (want_n, want_res) = moe(x), moe(x, residual=res, norm=norm)
    moe.ep_size, moe.ep_moe, moe.experts = 2, bank, None   # the path of a rank, on a group of one
    try:
        out = moe(x)
        got_n, got_res = moe(x, residual=res, norm=norm)
        bank.check_device_error()
        assert torch.equal(out, want)
        assert torch.equal(got_n, want_n) and torch.equal(got_res, want_res)
        with pytest.raises(RuntimeError, match="not the bank's"):
            _, ids, w = moe.route(x)
            torch.ops.prism_moe.ep_forward_routed(x, ids, w, bank.w_gate_up.clone(), bank.w_down,
                                                  bank.op_id)
    finally:
        bank.release()
