"""The scored router under expert parallelism as operators, traced without a GPU."""
import pytest
import torch

from prism_infer_b200 import ops  # noqa: F401
from prism_infer_b200.engine.parallel import set_expert_parallel_size
from prism_infer_b200.engine.parallel.expert_parallel import ExpertParallelMoE
from prism_infer_b200.layers.layernorm import RMSNorm
from prism_infer_b200.layers.moe import MoE

H, I, E, K = 128, 64, 8, 2


class Step(torch.nn.Module):
    def __init__(self, fuse):
        super().__init__()
        set_expert_parallel_size(1)
        self.moe = MoE(H, I, E, K, scoring="sigmoid", num_groups=4, topk_groups=2)
        # what rank 0 of two builds
        self.moe.ep_size, self.moe.experts = 2, None
        self.moe.ep_moe = ExpertParallelMoE(H, I, E, 2, 0, transport="p2p")
        self.norm = RMSNorm(H) if fuse else None

    def forward(self, x, residual):
        return self.moe(x, residual=residual, norm=self.norm) if self.norm is not None else self.moe(x)


@pytest.mark.parametrize("fuse", [False, True])
def test_scored_expert_parallel_step_is_one_graph(fuse):
    step = Step(fuse).to("meta", torch.bfloat16)
    x = torch.empty(2, 5, H, device="meta", dtype=torch.bfloat16)
    out = step(x, x)
    assert all(o.shape == x.shape and o.dtype == x.dtype for o in (out if fuse else (out,)))
    called = [str(n.target) for n in torch.export.export(step, (x, x)).graph.nodes
              if n.op == "call_function"]
    assert "prism_moe.route_scored.default" in called
    assert f"prism_moe.ep_forward_routed{'_norm' if fuse else ''}.default" in called


def test_choices_that_do_not_fit_the_step():
    """The step's kernels read [T, k] int64 ids and [T, E] logits, whatever they are given."""
    bank = ExpertParallelMoE(H, I, E, 2, 0, transport="p2p").to(torch.bfloat16)
    bf16 = torch.bfloat16
    x = torch.zeros(5, H, dtype=bf16)
    ids, w = torch.zeros(5, K, dtype=torch.int64), torch.zeros(5, K, dtype=bf16)
    choice = dict(topk_ids=ids, topk_weights=w)
    for bad in (dict(choice, topk_ids=ids.int()), dict(choice, topk_ids=ids[:4]),
                dict(choice, topk_weights=w[:, :1]), dict(choice, topk_weights=None),
                dict(choice, topk_ids=ids[0]), dict(choice, top_k=K + 1),
                dict(choice, topk_ids=ids.to("meta")),
                dict(router_logits=torch.zeros(5, E, dtype=bf16)), dict(top_k=K),
                dict(router_logits=torch.zeros(5, E), top_k=K),
                dict(router_logits=torch.zeros(5, E - 1, dtype=bf16), top_k=K)):
        with pytest.raises(RuntimeError, match="ep_forward"):
            bank.forward_p2p(x, **bad)
    for bad in (x.float(), x[:, :-1], x[0]):
        with pytest.raises(RuntimeError, match="ep_forward: x must be"):
            bank.forward_p2p(bad, **choice)
    with pytest.raises(RuntimeError, match="CUDA"):
        bank.forward_p2p(x, **choice)


def test_a_bank_that_is_not_there():
    x = torch.zeros(2, H, dtype=torch.bfloat16)
    ids, w = torch.zeros(2, K, dtype=torch.int64), torch.zeros(2, K, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="unknown expert-parallel bank"):
        torch.ops.prism_moe.ep_forward_routed(x, ids, w, x, x, -1)
