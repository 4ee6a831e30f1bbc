"""The scored router and 4-bit experts together, as a model runs them: the routed block, the modules
on it, its graphs and streams. The oracle is 64-bit arithmetic on the choice that the router's own
tests pin; bounds are those of the 4-bit products (tests/test_w4_gpu.py) and the combine's: each of
the k products and the sum are rounded to bf16 (2^-8 each, of the terms and of the result)."""
import pytest
import torch

from oracle.scored_routing import route_scored_ref
from prism_infer_b200 import capi, ops  # noqa: F401
from prism_infer_b200.engine.parallel import set_expert_parallel_size
from prism_infer_b200.engine.parallel.expert_parallel import ExpertParallelMoE
from prism_infer_b200.layers.layernorm import RMSNorm
from prism_infer_b200.layers.mlp import Qwen3MLP
from prism_infer_b200.layers.moe import MoE
from prism_infer_b200.layers.w4 import W4Linear
from prism_infer_b200.quant import dequantize_w4

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, I, E, K = 256, 128, 32, 4
HALF = 2.0 ** -8


def block(seed=0, w4=True, group=64, symmetric=True, **kw):
    set_expert_parallel_size(1)
    torch.manual_seed(seed)
    kw = dict(scoring="sigmoid", score_bias=True, num_groups=8, topk_groups=3, group_score="top2",
              routed_scale=2.5) | kw
    moe = MoE(H, I, E, K, **kw)
    with torch.no_grad():
        moe.gate.weight.normal_(std=H ** -0.5)
        if moe.gate.e_score_correction_bias is not None:
            moe.gate.e_score_correction_bias.normal_(std=0.1)
        moe.w_gate_up.normal_(std=H ** -0.5)
        moe.w_down.normal_(std=I ** -0.5)
    moe = moe.to(DEV, torch.bfloat16)
    return moe.quantize_experts_(group, symmetric=symmetric) if w4 else moe


def tokens(T, seed=1):
    return torch.randn(T, H, generator=torch.Generator(device=DEV).manual_seed(seed),
                       device=DEV).to(torch.bfloat16)


def weights_of(moe):
    if moe.w4_gate_up is None:
        return moe.w_gate_up.double(), moe.w_down.double()
    return (dequantize_w4(moe.w4_gate_up.weight, torch.float64),
            dequantize_w4(moe.w4_down.weight, torch.float64))


def check(moe, x, out):
    """Output against 64-bit experts on the block's own choice, and that choice against the oracle."""
    logits, ids, w = moe.route(x)
    if moe.scoring is not None:
        r_ids, r_w = route_scored_ref(
            logits, K, scoring=moe.scoring, bias=moe.gate.e_score_correction_bias,
            num_groups=moe.num_groups, topk_groups=moe.topk_groups, group_score=moe.group_score,
            renorm=moe.norm_topk_prob, scale=moe.routed_scale)
        assert torch.equal(ids, r_ids)
        torch.testing.assert_close(w.double(), r_w, rtol=HALF + 2.0 ** -18, atol=1e-30)
    gu, dn = weights_of(moe)
    ref = torch.zeros(x.shape[0], H, dtype=torch.float64, device=DEV)
    slack = torch.zeros_like(ref)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        g, u = (x[t].double() @ gu[e].t()).chunk(2, dim=-1)
        h = g * torch.sigmoid(g) * u
        y = h @ dn[e].t()
        we = w[t, j].double().unsqueeze(1)
        ref.index_put_((t,), we * y, accumulate=True)
        # dense experts round g, u and h to bf16, 4-bit ones h: at most 3.2 roundings of |h|
        wide = 3.2 * HALF * (h.abs() + u.abs() * HALF) @ dn[e].abs().t()
        slack.index_put_((t,), we.abs() * (wide + 2 * HALF * y.abs()), accumulate=True)
    off = (out.double() - ref).abs()
    assert (off <= slack + HALF * ref.abs() + 1e-6).all(), (off - slack).max()
    assert off.norm() <= 3 * HALF * ref.norm()


@pytest.mark.parametrize("T", [0, 1, 2, 7, 64, 300, 2000])
@pytest.mark.parametrize("w4", [False, True])
def test_routed_block(T, w4):
    moe, x = block(w4=w4), tokens(T)
    out = moe(x)
    assert out.shape == x.shape
    if T:
        moe.check_device_error()
        check(moe, x, out)


@pytest.mark.parametrize("kw", [dict(scoring="softmax", score_bias=False, group_score="max"),
                                dict(scoring=None, score_bias=False, num_groups=1, topk_groups=1,
                                     routed_scale=1.0),
                                dict(scoring="sigmoid", num_groups=1, topk_groups=1,
                                     norm_topk_prob=False)])
def test_other_routers_on_4_bit_experts(kw):
    moe, x = block(symmetric=False, group=32, **kw), tokens(90)
    check(moe, x, moe(x.view(9, 10, H)).view(90, H))


@pytest.mark.parametrize("w4", [False, True])
def test_norm_fused_equals_norm_after(w4):
    moe, x, res = block(w4=w4), tokens(77), tokens(77, 2)
    norm = RMSNorm(H).to(DEV, torch.bfloat16)
    norm.weight.data.normal_()
    got, got_res = moe(x, residual=res, norm=norm)
    want, want_res = norm(moe(x), res)
    assert torch.equal(got, want) and torch.equal(got_res, want_res)


def test_steps_one_by_one_equal_the_block():
    """route_scored -> dispatch_plan -> permute_rows -> expert_swiglu_w4 -> combine."""
    moe, x = block(), tokens(128)
    _, ids, w = moe.route(x)
    plan = capi.dispatch_plan(ids, E, 1, want_perm=False)
    xs = capi.permute_rows(x, K, plan["entry_row"])
    y = capi.expert_swiglu_w4(xs, plan["expert_offsets"], moe.w4_gate_up.weight, moe.w4_down.weight)
    assert torch.equal(capi.combine(y, w, entry_row=plan["entry_row"]), moe(x))


def test_two_graphs_share_nothing():
    """Two captured steps replayed at once on two streams, with new tokens each time."""
    moe = block()
    inputs = [tokens(64, s) for s in (3, 4)]
    moe(inputs[0])
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(moe(x))
        graphs.append(g)
    for turn in range(5):
        for i, x in enumerate(inputs):
            x.copy_(tokens(64, 10 * turn + i))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        moe(tokens(500, 99))                    # an eager call of another size between replays
        for x, out in zip(inputs, outs):
            assert torch.equal(out, moe(x))


def test_ids_of_no_expert_add_nothing():
    moe, x = block(), tokens(6)
    _, ids, w = moe.route(x)
    gu, dn = moe.w4_gate_up.weight, moe.w4_down.weight
    wrong = ids.clone()
    wrong[2, 1], wrong[4, 0] = -1, E
    out = capi.block_forward_routed(x, wrong, w, gu, dn)
    assert capi.read_device_error(capi.block_error_word(x.device)) == capi.ERR_ARG
    none = w.clone()
    none[2, 1] = none[4, 0] = 0
    assert torch.equal(out, capi.block_forward_routed(x, ids, none, gu, dn))
    same = ids.clone()
    same[:] = ids[:, :1]                        # one expert four times
    check_same = capi.block_forward_routed(x, same, w, gu, dn)
    assert check_same.isfinite().all()


def test_scored_choice_through_the_expert_parallel_step():
    """A group of one: the NVLink step fed with the scored router's choice."""
    moe, x = block(w4=False), tokens(70)
    _, ids, w = moe.route(x)
    bank = ExpertParallelMoE(H, I, E, 1, 0).to(DEV, torch.bfloat16)
    with torch.no_grad():
        bank.w_gate_up.copy_(moe.w_gate_up)
        bank.w_down.copy_(moe.w_down)
    out = bank(x, ids, w)
    bank.check_device_error()
    assert torch.equal(out, moe(x))
    bank.release()


@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_dense_modules(T):
    torch.manual_seed(3)
    mlp = Qwen3MLP(H, I).to(DEV, torch.bfloat16)
    for p in mlp.parameters():
        p.data.normal_(std=p.shape[1] ** -0.5)
    mlp.quantize_(64, symmetric=False)
    x = tokens(T).view(T, 1, H)
    gu = dequantize_w4(mlp.w4_gate_up.weight, torch.float64)[0]
    dn = dequantize_w4(mlp.w4_down.weight, torch.float64)[0]
    g, u = (x.double() @ gu.t()).chunk(2, dim=-1)
    h = g * torch.sigmoid(g) * u
    ref, y = h @ dn.t(), mlp(x)
    assert y.shape == x.shape
    assert ((y.double() - ref).abs() <= HALF * ref.abs() + 1.1 * HALF * (h.abs() @ dn.abs().t())).all()
    lin = W4Linear.from_weight(torch.randn(40, H, device=DEV), 32)
    ref = x.double() @ dequantize_w4(lin.weight, torch.float64).t()
    out = lin(x)
    assert out.shape == (T, 1, 40)
    assert (out.double() - ref).abs().norm() <= HALF * ref.norm()


@pytest.mark.parametrize("T", [3, 37, 150])
def test_dense_mlp_captured_at_its_first_call_with_these_rows(T):
    """Nothing that a replay needs is kept from, or made by, another call."""
    torch.manual_seed(4)
    mlp = Qwen3MLP(H, I).to(DEV, torch.bfloat16)
    for p in mlp.parameters():
        p.data.normal_(std=p.shape[1] ** -0.5)
    mlp.quantize_(64)
    mlp(tokens(T + 1000))
    x = tokens(T)
    static = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mlp(static)
    eager = mlp(x)            # between capture and first replay
    static.copy_(x)
    graph.replay()
    assert torch.equal(y, eager)


def test_refusals_on_the_device():
    moe, x = block(), tokens(4)
    gu, dn = moe.w4_gate_up.weight, moe.w4_down.weight
    _, ids, w = moe.route(x)
    for call in (lambda: capi.block_forward_routed(x, ids.int(), w, gu, dn),
                 lambda: capi.block_forward_routed(x, ids, w.float(), gu, dn),
                 lambda: capi.block_forward_routed(x[:3], ids, w, gu, dn),
                 lambda: capi.block_forward_routed(x.t().contiguous().t(), ids, w, gu, dn),
                 lambda: capi.route_scored(x, 2, bias=torch.zeros(H, device=DEV).bfloat16()),
                 lambda: capi.route_scored(x, 2, bias=torch.zeros(H)),
                 lambda: capi.route_scored(x, 33), lambda: capi.route_scored(x, 0),
                 lambda: capi.route_scored(x.half(), 2),
                 lambda: capi.linear_w4(x.cpu(), W4Linear.from_weight(torch.randn(8, H)).weight),
                 lambda: capi.linear_w4(x, W4Linear.from_weight(torch.randn(8, H)).weight),
                 lambda: capi.expert_swiglu_w4(x, torch.zeros(4, dtype=torch.int32, device=DEV), gu, dn),
                 lambda: moe(x.float())):
        with pytest.raises(RuntimeError):
            call()
