"""4-bit weights and the scored router without a GPU: the layout against its definition, the
quantiser, the refusals of the C ABI, of ``capi`` and of the modules, and shapes under tracing."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from prism_infer_b200 import build, capi, ops  # noqa: F401
from prism_infer_b200.layers.mlp import Qwen3MLP
from prism_infer_b200.layers.moe import MoE
from prism_infer_b200.layers.w4 import W4Linear
from prism_infer_b200.quant import W4Weight, dequantize_w4, pack_w4, quantize_w4


def parts(lead, N, K, G, zeros=True):
    codes = torch.randint(0, 16, (*lead, N, K))
    scales = torch.rand(*lead, N, K // G).bfloat16()
    z = torch.randint(0, 16, (*lead, N, K // G)) if zeros else None
    return codes, scales, z


@pytest.mark.parametrize("N,K,G", [(8, 32, 32), (40, 96, 32), (24, 192, 64), (136, 384, 128),
                                   (16, 128, 128), (1000, 160, 32)])
def test_layout_is_the_documented_one(N, K, G):
    """Every code, scale and zero point at the place that prism_moe_w4's comment gives."""
    codes, scales, z = parts((), N, K, G)
    w = pack_w4(codes, scales, z, group_size=G)
    assert w.qweight.shape == (-(-N // 16), -(-K // 128), 16, 64)
    for n, k in [(0, 0), (N - 1, K - 1), (N // 2, K // 3), (N // 3, K // 2), (7 % N, 31)] + \
            [(int(torch.randint(N, ())), int(torch.randint(K, ()))) for _ in range(50)]:
        r = k % 128
        word = 4 * ((r % 32) // 8) + r // 32
        nibble = [0, 2, 4, 6, 1, 3, 5, 7].index(r % 8)
        byte = int(w.qweight[n // 16, k // 128, n % 16, 4 * word + nibble // 2])
        assert (byte >> 4 * (nibble % 2)) & 15 == codes[n, k]
        assert w.scales[n // 16, k // 128, n % 16, r // G] == scales[n, k // G]
        assert w.zeros[n // 16, k // 128, n % 16, r // G] == z[n, k // G]


@pytest.mark.parametrize("gate_up", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
def test_values_come_back(gate_up, zeros):
    codes, scales, z = parts((3,), 48, 192, 64, zeros)
    w = pack_w4(codes, scales, z, group_size=64, gate_up=gate_up)
    per = lambda t: t.double().repeat_interleave(64, -1)
    ref = (codes.double() - (per(z) if zeros else 8)) * per(scales)
    assert torch.equal(dequantize_w4(w, torch.float64), ref)
    if gate_up:   # 8 gate rows and 8 up rows by turns
        assert torch.equal(w.scales[0, 0, 0, :, 0],
                           torch.cat([scales[0, :8, 0], scales[0, 24:32, 0]]))


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_quantiser_rounds_to_nearest(symmetric, G):
    w = torch.randn(2, 16, 256)
    w[0, 3] = 0
    w[1, 4, :G] = w[1, 4, :G].abs() + 1
    q = quantize_w4(w, G, symmetric=symmetric)
    back = dequantize_w4(q)
    assert (back[0, 3] == 0).all()
    step = torch.repeat_interleave(_scales(q), G, -1)
    # half a step, and what the scale's own rounding to bf16 (2^-8) moves the largest code by
    assert ((back - w).abs() <= step * (0.5 + 15 * 2.0 ** -8)).all()
    assert (q.zeros is None) == symmetric


def _scales(q):
    n16, c, _, per = q.scales.shape[-4:]
    s = q.scales.transpose(-3, -2).reshape(*q.scales.shape[:-4], n16 * 16, c * per)
    return s[..., :q.out_features, :q.in_features // q.group_size].float()


def test_weights_that_do_not_fit_are_refused():
    codes, scales, z = parts((), 32, 128, 64)
    bad = [dict(codes=codes + 1 - codes.min() + 15), dict(codes=-codes - 1), dict(codes=codes.float()),
           dict(scales=scales[:, :1]), dict(zeros=z + 16), dict(group_size=48),
           dict(codes=codes[:, :96]), dict(codes=codes[:12], scales=scales[:12], zeros=z[:12])]
    for change in bad:
        kw = dict(codes=codes, scales=scales, zeros=z, group_size=64) | change
        with pytest.raises(RuntimeError):
            pack_w4(kw.pop("codes"), kw.pop("scales"), kw.pop("zeros"), **kw)
    with pytest.raises(RuntimeError):
        pack_w4(codes[:24], scales[:24], z[:24], group_size=64, gate_up=True)
    w = pack_w4(codes, scales, z, group_size=64)
    with pytest.raises(RuntimeError):
        W4Weight(w.qweight, w.scales.float(), w.zeros, 32, 128, 64)
    with pytest.raises(RuntimeError):
        W4Weight(w.qweight, w.scales, w.zeros, 64, 128, 64)
    with pytest.raises(RuntimeError):
        W4Weight(w.qweight, w.scales, w.zeros.transpose(0, 1), 32, 128, 64)
    with pytest.raises(RuntimeError):
        quantize_w4(torch.randn(8, 100), 32)


def test_capi_refuses_before_any_kernel():
    codes, scales, _ = parts((), 32, 128, 64)
    w = pack_w4(codes, scales, group_size=64)
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    for call in (lambda: capi.linear_w4(x.float(), w), lambda: capi.linear_w4(x[:, :64], w),
                 lambda: capi.linear_w4(x, w),
                 lambda: capi.linear_w4(x, pack_w4(codes, scales, group_size=64, gate_up=True)),
                 lambda: capi.route_scored(x, 2, scoring="tanh"),
                 lambda: capi.route_scored(x, 2, group_score="sum"),
                 lambda: capi.route_scored(x, 2), lambda: capi.route_scored(x[0], 2)):
        with pytest.raises(RuntimeError):
            call()
    stack = lambda N, K, gu: pack_w4(*parts((2,), N, K, 64, False)[:2], group_size=64, gate_up=gu)
    gu, dn = stack(256, 128, True), stack(128, 128, False)
    seg = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: capi.expert_swiglu_w4(x, seg, gu, stack(64, 128, False)),
                 lambda: capi.expert_swiglu_w4(x, seg, dn, dn),
                 lambda: capi.expert_swiglu_w4(x, seg, gu, dn),
                 lambda: capi.expert_swiglu_w4(x.float(), seg, gu, dn),
                 lambda: capi.block_forward_routed(x, seg, x, gu, torch.zeros(1)),
                 lambda: capi.block_forward_routed(x.float(), seg, x, gu, dn)):
        with pytest.raises(RuntimeError):
            call()


@pytest.fixture(scope="module")
def lib():
    build.build()
    return capi.load()


def test_c_abi_refusals_need_no_gpu(lib):
    P = 1 << 20   # an aligned address that no refused call looks at

    def route(E=64, k=4, scoring=0, groups=1, keep=1, score=0, dtype=capi.F32, out=capi.F32, T=4,
              router=True, logits=P):
        r = capi.Router(scoring, None, groups, keep, score, 1, 1.0)
        return lib.prism_moe_route_scored(logits, dtype, T, E, k, ctypes.byref(r) if router else None,
                                          P, P, out, None, None)

    for bad in (dict(dtype=7), dict(out=7), dict(T=-1), dict(router=False), dict(E=0), dict(E=1025),
                dict(scoring=2), dict(score=2), dict(groups=0), dict(groups=33, E=66),
                dict(groups=3), dict(groups=4, keep=5), dict(groups=4, keep=0), dict(k=0),
                dict(k=33), dict(k=5, E=4), dict(k=9, groups=8, keep=1), dict(logits=None)):
        assert route(**bad) == capi.ERR_ARG, bad

    def linear(M=4, K=128, N=64, G=64, q=P, s=P, z=None, x=P, w=True):
        st = capi.W4(q, s, z, G)
        return lib.prism_moe_linear_w4(x, M, K, N, ctypes.byref(st) if w else None, P, None,
                                       None)

    for bad in (dict(M=-1), dict(K=0), dict(N=0), dict(G=16), dict(G=96), dict(K=96), dict(N=12),
                dict(q=None), dict(s=None), dict(w=False), dict(x=None), dict(x=P + 2), dict(q=P + 4),
                dict(s=P + 2), dict(z=P + 1), dict(M=1 << 31), dict(K=1 << 30), dict(),
                dict(x=P + 64 * 2 * 4 - 16)):   # the last two: x is y, or starts inside it
        assert linear(**bad) == capi.ERR_ARG, bad

    def experts(R=4, H=128, I=64, nseg=2, El=2, ws=1 << 20, seg=P, Gu=64, Gd=64, y=P, x=P, wsp=P):
        gu, dn = capi.W4(P, P, None, Gu), capi.W4(P, P, None, Gd)
        return lib.prism_moe_expert_swiglu_w4(x, R, H, I, seg, None, nseg, El, ctypes.byref(gu),
                                              ctypes.byref(dn), y, wsp, ws, None, None)

    assert experts(seg=None, nseg=2) == experts(seg=None, nseg=2, El=1) == capi.ERR_ARG
    for bad in (dict(R=-1), dict(H=0), dict(I=0), dict(nseg=0), dict(nseg=1025), dict(El=0),
                dict(ws=16), dict(seg=None), dict(Gu=48), dict(Gd=128), dict(H=96), dict(y=None),
                dict(x=P + 8), dict(wsp=P + 4), dict(R=1 << 31)):
        assert experts(**bad) == capi.ERR_ARG, bad
    assert lib.prism_moe_expert_w4_workspace_size(10, 64) >= 10 * 64 * 2
    assert lib.prism_moe_expert_w4_workspace_size(-1, 64) == 0

    q = capi.W4(P, P, None, 64)

    def block(T=2, H=128, I=64, E=4, k=2, dense=False, quant=True, dtype=capi.BF16, ws=1 << 30):
        d = (P, P) if dense else (None, None)
        w = (ctypes.byref(q), ctypes.byref(q)) if quant else (None, None)
        return lib.prism_moe_block_forward_routed(P, P, P, dtype, T, H, I, E, k, *d, *w, P, P, ws,
                                                  None, None)

    for bad in (dict(T=-1), dict(E=0), dict(k=5), dict(dense=True), dict(quant=False),
                dict(dtype=capi.F32), dict(H=96), dict(ws=16), dict(dtype=9)):
        assert block(**bad) == capi.ERR_ARG, bad


def test_fake_shapes():
    with FakeTensorMode():
        e = lambda *s, dt=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dt)
        x, u8 = e(6, 128), torch.uint8
        ids, w = torch.ops.prism_moe.route_scored(e(6, 64, dt=torch.float32), 4, "sigmoid",
                                                  e(64, dt=torch.float32), 8, 2, "top2", True, 2.0,
                                                  torch.bfloat16)
        assert ids.shape == w.shape == (6, 4) and ids.dtype == torch.int64
        assert w.dtype == torch.bfloat16
        y = torch.ops.prism_moe.linear_w4(x, e(2, 1, 16, 64, dt=u8), e(2, 1, 16, 2), None, 24, 64)
        assert y.shape == (6, 24) and y.dtype == x.dtype
        gu = (e(4, 8, 1, 16, 64, dt=u8), e(4, 8, 1, 16, 2), None)
        dn = (e(4, 8, 1, 16, 64, dt=u8), e(4, 8, 1, 16, 2), None)
        seg = e(5, dt=torch.int32)
        assert torch.ops.prism_moe.expert_swiglu_w4(x, seg, *gu, *dn, 64, 64, 64, None).shape == x.shape
        assert torch.ops.prism_moe.block_forward_w4(x, ids, w, *gu, *dn, 64, 64, 64).shape == x.shape
        o, r = torch.ops.prism_moe.block_forward_w4_norm(x, ids, w, *gu, *dn, 64, 64, 64, x, e(128),
                                                         1e-6)
        assert o.shape == r.shape == x.shape
        wgu, wd = e(4, 128, 128), e(4, 128, 64)
        assert torch.ops.prism_moe.block_forward_routed(x, ids, w, wgu, wd).shape == x.shape
        o, r = torch.ops.prism_moe.block_forward_routed_norm(x, ids, w, wgu, wd, x, e(128), 1e-6)
        assert o.shape == r.shape == x.shape


def test_modules_refuse_and_keep_types():
    for kw in (dict(score_bias=True), dict(num_groups=2), dict(routed_scale=2.0),
               dict(scoring="tanh"), dict(scoring="sigmoid", group_score="mean"),
               dict(scoring="sigmoid", num_groups=3), dict(scoring="sigmoid", num_groups=4, topk_groups=5),
               dict(scoring="sigmoid", num_groups=8, topk_groups=1)):
        with pytest.raises(RuntimeError):
            MoE(128, 64, 8, 2, **kw)
    moe = MoE(128, 64, 8, 2, scoring="sigmoid", score_bias=True, num_groups=4, topk_groups=2)
    bias = torch.randn(8)
    p = moe.gate.e_score_correction_bias
    p.weight_loader(p, bias)
    with torch.no_grad():
        moe.w_gate_up.normal_()
        moe.w_down.normal_()
    moe = moe.to(torch.bfloat16)
    assert moe.gate.e_score_correction_bias.dtype == torch.float32
    assert torch.equal(moe.gate.e_score_correction_bias, bias)
    dense = moe.w_down.float()
    moe.quantize_experts_(32, symmetric=False)
    assert not any(n.startswith("experts.") for n in moe.state_dict())
    assert (dequantize_w4(moe.w4_down.weight) - dense).abs().max() < 0.5
    with pytest.raises(RuntimeError):
        moe.quantize_experts_(32)
    scales = moe.w4_down.scales.clone().mul_(1e-6)      # below the range of float16
    moe.w4_down.scales.copy_(scales)
    again = moe.to(torch.float32).to(torch.float16).to(torch.bfloat16)
    assert torch.equal(again.w4_down.scales, scales)
    mlp = Qwen3MLP(128, 64)
    for q in mlp.parameters():
        q.data.normal_()
    mlp.quantize_(32)
    with pytest.raises(RuntimeError):
        mlp.quantize_(32)
    with pytest.raises(RuntimeError):
        W4Linear(moe.w4_gate_up.weight)
    # 96 and 128 inputs have the same number of tiles: the modules know which it is
    lin = W4Linear.from_weight(torch.nn.Parameter(torch.randn(16, 96)), 32)
    assert not lin.scales.requires_grad
    with pytest.raises(RuntimeError):
        lin(torch.zeros(1, 128, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        mlp(torch.zeros(1, 96, dtype=torch.bfloat16))


def test_quantised_scored_block_exports_as_one_graph():
    moe = MoE(128, 64, 8, 2, scoring="softmax", num_groups=4, topk_groups=2, routed_scale=2.0)
    with torch.no_grad():
        moe.w_gate_up.normal_()
        moe.w_down.normal_()
    moe = moe.to(torch.bfloat16).quantize_experts_(64).to("meta")
    x = torch.empty(2, 5, 128, device="meta", dtype=torch.bfloat16)
    assert moe(x).shape == x.shape
    called = [str(n.target) for n in torch.export.export(moe, (x,)).graph.nodes
              if n.op == "call_function"]
    assert "prism_moe.route_scored.default" in called
    assert "prism_moe.block_forward_w4.default" in called
