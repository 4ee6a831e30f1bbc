"""Products with 4-bit weights on the GPU against 64-bit arithmetic on the same codes and scales.

Bounds, element by element. The kernels multiply small integers by bf16 activations, exactly, and
sum in fp32: a sum of n partial sums in whatever order is off by at most n * 2^-22 of the sum of the
terms' magnitudes (2^-24 for each rounding, four times that for the tensor cores' alignment of their
addends). n is the 16-input steps of one group, the groups, and the joining of up to 16 parts. The
integers are code - zero for many rows; for few rows offset + code and offset + zero are summed apart,
128 + 15 at most each: terms of up to 286 * scale * |x| in all.
Outputs are rounded to bf16: 2^-8 of the value. In the experts, silu(g) * u is rounded to bf16
between the products (2^-8 of each h, passed on by |w_down|); the fast exponential (2 + 1.2 |g| ulp)
and division (2 ulp) before it are off by 2^-16 of h while |g| <= 87; and |silu'| <= 1.1.
Over a whole output the 2-norm of the difference stays below 2^-8 of the result's: a rounding's
error is spread over [-2^-8, 2^-8] at most, so its rms is at most 2^-8 / sqrt(3), and two of them
(h and y) come to 2^-8 * sqrt(2/3).
"""
from dataclasses import replace

import pytest
import torch

from prism_infer_b200 import capi, ops  # noqa: F401
from prism_infer_b200.quant import W4Weight, dequantize_w4, pack_w4, quantize_w4

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8


def gen_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def weights(seed, lead, N, K, G, zeros, gate_up=False):
    g = gen_of(seed)
    codes = torch.randint(0, 16, (*lead, N, K), generator=g, device=DEV)
    s = (0.5 + torch.rand(*lead, N, K // G, generator=g, device=DEV)) / (4.6 * K ** 0.5)
    z = torch.randint(0, 16, (*lead, N, K // G), generator=g, device=DEV) if zeros else None
    return pack_w4(codes, s, z, group_size=G, gate_up=gate_up)


def rows(seed, M, K):
    return torch.randn(M, K, generator=gen_of(seed), device=DEV).to(torch.bfloat16)


def most(w):
    """286 * scale of every weight, rows as dequantize_w4 gives them."""
    zeros = torch.zeros(w.scales.shape, dtype=torch.uint8, device=w.device)
    ones = replace(w, qweight=torch.full_like(w.qweight, 0xff), zeros=zeros)
    return dequantize_w4(ones, torch.float64) * (286 / 15)


def steps(w):
    return (w.group_size // 16 + w.in_features // w.group_size + 16) * 2.0 ** -22


def check_linear(x, w, y):
    wd, xd = dequantize_w4(w, torch.float64), x.double()
    ref, mag = xd @ wd.t(), xd.abs() @ most(w).t()
    off = (y.double() - ref).abs()
    assert (off <= HALF * ref.abs() + steps(w) * mag * (1 + HALF)).all(), off.max()
    if ref.numel() >= 256:
        assert off.norm() <= HALF * ref.norm()


def check_experts(x, bounds, experts, gu, dn, y):
    """``experts[s]`` is segment s's expert (None: the segment is left alone)."""
    all_gu, all_dn = dequantize_w4(gu, torch.float64), dequantize_w4(dn, torch.float64)
    most_gu, most_dn = most(gu), most(dn)
    diff = total = 0.0
    for s, e in enumerate(experts):
        a, b = bounds[s], bounds[s + 1]
        if a >= b or e is None:
            continue
        wg, wu = all_gu[e].chunk(2)
        wd, xd = all_dn[e], x[a:b].double()
        g, u = xd @ wg.t(), xd @ wu.t()
        dg, du = (steps(gu) * (xd.abs() @ w.t()) for w in most_gu[e].chunk(2))
        sg = g * torch.sigmoid(g)
        h = sg * u
        dh = (HALF + 2.0 ** -16) * h.abs() + (1.1 * u.abs() * dg + (sg.abs() + 1.1 * dg) * du) * 1.01
        ref = h @ wd.t()
        mag = (h.abs() + dh) @ most_dn[e].t()
        off = (y[a:b].double() - ref).abs()
        tol = (dh @ wd.abs().t() + steps(dn) * mag) * (1 + HALF) + HALF * ref.abs()
        assert (off <= tol).all(), (s, e, (off - tol).max().item())
        diff, total = diff + (off ** 2).sum().item(), total + (ref ** 2).sum().item()
    assert diff ** 0.5 <= HALF * total ** 0.5


# ------------------------------------------------------------------------------------ linear

LINEAR = [(1, 8, 32, 32), (1, 4096, 4096, 128), (2, 24, 96, 32), (3, 2056, 1440, 32),
          (8, 136, 192, 64), (9, 1000, 128, 64), (16, 264, 2176, 128), (17, 512, 640, 128),
          (33, 72, 352, 32), (64, 520, 4224, 64), (100, 1536, 2048, 128), (127, 40, 256, 128),
          (128, 128, 1024, 32), (129, 136, 1088, 64), (255, 96, 32, 32), (256, 384, 512, 64),
          (257, 392, 576, 64), (700, 1032, 1152, 128), (2048, 256, 768, 32), (5, 640, 9216, 128),
          # more tiles than SMs, of 64 and of 256 rows; exactly as many of 64; deep sums on few tiles
          (40, 19208, 96, 32), (64, 20000, 704, 64), (33, 19000, 1152, 128), (300, 19208, 192, 64),
          (64, 18944, 256, 128), (128, 9472, 320, 32), (250, 4096, 8192, 128), (190, 776, 5120, 64)]


@pytest.mark.parametrize("M,N,K,G", LINEAR)
@pytest.mark.parametrize("zeros", [False, True])
def test_linear(M, N, K, G, zeros):
    w, x = weights(M + N, (), N, K, G, zeros), rows(K, M, K)
    out = torch.full((M, N), float("nan"), device=DEV).to(torch.bfloat16)
    y = capi.linear_w4(x, w, out=out)
    assert y.data_ptr() == out.data_ptr()
    check_linear(x, w, y)
    assert torch.equal(capi.linear_w4(x, w), y), "the same call gives the same bits"


def test_linear_no_rows_and_operator():
    w = weights(1, (), 64, 128, 64, True)
    assert capi.linear_w4(rows(1, 0, 128), w).shape == (0, 64)
    x = rows(2, 5, 128)
    y = torch.ops.prism_moe.linear_w4(x, w.qweight, w.scales, w.zeros, 64, 64)
    assert torch.equal(y, capi.linear_w4(x, w))


@pytest.mark.parametrize("M", [3, 16, 40])
def test_linear_extreme_magnitudes(M):
    """Rows far from one another in size, and elements far from one another within a row."""
    w = weights(5, (), 264, 1024, 128, True)
    x = rows(6, M, 1024).float()
    x *= torch.logspace(-30, 30, M, device=DEV).unsqueeze(1)
    x[:, ::7] *= 2.0 ** -30
    x[1] = 0
    x = x.to(torch.bfloat16)
    y = capi.linear_w4(x, w)
    check_linear(x, w, y)
    assert (y[1] == 0).all()


def test_linear_rows_do_not_meet():
    """Infinities and NaN stay in their own row; a row's value does not depend on the others."""
    w = weights(3, (), 264, 512, 128, True)
    for M in (3, 40, 300):
        x = rows(4, M, 512)
        clean = capi.linear_w4(x, w)
        x[1, 7] = float("nan")
        x[2, 9] = float("inf")
        y = capi.linear_w4(x, w)
        keep = [i for i in range(M) if i not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])
        assert y[1].isnan().all() and not y[2].isfinite().all()


@pytest.mark.parametrize("M,N,K,G", [(8192, 4096, 1024, 128), (4096, 4096, 1024, 64),
                                     (4096, 2048, 2048, 32), (64, 16384, 2048, 128),
                                     (48, 16384, 2048, 32), (16, 16384, 2048, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_large_grids_repeat(M, N, K, G, zeros):
    """Thousands of tiles, many times: a hand-over between warps that is one instruction early shows in
    a few tiles of a large grid only."""
    w, x = weights(7, (), N, K, G, zeros), rows(8, M, K)
    y = capi.linear_w4(x, w)
    check_linear(x, w, y)
    for _ in range(20):
        assert torch.equal(capi.linear_w4(x, w), y)


# ------------------------------------------------------------------------------------ experts

EXPERTS = [
    (256, 128, 128, 64, [1, 0, 1, 1]), (2048, 768, 128, 128, [1] * 8 + [0] * 24),
    (2048, 768, 64, 64, [5, 0, 8, 9, 16, 17, 31, 33, 0, 1]), (160, 96, 32, 32, [3, 40, 0, 128, 1]),
    (1440, 736, 32, 32, [22, 0, 150, 7, 64]), (320, 192, 64, 32, [129, 64, 15]),
    (512, 256, 128, 64, [130, 0, 255, 256, 257, 3]), (256, 1024, 64, 128, [600, 2, 0, 1]),
    (32, 32, 32, 32, [0, 1, 0, 300]), (128, 128, 128, 128, [0, 0, 0]),
    (512, 512, 128, 64, [30, 17, 64, 0, 65, 16, 100, 2] * 5), (320, 1088, 32, 64, [40, 33, 20] * 12),
    (1024, 768, 128, 128, [200, 300, 16, 17, 90, 500] * 2),
]


def bounds_of(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return off


@pytest.mark.parametrize("H,I,Gu,Gd,counts", EXPERTS)
@pytest.mark.parametrize("zeros", [False, True])
def test_experts(H, I, Gu, Gd, counts, zeros):
    E, off = len(counts), bounds_of(counts)
    gu = weights(H, (E,), 2 * I, H, Gu, zeros, gate_up=True)
    dn = weights(I, (E,), H, I, Gd, zeros)
    R = off[-1] + 3                                   # three rows behind the last segment
    x = rows(H + I, R, H)
    seg = torch.tensor(off, dtype=torch.int32, device=DEV)
    y = torch.full((R, H), 7.0, device=DEV).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    capi.expert_swiglu_w4(x, seg, gu, dn, y=y, device_error=err)
    assert capi.read_device_error(err) == 0
    assert (y[off[-1]:] == 7).all(), "rows of no segment are left as they were"
    check_experts(x, off, range(E), gu, dn, y)
    again = y.clone().fill_(7)
    capi.expert_swiglu_w4(x, seg, gu, dn, y=again)
    assert torch.equal(again, y), "the same call gives the same bits"


def test_experts_segment_map_and_bad_ids():
    """Segments name any expert, the same twice; one with an id of no expert is left alone and
    recorded; offsets past the rows end at the last row."""
    H, I, El = 256, 128, 3
    gu, dn = weights(1, (El,), 2 * I, H, 64, True, gate_up=True), weights(2, (El,), H, I, 64, True)
    counts = [5, 0, 40, 300, 9, 2]
    off = bounds_of(counts)
    x = rows(3, off[-1], H)
    seg = torch.tensor(off, dtype=torch.int32, device=DEV)
    ids = [2, 1, 0, 2, 0, 0]
    y = capi.expert_swiglu_w4(x, seg, gu, dn,
                              seg_expert=torch.tensor(ids, dtype=torch.int32, device=DEV))
    check_experts(x, off, ids, gu, dn, y)
    for bad in (-1, El, 2 ** 31 - 1):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full_like(x, 3.0)
        wrong = torch.tensor([2, 1, bad, bad, 0, 0], dtype=torch.int32, device=DEV)
        capi.expert_swiglu_w4(x, seg, gu, dn, seg_expert=wrong, y=out, device_error=err)
        assert capi.read_device_error(err) == capi.ERR_ARG
        assert (out[off[2]:off[4]] == 3).all()
        check_experts(x, off, [2, 1, None, None, 0, 0], gu, dn, out)
    over = seg.clone()
    over[-1] = 10 ** 6
    y2 = capi.expert_swiglu_w4(x, over, gu, dn,
                               seg_expert=torch.tensor(ids, dtype=torch.int32, device=DEV))
    assert torch.equal(y, y2)


def test_experts_operator_stream_and_graph():
    H, I, E = 512, 256, 6
    gu, dn = weights(1, (E,), 2 * I, H, 128, False, gate_up=True), weights(2, (E,), H, I, 128, False)
    off = bounds_of([4, 0, 30, 1, 90, 2])
    seg = torch.tensor(off, dtype=torch.int32, device=DEV)
    x = rows(5, off[-1], H)
    y = torch.ops.prism_moe.expert_swiglu_w4(x, seg, gu.qweight, gu.scales, gu.zeros, dn.qweight,
                                             dn.scales, dn.zeros, I, 128, 128, None)
    check_experts(x, off, range(E), gu, dn, y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2 = capi.expert_swiglu_w4(x, seg, gu, dn)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, y2)
    static, table = x.clone(), seg.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy = capi.expert_swiglu_w4(static, table, gu, dn)
    other = bounds_of([0, 100, 3, 0, 20, 4])           # the table may change between replays
    for src, o in ((rows(6, off[-1], H), other), (x, off)):
        static.copy_(src)
        table.copy_(torch.tensor(o, dtype=torch.int32))
        graph.replay()
        check_experts(src, o, range(E), gu, dn, gy)
    assert torch.equal(gy, y)


@pytest.mark.parametrize("R,H,I", [(1, 384, 160), (17, 384, 160), (64, 384, 160), (65, 384, 160),
                                   (700, 384, 160), (20, 256, 5632)])
def test_experts_one_segment_of_all_rows(R, H, I):
    """Without a table (the last case's two products run on different kernels); y may be the input."""
    gu = weights(1, (1,), 2 * I, H, 64, True, gate_up=True)
    dn = weights(2, (1,), H, I, 32, True)
    x = rows(R, R, H)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = capi.expert_swiglu_w4(x, None, gu, dn, device_error=err)
    check_experts(x, [0, R], [0], gu, dn, y)
    same = x.clone()
    capi.expert_swiglu_w4(same, None, gu, dn, y=same)
    assert torch.equal(same, y) and capi.read_device_error(err) == 0
    two = weights(3, (2,), H, I, 32, True)
    with pytest.raises(RuntimeError):                 # two experts, one segment: which one?
        capi.expert_swiglu_w4(x, None, weights(1, (2,), 2 * I, H, 64, True, gate_up=True), two)


@pytest.mark.parametrize("counts", [[2, 0, 3, 1], [200, 3, 0, 40], [700, 16, 900, 17], [30, 40, 1, 20]])
def test_experts_follow_each_other_and_run_side_by_side(counts):
    """A call's kernels overlap; a call that reads what the one before it wrote, in the same buffers,
    still sees all of it, and calls on two streams do not meet."""
    H, I, E = 256, 192, len(counts)
    gu, dn = weights(1, (E,), 2 * I, H, 64, True, gate_up=True), weights(2, (E,), H, I, 64, True)
    seg = torch.tensor(bounds_of(counts), dtype=torch.int32, device=DEV)
    xs = [rows(s, sum(counts), H) for s in (3, 4)]

    def chain(x, wait):
        y = x.clone()
        for _ in range(6):
            capi.expert_swiglu_w4(y, seg, gu, dn, y=y)
            if wait:
                torch.cuda.synchronize()
            # a reader and writer in between, which also keeps rows at a length of sqrt(H)
            y.copy_(torch.nn.functional.normalize(y.float(), dim=1) * 16)
            capi.expert_swiglu_w4(y, seg, gu, dn, y=y)
            if wait:
                torch.cuda.synchronize()
        return y

    want = [chain(x, True) for x in xs]
    assert all(w.abs().max() > 0 and w.isfinite().all() for w in want)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(10):
        got = []
        for x, s in zip(xs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(chain(x, False))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_linear_outputs_past_32_bits():
    M, N, K = 540_000, 4096, 128                     # 2.2e9 outputs
    w = weights(1, (), N, K, 128, False)
    x = rows(2, M, K)
    y = capi.linear_w4(x, w)
    for at in (0, M // 2, 2 ** 31 // N - 100, M - 300):
        check_linear(x[at:at + 300], w, y[at:at + 300])


@pytest.mark.parametrize("counts", [[3, 1], [40, 700]])
def test_experts_of_a_stack_past_32_bits(counts):
    """The last experts of stacks whose codes take 2.5 GB."""
    E, H, I, G = 1200, 2048, 1024, 128
    g = gen_of(5)

    def stack(N, K, gate_up):
        shape = (E, N // 16, K // 128, 16)
        q = torch.randint(0, 256, (*shape, 64), generator=g, device=DEV, dtype=torch.uint8)
        s = ((0.5 + torch.rand(*shape, 1, generator=g, device=DEV)) / (4.6 * K ** 0.5)).bfloat16()
        return W4Weight(q, s, None, N, K, G, gate_up)

    def some(w, ids):
        return W4Weight(w.qweight[ids], w.scales[ids], None, w.out_features, w.in_features, G,
                        w.gate_up)

    gu, dn = stack(2 * I, H, True), stack(H, I, False)
    ids = [E - 1, E - 150]
    off = bounds_of(counts)
    x = rows(6, off[-1], H)
    y = capi.expert_swiglu_w4(x, torch.tensor(off, dtype=torch.int32, device=DEV), gu, dn,
                              seg_expert=torch.tensor(ids, dtype=torch.int32, device=DEV))
    check_experts(x, off, [0, 1], some(gu, ids), some(dn, ids), y)


def test_linear_out_and_error_word():
    w = weights(1, (), 256, 256, 64, False)
    x = rows(2, 40, 256)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = capi.linear_w4(x, w, device_error=err)
    check_linear(x, w, y)
    assert capi.read_device_error(err) == 0
    both = torch.zeros(60, 256, device=DEV, dtype=torch.bfloat16)
    for out in (x, both[10:50]):
        with pytest.raises(RuntimeError):
            capi.linear_w4(both[:40] if out is not x else x, w, out=out)
    with pytest.raises(RuntimeError):
        capi.linear_w4(x, w, device_error=err.long())


def test_quantised_close_to_the_weights():
    """Round-to-nearest: every value within half a step of its group's scale (and the bf16 scale's
    own rounding of the largest code)."""
    w = torch.randn(3, 64, 256, generator=gen_of(1), device=DEV)
    for symmetric in (True, False):
        q = quantize_w4(w, 64, symmetric=symmetric, gate_up=True)
        step = q.scales.float().max().item()
        assert (dequantize_w4(q) - w).abs().max().item() <= step * (0.5 + 15 * HALF)
