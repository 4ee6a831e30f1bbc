"""Scored routing on the GPU (``capi.route_scored`` / ``torch.ops.prism_moe.route_scored``) against a
plain implementation in 64 bits: choices exactly, weights to the rounding of their type.

Weights, in fp32: expf is off by 2 ulp (2^-22), twice in a softmax; its sum of up to 1024 terms goes
through 11 roundings, that of the chosen through 6, and there are three divisions and products: at
most 2^-22 * 2 + 20 * 2^-24 < 2^-18 of the value, before the rounding to the output's type.
"""
import pytest
import torch

from prism_infer_b200 import capi, ops  # noqa: F401
from oracle.scored_routing import route_scored_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
RTOL = {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -8 + 2.0 ** -18}


def check(logits, k, out_dtype=None, **kw):
    ids, w, counts = capi.route_scored(logits, k, out_dtype=out_dtype, with_counts=True, **kw)
    r_ids, r_w = route_scored_ref(logits, k, **kw)
    assert torch.equal(ids, r_ids), (ids != r_ids).sum().item()
    assert w.dtype == (out_dtype or logits.dtype)
    torch.testing.assert_close(w.double(), r_w, rtol=RTOL[w.dtype], atol=1e-30, equal_nan=True)
    E = logits.shape[1]
    assert torch.equal(counts.long(), torch.bincount(ids.flatten(), minlength=E))
    return ids, w


def logits_of(T, E, dtype, seed, spread=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(T, E, generator=gen, device=DEV)).to(dtype)


def bias_of(E, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return 0.1 * torch.randn(E, generator=gen, device=DEV)


SHAPES = [(1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (777, 128, 8, 1, 1), (333, 256, 8, 8, 4),
          (65, 60, 4, 3, 2), (5, 60, 6, 5, 1), (129, 160, 6, 8, 3), (33, 31, 31, 1, 1),
          (7, 34, 2, 17, 9), (9, 1024, 32, 1, 1), (4, 1008, 16, 18, 5), (50, 32, 20, 32, 20),
          (11, 513, 3, 1, 1), (6, 96, 5, 32, 2)]


@pytest.mark.parametrize("T,E,k,groups,keep", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_choice_and_weights(T, E, k, groups, keep, scoring, dtype):
    logits = logits_of(T, E, dtype, E + k)
    for bias in (None, bias_of(E, 3)):
        for score in ("max", "top2"):
            check(logits, k, scoring=scoring, bias=bias, num_groups=groups, topk_groups=keep,
                  group_score=score, renorm=True, scale=2.5)
    check(logits, k, scoring=scoring, num_groups=groups, topk_groups=keep, renorm=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_ties_go_to_the_lowest_index(scoring, groups, keep):
    gen = torch.Generator(device=DEV).manual_seed(5)
    logits = (torch.randint(0, 3, (300, 64), generator=gen, device=DEV) * 0.5).to(torch.bfloat16)
    for bias in (None, torch.zeros(64, device=DEV)):
        for score in ("max", "top2"):
            check(logits, 8, scoring=scoring, bias=bias, num_groups=groups, topk_groups=keep,
                  group_score=score)
    check(torch.zeros(3, 64, device=DEV), 8, scoring=scoring, num_groups=groups, topk_groups=keep)


def near_ties(T, E, seed):
    """fp32 logits and biases whose keys differ by less than 32-bit scores resolve."""
    logits = logits_of(1, E, torch.float32, seed).expand(T, E).clone()
    step = torch.arange(E, device=DEV) % 5 - 2
    bias = (0.75 - torch.sigmoid(logits[0].double())).float()
    ulps = logits.view(torch.int32) + torch.randint(-3, 4, (T, E), device=DEV).int()
    return ulps.view(torch.float32), bias + step * 2.0 ** -26


@pytest.mark.parametrize("groups,keep", [(1, 1), (8, 3)])
def test_keys_closer_than_32_bits_resolve(groups, keep):
    logits, bias = near_ties(200, 128, 11)
    for score in ("max", "top2"):
        check(logits, 8, scoring="sigmoid", bias=bias, num_groups=groups, topk_groups=keep,
              group_score=score)
    sm = logits_of(1, 128, torch.float32, 2).expand(200, 128) * 1e-4
    sm = (sm.contiguous().view(torch.int32) + torch.randint(-3, 4, (200, 128), device=DEV).int())
    check(sm.view(torch.float32), 8, scoring="softmax", num_groups=groups, topk_groups=keep)


def test_saturated_scores():
    logits = torch.linspace(-120, 120, 128, device=DEV).repeat(4, 1)
    logits[1] = logits[1].flip(0)
    logits[2] = 20 + 0.01 * torch.arange(128, device=DEV)       # 1 - s below 32-bit resolution
    logits[3] = 40 + torch.arange(128, device=DEV)              # s is 1 in 64 bits too: ties
    check(logits, 8, scoring="sigmoid")
    check(logits, 8, scoring="sigmoid", bias=torch.zeros(128, device=DEV), num_groups=4,
          topk_groups=2, group_score="top2")
    check(logits, 8, scoring="softmax")


def test_masked_experts_and_infinities():
    logits = logits_of(20, 32, torch.float32, 4)
    bias = torch.zeros(32, device=DEV)
    bias[4:] = float("-inf")                        # four experts left, eight wanted
    check(logits, 8, scoring="sigmoid", bias=bias)
    low = logits.clone()
    low[:, 3:] = float("-inf")
    check(low, 6, scoring="softmax")
    check(low, 6, scoring="sigmoid")
    lowest = logits.clone()
    lowest[:, 3:] = torch.finfo(torch.float32).min
    check(lowest, 6, scoring="softmax")
    check(lowest, 6, scoring="sigmoid")
    bias[4:] = 1e30                                 # a bias so large that it hides the scores
    check(logits, 6, scoring="sigmoid", bias=bias)


def test_nan_ranks_first_and_shows():
    logits = logits_of(8, 32, torch.float32, 6)
    logits[2, 17] = float("nan")
    logits[5, :] = float("nan")
    logits[6, 3] = float("inf")
    logits[7, :] = float("-inf")
    for scoring in ("sigmoid", "softmax"):
        ids, w = check(logits, 4, scoring=scoring, num_groups=4, topk_groups=2)
        assert ids[2, 0] == (17 if scoring == "sigmoid" else 0)
        assert w[2].isnan().all() and w[5].isnan().all()
        assert not w[:2].isnan().any()


def test_output_type_and_operator():
    logits = logits_of(17, 64, torch.float32, 8)
    bias = bias_of(64, 1)
    check(logits, 6, out_dtype=torch.bfloat16, scoring="sigmoid", bias=bias)
    check(logits.bfloat16(), 6, out_dtype=torch.float32, scoring="softmax", bias=bias)
    ids, w = torch.ops.prism_moe.route_scored(logits, 6, "sigmoid", bias, 4, 2, "top2", True, 2.0,
                                              torch.bfloat16)
    r_ids, _, _ = capi.route_scored(logits, 6, scoring="sigmoid", bias=bias, num_groups=4,
                                    topk_groups=2, group_score="top2", scale=2.0)
    assert torch.equal(ids, r_ids) and w.dtype == torch.bfloat16


def test_no_tokens():
    ids, w, counts = capi.route_scored(torch.empty(0, 64, device=DEV), 4, with_counts=True)
    assert ids.shape == w.shape == (0, 4) and counts.sum() == 0


def test_other_stream_and_graph():
    logits = logits_of(100, 128, torch.float32, 9)
    other = logits_of(100, 128, torch.float32, 10)
    bias = bias_of(128, 2)
    kw = dict(scoring="sigmoid", bias=bias, num_groups=8, topk_groups=4, group_score="top2")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ids, w, _ = capi.route_scored(logits, 8, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(ids, route_scored_ref(logits, 8, **kw)[0])
    graph = torch.cuda.CUDAGraph()
    static = logits.clone()
    with torch.cuda.graph(graph):
        g_ids, g_w, g_counts = capi.route_scored(static, 8, with_counts=True, **kw)
    for src in (other, logits):
        static.copy_(src)
        graph.replay()
        r_ids, _ = route_scored_ref(src, 8, **kw)
        assert torch.equal(g_ids, r_ids)
        assert torch.equal(g_counts.long(), torch.bincount(r_ids.flatten(), minlength=128))
