"""Scored routing where 32-bit keys do not decide: the choice is that of 64-bit keys, exactly."""
import pytest
import torch

from prism_infer_b200 import capi
from oracle.scored_routing import route_scored_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check_ids(logits, k, **kw):
    ids, w, _ = capi.route_scored(logits, k, **kw)
    r_ids, r_w = route_scored_ref(logits, k, **kw)
    wrong = (ids != r_ids).any(-1)
    assert not wrong.any(), (int(wrong.sum()), ids[wrong][:3].tolist(), r_ids[wrong][:3].tolist())
    return w, r_w


# ------------------------------------------------------------------------------ ties at the cut

def test_tie_at_the_cut_with_a_better_third():
    """Two equal keys meet at the cut; a third, equal in 32 bits, is larger in 64."""
    for dtype in (torch.bfloat16, torch.float32):
        logits = torch.tensor([[14, 14, 14.0625], [14, 14.0625, 14], [14.0625, 14, 14]],
                              device=DEV, dtype=dtype)
        check_ids(logits, 1, scoring="sigmoid", bias=torch.zeros(3, device=DEV))


@pytest.mark.parametrize("k", [1, 3, 8, 29, 32])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("ties", [2, 3, 9])
def test_tie_at_the_cut_among_biased_keys(k, scoring, ties):
    """k - 1 certain choices, then ``ties`` equal keys and one 2^-24 of a key above them."""
    E, T, g = 160, 40, gen_of(k)
    order = torch.rand(T, E, generator=g, device=DEV).argsort(-1)
    logits = torch.full((T, E), -3.0, device=DEV)
    where = order[:, :ties + 1]
    logits.scatter_(1, where, 2.0)
    logits.scatter_(1, where[:, :1], 2.0 + 2.0 ** -22)
    bias = torch.full((E,), 0.5, device=DEV)
    for row in range(T):                 # a bias belongs to an expert: rows one by one
        b = bias.clone()
        b[order[row, ties + 1:ties + k]] = 1.5 + 0.01 * torch.arange(k - 1, device=DEV)
        check_ids(logits[row:row + 1], k, scoring=scoring, bias=b)


@pytest.mark.parametrize("k", [1, 2, 5, 8, 27, 29, 32])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 3), (3, 2)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_ties_and_close_keys_together(k, groups, keep, scoring):
    """bf16 logits of few values and biases in fixed steps: many equal keys, many within a rounding."""
    g = gen_of(100 * k + groups)
    steps = torch.randint(0, 24, (600, 96), generator=g, device=DEV)
    high = 12 if scoring == "sigmoid" else 0
    logits = (high + 0.0625 * steps).to(torch.bfloat16)
    if scoring == "softmax":   # all scores small beside the biases
        logits[:, 7] = 14
    bias = 0.5 + 0.001 * torch.randint(-2, 3, (96,), generator=g, device=DEV)
    for b in (torch.zeros(96, device=DEV), bias):
        for score in ("max", "top2"):
            check_ids(logits, k, scoring=scoring, bias=b, num_groups=groups, topk_groups=keep,
                      group_score=score)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_logits_that_only_32_bits_tell_apart(scoring):
    """Logits so small that their 64-bit scores are equal: ties, which go to the lowest index."""
    logits = torch.full((4, 16), -5.0, device=DEV)
    logits[0, :3] = torch.tensor([0.0, 1e-20, 1e-20])
    logits[1, 4:8] = torch.tensor([1e-20, 1e-20, 0.0, 2e-20])
    logits[2, 1:16:4] = torch.tensor([0.0, 1e-20, 1e-20, 1e-20], device=DEV)
    logits[3, 1:16:4] = torch.tensor([1e-20, 1e-20, 2e-20, -1e-20], device=DEV)
    for k in (1, 2, 3):
        check_ids(logits, k, scoring=scoring)
        for keep in (1, 2, 3):
            check_ids(logits, k, scoring=scoring, num_groups=4, topk_groups=keep)


@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min, -100.0, -17.0])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(8, 3), (6, 4), (5, 2)])
def test_groups_that_are_masked(value, scoring, groups, keep):
    """Whole groups at a masking value, more of them than go, and by rows also less."""
    E = 240
    g = gen_of(groups)
    logits = torch.randn(200, E, generator=g, device=DEV)
    masked = torch.rand(200, groups, generator=g, device=DEV) < 0.5
    logits[masked.repeat_interleave(E // groups, 1)] = value
    logits[0] = value
    bias = 0.1 * torch.randn(E, generator=g, device=DEV)
    for b in (None, bias, torch.zeros(E, device=DEV)):
        for score in ("max", "top2"):
            ids, w, _ = capi.route_scored(logits, 8, scoring=scoring, bias=b, num_groups=groups,
                                          topk_groups=keep, group_score=score)
            r_ids, r_w = route_scored_ref(logits, 8, scoring=scoring, bias=b, num_groups=groups,
                                          topk_groups=keep, group_score=score)
            assert torch.equal(ids, r_ids)
            torch.testing.assert_close(w.double(), r_w, rtol=2.0 ** -18, atol=9 * 2.0 ** -148 / 1e-20,
                                       equal_nan=True)


# ------------------------------------------------------------------------------ the bottom of the range

@pytest.mark.parametrize("score", ["max", "top2"])
def test_keys_at_the_bottom_of_the_range(score):
    """Sigmoid scores around the smallest normal fp32 number, which 32 bits round to 0 or nearly so."""
    logits = torch.tensor([[-87.3, -200.0, -87.4, -87.4]], device=DEV)
    check_ids(logits, 2, scoring="sigmoid", num_groups=2, group_score=score)
    logits = -104 + 18 * torch.rand(300, 64, generator=gen_of(1), device=DEV)
    tiny = 1e-38 * torch.randn(64, generator=gen_of(2), device=DEV)
    for bias in (None, torch.zeros(64, device=DEV), tiny):
        for groups, keep in ((1, 1), (8, 3), (8, 8)):
            check_ids(logits, 6, scoring="sigmoid", bias=bias, num_groups=groups, topk_groups=keep,
                      group_score=score)


@pytest.mark.parametrize("renorm", [False, True])
def test_weights_of_scores_that_underflow(renorm):
    """A subnormal score is within 2^-148 (expf's 2 ulp); the sum of 8 of them is within 2^-145, and
    renormalising divides either by 1e-20 at least: 9 * 2^-148 / 1e-20 for a weight."""
    k = 8
    logits = -104 + 16 * torch.rand(300, 64, generator=gen_of(5), device=DEV)
    w, ref = check_ids(logits, k, scoring="sigmoid", renorm=renorm)
    atol = 9 * 2.0 ** -148 / 1e-20 if renorm else 2.0 ** -148
    torch.testing.assert_close(w.double(), ref, rtol=2.0 ** -18, atol=atol)
    assert (ref > 1e3 * atol).any()


@pytest.mark.parametrize("scoring,renorm", [("softmax", False), ("softmax", True), ("sigmoid", False),
                                            ("sigmoid", True)])
def test_which_weights_a_nan_logit_reaches(scoring, renorm):
    logits = torch.randn(4, 32, generator=gen_of(6), device=DEV)
    logits[1, 9] = float("nan")
    w, ref = check_ids(logits, 4, scoring=scoring, renorm=renorm)
    assert torch.equal(w.isnan(), ref.isnan())
    assert w[1].isnan().sum() == (1 if scoring == "sigmoid" and not renorm else 4)


# ------------------------------------------------------------------------------ who looks again

SWEEP = [(300, 33, 8, 3, 2), (300, 60, 6, 5, 3), (300, 60, 6, 6, 4), (200, 384, 8, 3, 2),
         (200, 102, 29, 17, 9), (200, 40, 32, 5, 4), (200, 9, 6, 3, 2), (200, 64, 8, 8, 8),
         (200, 512, 8, 1, 1), (100, 1008, 16, 18, 5)]


@pytest.mark.parametrize("T,E,k,groups,keep", SWEEP)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_near_ties_at_every_count(T, E, k, groups, keep, scoring):
    """Keys a few ulp apart, at group counts of no power of two, all groups kept, k + 4 above 32 or
    above the experts that stay."""
    g = gen_of(E + k)
    row = torch.randn(1, E, generator=g, device=DEV).expand(T, E).clone()
    logits = (row.view(torch.int32) +
              torch.randint(-3, 4, (T, E), generator=g, device=DEV, dtype=torch.int32)).view(torch.float32)
    score = torch.sigmoid(row[0].double()) if scoring == "sigmoid" else \
        torch.softmax(row[0].double(), -1)
    level = (0.75 - score).float() + 2.0 ** -26 * (torch.arange(E, device=DEV) % 5 - 2)
    bf16 = row.to(torch.bfloat16)
    for l, bias in ((logits, None), (logits, level), (bf16, None), (bf16, level)):
        for group_score in ("max", "top2"):
            check_ids(l, k, scoring=scoring, bias=bias, num_groups=groups, topk_groups=keep,
                      group_score=group_score)


def time_of(logits, **kw):
    """Shortest of some graph replays of ten calls."""
    capi.route_scored(logits, 8, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            capi.route_scored(logits, 8, **kw)
    best = float("inf")
    for _ in range(20):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def test_ordinary_rows_are_decided_in_32_bits():
    """Three groups, or all groups kept, cost no more than their neighbours: when every row of them
    took the 64-bit path the times were 3.4 and 4.1 apart."""
    logits = torch.randn(8192, 384, generator=gen_of(3), device=DEV)
    kw = dict(scoring="sigmoid", group_score="top2", bias=0.1 * torch.randn(384, generator=gen_of(4), device=DEV))
    assert time_of(logits, num_groups=3, topk_groups=2, **kw) < \
        2 * time_of(logits, num_groups=4, topk_groups=2, **kw)
    logits = logits[:, :256].contiguous()
    assert time_of(logits, scoring="sigmoid", num_groups=8, topk_groups=8) < \
        2 * time_of(logits, scoring="sigmoid")
