"""Scored routing in plain 64-bit torch, straight from its definition (test infrastructure)."""
import torch


def route_scored_ref(logits, k, *, scoring="softmax", bias=None, num_groups=1, topk_groups=1,
                     group_score="max", renorm=True, scale=1.0):
    """(ids int64 [T, k], weights float64 [T, k])."""
    l = logits.double()
    T, E = l.shape
    if scoring == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        e = torch.exp(l - l.max(-1, keepdim=True).values)
        s = e / e.sum(-1, keepdim=True)
    key = s if bias is None else s + bias.double()
    best = torch.sort(key.view(T, num_groups, -1), dim=-1, descending=True).values
    gs = best[..., 0]
    if group_score == "top2" and best.shape[-1] > 1:
        gs = gs + best[..., 1]
    order = torch.sort(gs, dim=-1, descending=True, stable=True).indices[:, :topk_groups]
    stays = torch.zeros(T, num_groups, dtype=torch.bool, device=l.device).scatter_(1, order, True)
    stays = stays.repeat_interleave(E // num_groups, 1)
    # all keys in order, then those that stay first, order kept
    by_key = torch.sort(key, dim=-1, descending=True, stable=True).indices
    first = torch.sort(~stays.gather(1, by_key), dim=-1, stable=True).indices
    ids = by_key.gather(1, first)[:, :k].contiguous()
    w = s.gather(1, ids)
    if renorm:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return ids, w * scale
