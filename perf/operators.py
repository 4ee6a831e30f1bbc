"""What the block's scored router and its 4-bit weight products are measured on.

``listed()`` names the cases, ``draw()`` gives more of the same ranges. ``run`` computes a case in
its plain form (elementary torch operations in 32 or 64 bits) or, where ``own`` is set, through
the package's entry points. ``exact`` is the definition in 64 bits.

Operators (T tokens, E experts, k chosen; M or R rows, N outputs, K inputs, groups of G inputs):

* ``route``    scores s = softmax(l) or sigmoid(l); selection keys s + bias; the best expert groups by
               their largest key or by the sum of their two largest; the k largest keys in them, ties
               to the lowest index; weights s[ids] / (sum + 1e-20) * scale.
* ``linear``   y = x W^T with W[n, k] = (code - zero) * scale, one scale (and zero) per row and G
               inputs; zero is 8 where the weights carry none.
* ``experts``  rows of x, grouped by expert: y = (silu(x Wg^T) * (x Wu^T)) Wd^T on such weights.

4-bit weights are held as the package holds them: tiles of 16 rows by 128 inputs, 1 KB each; a row's
64 bytes are 16 words of 8 codes, the word at 4 t + j holding inputs 32 j + 8 t and on, nibbles in
the order 0 2 4 6 1 3 5 7. Scales and zeros follow the tiles. Gate and up rows alternate by 8.
"""
from __future__ import annotations

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------ cases

def _route(name, T, E, k, scoring, dtype, bias, groups, keep, group_score, renorm, scale):
    return dict(name=name, op="route", T=T, E=E, k=k, scoring=scoring, dtype=dtype, bias=bias,
                groups=groups, keep=keep, group_score=group_score, renorm=renorm, scale=scale)


def _linear(name, M, N, K, G, zeros):
    return dict(name=name, op="linear", M=M, N=N, K=K, G=G, zeros=zeros)


def _experts(name, T, E, k, H, I, G, zeros, skew):
    return dict(name=name, op="experts", T=T, E=E, k=k, H=H, I=I, G=G, zeros=zeros, skew=skew)


def listed():
    return [
        # one token of a decode step, grouped sigmoid routing with a balance bias: latency
        _route("route_one_token", 1, 256, 8, "sigmoid", "float32", True, 8, 4, "top2", True, 2.5),
        # a decode batch routed by plain sigmoid scores, the block's own expert count
        _route("route_decode", 64, 128, 8, "sigmoid", "bfloat16", True, 1, 1, "max", True, 1.0),
        # a prefill batch, grouped sigmoid routing from fp32 logits
        _route("route_prefill", 8192, 256, 8, "sigmoid", "float32", True, 8, 4, "top2", True, 2.5),
        # ragged prefill, softmax scores limited to the best groups, weights kept unnormalised
        _route("route_softmax_groups", 4097, 160, 6, "softmax", "bfloat16", False, 8, 3, "max",
               False, 16.0),
        # one token through a square projection: a matrix-vector product
        _linear("linear_one_token", 1, 4096, 4096, 128, False),
        # a small ragged batch, inputs that end inside a tile, zero points, small groups
        _linear("linear_ragged", 17, 2056, 1440, 32, True),
        # a prefill batch through a wide projection
        _linear("linear_prefill", 2048, 4096, 2048, 128, False),
        # one token through its 8 experts
        _experts("experts_one_token", 1, 128, 8, 2048, 768, 128, False, 0.0),
        # the decode batch of the benchmark: nearly every expert's weights are read
        _experts("experts_decode", 64, 128, 8, 2048, 768, 128, False, 0.0),
        # uneven loads (some experts empty), odd sizes, zero points, small groups
        _experts("experts_ragged", 333, 60, 4, 1440, 736, 32, True, 1.5),
        # the benchmark's skewed batch: long and short experts in one call
        _experts("experts_skewed", 4096, 128, 8, 2048, 768, 64, True, 0.7),
        # a long prefill of wide experts: bound by the tensor cores
        _experts("experts_prefill", 8192, 32, 4, 4096, 1024, 128, False, 0.0),
    ]


def _log_int(rng, lo, hi):
    import math
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "linear", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log_int(rng, 4, 256 // groups)
        E = groups * per
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(16, keep * per))
        case = _route("", _log_int(rng, 1, 8192), E, k, rng.choice(["softmax", "sigmoid"]),
                      rng.choice(["bfloat16", "float32"]), rng.random() < 0.6, groups, keep,
                      rng.choice(["max", "top2"]), rng.random() < 0.7,
                      rng.choice([1.0, 2.5, 16.0]))
    elif op == "linear":
        G = rng.choice([32, 64, 128])
        case = _linear("", _log_int(rng, 1, 2048), 8 * _log_int(rng, 4, 512),
                       G * _log_int(rng, 1, 4096 // G), G, rng.random() < 0.5)
    else:
        G = rng.choice([32, 64, 128])
        E = _log_int(rng, 4, 128)
        H = G * _log_int(rng, 1, 2048 // G)
        I = G * _log_int(rng, 1, 1024 // G)
        case = _experts("", _log_int(rng, 1, 4096), E, rng.randint(1, min(8, E)), H, I, G,
                        rng.random() < 0.5, rng.choice([0.0, 0.7, 1.5]))
    del case["name"]
    return case


# ------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pack(codes):
    """uint8 codes [..., N, K] -> tiles [..., N/16, K/128, 16, 64], both sizes padded with code 8."""
    N, K = codes.shape[-2:]
    codes = torch.nn.functional.pad(codes, (0, -K % 128, 0, -N % 16), value=8)
    lead = codes.shape[:-2]
    n16, c = codes.shape[-2] // 16, codes.shape[-1] // 128
    # from [row tile, row, chunk, j, t, pair, half] to [row tile, chunk, row, t, j, half, pair]
    v = codes.view(*lead, n16, 16, c, 4, 4, 4, 2)
    d = len(lead)
    v = v.permute(*range(d), d, d + 2, d + 1, d + 4, d + 3, d + 6, d + 5).reshape(*lead, -1, 8)
    b = v[..., 0::2] | (v[..., 1::2] << 4)          # two nibbles to a byte, low first
    return b.reshape(*lead, n16, c, 16, 64)


def _tile_groups(v, G):
    """Per-group values [..., N, K/G] -> [..., N/16, K/128, 16, 128/G], padded with 0."""
    N, n_groups = v.shape[-2:]
    per = 128 // G
    v = torch.nn.functional.pad(v, (0, -n_groups % per, 0, -N % 16))
    lead = v.shape[:-2]
    return v.view(*lead, v.shape[-2] // 16, 16, v.shape[-1] // per, per).transpose(-3, -2).contiguous()


def _weights(gen, lead, N, K, G, zeros):
    """4-bit weights of the spread that round-to-nearest gives: values near N(0, 1/sqrt(K))."""
    n_groups = K // G
    q = torch.randn(*lead, N, K, generator=gen, device=DEV, dtype=torch.bfloat16)
    codes = (q.mul_(2.7).round_() + 8).clamp_(0, 15).to(torch.uint8)
    spread = 0.5 + torch.rand(*lead, N, n_groups, generator=gen, device=DEV)
    scales = (spread / (2.7 * K ** 0.5)).to(torch.bfloat16)
    z = None
    if zeros:
        z = torch.randint(6, 11, (*lead, N, n_groups), generator=gen, device=DEV).to(torch.uint8)
        z = _tile_groups(z, G)
    return dict(q=_pack(codes), s=_tile_groups(scales, G), z=z, N=N, K=K, G=G)


def prepare(case, seed):
    gen = _gen(seed)
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        dtype = getattr(torch, case["dtype"])
        logits = torch.randn(T, E, generator=gen, device=DEV)
        # experts differ in popularity, as a trained router's do
        logits = (logits + 0.5 * torch.randn(E, generator=gen, device=DEV)).to(dtype)
        bias = 0.1 * torch.randn(E, generator=gen, device=DEV) if case["bias"] else None
        return dict(case=case, logits=logits, bias=bias)
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x = torch.randn(M, K, generator=gen, device=DEV).to(torch.bfloat16)
        st = dict(case=case, x=x, w=_weights(gen, (), N, K, case["G"], case["zeros"]))
    else:
        T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
        pull = torch.randn(T, E, generator=gen, device=DEV)
        pull += case["skew"] * torch.randn(E, generator=gen, device=DEV)
        ids = torch.topk(pull, k, dim=-1).indices
        counts = torch.bincount(ids.flatten(), minlength=E)
        off = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        off[1:] = torch.cumsum(counts, 0)
        x = torch.randn(T * k, H, generator=gen, device=DEV).to(torch.bfloat16)
        st = dict(case=case, x=x, off=off, bounds=off.tolist(),
                  gu=_weights(gen, (E,), 2 * I, H, case["G"], case["zeros"]),
                  dn=_weights(gen, (E,), H, I, case["G"], case["zeros"]))
    if own:
        from prism_infer_b200.quant import W4Weight
        for key in ("w", "gu", "dn"):
            if key in st:
                w = st[key]
                st["own_" + key] = W4Weight(w["q"], w["s"], w["z"], w["N"], w["K"], w["G"],
                                            gate_up=key == "gu")
    return st


# ------------------------------------------------------------------------------------ the passes

def run(state):
    case = state["case"]
    if own:
        from prism_infer_b200 import capi
        if case["op"] == "route":
            ids, w, _ = capi.route_scored(
                state["logits"], case["k"], scoring=case["scoring"], bias=state["bias"],
                num_groups=case["groups"], topk_groups=case["keep"],
                group_score=case["group_score"], renorm=case["renorm"], scale=case["scale"])
            return [ids, w]
        if case["op"] == "linear":
            return capi.linear_w4(state["x"], state["own_w"])
        return capi.expert_swiglu_w4(state["x"], state["off"], state["own_gu"], state["own_dn"])
    if case["op"] == "route":
        return _plain_route(state)
    if case["op"] == "linear":
        w = _plain_weight(state["w"], state["w"]["q"], state["w"]["s"], state["w"]["z"])
        return (state["x"].float() @ w.t()).to(torch.bfloat16)
    return _plain_experts(state)


def _plain_route(state):
    case = state["case"]
    # selection compares values that may lie close to one another: in 64 bits
    l = state["logits"].double()
    T, E = l.shape
    if case["scoring"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.max(dim=-1, keepdim=True).values)
        s = e / e.sum(dim=-1, keepdim=True)
    key = s if state["bias"] is None else s + state["bias"].double()
    if case["groups"] > 1:
        grouped = key.view(T, case["groups"], -1).sort(dim=-1, descending=True).values
        score = grouped[..., 0]
        if case["group_score"] == "top2" and grouped.shape[-1] > 1:
            score = score + grouped[..., 1]
        order = torch.sort(score, dim=-1, descending=True, stable=True).indices
        kept = torch.zeros_like(score, dtype=torch.bool)
        kept.scatter_(1, order[:, :case["keep"]], True)
        out = ~kept.repeat_interleave(E // case["groups"], dim=1)
        key = key.masked_fill(out, float("-inf"))
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :case["k"]].contiguous()
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / (w.sum(dim=-1, keepdim=True) + 1e-20)
    return [ids, (w * case["scale"]).to(state["logits"].dtype)]


def _plain_weight(w, q, s, z):
    """The 32-bit values [N, K] that one matrix's tiles stand for, in packed row order."""
    n16, c = q.shape[:2]
    nib = torch.stack([q & 15, q >> 4], dim=-1)               # byte, nibble of the byte
    nib = nib.view(n16, c, 16, 4, 4, 2, 4)                    # t, j, odd/even half, pair
    v = nib.permute(0, 2, 1, 4, 3, 6, 5).reshape(n16 * 16, c * 128).float()
    per_group = lambda a: a.permute(0, 2, 1, 3).reshape(n16 * 16, -1).float().repeat_interleave(
        w["G"], dim=1)
    zero = per_group(z) if z is not None else 8.0
    return ((v - zero) * per_group(s))[:w["N"], :w["K"]]


def _plain_experts(state):
    x, gu, dn = state["x"], state["gu"], state["dn"]
    y = torch.empty_like(x)
    at = lambda w, e: _plain_weight(w, w["q"][e], w["s"][e], None if w["z"] is None else w["z"][e])
    for e, (a, b) in enumerate(zip(state["bounds"][:-1], state["bounds"][1:])):
        if a == b:
            continue
        pairs = (x[a:b].float() @ at(gu, e).t()).view(b - a, -1, 2, 8)   # gate, up by 8
        g, u = pairs[:, :, 0].reshape(b - a, -1), pairs[:, :, 1].reshape(b - a, -1)
        h = g / (1.0 + torch.exp(-g)) * u
        y[a:b] = (h @ at(dn, e).t()).to(x.dtype)
    return y


# ------------------------------------------------------------------------------------ definition

def _exact_weight(w, e=None):
    """The values of one matrix in 64 bits, each code read at its own place."""
    q, s, z = (None if t is None else (t if e is None else t[e]) for t in (w["q"], w["s"], w["z"]))
    N, K, G = w["N"], w["K"], w["G"]
    n = torch.arange(N, device=DEV).view(-1, 1)
    k = torch.arange(K, device=DEV).view(1, -1)
    r = k % 128
    word = 4 * ((r % 32) // 8) + r // 32
    nibble = (r % 8) // 2 + 4 * (r % 2)
    byte = q[n // 16, k // 128, n % 16, 4 * word + nibble // 2].to(torch.int16)
    code = torch.bitwise_right_shift(byte, (4 * (nibble % 2)).to(torch.int16).expand_as(byte)) & 15
    where = (n // 16, k // 128, n % 16, r // G)
    zero = z[where].double() if z is not None else 8.0
    return (code.double() - zero) * s[where].double()


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(st)
    if case["op"] == "linear":
        return torch.einsum("mk,nk->mn", st["x"].double(), _exact_weight(st["w"]))
    if 6.0 * case["T"] * case["k"] * case["H"] * case["I"] > 4e13:
        return None
    x, H = st["x"], case["H"]
    y = torch.zeros(x.shape[0], H, dtype=torch.float64, device=DEV)
    for e in range(case["E"]):
        a, b = st["bounds"][e], st["bounds"][e + 1]
        if b > a:
            gu = _exact_weight(st["gu"], e)
            rows = torch.arange(2 * case["I"], device=DEV)
            is_up = (rows % 16) >= 8
            xe = x[a:b].double()
            g = torch.einsum("mk,nk->mn", xe, gu[~is_up])
            u = torch.einsum("mk,nk->mn", xe, gu[is_up])
            y[a:b] = torch.einsum("mk,nk->mn", g * torch.sigmoid(g) * u, _exact_weight(st["dn"], e))
    return y


def _exact_route(st):
    case, l = st["case"], st["logits"].double()
    T, E = l.shape
    k, groups, keep = case["k"], case["groups"], case["keep"]
    s = torch.sigmoid(l) if case["scoring"] == "sigmoid" else torch.softmax(l, dim=-1)
    key = s.clone() if st["bias"] is None else s + st["bias"].double()
    first = torch.arange(E, device=DEV)
    if groups > 1:
        per = E // groups
        parts = key.view(T, groups, per)
        best = parts.max(dim=-1)
        score = best.values.clone()
        if case["group_score"] == "top2" and per > 1:
            score += parts.scatter(2, best.indices.unsqueeze(-1), float("-inf")).max(dim=-1).values
        gi = torch.arange(groups, device=DEV)
        # a group stays when fewer than ``keep`` groups come before it
        before = (score.unsqueeze(1) > score.unsqueeze(2)) | (
            (score.unsqueeze(1) == score.unsqueeze(2)) & (gi.view(1, 1, -1) < gi.view(1, -1, 1)))
        stays = before.sum(dim=-1) < keep
        key[~stays.gather(1, (first // per).expand(T, E))] = float("-inf")
    ids = torch.empty(T, k, dtype=torch.int64, device=DEV)
    for j in range(k):
        top = key.max(dim=-1, keepdim=True).values
        ids[:, j] = torch.where(key == top, first, E).min(dim=-1).values
        key.scatter_(1, ids[:, j:j + 1], float("-inf"))
    w = s.gather(1, ids)
    if case["renorm"]:
        w = w / (w.sum(dim=-1, keepdim=True) + 1e-20)
    return [ids, w * case["scale"]]


# ------------------------------------------------------------------------------------ cost

def _w4_bytes(N, K, G, zeros):
    return N * K // 2 + N * (K // G) * (3 if zeros else 2)


def work(case):
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        es = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": T * E * es + (4 * E if case["bias"] else 0) + T * k * (8 + es),
                "flops": 4 * T * E}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": _w4_bytes(N, K, case["G"], case["zeros"]) + 2 * M * (N + K),
                "flops": 2 * M * N * K}
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    # experts that T tokens reach when each picks k of E evenly
    hit = E * (1.0 - (1.0 - k / E) ** T)
    per = _w4_bytes(2 * I, H, case["G"], case["zeros"]) + _w4_bytes(H, I, case["G"], case["zeros"])
    return {"bytes": int(hit * per) + 4 * T * k * H, "flops": 6 * T * k * H * I}
