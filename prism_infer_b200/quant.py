"""4-bit weights with group scales: the values they stand for and the layout the kernels read.

``W[n, k] = (code[n, k] - zero[n, k // G]) * scale[n, k // G]`` with codes 0..15, bf16 scales, one
scale per row and group of G = 32, 64 or 128 inputs, and optional 4-bit zero points (8 without).
``W4Weight`` holds one matrix, or a stack of one per expert, in the tiled layout that
``include/prism_moe.h`` (``prism_moe_w4``) defines. Weights are laid out once, when a model is
loaded; everything here is plain torch and runs on any device.

The reference keeps its linear weights in bf16 (prism_infer/layers/linear.py:63-182) and has no
quantised form.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

GROUP_SIZES = (32, 64, 128)
_TILE_N, _TILE_K = 16, 128


@dataclass(frozen=True)
class W4Weight:
    """A 4-bit matrix [out_features, in_features], or a stack of them (leading dimension).

    ``qweight`` uint8 [.., N/16, ceil(K/128), 16, 64], ``scales`` bf16 and ``zeros`` uint8 (or None)
    [.., N/16, ceil(K/128), 16, 128/G]. With ``gate_up`` the rows are those of a gate_up matrix
    [2I, K], 8 gate rows and 8 up rows by turns. ``out_features`` is 2I then.
    """
    qweight: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None
    out_features: int
    in_features: int
    group_size: int
    gate_up: bool = False

    def __post_init__(self):
        N, K, G = self.out_features, self.in_features, self.group_size
        if G not in GROUP_SIZES:
            raise RuntimeError(f"group_size {G} is not one of {GROUP_SIZES}")
        if K < 1 or N < 1 or K % G:
            raise RuntimeError(f"{K} inputs are not a multiple of group_size {G}")
        if N % (16 if self.gate_up else 8):
            raise RuntimeError(f"{N} outputs: 4-bit weights need a multiple of 8 (gate_up: 16)")
        tiles = (-(-N // _TILE_N), -(-K // _TILE_K), _TILE_N)
        lead = tuple(self.qweight.shape[:-4])
        if len(lead) > 1 or tuple(self.qweight.shape) != lead + tiles + (64,):
            raise RuntimeError(f"qweight {tuple(self.qweight.shape)} does not hold [{N}, {K}]")
        for name, t, dt in (("qweight", self.qweight, torch.uint8),
                            ("scales", self.scales, torch.bfloat16),
                            ("zeros", self.zeros, torch.uint8)):
            if t is None and name == "zeros":
                continue
            if t.dtype != dt:
                raise RuntimeError(f"{name} must be {dt}, got {t.dtype}")
            if name != "qweight" and tuple(t.shape) != lead + tiles + (_TILE_K // G,):
                raise RuntimeError(f"{name} {tuple(t.shape)} does not match the weight")
            if t.device != self.qweight.device:
                raise RuntimeError("4-bit weight parts are on different devices")
            if not t.is_contiguous():
                raise RuntimeError("4-bit weights must be contiguous")

    @property
    def stack(self) -> int | None:
        """Matrices in the stack (None: a single matrix)."""
        return self.qweight.shape[0] if self.qweight.dim() == 5 else None

    @property
    def device(self) -> torch.device:
        return self.qweight.device

    def to(self, device) -> "W4Weight":
        z = None if self.zeros is None else self.zeros.to(device)
        return W4Weight(self.qweight.to(device), self.scales.to(device), z, self.out_features,
                        self.in_features, self.group_size, self.gate_up)


def _turns(v: torch.Tensor) -> torch.Tensor:
    """Rows [gate; up] (dimension -2) -> 8 gate and 8 up rows by turns."""
    *lead, n, c = v.shape
    return v.view(*lead, 2, n // 16, 8, c).transpose(-4, -3).reshape(*lead, n, c)


def _unturn(v: torch.Tensor) -> torch.Tensor:
    *lead, n, c = v.shape
    return v.view(*lead, n // 16, 2, 8, c).transpose(-4, -3).reshape(*lead, n, c)


def _pack_codes(codes: torch.Tensor) -> torch.Tensor:
    *lead, N, K = codes.shape
    codes = F.pad(codes, (0, -K % _TILE_K, 0, -N % _TILE_N), value=8)
    n16, c = codes.shape[-2] // _TILE_N, codes.shape[-1] // _TILE_K
    # [row tile, row, chunk, j, t, pair, half] -> [row tile, chunk, row, t, j, half, pair]
    v = codes.reshape(-1, n16, 16, c, 4, 4, 4, 2).permute(0, 1, 3, 2, 5, 4, 7, 6)
    v = v.reshape(*lead, n16, c, 16, 16, 8)
    return (v[..., 0::2] | (v[..., 1::2] << 4)).reshape(*lead, n16, c, 16, 64)


def _unpack_codes(q: torch.Tensor, N: int, K: int) -> torch.Tensor:
    *lead, n16, c, _, _ = q.shape
    v = torch.stack([q & 15, q >> 4], dim=-1).reshape(-1, n16, c, 16, 4, 4, 2, 4)
    v = v.permute(0, 1, 3, 2, 5, 4, 7, 6).reshape(*lead, n16 * 16, c * 128)
    return v[..., :N, :K]


def _pack_groups(v: torch.Tensor, G: int) -> torch.Tensor:
    *lead, N, n_groups = v.shape
    per = _TILE_K // G
    v = F.pad(v, (0, -n_groups % per, 0, -N % _TILE_N))
    return v.reshape(*lead, v.shape[-2] // 16, 16, v.shape[-1] // per,
                     per).transpose(-3, -2).contiguous()


def _unpack_groups(v: torch.Tensor, N: int, n_groups: int) -> torch.Tensor:
    *lead, n16, c, _, per = v.shape
    return v.transpose(-3, -2).reshape(*lead, n16 * 16, c * per)[..., :N, :n_groups]


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
            group_size: int, gate_up: bool = False) -> W4Weight:
    """Lay out ``codes`` [.., N, K] (integers 0..15), ``scales`` and ``zeros`` [.., N, K/G] (any
    quantiser's result); scales are rounded to bf16 and must be finite there. With ``gate_up`` the N
    rows are the I gate rows, then the I up rows."""
    N, K = codes.shape[-2:]
    if group_size not in GROUP_SIZES:
        raise RuntimeError(f"group_size {group_size} is not one of {GROUP_SIZES}")
    if K % group_size:
        raise RuntimeError(f"{K} inputs are not a multiple of group_size {group_size}")
    if N % (16 if gate_up else 8):
        raise RuntimeError(f"{N} outputs: 4-bit weights need a multiple of 8 (gate_up: 16)")
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t is not None and tuple(t.shape) != (*codes.shape[:-1], K // group_size):
            raise RuntimeError(f"{name} {tuple(t.shape)} do not match codes {tuple(codes.shape)}")
    for name, t in (("codes", codes), ("zeros", zeros)):
        if t is not None and t.numel() and (t.is_floating_point() or int(t.min()) < 0
                                            or int(t.max()) > 15):
            raise RuntimeError(f"{name} must be integers in 0..15")
    scales = scales.to(torch.bfloat16)
    if not bool(scales.isfinite().all()):
        raise RuntimeError("scales must be finite in bfloat16")
    parts = [codes.to(torch.uint8), scales,
             None if zeros is None else zeros.to(torch.uint8)]
    if gate_up:
        parts = [None if t is None else _turns(t) for t in parts]
    q, s, z = parts
    return W4Weight(_pack_codes(q), _pack_groups(s, group_size),
                    None if z is None else _pack_groups(z, group_size), N, K, group_size, gate_up)


def quantize_w4(weight: torch.Tensor, group_size: int = 128, *, symmetric: bool = True,
                gate_up: bool = False) -> W4Weight:
    """Round a weight [.., N, K] to the nearest 4-bit values of its groups.

    ``symmetric``: codes 1..15 around zero point 8, scale = largest magnitude / 7. Otherwise a zero
    point per group, scale = (max - min) / 15 over the group and zero, so that zero stays exact.
    The scale is rounded to bf16 before the codes are chosen. A group of zeros gets scale 1. Weights
    that are not finite, or whose scale is not, are refused.
    """
    if group_size not in GROUP_SIZES:
        raise RuntimeError(f"group_size {group_size} is not one of {GROUP_SIZES}")
    weight = weight.detach()
    *lead, N, K = weight.shape
    if K % group_size:
        raise RuntimeError(f"{K} inputs are not a multiple of group_size {group_size}")

    def one(w):   # a matrix at a time: the fp32 copies of a whole stack need not fit
        w = w.float().view(N, K // group_size, group_size)
        if symmetric:
            s = w.abs().amax(-1) / 7
        else:
            lo, hi = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
            s = (hi - lo) / 15
        if not bool(s.to(torch.bfloat16).isfinite().all()):   # a NaN weight makes its scale NaN
            raise RuntimeError("quantize_w4: weights and their scales must be finite")
        s = torch.where(s > 0, s, torch.ones_like(s)).to(torch.bfloat16)
        s = s.clamp_min(torch.finfo(torch.bfloat16).tiny)
        sf = s.float().unsqueeze(-1)
        z = torch.full_like(s, 8, dtype=torch.float32) if symmetric else \
            (-lo / sf[..., 0]).round().clamp_(0, 15)
        q = ((w / sf).round() + z.unsqueeze(-1)).clamp_(0, 15)
        return q.view(N, K).to(torch.uint8), s, None if symmetric else z.to(torch.uint8)

    parts = [one(w) for w in weight.reshape(-1, N, K)]
    codes, scales, zeros = (None if p[0] is None else torch.stack(p).view(*lead, N, -1)
                            for p in zip(*parts))
    return pack_w4(codes, scales, zeros, group_size=group_size, gate_up=gate_up)


def dequantize_w4(w: W4Weight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [.., N, K] a 4-bit weight stands for; gate_up rows come back as [gate; up]."""
    N, K, G = w.out_features, w.in_features, w.group_size
    codes = _unpack_codes(w.qweight, N, K).to(dtype)
    s = _unpack_groups(w.scales, N, K // G).to(dtype).repeat_interleave(G, dim=-1)
    z = 8.0 if w.zeros is None else \
        _unpack_groups(w.zeros, N, K // G).to(dtype).repeat_interleave(G, dim=-1)
    v = (codes - z) * s
    return _unturn(v) if w.gate_up else v
