"""ctypes binding of ``libprism_moe.so`` (the C ABI declared in ``include/prism_moe.h``).

The library is loaded on first use. There is no fallback: if the library is missing, or the
current device is not an sm_100 GPU, calls raise ``RuntimeError``.

The torch-facing helpers below validate dtype / device / contiguity, pass raw pointers and the
current CUDA stream, and raise ``RuntimeError`` with the library's message on a non-zero
status (the reference surfaces torch ``RuntimeError`` the same way, prism_infer
layers/moe.py:69-100).
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libprism_moe.so"
HEADER = Path(__file__).resolve().parent.parent / "include" / "prism_moe.h"

OK, ERR_ARG, ERR_CUDA, ERR_TIMEOUT, ERR_UNSUPPORTED, ERR_DEVICE = range(6)
F32, BF16 = 0, 1
ENGINES = {"auto": 0, "fused": 1, "single": 2, "pair": 3}
EP_STATS_FIELDS = ("epoch", "counter", "dispatch_t0_ns", "dispatch_t1_ns", "fused_t0_ns",
                   "fused_t1_ns", "send_rows", "recv_rows")

_vp, _i32, _i64, _sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t


class NormEpilogue(ctypes.Structure):
    """``prism_moe_norm_epilogue``: the decoder layer's residual add + RMSNorm fused into the
    block's combine."""
    _fields_ = [("residual", ctypes.c_void_p), ("norm_weight", ctypes.c_void_p),
                ("eps", ctypes.c_float), ("residual_out", ctypes.c_void_p)]


class Router(ctypes.Structure):
    """``prism_moe_router``: how prism_moe_route_scored scores, groups and weighs."""
    _fields_ = [("scoring", ctypes.c_int32), ("bias", ctypes.c_void_p),
                ("num_groups", ctypes.c_int32), ("topk_groups", ctypes.c_int32),
                ("group_score", ctypes.c_int32), ("renorm", ctypes.c_int32),
                ("scale", ctypes.c_float)]


class W4(ctypes.Structure):
    """``prism_moe_w4``: a 4-bit matrix or stack of matrices."""
    _fields_ = [("qweight", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("zeros", ctypes.c_void_p), ("group_size", ctypes.c_int32)]


_ep = ctypes.POINTER(NormEpilogue)
_w4p = ctypes.POINTER(W4)
SCORINGS = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}
_SIGNATURES = {
    "prism_moe_version": (ctypes.c_int, []),
    "prism_moe_last_error": (ctypes.c_char_p, []),
    "prism_moe_route_topk": (ctypes.c_int, [_vp, ctypes.c_int, _i64, _i32, _i32, _i32, _vp, _vp,
                                            _vp, _vp]),
    "prism_moe_route_scored": (ctypes.c_int, [_vp, ctypes.c_int, _i64, _i32, _i32,
                                              ctypes.POINTER(Router), _vp, _vp, ctypes.c_int,
                                              _vp, _vp]),
    "prism_moe_linear_w4": (ctypes.c_int, [_vp, _i64, _i64, _i64, _w4p, _vp, _vp, _vp]),
    "prism_moe_expert_w4_workspace_size": (_sz, [_i64, _i64]),
    "prism_moe_expert_swiglu_w4": (ctypes.c_int, [_vp, _i64, _i64, _i64, _vp, _vp, _i32, _i32,
                                                  _w4p, _w4p, _vp, _vp, _sz, _vp, _vp]),
    "prism_moe_block_forward_routed": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_int, _i64, _i64,
                                                      _i64, _i32, _i32, _vp, _vp, _w4p, _w4p, _vp,
                                                      _vp, _sz, _vp, _ep]),
    "prism_moe_block_forward_routed_reporting": (
        ctypes.c_int, [_vp, _vp, _vp, ctypes.c_int, _i64, _i64, _i64, _i32, _i32, _vp, _vp, _w4p,
                       _w4p, _vp, _vp, _sz, _vp, _vp, _ep]),
    "prism_moe_device_error_word": (ctypes.c_int, [ctypes.POINTER(_vp)]),
    "prism_moe_dispatch_workspace_size": (_sz, [_i64, _i32, _i32, _i32]),
    "prism_moe_build_dispatch_plan": (ctypes.c_int, [_vp, _i64, _i32, _i32, _i32, _vp, _vp, _vp,
                                                     _vp, _vp, _vp, _vp, _sz, _vp]),
    "prism_moe_build_dispatch_plan_static": (ctypes.c_int, [_vp, _i64, _i32, _i32, _i32, _vp,
                                                            _vp, _vp, _vp, _vp, _vp, _vp]),
    "prism_moe_permute_rows": (ctypes.c_int, [_vp, ctypes.c_int, _i64, _i64, _i32, _vp, _vp,
                                              _vp]),
    "prism_moe_expert_workspace_size": (_sz, [_i64, _i64, _i64, ctypes.c_int]),
    "prism_moe_expert_swiglu": (ctypes.c_int, [_vp, ctypes.c_int, _i64, _i64, _i64, _vp, _vp,
                                               _i32, _i32, _vp, _vp, _vp, _vp, _sz, _vp, _vp]),
    "prism_moe_combine": (ctypes.c_int, [_vp, ctypes.c_int, _vp, _vp, _i64, _i32, _i64, _vp,
                                         _vp]),
    "prism_moe_block_workspace_size": (_sz, [_i64, _i64, _i64, _i32, _i32, ctypes.c_int]),
    "prism_moe_block_forward": (ctypes.c_int, [_vp, _vp, ctypes.c_int, _i64, _i64, _i64, _i32,
                                               _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                                               _vp]),
    "prism_moe_ep_landing_bytes": (_sz, [_i32, _i64, _i32, _i64, _i32, ctypes.c_int]),
    "prism_moe_ep_alloc_landing": (ctypes.c_int, [_sz, ctypes.POINTER(_vp), _vp]),
    "prism_moe_ep_free_landing": (ctypes.c_int, [_vp]),
    "prism_moe_ep_ipc_handle_bytes": (ctypes.c_int, []),
    "prism_moe_ep_open_peer": (ctypes.c_int, [_vp, ctypes.POINTER(_vp)]),
    "prism_moe_ep_close_peer": (ctypes.c_int, [_vp]),
    "prism_moe_ep_workspace_size": (_sz, [_i64, _i64, _i64, _i32, _i32, _i32, ctypes.c_int]),
    "prism_moe_ep_forward": (ctypes.c_int, [_vp, _vp, _vp, _vp, ctypes.c_int, _i64, _i64, _i64,
                                            _i64, _i32, _i32, _i32, _i32, _i32, _vp, _vp, _vp,
                                            _vp, ctypes.c_uint64, _vp, _vp, _sz, _vp]),
    "prism_moe_ep_read_stats": (ctypes.c_int, [_vp, ctypes.POINTER(ctypes.c_uint64), _vp]),
    "prism_moe_set_expert_engine": (ctypes.c_int, [ctypes.c_int]),
    "prism_moe_set_wait_limits": (ctypes.c_int, [_i64, _i64]),
    "prism_moe_rmsnorm": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_float, ctypes.c_int, _i64, _i64,
                                         _vp, _vp, _vp]),
    "prism_moe_block_forward_norm": (ctypes.c_int, [_vp, _vp, ctypes.c_int, _i64, _i64, _i64, _i32,
                                                    _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _sz,
                                                    _vp, _ep]),
    "prism_moe_ep_forward_norm": (ctypes.c_int, [_vp, _vp, _vp, _vp, ctypes.c_int, _i64, _i64,
                                                 _i64, _i64, _i32, _i32, _i32, _i32, _i32, _vp,
                                                 _vp, _vp, _vp, ctypes.c_uint64, _vp, _vp, _sz,
                                                 _vp, _ep]),
    "prism_moe_profile_events": (ctypes.c_int, [ctypes.POINTER(_vp), _i32]),
    "prism_moe_read_device_error": (ctypes.c_int, [_vp, _vp]),
}

_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load libprism_moe.so (once) and declare every entry point's signature."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(
                    f"{LIB_PATH} is missing: build it with `python -m prism_infer_b200.build` "
                    "(the MoE block has no CPU or eager fallback)")
            lib = ctypes.CDLL(str(LIB_PATH))
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def last_error() -> str:
    msg = load().prism_moe_last_error()
    return msg.decode() if msg else ""


def check(status: int, what: str) -> None:
    if status != OK:
        raise RuntimeError(f"{what} failed with status {status}: {last_error()}")


# ---------------------------------------------------------------------------------- torch glue

_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def dtype_code(dt) -> int:
    torch = _torch()
    if dt == torch.bfloat16:
        return BF16
    if dt == torch.float32:
        return F32
    raise RuntimeError(f"prism MoE kernels support bfloat16 and float32, got {dt}")


def ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def stream_of(device) -> int:
    torch = _torch()
    return torch.cuda.current_stream(device).cuda_stream


def _need_cuda(*ts):
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("prism MoE kernels run on CUDA tensors only (no CPU fallback)")
        if not t.is_contiguous():
            raise RuntimeError("prism MoE kernels need contiguous tensors")


def route_topk(logits, top_k: int, renorm: bool, with_counts: bool = False):
    """Kernel 1 on ``logits`` [T, E]: returns (topk_ids int64 [T,k], topk_weights [T,k],
    expert_counts int32 [E] or None)."""
    torch = _torch()
    _need_cuda(logits)
    T, E = logits.shape
    ids = torch.empty(T, top_k, dtype=torch.int64, device=logits.device)
    w = torch.empty(T, top_k, dtype=logits.dtype, device=logits.device)
    counts = torch.empty(E, dtype=torch.int32, device=logits.device) if with_counts else None
    check(load().prism_moe_route_topk(ptr(logits), dtype_code(logits.dtype), T, E, top_k,
                                      int(bool(renorm)), ptr(ids), ptr(w), ptr(counts),
                                      stream_of(logits.device)), "prism_moe_route_topk")
    return ids, w, counts


def _one_device(first, *others) -> int:
    """Index of the device all given CUDA tensors are on (contiguous, or RuntimeError)."""
    index = first.get_device()
    for t in (first, *others):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("prism MoE kernels run on CUDA tensors only (no CPU fallback)")
        if not t.is_contiguous():
            raise RuntimeError("prism MoE kernels need contiguous tensors")
        if t.get_device() != index:
            raise RuntimeError(f"tensors are on different devices: cuda:{index} and "
                               f"cuda:{t.get_device()}")
    return index


_error_words: dict = {}


def device_error_word(index: int) -> int:
    """Address of the library's error word on device ``index``, where calls that are given none record
    a failing kernel's status, captured ones included (prism_moe_device_error_word)."""
    at = _error_words.get(index)
    if at is None:
        word = ctypes.c_void_p()
        with _torch().cuda.device(index):
            check(load().prism_moe_device_error_word(ctypes.byref(word)),
                  "prism_moe_device_error_word")
        at = _error_words[index] = word.value
    return at


def check_device_error(device=None) -> None:
    """Synchronise the current stream of ``device`` and raise (once) if a kernel recorded a failure in
    its ``device_error_word``: any call's on that device, so what ran on other streams too, as far as
    it has ended."""
    torch = _torch()
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    with torch.cuda.device(index):
        check(load().prism_moe_read_device_error(device_error_word(torch.cuda.current_device()),
                                                 stream_of(None)), "kernels on this device")


def _launch(index: int, what: str, fn, *args) -> None:
    """``fn(*args, stream)`` with device ``index`` current, on its current torch stream (the raw
    handle: a Stream object costs more host time than the launch)."""
    torch = _torch()
    if torch.cuda.current_device() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status != OK:
        check(status, what)


def route_scored(logits, top_k: int, *, scoring: str = "softmax", bias=None, num_groups: int = 1,
                 topk_groups: int = 1, group_score: str = "max", renorm: bool = True,
                 scale: float = 1.0, out_dtype=None, with_counts: bool = False):
    """Routing by ``scoring`` ("softmax" or "sigmoid") scores of ``logits`` [T, E]: the ``top_k``
    largest scores + ``bias`` (fp32 [E], for the choice only) among the ``topk_groups`` best of
    ``num_groups`` groups (by ``group_score`` "max" or "top2"), equal keys to the lowest index; the
    weights are the chosen scores, divided by their sum with ``renorm``, times ``scale``
    (prism_moe_route_scored). Returns (topk_ids int64 [T,k], topk_weights [T,k] in ``out_dtype``,
    by default the logits' dtype, expert_counts int32 [E] or None)."""
    torch = _torch()
    if scoring not in SCORINGS:
        raise RuntimeError(f"unknown scoring {scoring!r}; one of {sorted(SCORINGS)}")
    if group_score not in GROUP_SCORES:
        raise RuntimeError(f"unknown group_score {group_score!r}; one of {sorted(GROUP_SCORES)}")
    if logits.dim() != 2:
        raise RuntimeError("route_scored: logits must be [T, E]")
    dev = _one_device(logits, bias)
    T, E = logits.shape
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (E,)):
        raise RuntimeError(f"route_scored: bias must be float32 [{E}]")
    out_dtype = logits.dtype if out_dtype is None else out_dtype
    shape = (T, max(int(top_k), 0))
    ids = logits.new_empty(shape, dtype=torch.int64)
    w = logits.new_empty(shape, dtype=out_dtype)
    counts = logits.new_empty((E,), dtype=torch.int32) if with_counts else None
    router = Router(SCORINGS[scoring], ptr(bias), num_groups, topk_groups,
                    GROUP_SCORES[group_score], 1 if renorm else 0, scale)
    _launch(dev, "prism_moe_route_scored", load().prism_moe_route_scored, logits.data_ptr(),
            dtype_code(logits.dtype), T, E, top_k, ctypes.byref(router), ids.data_ptr(),
            w.data_ptr(), dtype_code(out_dtype), ptr(counts))
    return ids, w, counts


def dispatch_plan(topk_ids, num_experts: int, ep_size: int, want_perm: bool = True):
    """Kernel 2 (plan) on ``topk_ids`` [T, k] int64. Returns a dict of int tensors: perm,
    input_splits, sorted_local_eid (int64, reference layout) and expert_counts,
    expert_offsets, entry_row (int32, expert-major layout)."""
    torch = _torch()
    _need_cuda(topk_ids)
    if topk_ids.dtype != torch.int64:
        raise RuntimeError("topk_ids must be int64")
    T, k = topk_ids.shape
    dev = topk_ids.device
    N = T * k
    lib = load()
    ws_bytes = lib.prism_moe_dispatch_workspace_size(T, k, num_experts, ep_size)
    ws = torch.zeros(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    out = dict(
        perm=torch.empty(N, dtype=torch.int64, device=dev) if want_perm else None,
        input_splits=torch.empty(ep_size, dtype=torch.int64, device=dev) if want_perm else None,
        sorted_local_eid=torch.empty(N, dtype=torch.int64, device=dev) if want_perm else None,
        expert_counts=torch.empty(num_experts, dtype=torch.int32, device=dev),
        expert_offsets=torch.empty(num_experts + 1, dtype=torch.int32, device=dev),
        entry_row=torch.empty(N, dtype=torch.int32, device=dev),
    )
    check(lib.prism_moe_build_dispatch_plan(
        ptr(topk_ids), T, k, num_experts, ep_size, ptr(out["perm"]), ptr(out["input_splits"]),
        ptr(out["sorted_local_eid"]), ptr(out["expert_counts"]), ptr(out["expert_offsets"]),
        ptr(out["entry_row"]), ptr(ws), ws_bytes, stream_of(dev)), "prism_moe_build_dispatch_plan")
    return out


def permute_rows(x, top_k: int, entry_row, out=None):
    """x_sorted[entry_row[t*k+j]] = x[t] (rows not named by entry_row are left as they are)."""
    torch = _torch()
    _need_cuda(x, entry_row)
    T, H = x.shape
    if out is None:
        out = torch.empty(T * top_k, H, dtype=x.dtype, device=x.device)
    check(load().prism_moe_permute_rows(ptr(x), dtype_code(x.dtype), T, H, top_k, ptr(entry_row),
                                        ptr(out), stream_of(x.device)), "prism_moe_permute_rows")
    return out


def expert_swiglu(x_sorted, seg_offsets, w_gate_up, w_down, seg_expert=None, y=None,
                  device_error=None):
    """Kernel 4: grouped SwiGLU experts over the segment table (int32 device tensors).
    ``device_error`` None: errors go to ``device_error_word``'s word."""
    torch = _torch()
    _need_cuda(x_sorted, seg_offsets, w_gate_up, w_down, seg_expert)
    R, H = x_sorted.shape
    El, twoI, H2 = w_gate_up.shape
    I = twoI // 2
    if H2 != H or tuple(w_down.shape) != (El, H, I):
        raise RuntimeError("expert weight shapes do not match x_sorted")
    if w_gate_up.dtype != x_sorted.dtype or w_down.dtype != x_sorted.dtype:
        raise RuntimeError("expert weights must have the activations' dtype")
    lib = load()
    dt = dtype_code(x_sorted.dtype)
    ws_bytes = lib.prism_moe_expert_workspace_size(R, H, I, dt)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=x_sorted.device)
    if y is None:
        y = torch.empty_like(x_sorted)
    nseg = seg_offsets.numel() - 1
    check(lib.prism_moe_expert_swiglu(ptr(x_sorted), dt, R, H, I, ptr(seg_offsets),
                                      ptr(seg_expert), nseg, El, ptr(w_gate_up), ptr(w_down),
                                      ptr(y), ptr(ws), ws_bytes,
                                      device_error_word(x_sorted.get_device())
                                      if device_error is None else ptr(device_error),
                                      stream_of(x_sorted.device)), "prism_moe_expert_swiglu")
    return y


def _w4(weight) -> W4:
    return W4(ptr(weight.qweight), ptr(weight.scales), ptr(weight.zeros), weight.group_size)


def _need_bf16(x, what: str) -> None:
    if x.dtype != _torch().bfloat16:
        raise RuntimeError(f"{what}: 4-bit weights take bfloat16 activations, got {x.dtype}")


def linear_w4(x, weight, out=None, device_error=None):
    """y = x W^T for a 4-bit ``weight`` (``quant.W4Weight``, a single matrix): ``x`` [M, K] bf16, any
    M from 0; returns [M, N] bf16 (``out``, which must not overlap ``x``). ``device_error``: an int32
    device word that a failing kernel records its status in (None: ``device_error_word``'s;
    prism_moe_linear_w4)."""
    torch = _torch()
    _need_bf16(x, "linear_w4")
    if weight.stack is not None or weight.gate_up:
        raise RuntimeError("linear_w4: takes a single matrix, no stack and no gate_up rows")
    if x.dim() != 2 or x.shape[1] != weight.in_features:
        raise RuntimeError(f"linear_w4: x {tuple(x.shape)} does not match {weight.in_features} "
                           "inputs")
    dev = _one_device(x, weight.qweight, out, device_error)
    if device_error is not None and device_error.dtype != torch.int32:
        raise RuntimeError("linear_w4: device_error must be int32")
    M, N = x.shape[0], weight.out_features
    if out is None:
        out = x.new_empty((M, N))
    elif tuple(out.shape) != (M, N) or out.dtype != x.dtype:
        raise RuntimeError("linear_w4: out must be [M, N] in x's dtype")
    _launch(dev, "prism_moe_linear_w4", load().prism_moe_linear_w4, x.data_ptr(), M,
            weight.in_features, N, ctypes.byref(_w4(weight)), out.data_ptr(),
            device_error_word(dev) if device_error is None else ptr(device_error))
    return out


def _expert_shapes(what: str, H: int, w_gate_up, w_down):
    """(experts, inter) of a pair of 4-bit expert stacks for hidden size ``H``."""
    El, I = w_gate_up.stack, w_gate_up.out_features // 2
    if El is None or not w_gate_up.gate_up or w_down.gate_up or w_down.stack != El or \
            w_gate_up.in_features != H or \
            (w_down.out_features, w_down.in_features) != (H, I):
        raise RuntimeError(f"{what}: 4-bit expert weights do not match each other or hidden {H}")
    return El, I


def expert_swiglu_w4(x_sorted, seg_offsets, w_gate_up, w_down, seg_expert=None, y=None,
                     device_error=None):
    """Grouped SwiGLU experts on 4-bit weights (``quant.W4Weight`` stacks) over the segment table:
    ``expert_swiglu`` with ``w_gate_up`` [El, 2I, H] and ``w_down`` [El, H, I] in 4 bits and bf16
    activations (prism_moe_expert_swiglu_w4). ``seg_offsets`` None: all rows are one segment.
    ``device_error`` None: errors go to ``device_error_word``'s word."""
    torch = _torch()
    _need_bf16(x_sorted, "expert_swiglu_w4")
    if x_sorted.dim() != 2:
        raise RuntimeError("expert_swiglu_w4: x_sorted must be [R, H]")
    R, H = x_sorted.shape
    El, I = _expert_shapes("expert_swiglu_w4", H, w_gate_up, w_down)
    dev = _one_device(x_sorted, seg_offsets, seg_expert, w_gate_up.qweight, w_down.qweight, y,
                      device_error)
    nseg = 1 if seg_offsets is None else seg_offsets.numel() - 1
    for name, t in (("seg_offsets", seg_offsets), ("seg_expert", seg_expert),
                    ("device_error", device_error)):
        if t is not None and t.dtype != torch.int32:
            raise RuntimeError(f"expert_swiglu_w4: {name} must be int32")
    if seg_expert is None and nseg != El:
        raise RuntimeError(f"expert_swiglu_w4: {nseg} segments for {El} experts need seg_expert")
    if seg_expert is not None and seg_expert.numel() != nseg:
        raise RuntimeError("expert_swiglu_w4: seg_expert must name one expert per segment")
    if y is None:
        y = torch.empty_like(x_sorted)
    elif y.shape != x_sorted.shape or y.dtype != x_sorted.dtype:
        raise RuntimeError("expert_swiglu_w4: y must look like x_sorted")
    lib = load()
    ws_bytes = lib.prism_moe_expert_w4_workspace_size(R, I)
    ws = x_sorted.new_empty((max(ws_bytes, 1),), dtype=torch.uint8)
    _launch(dev, "prism_moe_expert_swiglu_w4", lib.prism_moe_expert_swiglu_w4,
            x_sorted.data_ptr(), R, H, I, ptr(seg_offsets), ptr(seg_expert), nseg, El,
            ctypes.byref(_w4(w_gate_up)), ctypes.byref(_w4(w_down)), y.data_ptr(), ws.data_ptr(),
            ws_bytes, device_error_word(dev) if device_error is None else ptr(device_error))
    return y


def combine(expert_out, topk_weights, entry_row=None, out=None):
    """Kernel 5: out[t] = sum_j w[t,j] * expert_out[row(t*k+j)]."""
    torch = _torch()
    _need_cuda(expert_out, topk_weights, entry_row)
    T, k = topk_weights.shape
    H = expert_out.shape[-1]
    if topk_weights.dtype != expert_out.dtype:
        raise RuntimeError("topk_weights must have the expert outputs' dtype")
    if out is None:
        out = torch.empty(T, H, dtype=expert_out.dtype, device=expert_out.device)
    check(load().prism_moe_combine(ptr(expert_out), dtype_code(expert_out.dtype), ptr(entry_row),
                                   ptr(topk_weights), T, k, H, ptr(out),
                                   stream_of(expert_out.device)), "prism_moe_combine")
    return out


_ws_lock = threading.Lock()
_workspaces: dict = {}


def block_workspace(device, nbytes: int):
    """Per-(device, stream) scratch for ``prism_moe_block_forward``; grows on demand. The first
    four bytes are the kernels' device error word (kept zero)."""
    torch = _torch()
    stream = torch.cuda.current_stream(device).cuda_stream
    key = (device.index, stream)
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            _workspaces[key] = ws
    return ws


def block_error_word(device):
    """The device error word of the current stream's block workspace (None before any call)."""
    torch = _torch()
    ws = _workspaces.get((device.index, torch.cuda.current_stream(device).cuda_stream))
    return None if ws is None else ws[:4].view(torch.int32)


def norm_epilogue(residual, norm_weight, eps: float, residual_out):
    """A ``prism_moe_norm_epilogue`` for the *_norm entry points (None when ``norm_weight`` is
    None): ``residual`` and ``residual_out`` [T,H] and ``norm_weight`` [H], of the hidden states' dtype
    and device. It holds the tensors."""
    if norm_weight is None:
        return None
    if residual.dim() != 2 or residual_out.shape != residual.shape or \
            norm_weight.shape != residual.shape[1:]:
        raise RuntimeError("norm epilogue: residual and residual_out must be [T, H], the weight [H]")
    if not residual.dtype == norm_weight.dtype == residual_out.dtype:
        raise RuntimeError("norm epilogue: residual, weight and residual_out differ in dtype")
    _one_device(residual, norm_weight, residual_out)
    epilogue = NormEpilogue(residual.data_ptr(), norm_weight.data_ptr(), float(eps),
                            residual_out.data_ptr())
    epilogue.held = (residual, norm_weight, residual_out)
    return epilogue


def _check_block_outputs(what: str, x, out, epilogue) -> None:
    """What a block call writes beside its workspace looks like ``x``."""
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype):
        raise RuntimeError(f"{what}: out must be {tuple(x.shape)} in {x.dtype}, got "
                           f"{tuple(out.shape)} in {out.dtype}")
    held = getattr(epilogue, "held", None)   # None: the caller filled the struct
    if held is not None and (held[0].shape != x.shape or held[0].dtype != x.dtype or
                             held[0].device != x.device):
        raise RuntimeError(f"{what}: the norm epilogue's residual must be {tuple(x.shape)} in "
                           f"{x.dtype} on {x.device}")


def rmsnorm(x, weight, eps: float, residual=None):
    """RMSNorm of ``x`` [T,H] (prism_moe_rmsnorm); with ``residual``, of ``x + residual``, and
    returns (out, residual_out) as the reference's add_rms_forward does."""
    torch = _torch()
    _need_cuda(x, weight, residual)
    T, H = x.shape
    if weight.shape != (H,) or weight.dtype != x.dtype or (
            residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype)):
        raise RuntimeError("rmsnorm: inconsistent shapes or dtypes")
    out = torch.empty_like(x)
    res_out = torch.empty_like(x) if residual is not None else None
    check(load().prism_moe_rmsnorm(ptr(x), ptr(residual), ptr(weight), float(eps),
                                   dtype_code(x.dtype), T, H, ptr(out), ptr(res_out),
                                   stream_of(x.device)), "prism_moe_rmsnorm")
    return out if residual is None else (out, res_out)


def block_forward(x, router_logits, w_gate_up, w_down, top_k: int, renorm: bool, out=None,
                  epilogue=None):
    """The single-GPU block after the router GEMM (prism_moe_block_forward): route, plan,
    gather, grouped SwiGLU experts, combine. ``x`` [T,H], ``router_logits`` [T,E],
    ``w_gate_up`` [E,2I,H], ``w_down`` [E,H,I]; returns [T,H]. ``epilogue`` (a NormEpilogue)
    fuses the decoder layer's next residual add + RMSNorm into the combine."""
    torch = _torch()
    _need_cuda(x, router_logits, w_gate_up, w_down)
    T, H = x.shape
    E, twoI, H2 = w_gate_up.shape
    I = twoI // 2
    if H2 != H or tuple(w_down.shape) != (E, H, I) or tuple(router_logits.shape) != (T, E):
        raise RuntimeError("block_forward: inconsistent shapes")
    for t in (router_logits, w_gate_up, w_down):
        if t.dtype != x.dtype:
            raise RuntimeError(f"block_forward: dtype {t.dtype} != hidden dtype {x.dtype}")
    _check_block_outputs("block_forward", x, out, epilogue)
    _need_cuda(out)
    if out is None:
        out = torch.empty_like(x)
    if T == 0:
        return out
    lib = load()
    dt = dtype_code(x.dtype)
    nbytes = lib.prism_moe_block_workspace_size(T, H, I, E, top_k, dt)
    ws = block_workspace(x.device, nbytes)
    check(lib.prism_moe_block_forward_norm(
        ptr(x), ptr(router_logits), dt, T, H, I, E, top_k, int(bool(renorm)), ptr(w_gate_up),
        ptr(w_down), ptr(out), None, None, ptr(ws), ws.numel(), stream_of(x.device),
        ctypes.byref(epilogue) if epilogue is not None else None),
        "prism_moe_block_forward")
    return out


def _routed_workspace(device, nbytes: int):
    """The block's scratch and the address of its error word: the (device, stream) workspace and its own
    (None), or, while a CUDA graph is captured, memory of that graph's own (two graphs never share
    it) and ``device_error_word``'s."""
    torch = _torch()
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device), device_error_word(device.index)
    return block_workspace(device, nbytes), None


def block_forward_routed(x, topk_ids, topk_weights, w_gate_up, w_down, out=None, epilogue=None):
    """The block after its router for a given choice: ``topk_ids`` [T,k] int64 and ``topk_weights``
    [T,k] in x's dtype; plan, gather, experts, combine (prism_moe_block_forward_routed). The experts
    are tensors [E,2I,H] and [E,H,I], or two 4-bit stacks (``quant.W4Weight``)."""
    torch = _torch()
    from prism_infer_b200.quant import W4Weight
    T, H = x.shape
    k = topk_ids.shape[-1]
    w4 = isinstance(w_gate_up, W4Weight)
    if w4 != isinstance(w_down, W4Weight):
        raise RuntimeError("block_forward_routed: give either dense or 4-bit expert weights")
    if w4:
        _need_bf16(x, "block_forward_routed")
        E, I = _expert_shapes("block_forward_routed", H, w_gate_up, w_down)
        held = (w_gate_up.qweight, w_down.qweight)
    else:
        E, twoI, H2 = w_gate_up.shape
        I = twoI // 2
        if H2 != H or tuple(w_down.shape) != (E, H, I):
            raise RuntimeError("block_forward_routed: inconsistent shapes")
        if w_gate_up.dtype != x.dtype or w_down.dtype != x.dtype:
            raise RuntimeError("block_forward_routed: weights must have the hidden dtype")
        held = (w_gate_up, w_down)
    _check_block_outputs("block_forward_routed", x, out, epilogue)
    dev = _one_device(x, topk_ids, topk_weights, out, *held)
    if topk_ids.dtype != torch.int64 or topk_weights.dtype != x.dtype or \
            tuple(topk_ids.shape) != (T, k) or tuple(topk_weights.shape) != (T, k):
        raise RuntimeError("block_forward_routed: topk_ids must be int64 [T, k], topk_weights "
                           "[T, k] in the hidden dtype")
    if out is None:
        out = torch.empty_like(x)
    if T == 0:
        return out
    lib = load()
    dt = dtype_code(x.dtype)
    dense = (None, None) if w4 else (ptr(w_gate_up), ptr(w_down))
    quant = (ctypes.byref(_w4(w_gate_up)), ctypes.byref(_w4(w_down))) if w4 else (None, None)
    with torch.cuda.device(dev):
        nbytes = lib.prism_moe_block_workspace_size(T, H, I, E, k, dt)
        ws, word = _routed_workspace(x.device, nbytes)
        check(lib.prism_moe_block_forward_routed_reporting(
            ptr(x), ptr(topk_ids), ptr(topk_weights), dt, T, H, I, E, k, *dense, *quant, ptr(out),
            ptr(ws), ws.numel(), word, stream_of(x.device),
            ctypes.byref(epilogue) if epilogue is not None else None),
            "prism_moe_block_forward_routed")
    return out


def ep_alloc_landing(nbytes: int):
    """Allocate this rank's landing zone; returns (device address, IPC handle bytes)."""
    lib = load()
    buf = ctypes.create_string_buffer(lib.prism_moe_ep_ipc_handle_bytes())
    p = _vp()
    check(lib.prism_moe_ep_alloc_landing(nbytes, ctypes.byref(p), buf),
          "prism_moe_ep_alloc_landing")
    return p.value, buf.raw


def ep_open_peer(handle: bytes) -> int:
    """Map a peer's landing zone from its IPC handle; returns the device address."""
    lib = load()
    p = _vp()
    check(lib.prism_moe_ep_open_peer(ctypes.create_string_buffer(handle, len(handle)),
                                     ctypes.byref(p)), "prism_moe_ep_open_peer")
    return p.value


def set_profile_events(events) -> None:
    """Record ``events`` (torch.cuda.Event, already created) at the kernels' stage boundaries on
    this thread; ``None`` or an empty list turns the hook off."""
    events = list(events or [])
    arr = (_vp * max(len(events), 1))(*[ctypes.c_void_p(e.cuda_event) for e in events])
    check(load().prism_moe_profile_events(arr, len(events)), "prism_moe_profile_events")


def read_device_error(word, device=None) -> int:
    """Synchronise and return (and clear) the status in a device error word."""
    dev = word.device if device is None else device
    return load().prism_moe_read_device_error(ptr(word), stream_of(dev))


def set_expert_engine(name: str) -> None:
    """Expert GEMM engine for calls without an expert-parallel exchange: ``auto`` (default),
    ``fused``, ``single`` or ``pair`` (prism_moe_set_expert_engine)."""
    if name not in ENGINES:
        raise RuntimeError(f"unknown expert engine {name!r}; one of {sorted(ENGINES)}")
    check(load().prism_moe_set_expert_engine(ENGINES[name]), "prism_moe_set_expert_engine")


def set_wait_limits(wait_ns: int = 0, peer_wait_ns: int = 0) -> None:
    """Bounds of the kernels' waits on their own pipeline and on other ranks (0 = default)."""
    check(load().prism_moe_set_wait_limits(int(wait_ns), int(peer_wait_ns)),
          "prism_moe_set_wait_limits")


def ep_read_stats(workspace, device=None) -> dict:
    """Statistics of the last expert-parallel step that used ``workspace`` (synchronises)."""
    dev = workspace.device if device is None else device
    buf = (ctypes.c_uint64 * len(EP_STATS_FIELDS))()
    check(load().prism_moe_ep_read_stats(ptr(workspace), buf, stream_of(dev)),
          "prism_moe_ep_read_stats")
    return dict(zip(EP_STATS_FIELDS, (int(v) for v in buf)))
