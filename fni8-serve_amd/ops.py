"""Tensor-level entry points over the C ABI (libfni8amd.so).

`linear(x, qt, bias=None)` is the drop-in for `fni8.linear`, the one call the
reference's W8A8 seam makes (fni8serve/layers/linear.py:69): per-token int8
quantization of x, the int8 GEMM against a per_row_i8 QTensor, and the fused
dequant epilogue to fp16.  The other functions expose the pieces (for the
grouped MoE path and for parity checks).

Every function launches on `torch.cuda.current_stream()` of the operands'
device, allocates its outputs and scratch from torch's caching allocator, and
never synchronises, so the calls can be captured in a HIP graph.  GPU tensors
are required: there is no CPU or PyTorch fallback here.

`linear`, `gemm_w8a8`, `gemm_w4a8`, `rmsnorm`, `rmsnorm_quant`, `rope`, `qk_norm_rope`,
`rope_append`, `paged_attention`, `lora_add`, `sample` and the chains `gated_mlp` and `sparse_moe` run in native
host code (`_host`, csrc/host.cpp) when
every tensor is a plain GPU tensor in the layout the kernels take; the Python below
is the general way (strided, converted or refused arguments).  A LinearW8A8 call at
one token took 17 us of Python for 4.3 us of kernel on an MI355X host; natively a
pass takes 6.1 us.
"""
from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence
from typing import NamedTuple

import torch

from . import _lib
from .qtensor import QTensor

_f16 = torch.float16


def _group(qt: QTensor) -> int:
    """0 for a per_row_i8 weight, the group size of a per_group_i4 int4 one, else -1."""
    if qt.scheme == "per_row_i8":
        return 0
    if qt.scheme == "per_group_i4" and qt.codebook == "int4" and qt.group_size:
        return qt.group_size
    return -1


def _stream(dev: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _require_cuda(name: str, *ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name}: every tensor must be on the GPU (got {t.device})")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{name}: tensors on different devices ({dev} vs {t.device})")
    return dev


def _rows(x: torch.Tensor, K: int):
    """View x[..., K] as 2-D rows with unit inner stride; returns (x2, ldx)."""
    if x.stride(-1) != 1:
        x = x.contiguous()
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < K):
        x2 = x2.contiguous()
    ldx = x2.stride(0) if x2.shape[0] > 1 else K
    return x2, ldx


def _check_weight(qt: QTensor, K: int):
    if qt.scheme != "per_row_i8":
        raise ValueError(f"W8A8 linear cannot use scheme {qt.scheme!r}")
    w, s = qt.data, qt.scale
    if w.dtype != torch.int8 or w.dim() != 2 or not w.is_contiguous():
        raise ValueError("per_row_i8 data must be a contiguous int8 [N, K] tensor")
    if w.shape[1] != K:
        raise ValueError(f"in_features mismatch: x has K={K}, weight has {w.shape[1]}")
    if s is None or s.dtype != torch.float32 or s.numel() != w.shape[0] or not s.is_contiguous():
        raise ValueError("per_row_i8 scale must be a contiguous fp32 tensor with N entries")
    return w, s.reshape(-1)


def _check_bias(bias: torch.Tensor | None, N: int):
    if bias is None:
        return None
    if bias.dtype != _f16 or bias.numel() != N:
        raise ValueError("bias must be an fp16 tensor with N entries")
    return bias.reshape(-1).contiguous()


W4_GROUPS = (32, 64, 128, 256)


def _check_weight_i4(qt: QTensor, K: int):
    """per_group_i4 int4 weight (fni8serve/convert.py:69-79): packed uint8
    [N, K/2], fp32 scales [N, K/G]."""
    if qt.codebook != "int4":
        raise ValueError(f"the W4A8 kernel needs the int4 codebook (got {qt.codebook!r}); "
                         "NF4 weights take the dequantize path")
    w, s, G = qt.data, qt.scale, qt.group_size
    if w.dtype != torch.uint8 or w.dim() != 2 or not w.is_contiguous():
        raise ValueError("per_group_i4 data must be a contiguous uint8 [N, K/2] tensor")
    if 2 * w.shape[1] != K:
        raise ValueError(f"in_features mismatch: x has K={K}, weight packs {2 * w.shape[1]}")
    if G not in W4_GROUPS or K % G or K % 32:
        raise ValueError(f"group size {G} with K={K} not supported (G in {W4_GROUPS}, "
                         "dividing K; K a multiple of 32)")
    N = w.shape[0]
    if s is None or s.dtype != torch.float32 or s.numel() != N * (K // G) or not s.is_contiguous():
        raise ValueError("per_group_i4 scale must be a contiguous fp32 tensor of N * K/G entries")
    return w, s.reshape(N, K // G), G


def _linear_w4a8(x, qt, bias):
    K = x.shape[-1]
    w, ws, G = _check_weight_i4(qt, K)
    N = w.shape[0]
    bias = _check_bias(bias, N)
    dev = _require_cuda("linear", x, w, ws, bias)
    if x.dtype != _f16:
        raise ValueError(f"linear expects fp16 activations (got {x.dtype})")
    x2, ldx = _rows(x, K)
    M = x2.shape[0]
    y = torch.empty((*x.shape[:-1], N), dtype=_f16, device=dev)
    xq = torch.empty((M, K), dtype=torch.int8, device=dev)
    xs = torch.empty((M,), dtype=torch.float32, device=dev)
    if M:
        with torch.cuda.device(dev):
            _lib.call("fni8_linear_w4a8_f16", _ptr(x2), ldx, M, K, _ptr(w), _ptr(ws), N, G,
                      _ptr(bias), _ptr(y), N, _ptr(xq), _ptr(xs), _stream(dev))
    return y, xq, xs, None


def linear_with_intermediates(x: torch.Tensor, qt: QTensor, bias: torch.Tensor | None = None,
                              want_acc: bool = False):
    """`linear` that also returns the quantized activations, their scales and
    (if want_acc) the int32 accumulators: (y, xq [M, K], xs [M], acc [M, N] | None).
    For per_group_i4 weights the accumulators are per group and not returned."""
    if qt.scheme == "per_group_i4":
        return _linear_w4a8(x, qt, bias)
    K = x.shape[-1]
    w, ws = _check_weight(qt, K)
    N = w.shape[0]
    bias = _check_bias(bias, N)
    dev = _require_cuda("linear", x, w, ws, bias)
    if x.dtype != _f16:
        raise ValueError(f"linear expects fp16 activations (got {x.dtype})")
    x2, ldx = _rows(x, K)
    M = x2.shape[0]
    y = torch.empty((*x.shape[:-1], N), dtype=_f16, device=dev)
    xq = torch.empty((M, K), dtype=torch.int8, device=dev)
    xs = torch.empty((M,), dtype=torch.float32, device=dev)
    acc = torch.empty((M, N), dtype=torch.int32, device=dev) if want_acc else None
    if M == 0:
        return y, xq, xs, acc
    # 5..16 tokens on the narrower weights: the one-launch path exchanges the
    # quantized rows through a workspace; prefill shapes with too few output
    # tiles split K and exchange partial tiles through it.  It comes from the
    # caching allocator like every other buffer: torch hands a block back to the
    # same stream only, after the work queued on it, so no two calls that can
    # overlap share one; its contents never matter, so it is not cleared.
    nw = _lib.workspace_bytes(M, N, K)
    work = torch.empty(nw, dtype=torch.uint8, device=dev) if nw else None
    with torch.cuda.device(dev):
        _lib.call("fni8_linear_w8a8_f16_ws", _ptr(x2), ldx, M, K, _ptr(w), _ptr(ws), N,
                  _ptr(bias), _ptr(y), N, _ptr(xq), _ptr(xs), _ptr(acc), _ptr(work), nw,
                  _stream(dev))
    return y, xq, xs, acc


def linear(x: torch.Tensor, qt: QTensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """fni8.linear(x, qt, bias=None): x fp16 [..., K] on the GPU -> fp16 [..., N],
    for per_row_i8 (W8A8) and per_group_i4 int4 (W4A8) weights."""
    if x.is_cuda:
        G = _group(qt)
        if G >= 0:
            y = _lib.host().linear(x, qt.data, qt.scale, G, bias)
            if y is not None:
                return y
    return linear_with_intermediates(x, qt, bias)[0]


def quantize_rowwise(x: torch.Tensor):
    """Per-token quantization of fp16 x [..., K] -> (xq int8 [M, K], xs fp32 [M])."""
    K = x.shape[-1]
    dev = _require_cuda("quantize_rowwise", x)
    if x.dtype != _f16:
        raise ValueError(f"quantize_rowwise expects fp16 (got {x.dtype})")
    x2, ldx = _rows(x, K)
    M = x2.shape[0]
    xq = torch.empty((M, K), dtype=torch.int8, device=dev)
    xs = torch.empty((M,), dtype=torch.float32, device=dev)
    if M:
        with torch.cuda.device(dev):
            _lib.call("fni8_quantize_rowwise_f16", _ptr(x2), M, K, ldx, _ptr(xq), K, _ptr(xs),
                      _stream(dev))
    return xq, xs


def gemm_w8a8(xq: torch.Tensor, xs: torch.Tensor, qt: QTensor, bias: torch.Tensor | None = None,
              want_acc: bool = False):
    """`gemm_w8a8` on already-quantized activations: xq int8 [M, K], xs fp32 [M]
    -> y fp16 [M, N] (and the int32 accumulators if want_acc)."""
    if xq.is_cuda and not want_acc and qt.scheme == "per_row_i8":
        y = _lib.host().gemm(xq, xs, qt.data, qt.scale, 0, bias)
        if y is not None:
            return y
    if xq.dtype != torch.int8 or xq.dim() != 2 or xq.stride(1) != 1:
        raise ValueError("xq must be int8 [M, K] with unit inner stride")
    M, K = xq.shape
    w, ws = _check_weight(qt, K)
    N = w.shape[0]
    bias = _check_bias(bias, N)
    if xs.dtype != torch.float32 or xs.numel() != M or not xs.is_contiguous():
        raise ValueError("xs must be a contiguous fp32 tensor with M entries")
    dev = _require_cuda("gemm_w8a8", xq, xs, w, ws, bias)
    y = torch.empty((M, N), dtype=_f16, device=dev)
    acc = torch.empty((M, N), dtype=torch.int32, device=dev) if want_acc else None
    if M:
        ldq = xq.stride(0) if M > 1 else K
        # split-K workspace for prefill shapes with too few output tiles
        nw = _lib.workspace_bytes(M, N, K)
        work = torch.empty(nw, dtype=torch.uint8, device=dev) if nw else None
        with torch.cuda.device(dev):
            _lib.call("fni8_gemm_w8a8_ws", _ptr(xq), ldq, _ptr(xs), M, K, _ptr(w), _ptr(ws), N,
                      _ptr(bias), _ptr(y), N, _ptr(acc), _ptr(work), nw, _stream(dev))
    return (y, acc) if want_acc else y


def gemm_w4a8(xq: torch.Tensor, xs: torch.Tensor, qt: QTensor,
              bias: torch.Tensor | None = None) -> torch.Tensor:
    """`gemm_w4a8` on already-quantized activations: xq int8 [M, K], xs fp32 [M]
    and a per_group_i4 int4 QTensor -> y fp16 [M, N]."""
    if xq.is_cuda and qt.scheme == "per_group_i4" and _group(qt) > 0:
        y = _lib.host().gemm(xq, xs, qt.data, qt.scale, qt.group_size, bias)
        if y is not None:
            return y
    if xq.dtype != torch.int8 or xq.dim() != 2 or xq.stride(1) != 1:
        raise ValueError("xq must be int8 [M, K] with unit inner stride")
    M, K = xq.shape
    w, ws, G = _check_weight_i4(qt, K)
    N = w.shape[0]
    bias = _check_bias(bias, N)
    if xs.dtype != torch.float32 or xs.numel() != M or not xs.is_contiguous():
        raise ValueError("xs must be a contiguous fp32 tensor with M entries")
    dev = _require_cuda("gemm_w4a8", xq, xs, w, ws, bias)
    y = torch.empty((M, N), dtype=_f16, device=dev)
    if M:
        ldq = xq.stride(0) if M > 1 else K
        if ldq % 16 or xq.data_ptr() % 16:
            xq, ldq = xq.contiguous(), K
        with torch.cuda.device(dev):
            _lib.call("fni8_gemm_w4a8", _ptr(xq), ldq, _ptr(xs), M, K, _ptr(w), _ptr(ws), N, G,
                      _ptr(bias), _ptr(y), N, _stream(dev))
    return y


def gemm_quantized(xq: torch.Tensor, xs: torch.Tensor, qt: QTensor,
                   bias: torch.Tensor | None = None) -> torch.Tensor:
    """The GEMM of `linear` for either weight scheme on pre-quantized activations."""
    if qt.scheme == "per_group_i4":
        return gemm_w4a8(xq, xs, qt, bias)
    return gemm_w8a8(xq, xs, qt, bias)


def moe_sort(topi: torch.Tensor, num_experts: int):
    """Stable counting sort of routed (token, slot) pairs by expert.
    topi int [T, k] -> (seg_off int32 [E+1], row_token int32 [T*k], pos int32 [T, k])."""
    if topi.dim() != 2:
        raise ValueError("topi must be [T, k]")
    dev = _require_cuda("moe_sort", topi)
    topi = topi.to(torch.int32).contiguous()
    T, k = topi.shape
    seg_off = torch.empty((num_experts + 1,), dtype=torch.int32, device=dev)
    row_token = torch.empty((T * k,), dtype=torch.int32, device=dev)
    pos = torch.empty((T, k), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.call("fni8_moe_sort", _ptr(topi), T, k, num_experts, _ptr(seg_off), _ptr(row_token),
                  _ptr(pos), _stream(dev))
    return seg_off, row_token, pos


def gemm_w8a8_grouped(aq: torch.Tensor, as_: torch.Tensor, w: torch.Tensor, ws: torch.Tensor,
                      seg_off: torch.Tensor, rows: int, row_index: torch.Tensor | None = None,
                      bias: torch.Tensor | None = None, want_acc: bool = False):
    """Grouped W8A8 GEMM over expert segments.
    aq int8 [A, K], as_ fp32 [A]; w int8 [E, N, K]; ws fp32 [E, N]; seg_off int32 [E+1];
    row_index int32 [rows] or None -> y fp16 [rows, N] in sorted-row order."""
    if aq.dtype != torch.int8 or aq.dim() != 2 or not aq.is_contiguous():
        raise ValueError("aq must be a contiguous int8 [rows, K] tensor")
    if w.dtype != torch.int8 or w.dim() != 3 or not w.is_contiguous():
        raise ValueError("w must be a contiguous int8 [E, N, K] tensor")
    E, N, K = w.shape
    if aq.shape[1] != K:
        raise ValueError(f"in_features mismatch: {aq.shape[1]} vs {K}")
    if ws.dtype != torch.float32 or ws.shape != (E, N) or not ws.is_contiguous():
        raise ValueError("ws must be a contiguous fp32 [E, N] tensor")
    if as_.dtype != torch.float32 or as_.numel() != aq.shape[0] or not as_.is_contiguous():
        raise ValueError("as_ must be a contiguous fp32 tensor with one entry per row of aq")
    if seg_off.dtype != torch.int32 or seg_off.numel() != E + 1:
        raise ValueError("seg_off must be int32 [E+1]")
    if row_index is not None and (row_index.dtype != torch.int32 or row_index.numel() < rows):
        raise ValueError("row_index must be int32 with at least `rows` entries")
    if row_index is None and aq.shape[0] < rows:
        raise ValueError("aq has fewer rows than `rows`")
    if bias is not None and (bias.dtype != _f16 or bias.shape != (E, N)):
        raise ValueError("bias must be fp16 [E, N]")
    dev = _require_cuda("gemm_w8a8_grouped", aq, as_, w, ws, seg_off, row_index, bias)
    y = torch.empty((rows, N), dtype=_f16, device=dev)
    acc = torch.empty((rows, N), dtype=torch.int32, device=dev) if want_acc else None
    if rows:
        with torch.cuda.device(dev):
            _lib.call("fni8_gemm_w8a8_grouped", _ptr(aq), _ptr(as_), _ptr(row_index), rows, K,
                      _ptr(w), _ptr(ws), E, N, _ptr(seg_off), _ptr(bias), _ptr(y), _ptr(acc),
                      _stream(dev))
    return (y, acc) if want_acc else y


W4_GROUPED_GROUPS = (64, 128, 256)


def gemm_w4a8_grouped(aq: torch.Tensor, as_: torch.Tensor, w: torch.Tensor, ws: torch.Tensor,
                      G: int, seg_off: torch.Tensor, rows: int,
                      row_index: torch.Tensor | None = None,
                      bias: torch.Tensor | None = None) -> torch.Tensor:
    """Grouped W4A8 GEMM over expert segments (per_group_i4 int4 experts).
    aq int8 [A, K], as_ fp32 [A]; w uint8 [E, N, K/2]; ws fp32 [E, N, K/G];
    seg_off int32 [E+1]; row_index int32 [rows] or None -> y fp16 [rows, N] in
    sorted-row order.  G in (64, 128, 256), K a multiple of 256."""
    if aq.dtype != torch.int8 or aq.dim() != 2 or not aq.is_contiguous():
        raise ValueError("aq must be a contiguous int8 [rows, K] tensor")
    if w.dtype != torch.uint8 or w.dim() != 3 or not w.is_contiguous():
        raise ValueError("w must be a contiguous uint8 [E, N, K/2] tensor")
    E, N, Kh = w.shape
    K = 2 * Kh
    if aq.shape[1] != K:
        raise ValueError(f"in_features mismatch: {aq.shape[1]} vs {K}")
    if G not in W4_GROUPED_GROUPS or K % 256:
        raise ValueError(f"grouped W4A8 needs G in {W4_GROUPED_GROUPS} and K a multiple of 256 "
                         f"(G={G}, K={K})")
    if ws.dtype != torch.float32 or ws.shape != (E, N, K // G) or not ws.is_contiguous():
        raise ValueError("ws must be a contiguous fp32 [E, N, K/G] tensor")
    if as_.dtype != torch.float32 or as_.numel() != aq.shape[0] or not as_.is_contiguous():
        raise ValueError("as_ must be a contiguous fp32 tensor with one entry per row of aq")
    if seg_off.dtype != torch.int32 or seg_off.numel() != E + 1:
        raise ValueError("seg_off must be int32 [E+1]")
    if row_index is not None and (row_index.dtype != torch.int32 or row_index.numel() < rows):
        raise ValueError("row_index must be int32 with at least `rows` entries")
    if row_index is None and aq.shape[0] < rows:
        raise ValueError("aq has fewer rows than `rows`")
    if bias is not None and (bias.dtype != _f16 or bias.shape != (E, N)):
        raise ValueError("bias must be fp16 [E, N]")
    dev = _require_cuda("gemm_w4a8_grouped", aq, as_, w, ws, seg_off, row_index, bias)
    y = torch.empty((rows, N), dtype=_f16, device=dev)
    if rows:
        with torch.cuda.device(dev):
            _lib.call("fni8_gemm_w4a8_grouped", _ptr(aq), _ptr(as_), _ptr(row_index), rows, K,
                      _ptr(w), _ptr(ws), E, N, G, _ptr(seg_off), _ptr(bias), _ptr(y),
                      _stream(dev))
    return y


def moe_combine(y_sorted: torch.Tensor, topi: torch.Tensor, topw: torch.Tensor,
                pos: torch.Tensor) -> torch.Tensor:
    """out[t] = sum over slots (ascending expert id) of fp16(y_sorted[pos[t, j]] * topw[t, j]),
    accumulated in fp16 from zero, as the expert loop's index_add_ does."""
    T, k = topi.shape
    if y_sorted.dtype != _f16 or y_sorted.dim() != 2 or y_sorted.shape[0] < T * k:
        raise ValueError("y_sorted must be fp16 [T*k, H]")
    if topw.dtype != _f16 or topw.shape != (T, k):
        raise ValueError("topw must be fp16 [T, k]")
    dev = _require_cuda("moe_combine", y_sorted, topi, topw, pos)
    H = y_sorted.shape[1]
    y_sorted = y_sorted.contiguous()
    topi = topi.to(torch.int32).contiguous()
    topw = topw.contiguous()
    pos = pos.to(torch.int32).contiguous()
    out = torch.empty((T, H), dtype=_f16, device=dev)
    if T:
        with torch.cuda.device(dev):
            _lib.call("fni8_moe_combine_f16", _ptr(y_sorted), H, _ptr(topi), _ptr(topw), _ptr(pos),
                      T, k, _ptr(out), _stream(dev))
    return out


_ACTS = {"silu": 0, "gelu_tanh": 1}


def _act_code(act: str) -> int:
    try:
        return _ACTS[act]
    except KeyError:
        raise ValueError(f"unsupported fused activation {act!r} (silu, gelu_tanh)") from None


def _merged_rows(x: torch.Tensor, name: str):
    if x.dtype != _f16:
        raise ValueError(f"{name} expects fp16 (got {x.dtype})")
    if x.shape[-1] % 2:
        raise ValueError(f"{name}: last dimension {x.shape[-1]} is not 2 * intermediate")
    return _rows(x, x.shape[-1])


def act_and_mul(x: torch.Tensor, act: str = "silu") -> torch.Tensor:
    """fni8.act_and_mul(x, act): x fp16 [..., 2I] (gate | up) -> fp16 [..., I]
    (fni8serve/layers/activation.py:24, :40)."""
    dev = _require_cuda("act_and_mul", x)
    code = _act_code(act)
    x2, ldx = _merged_rows(x, "act_and_mul")
    M, I = x2.shape[0], x2.shape[1] // 2
    out = torch.empty((*x.shape[:-1], I), dtype=_f16, device=dev)
    if M and I:
        with torch.cuda.device(dev):
            _lib.call("fni8_act_and_mul_f16", _ptr(x2), ldx, M, I, code, _ptr(out), I,
                      _stream(dev))
    return out


def act_and_mul_quant(x: torch.Tensor, act: str = "silu"):
    """act_and_mul with the next linear's per-token quantization fused in:
    x fp16 [..., 2I] -> (xq int8 [M, I], xs fp32 [M]), bit-identical to
    quantize_rowwise(act_and_mul(x, act))."""
    dev = _require_cuda("act_and_mul_quant", x)
    code = _act_code(act)
    x2, ldx = _merged_rows(x, "act_and_mul_quant")
    M, I = x2.shape[0], x2.shape[1] // 2
    if I % 4:
        raise ValueError(f"act_and_mul_quant: intermediate size {I} is not a multiple of 4")
    xq = torch.empty((M, I), dtype=torch.int8, device=dev)
    xs = torch.empty((M,), dtype=torch.float32, device=dev)
    if M:
        # few rows: several workgroups share a row and exchange partial maxima
        # through a workspace (caching allocator; contents never matter)
        nw = int(_lib.load().fni8_act_and_mul_quant_workspace_bytes(M, I))
        work = torch.empty(nw, dtype=torch.uint8, device=dev) if nw else None
        with torch.cuda.device(dev):
            _lib.call("fni8_act_and_mul_quant_f16_ws", _ptr(x2), ldx, M, I, code, _ptr(xq), I,
                      _ptr(xs), _ptr(work), nw, _stream(dev))
    return xq, xs


def _norm_args(name, x, weight, residual):
    dev = _require_cuda(name, x, weight, residual)
    K = x.shape[-1]
    if x.dtype != _f16 or weight.dtype != _f16:
        raise ValueError(f"{name} expects fp16 x and weight (got {x.dtype}, {weight.dtype})")
    if weight.numel() != K:
        raise ValueError(f"{name}: weight has {weight.numel()} entries, x rows have {K}")
    if residual is not None and (residual.dtype != _f16 or residual.shape != x.shape):
        raise ValueError(f"{name}: residual must be fp16 with x's shape")
    x2, ldx = _rows(x, K)
    r2, ldr = (None, 0) if residual is None else _rows(residual, K)
    return dev, K, x2, ldx, r2, ldr, weight.contiguous()


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
            residual: torch.Tensor | None = None, unit_offset: bool = False):
    """fni8.rmsnorm(x, weight, eps, residual=, unit_offset=)
    (fni8serve/layers/norm.py:51-52): the normed fp16 tensor, or
    (normed, x + residual) when a residual is given."""
    if x.is_cuda:
        out = _lib.host().rmsnorm(x, weight, eps, residual, unit_offset, False)
        if out is not None:
            return out
    dev, K, x2, ldx, r2, ldr, w = _norm_args("rmsnorm", x, weight, residual)
    M = x2.shape[0]
    out = torch.empty(x.shape, dtype=_f16, device=dev)
    new_res = None if residual is None else torch.empty(x.shape, dtype=_f16, device=dev)
    if M:
        with torch.cuda.device(dev):
            _lib.call("fni8_rmsnorm_f16", _ptr(x2), ldx, _ptr(r2), ldr, _ptr(w),
                      ctypes.c_float(eps), int(bool(unit_offset)), M, K, _ptr(out), K,
                      _ptr(new_res), K, _stream(dev))
    return out if residual is None else (out, new_res)


def rmsnorm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                  residual: torch.Tensor | None = None, unit_offset: bool = False):
    """rmsnorm with the next linear's per-token quantization fused in:
    (xq int8 [M, K], xs fp32 [M]), or (xq, xs, x + residual) with a residual;
    bit-identical to quantize_rowwise(rmsnorm(...))."""
    if x.is_cuda:
        out = _lib.host().rmsnorm(x, weight, eps, residual, unit_offset, True)
        if out is not None:
            return out
    dev, K, x2, ldx, r2, ldr, w = _norm_args("rmsnorm_quant", x, weight, residual)
    if K % 4:
        raise ValueError(f"rmsnorm_quant: K={K} is not a multiple of 4")
    M = x2.shape[0]
    xq = torch.empty((M, K), dtype=torch.int8, device=dev)
    xs = torch.empty((M,), dtype=torch.float32, device=dev)
    new_res = None if residual is None else torch.empty(x.shape, dtype=_f16, device=dev)
    if M:
        with torch.cuda.device(dev):
            _lib.call("fni8_rmsnorm_quant_f16", _ptr(x2), ldx, _ptr(r2), ldr, _ptr(w),
                      ctypes.c_float(eps), int(bool(unit_offset)), M, K, _ptr(xq), K, _ptr(xs),
                      _ptr(new_res), K, _stream(dev))
    return (xq, xs) if residual is None else (xq, xs, new_res)


def gated_mlp(x: torch.Tensor, gate_up: QTensor, down: QTensor, act: str, bias_gate_up=None,
              bias_down=None, fuse_min_rows: int = 0):
    """down(act_and_mul(gate_up(x))) as one host call, the activation fused with down's
    quantization from `fuse_min_rows` rows; None when the general way has to take it."""
    g1, g2 = _group(gate_up), _group(down)
    if g1 < 0 or g2 < 0:
        return None
    return _lib.host().mlp(x, gate_up.data, gate_up.scale, g1, bias_gate_up, down.data,
                           down.scale, g2, bias_down, _act_code(act), fuse_min_rows)


_SCORES = {"softmax": 0, "sigmoid": 1}


def sparse_moe(x: torch.Tensor, gate: torch.Tensor, top_k: int, scoring: str, bias, num_groups,
               topk_group, renorm: bool, scale: float, w_gate_up, s_gate_up, g_gate_up: int,
               w_down, s_down, g_down: int, act: str):
    """Router, sort and the routed experts of x [T, H] as one host call (the chain of
    SparseMoE.experts_grouped; group size 0 for per_row_i8 experts); None when the
    general way has to take it."""
    if scoring not in _SCORES:
        return None
    groups = 0 if num_groups is None or topk_group is None else int(num_groups)
    return _lib.host().moe(x, gate, bias, _SCORES[scoring], groups,
                           int(topk_group) if groups else 0, top_k, bool(renorm), scale, w_gate_up,
                           s_gate_up, g_gate_up, w_down, s_down, g_down, _act_code(act))


def moe_route(logits: torch.Tensor, top_k: int, scoring: str = "softmax",
              bias: torch.Tensor | None = None, num_groups: int | None = None,
              topk_group: int | None = None, renorm: bool = True, scale: float = 1.0):
    """Router of SparseMoE (fni8serve/models/moe.py:62-91) in one launch:
    logits fp32 [T, E] -> (topw fp16 [T, k], topi int32 [T, k]), best first."""
    dev = _require_cuda("moe_route", logits, bias)
    if logits.dtype != torch.float32 or logits.dim() != 2:
        raise ValueError("moe_route expects fp32 logits [T, E]")
    if scoring not in _SCORES:
        raise ValueError(f"unsupported scoring function {scoring!r} (softmax, sigmoid)")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    T, E = logits.shape
    if bias is not None:
        if bias.numel() != E:
            raise ValueError(f"bias has {bias.numel()} entries, expected {E}")
        bias = bias.reshape(-1).float().contiguous()
    groups = 0 if num_groups is None or topk_group is None else int(num_groups)
    tg = 0 if groups == 0 else int(topk_group)
    topw = torch.empty((T, top_k), dtype=_f16, device=dev)
    topi = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    if T:
        ldl = logits.stride(0) if T > 1 else E
        with torch.cuda.device(dev):
            _lib.call("fni8_moe_route", _ptr(logits), T, E, ldl, _SCORES[scoring], _ptr(bias),
                      groups, tg, top_k, int(bool(renorm)), ctypes.c_float(scale), _ptr(topw),
                      _ptr(topi), _stream(dev))
    return topw, topi


def _heads(name: str, x: torch.Tensor):
    """x [T, H, D] fp16 with unit inner stride and 16-byte aligned rows (a copy where it is
    not): the tensor and its token and head strides."""
    if x.dtype != _f16 or x.dim() != 3:
        raise ValueError(f"{name} must be fp16 [tokens, heads, head_dim] (got {x.dtype}, "
                         f"{tuple(x.shape)})")
    T, H, D = x.shape
    if D == 0 or D % 8 or D > 256:
        raise ValueError(f"{name}: head_dim {D} must be a multiple of 8, at most 256")
    lt, lh = (x.stride(0) if T > 1 else H * D), (x.stride(1) if H > 1 else D)
    if x.numel() and (x.stride(2) != 1 or lt < D or lh < D or lt % 8 or lh % 8
                      or x.data_ptr() % 16):
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        lt, lh = H * D, D
    return x, max(lt, D), lh


def _index(name: str, t: torch.Tensor, n: int | None):
    if t.dtype not in (torch.int32, torch.int64) or t.dim() != 1 or (n is not None
                                                                   and t.numel() != n):
        raise ValueError(f"{name} must be int32 or int64 with {n if n is not None else 'one'} "
                         f"entries (got {t.dtype}, {tuple(t.shape)})")
    return _int32(t).contiguous()


def _int32(t: torch.Tensor):
    """64-bit positions, slots, pages or lengths in 32 bits; what lies outside stays outside
    every table and cache."""
    return t if t.dtype == torch.int32 else t.clamp(-1, 2 ** 31 - 1).to(torch.int32)


def _table(positions, cos_sin, T: int, D: int):
    """positions int32 [T] and cos_sin fp32 [P, R], or nothing: no rotation."""
    if (positions is None) != (cos_sin is None):
        raise ValueError("positions and cos_sin go together")
    if cos_sin is None:
        return None, None, 0, 0
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous fp32 [positions, rotary_dim] tensor")
    P, R = cos_sin.shape
    if R % 2 or not 0 < R <= D or P == 0:
        raise ValueError(f"cos_sin {tuple(cos_sin.shape)}: rotary_dim must be even and at most "
                         f"head_dim {D}, with one position at least")
    if cos_sin.data_ptr() % 16:
        cos_sin = cos_sin.clone()
    return _index("positions", positions, T), cos_sin, P, R


def _head_weight(name: str, w, D: int):
    if w is None:
        return None
    if w.dtype != _f16 or w.numel() != D:
        raise ValueError(f"{name} must be fp16 with {D} entries (got {w.dtype}, {w.numel()})")
    w = w.reshape(-1).contiguous()
    return w.clone() if w.data_ptr() % 16 else w


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                 k_weight: torch.Tensor | None, positions: torch.Tensor | None,
                 cos_sin: torch.Tensor | None, eps: float = 1e-6, interleaved: bool = False,
                 unit_offset: bool = False):
    """RMSNorm of every query and key head (a weight of None: none), then rotary positions,
    in one pass: q [T, Hq, D], k [T, Hk, D] fp16 -> (q', k'), rounded once.

    cos_sin fp32 [P, R] (RotaryEmbedding.cos_sin): row p holds the R/2 cosines, then the R/2
    sines of position p; the first R elements of a head turn, as halves (i, i + R/2) or, with
    interleaved, as pairs (2i, 2i + 1).  A position outside [0, P) gives NaN.  positions and
    cos_sin of None: norms only (fni8serve/layers/rotary.py:21-55,
    layers/gqa_attention.py:59-157)."""
    if q.is_cuda:
        out = _lib.host().norm_rope(q, k, q_weight, k_weight, positions, cos_sin, eps, interleaved,
                                    unit_offset)
        if out is not None:
            return out
    dev = _require_cuda("qk_norm_rope", q, k, q_weight, k_weight, positions, cos_sin)
    q, ldq, hsq = _heads("q", q)
    k, ldk, hsk = _heads("k", k)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    if k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in tokens or head_dim")
    pos, tab, P, R = _table(positions, cos_sin, T, D)
    q_weight = _head_weight("q_weight", q_weight, D)
    k_weight = _head_weight("k_weight", k_weight, D)
    q_out = torch.empty((T, Hq, D), dtype=_f16, device=dev)
    k_out = torch.empty((T, Hk, D), dtype=_f16, device=dev)
    if T and Hq + Hk:
        with torch.cuda.device(dev):
            _lib.call("fni8_qk_norm_rope_f16", _ptr(q), ldq, hsq, Hq, _ptr(k), ldk, hsk, Hk, T, D,
                      _ptr(q_weight), _ptr(k_weight), ctypes.c_float(eps), int(bool(unit_offset)),
                      _ptr(pos), _ptr(tab), P, R, int(bool(interleaved)), _ptr(q_out),
                      _ptr(k_out), _stream(dev))
    return q_out, k_out


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
         interleaved: bool = False):
    """`fni8.rope` (fni8serve/layers/rotary.py:52) into new tensors: qk_norm_rope without
    the norms."""
    if positions is None or cos_sin is None:
        raise ValueError("rope: positions and cos_sin are required")
    return qk_norm_rope(q, k, None, None, positions, cos_sin, interleaved=interleaved)


def _cache_args(k_cache, v_cache, k_scale, v_scale, Hk: int | None, D: int):
    """Checks of a paged cache [pages, heads, page_size, head_dim]: fp16, or int8 with fp32
    scales [pages, heads, page_size]."""
    if (k_scale is None) != (v_scale is None):
        raise ValueError("k_scale and v_scale go together")
    want = _f16 if k_scale is None else torch.int8
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dtype != want or c.dim() != 4 or not c.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {want} tensor [pages, heads, page_size, "
                             f"head_dim] (got {c.dtype}, {tuple(c.shape)}; 8 bits need k_scale "
                             "and v_scale, 16 bits none)")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} differ")
    N, H, page, dim = k_cache.shape
    if dim != D or (Hk is not None and H != Hk):
        raise ValueError(f"cache {tuple(k_cache.shape)} does not hold {Hk} heads of {D}")
    if D % 16:
        raise ValueError(f"head_dim {D} must be a multiple of 16 with a cache")
    if page < 16 or page > 65536 or page & (page - 1):
        raise ValueError(f"page_size {page} must be a power of two from 16 to 65536")
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s is not None and (s.dtype != torch.float32 or s.shape != (N, H, page)
                              or not s.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 tensor {(N, H, page)}")
    return N, H, page


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                positions: torch.Tensor | None, cos_sin: torch.Tensor | None,
                k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                eps: float = 1e-6, interleaved: bool = False,
                unit_offset: bool = False) -> torch.Tensor:
    """qk_norm_rope with the keys, and the values as they are, appended to the paged cache in
    the same pass: q [T, Hq, D], k and v [T, Hk, D] fp16 -> q'.

    k_cache, v_cache [pages, Hk, page_size, D] are written in place at slots [T] (page *
    page_size + offset): fp16, or int8 with the per-row scales k_scale, v_scale fp32 [pages,
    Hk, page_size], quantized as quantize_rowwise does.  A slot outside the cache (negative:
    padding) drops its token's rows; no slot may occur twice in a call
    (fni8serve/engine/kv_cache.py:265,681,700,730,826)."""
    if q.is_cuda:
        out = _lib.host().rope_append(q, k, v, k_cache, v_cache, k_scale, v_scale, slots, q_weight,
                                      k_weight, positions, cos_sin, eps, interleaved, unit_offset)
        if out is not None:
            return out
    dev = _require_cuda("rope_append", q, k, v, positions, cos_sin, k_cache, v_cache, slots,
                        k_scale, v_scale, q_weight, k_weight)
    q, ldq, hsq = _heads("q", q)
    k, ldk, hsk = _heads("k", k)
    v, ldv, hsv = _heads("v", v)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    if k.shape[0] != T or k.shape[2] != D or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} differ "
                         "in tokens, heads or head_dim")
    N, _, page = _cache_args(k_cache, v_cache, k_scale, v_scale, Hk, D)
    pos, tab, P, R = _table(positions, cos_sin, T, D)
    slots = _index("slots", slots, T)
    q_weight = _head_weight("q_weight", q_weight, D)
    k_weight = _head_weight("k_weight", k_weight, D)
    q_out = torch.empty((T, Hq, D), dtype=_f16, device=dev)
    if T:
        with torch.cuda.device(dev):
            _lib.call("fni8_rope_append_f16", _ptr(q), ldq, hsq, Hq, _ptr(k), ldk, hsk, Hk,
                      _ptr(v), ldv, hsv, T, D, _ptr(q_weight), _ptr(k_weight),
                      ctypes.c_float(eps), int(bool(unit_offset)), _ptr(pos), _ptr(tab), P, R,
                      int(bool(interleaved)), _ptr(q_out), _ptr(k_cache), _ptr(v_cache),
                      _ptr(k_scale), _ptr(v_scale), N, page, _ptr(slots), _stream(dev))
    return q_out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_tables: torch.Tensor, context_lens: torch.Tensor,
                    cu_seqlens: torch.Tensor | None = None, max_seqlen: int | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    scale: float | None = None, window: int | None = None) -> torch.Tensor:
    """Causal attention of new tokens over the paged cache, q [T, Hq, D] -> fp16 [T, Hq, D]
    (fni8serve/layers/gqa_attention.py:87,123,131,154,278).

    Sequence s owns tokens cu_seqlens[s] .. cu_seqlens[s + 1] of q (from 0 on, not
    decreasing; None: one token a sequence), the last of its context_lens[s] tokens; their keys
    and values are in the cache already, token c of the sequence in page
    block_tables[s, c // page_size].  Query head h
    reads key head h // (Hq / Hk).  max_seqlen bounds the new tokens of a sequence (None: not
    known; giving it saves time for decoded tokens; without cu_seqlens it is 1 whatever it
    says).  scale defaults to D ** -0.5; window
    is the number of keys that a query sees, itself among them.  A query without keys and
    tokens past cu_seqlens[-1] give 0; a token whose page is not in the cache, or past the block
    table, counts as NaN.  The weights of the values are rounded to fp16, sums are fp32."""
    if q.is_cuda:
        out = _lib.host().paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables,
                                          context_lens, cu_seqlens, max_seqlen, scale, window)
        if out is not None:
            return out
    dev = _require_cuda("paged_attention", q, k_cache, v_cache, block_tables, context_lens,
                        cu_seqlens, k_scale, v_scale)
    q, ldq, hsq = _heads("q", q)
    T, Hq, D = q.shape
    N, Hk, page = _cache_args(k_cache, v_cache, k_scale, v_scale, None, D)
    if Hq == 0 or Hk == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} key heads")
    if block_tables.dtype not in (torch.int32, torch.int64) or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 or int64 [sequences, pages]")
    B, width = block_tables.shape
    if cu_seqlens is None and T != B:
        raise ValueError(f"{T} tokens for {B} sequences: cu_seqlens is required")
    if window is not None and window < 1:
        raise ValueError(f"window {window} must be at least 1")
    if max_seqlen is not None and max_seqlen < 0:
        raise ValueError(f"max_seqlen {max_seqlen} is negative")
    lens = _index("context_lens", context_lens, B)
    cu = None if cu_seqlens is None else _index("cu_seqlens", cu_seqlens, B + 1)
    out = torch.empty((T, Hq, D), dtype=_f16, device=dev)
    if T == 0:
        return out
    if B == 0 or width == 0:
        if B:
            raise ValueError("block_tables has no pages")
        return out.zero_()
    tables = _int32(block_tables)
    if width > 1 and tables.stride(1) != 1 or B > 1 and tables.stride(0) < width:
        tables = tables.contiguous()
    ldt = tables.stride(0) if B > 1 else width
    most = 1 if cu is None else T if max_seqlen is None else max_seqlen
    nw = int(_lib.load().fni8_paged_attention_workspace_bytes(T, Hq, Hk, D, B, most, width * page))
    work = torch.empty(nw, dtype=torch.uint8, device=dev) if nw else None
    with torch.cuda.device(dev):
        _lib.call("fni8_paged_attention_f16", _ptr(q), ldq, hsq, T, Hq, Hk, D, _ptr(k_cache),
                  _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), N, page, _ptr(tables), ldt, width,
                  _ptr(lens), _ptr(cu), B, most,
                  ctypes.c_float(D ** -0.5 if scale is None else scale), window or 0, _ptr(out),
                  _ptr(work), nw, _stream(dev))
    return out


class LoraPlan(NamedTuple):
    """Which tokens belong to which adapter: those of adapter e are
    rows[seg_off[e]:seg_off[e + 1]], those without one segment S; both int32, on the GPU."""
    seg_off: torch.Tensor
    rows: torch.Tensor


def lora_plan(ids: torch.Tensor, num_adapters: int) -> LoraPlan:
    """The plan of a step's tokens, ids int [T]: each token's adapter, or any number outside
    [0, num_adapters) for none.  Made once a step: every projection of every layer shares it."""
    if not 0 < num_adapters <= 65534:
        raise ValueError(f"num_adapters {num_adapters} must be from 1 to 65534")
    _require_cuda("lora_plan", ids)
    ids = _index("ids", ids, None)
    if ids.numel() == 0:
        return LoraPlan(ids.new_zeros(num_adapters + 2), ids.new_empty(0))
    ids = torch.where((ids < 0) | (ids >= num_adapters), num_adapters, ids)
    seg_off, rows, _ = moe_sort(ids.unsqueeze(1), num_adapters + 1)
    return LoraPlan(seg_off, rows)


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan,
             scaling: torch.Tensor | None = None, splits: Sequence[int] | None = None,
             out: torch.Tensor | None = None, ranks: torch.Tensor | None = None) -> torch.Tensor:
    """y plus each token's own low-rank product, y fp16 [..., N] -> fp16 [..., N] in one call
    for all adapters (the unmerged forward of fni8serve/training/lora.py:14-170):

        out[t, n] = y[t, n] + scaling[e] * sum_j b[e, n, j] * (a[e] x[t])[p(n) * rank + j]

    x fp16 [..., K] (the input of the projection that made y), b fp16 [S, N, rank], a fp16
    [S, parts * rank, K], plan = lora_plan(ids, S).  splits: the widths of the parts of a
    merged projection, p(n) the part of column n (None: one part).  scaling fp32 [S] (None: 1).
    out: where the result goes; y itself adds in place and leaves rows without an adapter
    untouched, and nothing else may share elements with y; None allocates it.  rank is a multiple of 8, at most 256 (zeros fill up).
    ranks int32 [S, parts]: how many of a part's rank are the adapter's own; the others add
    nothing, also where x holds infinities, of which zeros make NaN (None: all).
    Sums are fp32; the result is rounded once."""
    if y.is_cuda and (out is None or out is y):
        z = _lib.host().lora_add(y, x, a, b, plan[0], plan[1], scaling, splits, ranks,
                                 out is y)
        if z is not None:
            return y if out is y else z
    for name, t, dims in (("y", y, 0), ("x", x, 0), ("a", a, 3), ("b", b, 3)):
        if t.dtype != _f16 or t.dim() < 1 or (dims and (t.dim() != dims or not t.is_contiguous())):
            raise ValueError(f"{name} must be {'a contiguous' if dims else 'an'} fp16 tensor"
                             f"{' of 3 dimensions' if dims else ''} (got {t.dtype}, "
                             f"{tuple(t.shape)})")
    S, N, rank = b.shape
    K = x.shape[-1]
    splits = [N] if splits is None else [int(n) for n in splits]
    if a.shape != (S, len(splits) * rank, K) or y.shape[-1] != N or sum(splits) != N:
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} do not fit x "
                         f"{tuple(x.shape)}, y {tuple(y.shape)} and splits {splits}")
    if scaling is not None:
        if scaling.dtype != torch.float32 or scaling.numel() != S:
            raise ValueError(f"scaling must be fp32 with {S} entries")
        scaling = scaling.reshape(-1).contiguous()
    if ranks is not None:
        if ranks.dtype != torch.int32 or ranks.shape != (S, len(splits)):
            raise ValueError(f"ranks must be int32 [{S}, {len(splits)}] (got {ranks.dtype}, "
                             f"{tuple(ranks.shape)})")
        ranks = ranks.contiguous()
    seg_off, rows = plan
    for name, t, n in (("seg_off", seg_off, S + 2), ("rows", rows, y.numel() // max(N, 1))):
        if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"plan.{name} must be a contiguous int32 tensor with {n} entries "
                             f"(got {t.dtype}, {tuple(t.shape)}): lora_plan({n} ids, {S})")
    if x.shape[:-1] != y.shape[:-1]:
        raise ValueError(f"x {tuple(x.shape)} and y {tuple(y.shape)} differ in tokens")
    if rank % 8 or not 0 < rank <= 256:
        raise ValueError(f"rank {rank} must be a multiple of 8, at most 256 (zeros fill up)")
    dev = _require_cuda("lora_add", y, x, a, b, seg_off, rows, scaling, ranks, out)
    x2, ldx = _rows(x, K)
    if out is None:
        y2, ldy = _rows(y, N)
        out = torch.empty(y.shape, dtype=_f16, device=dev)
        o2, ldo = out, N
    else:
        if out.dtype != _f16 or out.shape != y.shape:
            raise ValueError(f"out must be fp16 with y's shape {tuple(y.shape)}")
        o2, ldo = _rows(out, N)
        if o2.numel() and o2.data_ptr() != out.data_ptr():
            raise ValueError("out's rows must be evenly spaced, with unit inner stride")
        y2, ldy = (o2, ldo) if out is y else _rows(y, N)
        if y2.numel() and y2.data_ptr() == o2.data_ptr() and ldy != ldo:
            raise ValueError("out lies in y's memory with other strides")
    T = x2.shape[0]
    if T == 0:
        return out
    nw = int(_lib.load().fni8_lora_workspace_bytes(T, K, S, len(splits) * rank))
    work = torch.empty(nw, dtype=torch.uint8, device=dev) if nw else None
    with torch.cuda.device(dev):
        _lib.call("fni8_lora_add_ranks_f16", _ptr(x2), ldx, T, K, _ptr(a), _ptr(b), S, rank,
                  (ctypes.c_int64 * len(splits))(*splits), len(splits), _ptr(scaling),
                  _ptr(ranks), _ptr(seg_off), _ptr(rows), _ptr(y2), ldy, _ptr(o2), ldo,
                  _ptr(work), nw, _stream(dev))
    return out


def _setting(name: str, v, B: int, dtype: torch.dtype, least: float, most: float):
    """A sampling setting: one number for all rows (checked), or a tensor with one a row."""
    if torch.is_tensor(v):
        if v.numel() != B or v.dtype == torch.bool or v.is_complex() \
                or v.is_floating_point() != dtype.is_floating_point:
            raise ValueError(f"{name} must be a number or a {dtype} tensor with {B} entries (got "
                             f"{v.dtype}, {tuple(v.shape)})")
        v = _int32(v) if dtype == torch.int32 else v.to(dtype)
        return v.reshape(-1).contiguous(), 0
    if not least <= v <= most:
        raise ValueError(f"{name} {v} must be from {least} to {most}")
    return None, v


def sample(logits: torch.Tensor, u: torch.Tensor | None = None, temperature=1.0, top_k=0,
           top_p=1.0, min_p=0.0, return_logprobs: bool = False):
    """One token a row, logits fp16 or fp32 [..., V] -> int64 [...], drawn with the random
    numbers u fp32 [...] in [0, 1) (fni8serve/layers/sampler.py:20-87).

    Tokens are ordered by logit, ties by the lower index; their weights are exp((x - max) /
    temperature).  top_k keeps the first k, top_p a token while the mass before it is less than
    top_p times the mass that top_k keeps, min_p those with at least min_p times the largest
    weight: the shortest of these runs is kept, the first token always.  The token is the first
    kept one, in index order, at which the running mass exceeds u times the kept mass.

    Each setting is a number, or a tensor with one for each row.  temperature 0 takes the
    largest logit (u may be None where it is the number 0); top_k 0, top_p 1 and min_p 0 filter
    nothing; tensors may hold values outside these ranges, which mean the nearest one inside
    (a temperature that is NaN: see below).  A logit of minus infinity is never drawn.  A row
    with a NaN, or of minus infinity alone, gives -1 and the log-probability NaN.

    return_logprobs: (tokens, fp32 [...]), the logarithm of the token's share of the kept mass."""
    if logits.is_cuda:
        out = _lib.host().sample(logits, u, temperature, top_k, top_p, min_p, return_logprobs)
        if out is not None:
            return out
    if logits.dtype not in (_f16, torch.float32) or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be fp16 or fp32 [..., V] (got {logits.dtype}, "
                         f"{tuple(logits.shape)})")
    lead, V = logits.shape[:-1], logits.shape[-1]
    B = math.prod(lead)
    settings = [_setting(name, v, B, dtype, least, most) for name, v, dtype, least, most in (
        ("temperature", temperature, torch.float32, 0.0, 3e38),
        ("top_k", top_k, torch.int32, 0, 2 ** 31 - 1), ("top_p", top_p, torch.float32, 0.0, 1.0),
        ("min_p", min_p, torch.float32, 0.0, 1.0))]
    if u is None:
        if torch.is_tensor(temperature) or temperature != 0:
            raise ValueError("u is required where the temperature is not the number 0")
    elif u.dtype != torch.float32 or u.shape != lead:
        raise ValueError(f"u must be fp32 {tuple(lead)} (got {u.dtype}, {tuple(u.shape)})")
    dev = _require_cuda("sample", logits, u, *(t for t, _ in settings))
    x2, ldl = _rows(logits, V)
    u = None if u is None else u.reshape(-1).contiguous()
    tokens = torch.empty(lead, dtype=torch.int64, device=dev)
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev) if return_logprobs else None
    if B:
        (ts, t1), (ks, k1), (ps, p1), (ms, m1) = settings
        nw = int(_lib.load().fni8_sample_workspace_bytes(B, V))
        work = torch.empty(nw, dtype=torch.uint8, device=dev) if nw else None
        with torch.cuda.device(dev):
            _lib.call("fni8_sample", _ptr(x2), int(logits.dtype == torch.float32), B, V, ldl,
                      _ptr(u), _ptr(ts), ctypes.c_float(t1), _ptr(ks), int(k1), _ptr(ps),
                      ctypes.c_float(p1), _ptr(ms), ctypes.c_float(m1), _ptr(tokens),
                      _ptr(logprobs), _ptr(work), nw, _stream(dev))
    return (tokens, logprobs) if return_logprobs else tokens
