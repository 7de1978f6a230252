"""The step between two sub-layers of a residual stream as one operator: the norm behind a branch, its gate and scale, the sum with
the residual and the norm in front of the next sub-layer (``csrc/branch_norm.cu``). Models with norms before and after each
sub-layer, with scaled branches or with per-channel branch scales take it at every layer."""
from __future__ import annotations

import struct

import torch

from . import _lib, reference as ref

_ARGS = struct.Struct("PqPqPPPPPqPqiifffii")        # MxBranchNorm of csrc/api.h
_TYPES = (torch.bfloat16, torch.float32)


def _row_stride(t: torch.Tensor | None, rows: int, dim: int) -> int:
    if t is None:
        return dim
    ld, one = t.stride()
    if one != 1 and dim > 1 or rows > 1 and ld < dim:
        raise ValueError("the elements of a row have to be adjacent and rows apart")
    return ld


def branch_norm(x: torch.Tensor, residual: torch.Tensor | None = None, *, post_w: torch.Tensor | None = None,
                gate: torch.Tensor | None = None, scale: float = 1.0, pre_w: torch.Tensor | None = None,
                pre_b: torch.Tensor | None = None, layer_norm: bool = False, eps: float = 1e-6, w_bias: float = 0.0,
                out: torch.Tensor | None = None) -> tuple[torch.Tensor | None, torch.Tensor]:
    """``b = rmsnorm(x) * (post_w + w_bias)`` (``x`` itself without ``post_w``); ``h = residual + scale * gate * b``;
    ``y = norm(h) * (pre_w + w_bias) + pre_b`` → ``(y, h)``, ``y`` None without ``pre_w``.

    ``x`` and ``residual`` are [rows, dim] of one type (bf16 or fp32), their rows may be strided; ``gate`` (a factor per channel), the
    weights and ``pre_b`` are [dim] of the same type. ``layer_norm``: the last norm is a layer norm (``pre_b`` belongs to it), else an
    rms norm. Sums and statistics are fp32; ``h`` is rounded once and ``y`` is the norm of the rounded ``h``. ``out``: where ``h``
    goes (``x`` or ``residual`` itself is fine)."""
    if x.dim() != 2:
        raise ValueError(f"branch_norm takes rows [rows, dim], not {tuple(x.shape)}")
    rows, dim = shape = x.shape
    dtype, dev = x.dtype, x.get_device()
    if dtype not in _TYPES:
        raise ValueError(f"branch_norm takes bf16 or fp32 rows, not {dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype or residual.get_device() != dev) or (
            out is not None and (out.shape != shape or out.dtype != dtype or out.get_device() != dev)):
        raise ValueError(f"residual and out have to be like x: {tuple(shape)} {dtype} on {x.device}")
    for t in (post_w, gate, pre_w, pre_b):
        if t is not None and (t.dtype != dtype or t.dim() != 1 or t.numel() != dim or t.get_device() != dev or not t.is_contiguous()):
            raise ValueError(f"weights, gate and bias have to be contiguous [{dim}] {dtype} tensors on {x.device}")
    if pre_b is not None and (pre_w is None or not layer_norm):
        raise ValueError("pre_b belongs to a layer norm (pre_w, layer_norm=True)")
    if not 1 <= dim <= 32768:
        raise ValueError(f"rows of 1 to 32768 elements are covered, not {dim}")
    if not x.is_cuda:
        y, h = ref.branch_norm(x, residual, post_w, gate, scale, pre_w, pre_b, layer_norm, eps, w_bias)
        return y, h if out is None else out.copy_(h)
    dense = x.is_contiguous()
    ldx, ldr, ldh = (_row_stride(t, rows, dim) for t in (x, residual, out))
    h = out if out is not None else torch.empty_like(x) if dense else torch.empty(shape, dtype=dtype, device=x.device)
    y = None if pre_w is None else torch.empty_like(x) if dense else torch.empty(shape, dtype=dtype, device=x.device)
    if rows:
        at = lambda t: 0 if t is None else t.data_ptr()    # noqa: E731
        _lib.launch_on(x.device, "mx_branch_norm", _ARGS.pack(
            x.data_ptr(), ldx, at(residual), ldr, at(post_w), at(gate), at(pre_w), at(pre_b), h.data_ptr(), ldh, at(y), dim,
            rows, dim, scale, eps, w_bias, layer_norm, dtype == torch.float32))
    return y, h


def branch_step(x: torch.Tensor, residual: torch.Tensor, *, post_w=None, gate=None, scale: float = 1.0, pre_w=None, pre_b=None,
                layer_norm: bool = False, eps: float = 1e-6, w_bias: float = 0.0) -> tuple[torch.Tensor | None, torch.Tensor]:
    """:func:`branch_norm` as models take it: on the CPU, where they may hold other types, also for those and for weights of a type of
    their own (by the plain statement)."""
    if not x.is_cuda and (x.dtype not in _TYPES or any(t is not None and t.dtype != x.dtype for t in (post_w, gate, pre_w, pre_b))):
        return ref.branch_norm(x, residual, post_w, gate, scale, pre_w, pre_b, layer_norm, eps, w_bias)
    return branch_norm(x, residual, post_w=post_w, gate=gate, scale=scale, pre_w=pre_w, pre_b=pre_b, layer_norm=layer_norm, eps=eps, w_bias=w_bias)
