"""Rotary positions with several axes (``csrc/mrope.cu``): the language model's form, which rotates q and k of the fused projection
and appends k and v to the paged cache, and the vision towers' form, which lays q, k and v out for their attention.

Frequency ``i`` of the rotated half turns with the position of axis ``axes[i]``; :func:`section_axes` makes that list from a model's
sections."""
from __future__ import annotations

import struct

import torch

from . import KVLayer, _lib, reference as ref

MAX_DIM = 256                                             # of a head, on the GPU
_ARGS = struct.Struct("PqPqPqPPqPPPPPPPiiiiiiiiiff")        # MxMropeAppend of csrc/api.h


def section_axes(sections, half: int, interleaved: bool = False) -> torch.Tensor:
    """The axis of each of ``half`` frequencies, int32 on the CPU. ``sections``: frequencies per axis (time, height, width, and from
    the fourth on time, height, width again), one after the other; ``interleaved``: the axes take turns over the first
    ``3 * sections[1]`` (height) and ``3 * sections[2]`` (width) frequencies and the rest are time's."""
    return ref.section_axes(sections, half, interleaved)


def _check_angles(positions, axes, inv_freq, half, rows, device: int) -> None:
    if positions.dim() != 2 or positions.shape[1] != rows or positions.shape[0] < 1 or positions.dtype != torch.int32:
        raise ValueError(f"positions have to be int32 [axes, {rows}], not {positions.dtype} {tuple(positions.shape)}")
    if axes.dtype != torch.int32 or axes.dim() != 1 or axes.numel() < half or not axes.is_contiguous():
        raise ValueError(f"axes have to be a contiguous int32 tensor of {half} axis numbers")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or inv_freq.numel() < half or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq has to be a contiguous fp32 tensor of {half} frequencies")
    if not positions.get_device() == axes.get_device() == inv_freq.get_device() == device:
        raise ValueError("positions, axes and frequencies have to be on the device of the projection")


def mrope_append(qkv: torch.Tensor, positions: torch.Tensor, slot_mapping: torch.Tensor, inv_freq: torch.Tensor, axes: torch.Tensor,
                 kv: KVLayer, *, Hq: int, Hkv: int, D: int, rot_dim: int, traditional: bool = False, mscale: float = 1.0,
                 q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None, norm_eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotates q and k of ``qkv`` [T, (Hq + 2 Hkv) * D] by ``positions`` int32 [axes, T], appends k and v to the pool at
    ``slot_mapping`` int32 [T] (rows with a slot outside the pool, like -1, are not appended) → q [T, Hq * D].

    The first ``rot_dim`` columns of a head turn, as pairs (i, i + rot_dim / 2) or, ``traditional``, (2i, 2i + 1), and are scaled by
    ``mscale``. ``q_norm_w`` / ``k_norm_w`` [D]: rms norm of each head before it turns. Values are rounded once, at the end.
    ``out``: where q goes; q's own columns of ``qkv`` are fine, other overlap is not. No two rows may name one slot. A row's axis number
    outside ``positions`` takes the nearest axis."""
    if D < 1 or Hq < 0 or Hkv < 0 or Hq + Hkv == 0:
        raise ValueError(f"{Hq} + {Hkv} heads of {D} are no projection")
    T, width = qkv.shape[0], (Hq + 2 * Hkv) * D
    if qkv.dim() != 2 or qkv.shape[1] != width:
        raise ValueError(f"qkv has to be [T, {width}], not {tuple(qkv.shape)}")
    if rot_dim % 2 or not 0 <= rot_dim <= D:
        raise ValueError(f"rot_dim {rot_dim} is not an even part of a head of {D}")
    dev, dtype = qkv.get_device(), qkv.dtype
    _check_angles(positions, axes, inv_freq, rot_dim // 2, T, dev)
    if slot_mapping.dtype != torch.int32 or slot_mapping.shape != (T,) or not slot_mapping.is_contiguous() or slot_mapping.get_device() != dev:
        raise ValueError(f"slot_mapping has to be a contiguous int32 [{T}] tensor on the device of the projection")
    for name, t in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
        if t is not None and (t.shape != (D,) or t.dtype != dtype or t.get_device() != dev or not t.is_contiguous()):
            raise ValueError(f"{name} has to be a contiguous [{D}] {qkv.dtype} tensor on {qkv.device}")
    if out is not None and (out.shape != (T, Hq * D) or out.dtype != dtype or out.get_device() != dev):
        raise ValueError(f"out has to be a [{T}, {Hq * D}] {qkv.dtype} tensor on {qkv.device}")
    bits, k, v, block_size = kv.kv_bits, kv.k, kv.v, kv.block_size
    slabs = (k, v) if bits == 16 else (k, v, kv.k_meta, kv.v_meta)
    pool = (k.shape[0], Hkv, block_size)
    stored = (*pool, D if bits != 4 else D // 2)
    if k.shape != stored or v.shape != stored or (bits != 16 and (D % 64 or any(m is None or m.shape != (*pool, D // 64, 2) for m in slabs[2:]))):
        raise ValueError(f"the pool's slabs do not hold {Hkv} heads of {D} with {bits} bits in pages of {block_size}")
    if not qkv.is_cuda:
        q = ref.mrope_append(qkv, positions, slot_mapping, inv_freq, axes, kv, Hq=Hq, Hkv=Hkv, D=D, rot_dim=rot_dim,
                             traditional=traditional, mscale=mscale, q_norm_w=q_norm_w, k_norm_w=k_norm_w, norm_eps=norm_eps)
        return q if out is None else out.copy_(q)
    if dtype != torch.bfloat16 or D > MAX_DIM:
        raise ValueError(f"the kernel takes bf16 projections with heads of up to {MAX_DIM}, not {dtype} with {D}")
    ldqkv, one = qkv.stride()
    ldq, one_q = (Hq * D, 1) if out is None else out.stride()
    if one != 1 or one_q != 1 or T > 1 and (ldqkv < width or ldq < Hq * D):
        raise ValueError("the elements of a row of qkv and out have to be adjacent and its rows apart")
    if positions.stride(1) != 1 and T > 1:
        raise ValueError("an axis' positions have to be adjacent")
    for t in slabs:
        if t.get_device() != dev or not t.is_contiguous():
            raise ValueError("the pool's slabs have to be contiguous and on the device of the projection")
    if k.dtype != (torch.bfloat16 if bits == 16 else torch.uint8) or v.dtype != k.dtype or bits not in (16, 8, 4) or any(
            m.dtype != torch.bfloat16 for m in slabs[2:]):
        raise ValueError(f"a {bits}-bit pool of {k.dtype} is not covered")
    q = qkv.new_empty((T, Hq * D)) if out is None else out
    if T:
        at = lambda t: 0 if t is None else t.data_ptr()    # noqa: E731
        _lib.launch_on(qkv.device, "mx_mrope_append", _ARGS.pack(
            qkv.data_ptr(), ldqkv, q.data_ptr(), ldq, positions.data_ptr(), positions.stride(0), axes.data_ptr(), slot_mapping.data_ptr(),
            pool[0] * block_size, inv_freq.data_ptr(), k.data_ptr(), v.data_ptr(), *((0, 0) if bits == 16 else (slabs[2].data_ptr(), slabs[3].data_ptr())),
            at(q_norm_w), at(k_norm_w), positions.shape[0], T, Hq, Hkv, D, rot_dim, block_size, traditional, bits, norm_eps, mscale))
    return q


def axial_rope(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, axes: torch.Tensor, *, heads: int,
               D: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q, k, v of ``qkv`` [R, 3 * heads * D] (q of all heads, then k, then v) as fp32 [heads, R, D], q and k rotated as pairs
    (i, i + D / 2) by ``positions`` int32 [axes, R]."""
    R = qkv.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] != 3 * heads * D or D % 2:
        raise ValueError(f"qkv has to be [R, {3 * heads * D}] with heads of an even size, not {tuple(qkv.shape)}")
    _check_angles(positions, axes, inv_freq, D // 2, R, qkv.get_device())
    if not qkv.is_cuda:
        return ref.axial_rope(qkv, positions, inv_freq, axes, heads, D)
    if qkv.dtype != torch.bfloat16 or D > MAX_DIM:
        raise ValueError(f"the kernel takes bf16 projections with heads of up to {MAX_DIM}, not {qkv.dtype} with {D}")
    if qkv.stride(1) != 1 or R > 1 and (qkv.stride(0) < qkv.shape[1] or positions.stride(1) != 1):
        raise ValueError("the elements of a row and an axis' positions have to be adjacent")
    q, k, v = qkv.new_empty((3, heads, R, D), dtype=torch.float32).unbind()
    if R and heads:
        _lib.launch_on(qkv.device, "mx_axial_rope", qkv.data_ptr(), qkv.stride(0), q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(),
                       positions.stride(0), positions.shape[0], axes.data_ptr(), inv_freq.data_ptr(), R, heads, D)
    return q, k, v
