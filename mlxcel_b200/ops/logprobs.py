"""Log probabilities of given tokens, the entropy of every row's distribution and its most likely tokens, from logits
(``csrc/logprobs.cu``) or straight from hidden rows and the head's weights."""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import _lib, linear, reference as ref

MAX_TOP = 64
TYPES = (torch.bfloat16, torch.float32)           # of logits, hidden rows, weights and biases
_ARGS = struct.Struct("PqPPPPPPPiiiiiiiff")        # MxTokenLogprobs of csrc/api.h
# head_logprobs keeps its logits on the chip, unless few rows meet large weights: there both forms read the weights at the pace of the
# memory, and the smaller tiles of `linear` are the faster ones. us on the chip / through memory: 8 rows, 128256 x 4096 230 / 174, 64
# rows 226 / 194, 100 rows 231 / 229, 256 rows 251 / 437; 8 rows, 50257 x 1024 50 / 70, 5000 x 512 27 / 58.
FEW_ROWS, LARGE_WEIGHTS = 64, 1 << 28
PARTIAL_BYTES = 256 << 20        # of the column tiles' sums that are held at once


class TokenLogprobs(NamedTuple):
    """``logprob`` of the given tokens (shaped like them), ``entropy`` (nats) and log normaliser ``lse`` [R], ``top_ids`` int32 and
    ``top_logprobs`` [R, top], most likely first and equal ones by index; all but the ids fp32."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def _check(rows: int, vocab: int, device, ids, bias, scale: float, softcap: float, dim: int) -> None:
    if ids.dtype not in (torch.int32, torch.int64) or ids.dim() not in (1, 2)[:dim] or ids.shape[0] != rows or ids.device != device:
        raise ValueError(f"ids have to be int32 or int64 [{rows}]{f' or [{rows}, n]' if dim > 1 else ''} on {device}")
    if bias is not None and (bias.shape != (vocab,) or bias.dtype not in TYPES or bias.device != device
                             or not bias.is_contiguous()):
        raise ValueError(f"bias has to be a contiguous bf16 or fp32 [{vocab}] tensor on {device}")
    if not scale > 0.0 or not softcap >= 0.0:
        raise ValueError("scale has to be positive and softcap not negative")


def widened(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself, or in fp32 where it is of a type that is not covered here (models on the CPU run in others)."""
    return t if t.dtype in TYPES else t.float()


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0, *, bias: torch.Tensor | None = None, scale: float = 1.0,
                   softcap: float = 0.0) -> TokenLogprobs:
    """``logits`` [R, V] (bf16 or fp32, rows may be strided) and the tokens asked for, ``ids`` [R] or [R, n]. The distribution is that
    of ``softcap * tanh((logits + bias) * scale / softcap)`` (no cap: 0). NaN counts as -inf; a row with nothing left has log
    probabilities and ``lse`` of -inf and entropy 0; an id outside the vocabulary has log probability NaN. ``top``: up to 64."""
    if logits.dim() != 2 or logits.dtype not in TYPES:
        raise ValueError(f"logits have to be bf16 or fp32 [R, V], not {logits.dtype} {tuple(logits.shape)}")
    R, V = logits.shape
    _check(R, V, logits.device, ids, bias, scale, softcap, 2)
    if not 0 <= top <= min(V, MAX_TOP) or V < 1:
        raise ValueError(f"top {top} is not within 0 to {min(V, MAX_TOP)}")
    if not logits.is_cuda:
        return TokenLogprobs(*ref.token_logprobs(logits, ids, top, bias, scale, softcap))
    if logits.stride(1) != 1 and V > 1 or R > 1 and logits.stride(0) < V:
        raise ValueError("the logits of a row have to be adjacent and rows apart")
    ids = ids.contiguous()
    # one buffer for all results (they are a few words per row)
    n, k = ids.numel(), R * top
    logprob, entropy, lse, best, at = torch.empty(n + 2 * R + 2 * k, dtype=torch.float32, device=logits.device).split([n, R, R, k, k])
    r = TokenLogprobs(logprob if ids.dim() == 1 else logprob.view(ids.shape), entropy, lse, at.view(torch.int32).view(R, top), best.view(R, top))
    if R:
        _lib.launch_on(logits.device, "mx_token_logprobs", _ARGS.pack(
            logits.data_ptr(), logits.stride(0), ids.data_ptr(), 0 if bias is None else bias.data_ptr(), logprob.data_ptr(), entropy.data_ptr(),
            lse.data_ptr(), at.data_ptr(), best.data_ptr(), logits.dtype == torch.float32, ids.dtype == torch.int64, n // R,
            bias is not None and bias.dtype == torch.float32, top, R, V, scale, softcap))
    return r


def head_logprobs(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, *, bias: torch.Tensor | None = None, scale: float = 1.0,
                  softcap: float = 0.0) -> TokenLogprobs:
    """:func:`token_logprobs` (without alternatives) of the logits ``x @ w^T``, which are fp32 sums and never rounded to fewer bits.
    ``x`` [R, K] and the head's weights ``w`` [V, K] are bf16 (or both fp32); ``ids`` [R]."""
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1] or x.dtype != w.dtype or x.device != w.device:
        raise ValueError("hidden rows [R, K] and head weights [V, K] of one type are needed on one device")
    if x.dtype not in TYPES:
        raise ValueError(f"hidden rows have to be bf16 or fp32, not {x.dtype}")
    R, V = x.shape[0], w.shape[0]
    _check(R, V, x.device, ids, bias, scale, softcap, 1)
    if V < 1 or x.shape[1] < 1:
        raise ValueError("an empty vocabulary or width has no distribution")
    if not x.is_cuda:
        return TokenLogprobs(*ref.token_logprobs(x.float() @ w.float().t(), ids, 0, bias, scale, softcap))
    if any(t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1] for t in (x, w)):
        raise ValueError("the elements of a row have to be adjacent and rows apart")
    f = dict(dtype=torch.float32, device=x.device)
    r = TokenLogprobs(torch.empty(R, **f), torch.empty(R, **f), torch.empty(R, **f), torch.empty(R, 0, dtype=torch.int32, device=x.device),
                      torch.empty(R, 0, **f))
    K = x.shape[1]
    ldx, ldw = x.stride(0) if R > 1 else K, w.stride(0) if V > 1 else K
    if R and (R > FEW_ROWS or V * K <= LARGE_WEIGHTS) and x.dtype == torch.bfloat16 and not (K % 8 or ldx % 8 or ldw % 8 or (x.data_ptr() | w.data_ptr()) % 16):
        tiles, ids = -(-V // 256), ids.contiguous()
        part = min(R, max(256, PARTIAL_BYTES // (24 * tiles) // 256 * 256))
        partials = torch.empty((6 * tiles + 1) * part, **f)
        for r0 in range(0, R, part):
            _lib.launch_on(x.device, "mx_head_logprobs", x.data_ptr() + 2 * r0 * ldx, w.data_ptr(), ids.data_ptr() + r0 * ids.element_size(),
                           int(ids.dtype == torch.int64), _lib.ptr(bias), int(bias is not None and bias.dtype == torch.float32), float(scale),
                           float(softcap), partials.data_ptr(), r.logprob.data_ptr() + 4 * r0, r.entropy.data_ptr() + 4 * r0,
                           r.lse.data_ptr() + 4 * r0, min(part, R - r0), V, K, ldx, ldw, _lib.workspace(x.device).data_ptr())
        return r
    part = max(1, (1 << 26) // V)                 # rows whose logits are held at once: 256 MB
    if R == 0:
        return r
    with torch.cuda.device(x.device):
        if R <= part:
            return token_logprobs(linear(x, w, out_fp32=True, w_fresh=True), ids, bias=bias, scale=scale, softcap=softcap)
        for r0 in range(0, R, part):
            got = token_logprobs(linear(x[r0:r0 + part], w, out_fp32=True, w_fresh=True), ids[r0:r0 + part], bias=bias, scale=scale, softcap=softcap)
            for whole, piece in zip(r[:3], got[:3]):
                whole[r0:r0 + part] = piece
    return r
