"""Training ops: argument checks, autograd, dispatch to the HIP kernels.

The public entry points, with their documentation, are in ops/__init__.py.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _get_ext, reference


# ---------------------------------------------------------- packed attention

def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, or a dense copy where its rows of a head are not dense at 16-byte
    boundaries."""
    if (t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0
            and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, scale):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        out, lse, tiles = _get_ext().packed_attn_fwd(q, k, v, starts, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, tiles)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, tiles = ctx.saved_tensors
        dq, dk, dv = _get_ext().packed_attn_bwd(_rows16(dout), q, k, v, out, lse,
                                                tiles, ctx.scale)
        return dq, dk, dv, None, None


def packed_attention(q, k, v, seq_starts, scale: Optional[float] = None):
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, head dim]")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"shapes do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads are no multiple of "
                         f"{k.shape[1]} key/value heads")
    if not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device):
        raise ValueError("q, k and v must have one type and device")
    if (seq_starts.dim() != 1 or seq_starts.numel() < 1
            or seq_starts.dtype not in (torch.int32, torch.int64)):
        raise ValueError("seq_starts must be a vector of whole numbers, one more than sequences")
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, not {scale}")
    if not seq_starts.is_cuda:
        starts = seq_starts.tolist()
        if starts[0] < 0 or starts[-1] > q.shape[0] or starts != sorted(starts):
            raise ValueError(f"seq_starts must rise within 0 and {q.shape[0]}")
    if not q.is_cuda:
        return reference.packed_attention(q, k, v, seq_starts, scale)
    if q.dtype != torch.bfloat16:
        raise ValueError(f"on the GPU q, k and v must be bfloat16, not {q.dtype}")
    if q.shape[2] not in (64, 128):
        raise ValueError(f"on the GPU the head dim must be 64 or 128, not {q.shape[2]}")
    starts = seq_starts.to(device=q.device, dtype=torch.int32).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, starts, scale)
    return _get_ext().packed_attn_fwd(_rows16(q), _rows16(k), _rows16(v), starts, scale,
                                      False)[0]


# ------------------------------------------------------------- cross-entropy

_MODES = {"none": 0, "mean": 1, "sum": 2}


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore, mode):
        got = _get_ext().xent_fwd(logits, targets, ignore, mode, True)
        ctx.save_for_backward(logits, targets, got[1], *got[3:])
        ctx.ignore = ignore
        return got[2] if mode else got[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        logits, targets, stats, *factor = ctx.saved_tensors
        return (_get_ext().xent_bwd(gout, logits, targets, ctx.ignore, stats,
                                    factor[0] if factor else None), None, None, None)


def cross_entropy(logits, targets, ignore_index: int = -100, reduction: str = "mean"):
    if logits.dim() != 2 or logits.shape[1] < 1 or targets.shape != logits.shape[:1]:
        raise ValueError(f"logits must be [rows, vocabulary] with one label a row: logits "
                         f"{tuple(logits.shape)}, targets {tuple(targets.shape)}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"targets must be whole numbers, not {targets.dtype}")
    if targets.device != logits.device:
        raise ValueError("logits and targets must be on one device")
    if reduction not in _MODES:
        raise ValueError(f"reduction must be one of {sorted(_MODES)}, not {reduction!r}")
    targets = targets.long().contiguous()
    if not logits.is_cuda:
        return reference.cross_entropy(logits, targets, ignore_index, reduction)
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"on the GPU logits must be float32, bfloat16 or float16, "
                         f"not {logits.dtype}")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    mode = _MODES[reduction]
    if torch.is_grad_enabled() and logits.requires_grad:
        return _CrossEntropy.apply(logits, targets, ignore_index, mode)
    got = _get_ext().xent_fwd(logits, targets, ignore_index, mode, False)
    return got[2] if mode else got[0]


# ------------------------------------------------------------- gradient norm

_EPS = 1e-6   # in the divisor, so that a norm of zero divides


def _grads(parameters) -> list[torch.Tensor]:
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    for g in grads:
        if g.layout != torch.strided or g.dtype not in (torch.float32, torch.bfloat16,
                                                        torch.float16):
            raise ValueError(f"gradients must be dense float32, bfloat16 or float16, "
                             f"not {g.layout} {g.dtype}")
        if g.device != grads[0].device:
            raise ValueError("gradients must be on one device")
    return grads


@torch.no_grad()
def grad_norm(parameters) -> torch.Tensor:
    grads = _grads(parameters)
    if not grads:
        return torch.zeros(())
    if not grads[0].is_cuda:
        return reference.grad_norm(grads)
    return _get_ext().grad_norm(grads)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative: {max_norm}")
    if error_if_nonfinite:
        parameters = ([parameters] if isinstance(parameters, torch.Tensor)
                      else list(parameters))
        norm = grad_norm(parameters)
        if not torch.isfinite(norm):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}; "
                               "they are left as they were")
    grads = _grads(parameters)
    if not grads:
        return torch.zeros(())
    if not grads[0].is_cuda:
        return reference.grad_clip(grads, max_norm, _EPS)
    return _get_ext().grad_clip(grads, max_norm, _EPS)
