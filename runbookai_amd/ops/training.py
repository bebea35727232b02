"""Training ops: packed attention, cross-entropy, gradient norm and clipping.

On the GPU the kernels of csrc/packed_attn.hip, cross_entropy.hip and
grad_norm.hip, whose autograd nodes are in csrc/training.cpp; on the CPU the
references of reference.py. Arguments are checked here or, where all are on the
GPU, by the same rules in training.cpp (a short call is mostly host time).
On the GPU forward-mode derivatives and torch.jit.trace are refused
(NotImplementedError); the CPU's references have them.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _get_ext, reference


# ---------------------------------------------------------- packed attention

def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     seq_starts: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of packed sequences, with gradients for q, k and v.

    q [T, Hq, D], k and v [T, Hk, D] (Hq a multiple of Hk) hold sequences one
    after another; sequence b has rows seq_starts[b] up to seq_starts[b + 1],
    which may be none, and each row attends to its own sequence's rows up to
    itself. Rows in no sequence (a buffer's unused end) get zeros, in the
    output and in the gradients, whatever they hold. scale defaults to
    1 / sqrt(D).

    On the GPU: bfloat16, D 64 or 128. q, k and v may be views (slices of a
    fused projection, say): rows at 16-byte boundaries are read in place,
    others are copied first. The starts stay on the device and nothing waits
    for the host, so forward and backward can be captured into a graph (by
    autograd.grad, or while no eager step's graph of the same leaves lives).
    Starts are checked where they or q are on the host; with all on the device
    they cannot be without waiting for them: where they fall or leave [0, T],
    every output and gradient is NaN. A value that is not finite may reach any
    row of its own sequence (a shut place's product is 0 times the value), but
    no other's.

    The training counterpart of prefill_attention, which has no gradients."""
    if q.is_cuda and seq_starts.is_cuda:
        return _get_ext().packed_attention(q, k, v, seq_starts, scale)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [tokens, heads, head dim]")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"shapes do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")
    if q.shape[2] == 0:
        raise ValueError("the head dim must not be 0")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads are no multiple of "
                         f"{k.shape[1]} key/value heads")
    if (not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device)
            or not q.dtype.is_floating_point):
        raise ValueError("q, k and v must have one floating-point type and one device")
    if (seq_starts.dim() != 1 or seq_starts.numel() < 1
            or seq_starts.dtype not in (torch.int32, torch.int64)):
        raise ValueError("seq_starts must be a vector of whole numbers, one more than sequences")
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not 2.0 ** -126 <= scale < 2.0 ** 127:   # times log2(e) it is still an fp32 number
        raise ValueError(f"scale must be positive and a normal fp32 number, not {scale}")
    starts = seq_starts.tolist()
    if starts[0] < 0 or starts[-1] > q.shape[0] or starts != sorted(starts):
        raise ValueError(f"seq_starts must rise within 0 and {q.shape[0]}")
    if not q.is_cuda:
        return reference.packed_attention(q, k, v, seq_starts, scale)
    return _get_ext().packed_attention(q, k, v, seq_starts.to(q.device), scale)


# ------------------------------------------------------------- cross-entropy

_MODES = {"none": 0, "mean": 1, "sum": 2}


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100,
                  reduction: str = "mean") -> torch.Tensor:
    """Cross-entropy of logits [N, V] with integer labels [N], with its
    gradient; fp32 result.

    Rows labelled ignore_index count for nothing: their loss is 0, their
    gradient zeros, their logits are not read. reduction: "mean" over the
    labelled rows (NaN if there are none), "sum", or "none" for one loss a
    row. A label outside the vocabulary makes its row's loss and gradient NaN.
    Logits of -inf (vocabulary shut off) have probability and gradient 0.

    On the GPU: float32, bfloat16 or float16 logits. Rows of any distance and
    alignment are read in place (columns apart from each other are copied
    first); the sums are fp32 and over rows fp64."""
    if reduction not in _MODES:
        raise ValueError(f"reduction must be one of {sorted(_MODES)}, not {reduction!r}")
    if logits.is_cuda:
        return _get_ext().cross_entropy(logits, targets, ignore_index, _MODES[reduction])
    if logits.dim() != 2 or logits.shape[1] < 1 or targets.shape != logits.shape[:1]:
        raise ValueError(f"logits must be [rows, vocabulary] with one label a row: logits "
                         f"{tuple(logits.shape)}, targets {tuple(targets.shape)}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"targets must be whole numbers, not {targets.dtype}")
    if not logits.dtype.is_floating_point:
        raise ValueError(f"logits must be floating-point numbers, not {logits.dtype}")
    if targets.device != logits.device:
        raise ValueError("logits and targets must be on one device")
    return reference.cross_entropy(logits, targets.long(), ignore_index, reduction)


# ------------------------------------------------------------- gradient norm

_EPS = 1e-6   # in the divisor, so that a norm of zero divides


def _list(parameters) -> list[torch.Tensor]:
    return [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)


def _check_host(grads: list[torch.Tensor], write: bool = False) -> None:
    """What the kernels' bindings check of gradients on the GPU."""
    spans = []
    for g in grads:
        if g.layout != torch.strided or g.dtype not in (torch.float32, torch.bfloat16,
                                                        torch.float16):
            raise ValueError(f"gradients must be dense float32, bfloat16 or float16, "
                             f"not {g.layout} {g.dtype}")
        if g.device != grads[0].device:
            raise ValueError("gradients must be on one device")
        if g.numel():
            last = sum((n - 1) * step for n, step in zip(g.shape, g.stride()))
            spans.append((g.data_ptr(), g.data_ptr() + (last + 1) * g.element_size()))
    spans.sort()
    if write and any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
        raise ValueError("two of the gradients share or interleave their memory")


def _first(parameters: list[torch.Tensor]) -> Optional[torch.Tensor]:
    """The first gradient, whose device decides where the call runs."""
    return next((p.grad for p in parameters if p.grad is not None), None)


def _none(parameters: list[torch.Tensor]) -> torch.Tensor:
    """The norm where no parameter has a gradient."""
    return torch.zeros((), device=parameters[0].device if parameters else None)


def grad_norm(parameters) -> torch.Tensor:
    """2-norm of all parameters' gradients together (fp32 scalar on the
    gradients' device, or the first parameter's if there are none); parameters
    without a gradient are passed over, wherever they are."""
    parameters = _list(parameters)
    first = _first(parameters)
    if first is None:
        return _none(parameters)
    if first.is_cuda:
        return _get_ext().grad_norm(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    _check_host(grads)
    with torch.no_grad():
        return reference.grad_norm(grads)


def clip_grad_norm_(parameters, max_norm: float,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales all parameters' gradients in place by
    min(1, max_norm / (norm + 1e-6)) and returns their norm before that (as
    grad_norm). Two gradients whose memory overlaps or interleaves
    (the same one twice, columns of one buffer) are refused.

    On the GPU: any mix of float32, bfloat16 and float16 gradients of any
    sizes, strides and alignment on one device. The norm is summed in fp64 and
    the factor applied in fp64. The host waits for nothing (so it can be
    captured into a graph) unless error_if_nonfinite is set, which raises for a
    norm that is not finite and leaves the gradients as they were."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative: {max_norm}")
    parameters = _list(parameters)
    if error_if_nonfinite:
        norm = grad_norm(parameters)
        if not torch.isfinite(norm):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}; "
                               "they are left as they were")
    first = _first(parameters)
    if first is None:
        return _none(parameters)
    if first.is_cuda:
        return _get_ext().grad_clip(parameters, max_norm, _EPS)
    grads = [p.grad for p in parameters if p.grad is not None]
    _check_host(grads, write=True)
    with torch.no_grad():
        return reference.grad_clip(grads, max_norm, _EPS)
