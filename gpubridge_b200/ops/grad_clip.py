"""The global norm of many gradient tensors and clipping by it (``csrc/gb_grad_norm.cu``).

    norm = grad_norm(tensors)                              # 0-dim fp32 tensor, nothing waits
    norm = clip_grad_norm_(model.parameters(), 1.0)        # torch.nn.utils' arithmetic, in place

Squares and sums are held in 64 bits and added in a fixed order.  The list of tensors travels in
the launch itself, so both calls can be captured in a CUDA graph; whether the gradients are
rescaled is decided on the device (within the limit nothing is written).  The data-parallel
trainer clips without the second pass over the gradients: ``FlatAdamW.step(max_norm=...)`` takes
the factor into the update.

On CPU tensors the same results come from plain torch operations.
"""
from __future__ import annotations

import math
from collections.abc import Iterable

import torch

from gpubridge_b200.ops import _build_ops

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_EPS = 1e-6


def _norm_type(value) -> bool:
    """True for the largest magnitude, False for the 2-norm."""
    value = float(value)
    if value == 2.0:
        return False
    if value == math.inf:
        return True
    raise ValueError(f"norm_type must be 2 or inf, got {value}")


def _max_norm(value) -> float:
    value = float(value)
    if not value >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {value}")
    return value


def _checked(tensors) -> tuple[list[torch.Tensor], torch.device | None]:
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    tensors = list(tensors)
    device = None
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"gradients are tensors, got {type(t).__name__}")
        if t.is_sparse or t.layout is not torch.strided:
            raise ValueError("sparse gradients have no fused norm")
        if hasattr(t, "to_local"):
            raise TypeError("a DTensor's norm spans ranks: pass its local parts and join their norms, "
                            "or use torch.nn.utils.clip_grad_norm_")
        if t.dtype not in _FLOATS and not (t.device.type == "cpu" and t.is_floating_point()):
            raise ValueError(f"gradients are float32, bfloat16 or float16 on the GPU, got {t.dtype}")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"gradients are on one device, got {device} and {t.device}")
    return tensors, device


def _dense(t: torch.Tensor) -> bool:
    """Whether the values fill the memory from data_ptr on without gaps, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda pair: pair[1]):
        if size == 1:
            continue
        if stride != expected:
            return False
        expected *= size
    return True


def _cpu_norm(tensors, maximum: bool, scale: float = 1.0) -> torch.Tensor:
    if maximum:
        parts = [t.abs().max().double() for t in tensors if t.numel()]
        total = torch.stack(parts).max() if parts else torch.zeros((), dtype=torch.float64)
    else:
        parts = [t.double().square().sum() for t in tensors if t.numel()]
        total = torch.stack(parts).sum().sqrt() if parts else torch.zeros((), dtype=torch.float64)
    return (total * abs(scale)).float()


def _gpu_norm(tensors, maximum: bool, max_norm: float) -> torch.Tensor:
    """Device tensor of two floats: the norm, and the factor that clips it."""
    ops = _build_ops.load()
    result = ops.grad_norm(tensors, maximum, 1.0, max_norm)
    if result is None:                         # gaps between the values, or a list without tensors
        result = ops.grad_norm([t if _dense(t) else t.contiguous() for t in tensors], maximum, 1.0, max_norm)
    return result


def grad_norm(tensors: Iterable[torch.Tensor] | torch.Tensor, norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, with ``norm_type=inf``, the largest magnitude) over all values of
    ``tensors``, as a 0-dim float32 tensor on their device.  An empty list has norm 0."""
    maximum = _norm_type(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if tensors and isinstance(tensors[0], torch.Tensor) and tensors[0].is_cuda and \
            all(isinstance(t, torch.Tensor) for t in tensors):
        result = _build_ops.load().grad_norm(tensors, maximum, 1.0, 0.0)
        if result is not None:
            return result[0]
    tensors, device = _checked(tensors)
    with torch.no_grad():
        if device is None or device.type != "cuda":
            return _cpu_norm(tensors, maximum)
        return _gpu_norm(tensors, maximum, 0.0)[0]


def _refuse_overlap(tensors) -> None:
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors
                   if t.numel() and _dense(t))
    gappy = [t.data_ptr() for t in tensors if t.numel() and not _dense(t)]     # these may lie between one another
    if any(start < end for (_, end), (start, _) in zip(spans, spans[1:])) or len(set(gappy)) < len(gappy):
        raise ValueError("two of the gradients share memory: it would be scaled twice")


def _scale_(tensors, result: torch.Tensor) -> None:
    _build_ops.load().grad_scale([t for t in tensors if _dense(t)], result)
    for t in tensors:
        if not _dense(t):                      # gaps between the values: torch walks the strides
            t.copy_(t.float() * result[1])


def _grads(parameters) -> list[torch.Tensor]:
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [p.grad for p in parameters if p.grad is not None]


def clip_grads_with_norm_(parameters: Iterable[torch.Tensor] | torch.Tensor, max_norm: float,
                          total_norm: torch.Tensor) -> None:
    """Scale the parameters' gradients, in place, by ``min(1, max_norm / (total_norm + 1e-6))`` for
    a norm found elsewhere (over shards on several ranks): a float32 scalar tensor on their device."""
    max_norm = _max_norm(max_norm)
    tensors, device = _checked(_grads(parameters))
    if not isinstance(total_norm, torch.Tensor) or total_norm.numel() != 1 or total_norm.dtype != torch.float32:
        raise ValueError("total_norm is a float32 tensor of one value")
    if device is None:
        return
    if total_norm.device != device:
        raise ValueError(f"total_norm is on {total_norm.device}, the gradients on {device}")
    _refuse_overlap(tensors)
    with torch.no_grad():
        if device.type != "cuda":
            coef = (max_norm / (total_norm.double() + _EPS)).clamp(max=1.0).float()
            for t in tensors:
                t.mul_(coef.to(t.dtype) if t.dtype == torch.float64 else coef)
            return
        _scale_(tensors, _build_ops.load().grad_coef(total_norm.detach(), max_norm))


def clip_grad_norm_(parameters: Iterable[torch.Tensor] | torch.Tensor, max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` on the kernels: the gradients of ``parameters`` are scaled
    in place by ``min(1, max_norm / (norm + 1e-6))``; returns the norm before clipping as a 0-dim
    float32 tensor.  Nothing waits for the device unless ``error_if_nonfinite`` asks for the value.
    Gradients that share memory are refused (they would be scaled twice)."""
    max_norm, maximum = _max_norm(max_norm), _norm_type(norm_type)
    tensors, device = _checked(_grads(parameters))
    _refuse_overlap(tensors)
    with torch.no_grad():
        on_gpu = device is not None and device.type == "cuda"
        if on_gpu:
            result = _gpu_norm(tensors, maximum, max_norm)
            norm = result[0]
        else:
            norm = _cpu_norm(tensors, maximum)
        if error_if_nonfinite and not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the gradients' norm is {float(norm)}: not clipped")
        if on_gpu:
            _scale_(tensors, result)
        elif tensors:
            coef = (max_norm / (norm.double() + _EPS)).clamp(max=1.0).float()
            for t in tensors:
                t.mul_(coef.to(t.dtype) if t.dtype == torch.float64 else coef)
    return norm
