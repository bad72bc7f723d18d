"""Host helpers of the selective-mixer operators (``selective``, ``norm``, ``q4``):
argument checks, row strides, streams.

Each operator is a torch custom op with a fake impl and, where it trains, an
autograd formula, so ``torch.compile`` traces it. Eager calls run the same body
without the dispatcher: generation calls one of these operators every few
microseconds, where the dispatcher's cost exceeds the kernel's.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ._ops import _CODES


def code_of(name: str, t: Tensor) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {t.dtype} of {name}; expected float32, bfloat16 or float16")
    return code


def need_cuda(op: str, first: Tensor, *others: Tensor | None) -> None:
    if not first.is_cuda:
        raise NotImplementedError(f"spikegpt_b200.{op} runs on CUDA tensors only")
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"all tensors of {op} must be on {device}; got one on {t.device}")


def need_shape(name: str, t: Tensor | None, shape: tuple[int, ...]) -> None:
    if t is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}; got {list(t.shape)}")


def need_dtype(name: str, t: Tensor | None, dtype: torch.dtype, of: str) -> None:
    if t is not None and t.dtype != dtype:
        raise ValueError(f"{name} must have the dtype of {of} ({dtype}); got {t.dtype}")


def parameter(t: Tensor | None) -> Tensor | None:
    """A parameter as the kernels read it: float32 and contiguous."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def rows(t: Tensor | None) -> Tensor | None:
    """``t`` with unit stride of its last index (a copy only where it lacks that)."""
    if t is None or t.stride(-1) == 1 or t.shape[-1] == 1:
        return t
    return t.contiguous()


def lengths_of(lengths: Tensor | None, b: int) -> Tensor | None:
    if lengths is None:
        return None
    if lengths.shape != (b,) or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"lengths must be int32 or int64 of shape [{b}]; got {lengths.dtype} {list(lengths.shape)}")
    return lengths.to(torch.int32).contiguous()


def ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream(t: Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def on_device(t: Tensor):
    """A device guard where ``t`` is not on the current device, else None."""
    return None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def wants_grad(*tensors: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def no_grad_only(op: str, *tensors: Tensor | None) -> None:
    if wants_grad(*tensors):
        raise NotImplementedError(f"spikegpt_b200.{op} has no gradient; call it under torch.no_grad()")


def workspace(nbytes: int, like: Tensor) -> Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None
