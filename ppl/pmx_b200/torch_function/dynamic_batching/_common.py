"""Argument helpers shared by the operators of this package."""
from __future__ import annotations

import contextlib

import torch

_NULL = contextlib.nullcontext()


def on_device(device: torch.device):
    """Makes `device` current for a launch; free when it is already."""
    return _NULL if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def same_device(name: str, device: torch.device, **tensors) -> None:
    for key, t in tensors.items():
        if t is not None and t.device != device:
            if not t.is_cuda:
                raise RuntimeError(f"{name}: `{key}` is on {t.device}; this implementation runs on CUDA "
                                   "devices only and has no CPU fallback")
            raise ValueError(f"{name}: `{key}` is on {t.device}, the query or cache on {device}")


def index(name: str, key: str, t: torch.Tensor, count: int) -> torch.Tensor:
    """An index array as the kernels read it: `count` dense int64 values."""
    if t.numel() != count:
        raise ValueError(f"{name}: `{key}` has {t.numel()} entries, expected {count}")
    if t.dtype is torch.int64:
        return t if t.is_contiguous() else t.contiguous()
    if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
        raise TypeError(f"{name}: `{key}` must hold integers, not {t.dtype}")
    return t.to(torch.int64).contiguous()


def heads(name: str, key: str, t: torch.Tensor, num_heads: int, head_dim: int, dtype: torch.dtype,
          aligned: bool = False) -> torch.Tensor:
    """[tokens, num_heads, head_dim] with unit inner stride; views into a fused projection stay views.
    `aligned`: a view whose rows the 16-byte tensor copies cannot address is copied."""
    if t.dim() != 3 or t.shape[1] != num_heads or t.shape[2] != head_dim:
        raise ValueError(f"{name}: `{key}` must be [tokens, {num_heads}, {head_dim}], not {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name}: `{key}` is {t.dtype}, the query {dtype}: one dtype for all")
    a, b, c = t.stride()
    if c != 1 and head_dim != 1:
        return t.contiguous()
    if aligned:
        e = t.element_size()
        if a * e % 16 or b * e % 16 or a <= 0 or b <= 0 or t.data_ptr() % 16:
            return t.contiguous()
    return t


def host_int(name: str, key: str, v) -> int:
    """A host value: an int or a one-element tensor, as the reference passes them."""
    n = int(v.reshape(-1)[0]) if isinstance(v, torch.Tensor) else int(v)
    if n <= 0:
        raise ValueError(f"{name}: `{key}` must be positive, not {n}")
    return n


def wants_grad(*tensors) -> bool:
    """The operators have no backward pass: where a gradient would be asked for they go through
    autograd, which then says so, instead of returning results that silently carry none."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
