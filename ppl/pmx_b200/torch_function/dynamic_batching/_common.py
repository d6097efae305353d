"""Argument helpers shared by the operators of this package."""
from __future__ import annotations

import contextlib
import ctypes as C
import sys
import warnings

import torch
from torch.autograd import forward_ad

from ..._cabi import lib


class _GeneralPath:
    """Stands in for the host calls: no call is a regular one."""
    rotary = prompt = tree = compact = staticmethod(lambda *args: None)


def _host_calls():
    """The short way through the host (csrc/host_calls.cpp), where it was built for this torch and this Python.  It saves a call
    a few microseconds; without it the operators check and convert in Python."""
    try:
        from ... import _host_calls as calls
        built, here = calls.built_for, f"torch {torch.__version__}, python {sys.version_info[0]}.{sys.version_info[1]}"
        if built != here:
            raise ImportError(f"built for {built}, this is {here}")
        calls.bind(*(C.cast(getattr(lib, name), C.c_void_p).value for name in (
            "pmx_rotary_embedding", "pmx_prompt_attention", "pmx_tree_cache_attention", "pmx_compact_cache",
            "pmx_attention_workspace_bytes")))
        return calls
    except (ImportError, AttributeError) as e:
        warnings.warn(f"ppl/pmx_b200/_host_calls.so is not used, which costs each call of the attention block a few microseconds "
                      f"({e}); `python -m ppl.pmx_b200.build` builds it", RuntimeWarning)
        return _GeneralPath


host = _host_calls()

_NULL = contextlib.nullcontext()
# the raw stream handle and the current device without the objects that torch.cuda wraps them in: these
# calls cost a few microseconds of host time in all, which is what a decode step's launches are bound by
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def on_device(index: int):
    """Makes device `index` current for a launch; free when it is already."""
    return _NULL if torch.cuda.current_device() == index else torch.cuda.device(index)


is_tracing = torch.jit.is_tracing


def exporting() -> bool:
    return torch.jit.is_tracing() and torch.onnx.is_in_onnx_export()


def same_device(name: str, device: int, **tensors) -> None:
    """Raises for a tensor that is not on CUDA device `device` (-1: the operator's first tensor is not on one)."""
    for key, t in tensors.items():
        if t is not None and (device < 0 or t.get_device() != device):
            if not t.is_cuda:
                raise RuntimeError(f"{name}: `{key}` is on {t.device}; this implementation runs on CUDA "
                                   "devices only and has no CPU fallback")
            raise ValueError(f"{name}: `{key}` is on {t.device}, other arguments on device {device}")


def index(name: str, key: str, t: torch.Tensor, count: int) -> torch.Tensor:
    """An index array as the kernels read it: `count` dense int64 values."""
    if t.dtype is torch.int64 and t.numel() == count and t.is_contiguous():
        return t
    if t.numel() != count:
        raise ValueError(f"{name}: `{key}` has {t.numel()} entries, expected {count}")
    if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
        raise TypeError(f"{name}: `{key}` must hold integers, not {t.dtype}")
    return t.to(torch.int64).contiguous()


def heads(name: str, key: str, t: torch.Tensor, num_heads: int, head_dim: int, dtype: torch.dtype,
          aligned: bool = False) -> torch.Tensor:
    """[tokens, num_heads, head_dim] with unit inner stride; views into a fused projection stay views.
    `aligned`: a view whose rows the 16-byte tensor copies cannot address is copied."""
    if t.dim() != 3 or t.shape[1:] != (num_heads, head_dim):
        raise ValueError(f"{name}: `{key}` must be [tokens, {num_heads}, {head_dim}], not {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name}: `{key}` is {t.dtype}, the query {dtype}: one dtype for all")
    a, b, c = t.stride()
    if c != 1 and head_dim != 1:
        return t.contiguous()
    if aligned:
        e = t.element_size()
        if (a | b) * e % 16 or a == 0 or b == 0 or t.data_ptr() % 16:
            return t.contiguous()
    return t


def host_int(name: str, key: str, v) -> int:
    """A host value: an int or a one-element tensor, as the reference passes them."""
    n = v if type(v) is int else int(v.reshape(-1)[0]) if isinstance(v, torch.Tensor) else int(v)
    if n <= 0:
        raise ValueError(f"{name}: `{key}` must be positive, not {n}")
    return n


def has_tangent(t) -> bool:
    """Whether a tensor carries a tangent of forward-mode differentiation."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def wants_grad(*tensors) -> bool:
    """The operators have no backward pass and no tangents: where a gradient or a tangent would be asked for they go
    through autograd, which then says so, instead of returning results that silently carry none."""
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and ((grad and t.requires_grad) or has_tangent(t)):
            return True
    return False


def cache_strides(cache: torch.Tensor, cache_layout: int, num_layer: int, layer_idx: int):
    """-> (layer_offset, row_stride, kv_stride, head_stride, total_rows) in elements for the
    four cache layouts of cache_mode 0 (Pipeline.py:80-89 of the Mixtral model):
      0: [rows, layers, 2, heads, d]   1: [layers, rows, 2, heads, d]
      2: [layers, 2, rows, heads, d]   3: [layers, 2, heads, rows, d]"""
    if cache.dim() != 5 or not cache.is_contiguous():
        raise ValueError("the cache must be a contiguous 5-d tensor")
    d = cache.shape[-1]
    if cache_layout == 0:
        rows, layers, two, heads, _ = cache.shape
        st = (layer_idx * 2 * heads * d, layers * 2 * heads * d, heads * d, d)
    elif cache_layout == 1:
        layers, rows, two, heads, _ = cache.shape
        st = (layer_idx * rows * 2 * heads * d, 2 * heads * d, heads * d, d)
    elif cache_layout == 2:
        layers, two, rows, heads, _ = cache.shape
        st = (layer_idx * 2 * rows * heads * d, heads * d, rows * heads * d, d)
    elif cache_layout == 3:
        layers, two, heads, rows, _ = cache.shape
        st = (layer_idx * 2 * heads * rows * d, d, heads * rows * d, rows * d)
    else:
        raise ValueError(f"unsupported cache_layout: {cache_layout}")
    if two != 2 or layers != num_layer or not 0 <= layer_idx < layers:
        raise ValueError(f"cache shape {tuple(cache.shape)} does not fit layout {cache_layout} with {num_layer} layers")
    return st + (rows,)
