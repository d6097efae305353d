"""Moving the accepted rows of a drafted tree together inside the key/value cache."""
from __future__ import annotations

import torch

from ..._cabi import lib, check, COMPACT_CACHE_ARGS, DTYPE_CODE
from ._common import cache_strides, host, host_int, index, on_device, raw_stream, same_device, wants_grad


def compact_cache(cache: torch.Tensor, cachestarts: torch.Tensor, start_pos: torch.Tensor, accept_starts: torch.Tensor,
                  accept_index: torch.Tensor, max_accept, num_layer: int = 1, cache_layout: int = 0) -> torch.Tensor:
    """Keeps, of the rows that tree_cache_attention() stored, those of the accepted tokens -> `cache`, changed in place.

    Sequence b accepts the drafted tokens accept_index[accept_starts[b]..accept_starts[b+1]] (their places in the draft,
    at most max_accept <= 64: entries behind those are left out; normally a path from the root): row base + i takes the row
    base + accept_index[..i], with base = cachestarts[b] + start_pos[b], in all layers, keys and values.  All rows of a
    sequence are read before one is written, so the indices may come in any order and repeat; a negative index leaves its
    row alone, and so does one that leads outside the cache or in front of cachestarts[b].  The caller's next start_pos is
    start_pos + the number accepted.  Rows of different sequences must not overlap."""
    status = host.compact(cache, cachestarts, start_pos, accept_starts, accept_index, max_accept, num_layer, cache_layout)
    if status is not None:           # None: not the regular case
        check(status)
        return cache
    name = "compact_cache"
    dev = cache.get_device()
    for t in (cache, cachestarts, start_pos, accept_starts, accept_index):
        if dev < 0 or t.get_device() != dev:
            same_device(name, dev, cache=cache, cachestarts=cachestarts, start_pos=start_pos,
                        accept_starts=accept_starts, accept_index=accept_index)
    code = DTYPE_CODE.get(cache.dtype)
    if code is None:
        raise TypeError(f"{name}: dtype {cache.dtype} is not supported (float16, bfloat16, float32)")
    if wants_grad(cache):
        raise RuntimeError(f"{name}: changes the cache in place and has no backward pass and no forward-mode derivative")
    _, row_stride, kv_stride, head_stride, rows = cache_strides(cache, cache_layout, num_layer, 0)
    layer_stride = cache.stride(1 if cache_layout == 0 else 0)
    kv_heads = cache.shape[2 if cache_layout == 3 else 3]
    B = accept_starts.numel() - 1
    if B < 1:
        raise ValueError(f"{name}: `accept_starts` must hold the start of every sequence and the end")
    accept_starts = index(name, "accept_starts", accept_starts, B + 1)
    cachestarts, start_pos = index(name, "cachestarts", cachestarts, B), index(name, "start_pos", start_pos, B)
    accept_index = index(name, "accept_index", accept_index, accept_index.numel())
    max_accept = host_int(name, "max_accept", max_accept)
    if max_accept > 64:
        raise ValueError(f"{name}: at most 64 accepted rows a sequence")
    if accept_index.numel() == 0 or cache.numel() == 0:
        return cache
    with on_device(dev):
        check(lib.pmx_compact_cache(COMPACT_CACHE_ARGS.pack(
            cache.data_ptr(), cachestarts.data_ptr(), start_pos.data_ptr(), accept_starts.data_ptr(),
            accept_index.data_ptr(), B, accept_index.numel(), max_accept, num_layer, kv_heads, cache.shape[-1], rows,
            row_stride, layer_stride, kv_stride, head_stride, code), raw_stream(dev)))
    return cache
