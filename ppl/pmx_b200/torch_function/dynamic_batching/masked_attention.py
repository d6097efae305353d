"""Attention of several new tokens per sequence: packed prompts, and drafted trees over the cache.

`multi_head_cache_attention` covers decode steps; these cover what comes before and beside them.
The reference runs prompts as one small attention per sequence in a Python loop
(torch_function/dynamic_batching/MultiHeadAttention.py:76-109); here a batch is one launch, plus a
merge where a long key axis is split because there are few rows.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from ..._cabi import lib, check, workspace, DTYPE_CODE, PROMPT_ATTENTION_ARGS, TREE_ATTENTION_ARGS
from ._common import (cache_strides, exporting, heads, host, host_int, index, is_tracing, on_device, raw_stream,
                      same_device, wants_grad)


def _code(name: str, t: torch.Tensor) -> int:
    code = DTYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: dtype {t.dtype} is not supported (float16, bfloat16, float32)")
    return code


def _numbers(name: str, num_heads: int, kv_heads: int, head_dim: int, scale, logit_cap) -> float:
    if num_heads <= 0 or kv_heads <= 0 or num_heads % kv_heads:
        raise ValueError(f"{name}: num_heads ({num_heads}) must be a multiple of num_kv_heads ({kv_heads})")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"{name}: scale must be positive and finite, not {scale}")
    if not (logit_cap >= 0.0 and math.isfinite(logit_cap)):
        raise ValueError(f"{name}: logit_cap must be finite and not negative (0: no cap), not {logit_cap}")
    return scale


def attention_check(device=None) -> None:
    """Synchronises the current stream of the device and raises PmxError (status -6) if a bounded wait inside
    prompt_attention or tree_cache_attention ran out since the last check (their results are then undefined)."""
    dev = torch.device("cuda" if device is None else device)
    dev = torch.cuda.current_device() if dev.index is None else dev.index
    out = (C.c_int32 * 4)()
    with on_device(dev):
        check(lib.pmx_attention_check(C.byref(out), raw_stream(dev)))


def _prompt(query, key, value, seqstarts, kvstarts, max_seqlen, max_kvlen, num_heads, head_dim, is_causal, num_kv_heads,
            scale, logit_cap, alibi_slopes, prefix_lens):
    name = "prompt_attention"
    dev = query.get_device()
    for t in (query, key, value, seqstarts, kvstarts, alibi_slopes, prefix_lens):
        if t is not None and (dev < 0 or t.get_device() != dev):
            same_device(name, dev, query=query, key=key, value=value, seqstarts=seqstarts, kvstarts=kvstarts,
                        alibi_slopes=alibi_slopes, prefix_lens=prefix_lens)
    code = _code(name, query)
    kv_heads = num_kv_heads or num_heads
    scale = _numbers(name, num_heads, kv_heads, head_dim, scale, logit_cap)
    q = heads(name, "query", query, num_heads, head_dim, query.dtype, True)
    k = heads(name, "key", key, kv_heads, head_dim, query.dtype, True)
    v = heads(name, "value", value, kv_heads, head_dim, query.dtype, True)
    if k.shape[0] != v.shape[0]:
        raise ValueError(f"{name}: {k.shape[0]} keys and {v.shape[0]} values")
    B = seqstarts.numel() - 1
    if B < 1:
        raise ValueError(f"{name}: `seqstarts` must hold the start of every sequence and the end")
    seqstarts, kvstarts = index(name, "seqstarts", seqstarts, B + 1), index(name, "kvstarts", kvstarts, B + 1)
    if prefix_lens is not None:
        prefix_lens = index(name, "prefix_lens", prefix_lens, B)
    if alibi_slopes is not None:
        if tuple(alibi_slopes.shape) != (num_heads,):
            raise ValueError(f"{name}: `alibi_slopes` must be [{num_heads}]")
        alibi_slopes = alibi_slopes.to(torch.float32).contiguous()
    max_seqlen, max_kvlen = host_int(name, "max_seqlen", max_seqlen), host_int(name, "max_kvlen", max_kvlen)
    Tq, Tk = q.shape[0], k.shape[0]
    out = q.new_empty((Tq, num_heads, head_dim))
    if Tq == 0 or Tk == 0:
        return out.zero_()
    q0, q1, _ = q.stride()
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    with on_device(dev):
        nbytes = lib.pmx_attention_workspace_bytes(Tq, B, num_heads, kv_heads, head_dim, max_seqlen, max_kvlen, code)
        ws = workspace(nbytes, q.device) if nbytes else None
        check(lib.pmx_prompt_attention(PROMPT_ATTENTION_ARGS.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), seqstarts.data_ptr(), kvstarts.data_ptr(),
            0 if prefix_lens is None else prefix_lens.data_ptr(), 0 if alibi_slopes is None else alibi_slopes.data_ptr(),
            out.data_ptr(), ws.data_ptr() if nbytes else 0, Tq, Tk, B, num_heads, kv_heads, head_dim, q0, q1, k0, k1, v0, v1,
            max_seqlen, max_kvlen, 1 if is_causal else 0, code, nbytes, scale, logit_cap), raw_stream(dev)))
    return out


def _tree(query, current_key, current_value, seqstarts, cachestarts, start_pos, tree_mask, max_seqlen, max_kvlen, cache,
          num_heads, head_dim, num_kv_heads, num_layer, layer_idx, cache_layout, scale, logit_cap):
    name = "tree_cache_attention"
    dev = query.get_device()
    for t in (query, current_key, current_value, cache, seqstarts, cachestarts, start_pos, tree_mask):
        if dev < 0 or t.get_device() != dev:
            same_device(name, dev, query=query, current_key=current_key, current_value=current_value, cache=cache,
                        seqstarts=seqstarts, cachestarts=cachestarts, start_pos=start_pos, tree_mask=tree_mask)
    code = _code(name, query)
    kv_heads = num_kv_heads or num_heads
    scale = _numbers(name, num_heads, kv_heads, head_dim, scale, logit_cap)
    q = heads(name, "query", query, num_heads, head_dim, query.dtype, True)
    k = heads(name, "current_key", current_key, kv_heads, head_dim, query.dtype, True)
    v = heads(name, "current_value", current_value, kv_heads, head_dim, query.dtype, True)
    if cache.dtype is not query.dtype:
        raise TypeError(f"{name}: the cache is {cache.dtype}, the query {query.dtype}: one dtype for all")
    Tq = q.shape[0]
    if k.shape[0] != Tq or v.shape[0] != Tq:
        raise ValueError(f"{name}: query, current_key and current_value must have one row per drafted token")
    layer_off, row_stride, kv_stride, head_stride, rows = cache_strides(cache, cache_layout, num_layer, layer_idx)
    if cache.shape[-1] != head_dim or cache.shape[2 if cache_layout == 3 else 3] != kv_heads:
        raise ValueError(f"{name}: cache shape {tuple(cache.shape)} does not hold {kv_heads} heads of {head_dim}")
    B = seqstarts.numel() - 1
    if B < 1:
        raise ValueError(f"{name}: `seqstarts` must hold the start of every sequence and the end")
    seqstarts = index(name, "seqstarts", seqstarts, B + 1)
    cachestarts, start_pos = index(name, "cachestarts", cachestarts, B), index(name, "start_pos", start_pos, B)
    tree_mask = index(name, "tree_mask", tree_mask, Tq)
    max_seqlen, max_kvlen = host_int(name, "max_seqlen", max_seqlen), host_int(name, "max_kvlen", max_kvlen)
    out = q.new_empty((Tq, num_heads, head_dim))
    if Tq == 0:
        return out
    if rows == 0:
        raise ValueError(f"{name}: the cache has no rows")
    q0, q1, _ = q.stride()
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    with on_device(dev):
        nbytes = lib.pmx_attention_workspace_bytes(Tq, B, num_heads, kv_heads, head_dim, max_seqlen, max_kvlen, code)
        ws = workspace(nbytes, q.device) if nbytes else None
        check(lib.pmx_tree_cache_attention(TREE_ATTENTION_ARGS.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), cache.data_ptr(), seqstarts.data_ptr(), cachestarts.data_ptr(),
            start_pos.data_ptr(), tree_mask.data_ptr(), out.data_ptr(), ws.data_ptr() if nbytes else 0, Tq, B, num_heads,
            kv_heads, head_dim, q0, q1, k0, k1, v0, v1, rows, layer_off, row_stride, kv_stride, head_stride, max_seqlen,
            max_kvlen, code, nbytes, scale, logit_cap), raw_stream(dev)))
    return out


def _length(g, n):
    """A length of an exported call: an input of the node, a constant where the call has a number."""
    return n if isinstance(n, torch._C.Value) else g.op("Constant", value_t=torch.tensor([int(n)]))


class PromptAttention(torch.autograd.Function):
    """opmx.dynamic_batching::PromptAttention; no backward."""

    @staticmethod
    def symbolic(g, query, key, value, seqstarts, kvstarts, max_seqlen, max_kvlen, num_heads: int, head_dim: int,
                 is_causal: bool = True, num_kv_heads: int = 0, scale=None, logit_cap: float = 0.0, alibi_slopes=None,
                 prefix_lens=None):
        args = [query, key, value, seqstarts, kvstarts, _length(g, max_seqlen), _length(g, max_kvlen)]
        args += [t for t in (alibi_slopes, prefix_lens) if t is not None]
        return g.op("opmx.dynamic_batching::PromptAttention", *args, num_heads_i=num_heads, head_dim_i=head_dim,
                    is_causal_i=is_causal, num_kv_heads_i=num_kv_heads, scale_f=scale or 1.0 / math.sqrt(head_dim),
                    logit_cap_f=logit_cap, alibi_slopes_i=alibi_slopes is not None,
                    prefix_lens_i=prefix_lens is not None).setTypeAs(query)

    @staticmethod
    def forward(ctx, query, *args):
        if torch.onnx.is_in_onnx_export():
            return query
        return _prompt(query, *args)


class TreeCacheAttention(torch.autograd.Function):
    """opmx.dynamic_batching::TreeCacheAttention; no backward."""

    @staticmethod
    def symbolic(g, query, current_key, current_value, seqstarts, cachestarts, start_pos, tree_mask, max_seqlen,
                 max_kvlen, cache, num_heads: int, head_dim: int, num_kv_heads: int = 0, num_layer: int = 1,
                 layer_idx: int = 0, cache_layout: int = 0, scale=None, logit_cap: float = 0.0):
        return g.op("opmx.dynamic_batching::TreeCacheAttention", query, current_key, current_value, seqstarts,
                    cachestarts, start_pos, tree_mask, _length(g, max_seqlen), _length(g, max_kvlen), cache,
                    num_heads_i=num_heads, head_dim_i=head_dim,
                    num_kv_heads_i=num_kv_heads, num_layer_i=num_layer, layer_idx_i=layer_idx,
                    cache_layout_i=cache_layout, scale_f=scale or 1.0 / math.sqrt(head_dim),
                    logit_cap_f=logit_cap).setTypeAs(query)

    @staticmethod
    def forward(ctx, query, *args):
        if torch.onnx.is_in_onnx_export():
            return query
        return _tree(query, *args)


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, seqstarts: torch.Tensor,
                     kvstarts: torch.Tensor, max_seqlen, max_kvlen, num_heads: int, head_dim: int,
                     is_causal: bool = True, num_kv_heads: int = 0, scale: Optional[float] = None,
                     logit_cap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None,
                     prefix_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed ragged prompts -> [tokens, num_heads, head_dim].

    Sequence b holds the queries seqstarts[b]..seqstarts[b+1] and the keys kvstarts[b]..kvstarts[b+1]; its queries are the
    last of its positions (a chunk of a prompt behind what is there already).  No token sees another sequence: starts at
    document borders are a document mask.  is_causal: a token sees the positions up to its own, and with
    `prefix_lens` [B] all of the first prefix_lens[b] as well; otherwise its whole sequence, to which a prefix adds
    nothing.  Scores are scale * q.k (None: 1/sqrt(head_dim)), capped to logit_cap * tanh(score / logit_cap) where that is
    positive, less alibi_slopes[head] * |distance| where those are given.  A token that sees no key, and a row of no sequence, is zero;
    what a token may not see does not reach its result, whatever it holds.
    max_seqlen, max_kvlen (int or one-element tensor): at least the longest sequence's queries and keys.  The rows
    of a sequence behind its first max_seqlen are zero.
    query, key and value may be views with unit inner stride.  float16, bfloat16, float32, head_dim up to 256."""
    args = (query, key, value, seqstarts, kvstarts, max_seqlen, max_kvlen, num_heads, head_dim, is_causal, num_kv_heads,
            scale, float(logit_cap), alibi_slopes, prefix_lens)
    if not is_tracing():
        out = host.prompt(*args)
        if out is not None:          # None: not the regular case
            return out if type(out) is not int else check(out)
    if exporting() or wants_grad(query, key, value, alibi_slopes):
        return PromptAttention.apply(*args)
    return _prompt(*args)


def tree_cache_attention(query: torch.Tensor, current_key: torch.Tensor, current_value: torch.Tensor,
                         seqstarts: torch.Tensor, cachestarts: torch.Tensor, start_pos: torch.Tensor,
                         tree_mask: torch.Tensor, max_seqlen, max_kvlen, cache: torch.Tensor, num_heads: int,
                         head_dim: int, num_kv_heads: int = 0, num_layer: int = 1, layer_idx: int = 0,
                         cache_layout: int = 0, scale: Optional[float] = None, logit_cap: float = 0.0) -> torch.Tensor:
    """Attention of drafted tokens (a tree or a chain per sequence) over the cache -> [tokens, num_heads, head_dim].

    Sequence b brings the tokens seqstarts[b]..seqstarts[b+1], at most 64.  Token i of it sees the start_pos[b] cached
    rows from cachestarts[b] on, and drafted token j of its sequence where bit j of tree_mask[token] is set (int64
    [tokens]; a token that is to see itself needs its own bit).  The new keys and values are stored into `cache`, in place,
    at rows cachestarts[b] + start_pos[b] + i (rows outside the cache are neither seen nor stored, nor are rows stored in
    front of cachestarts[b], where a negative start_pos leads); compact_cache() then moves the accepted
    ones together.  max_seqlen: at least the most drafted tokens of a sequence, max_kvlen: at least the most cached plus
    drafted rows.  Cache layouts 0..3 as multi_head_cache_attention(); scores, types and empty rows as
    prompt_attention()."""
    args = (query, current_key, current_value, seqstarts, cachestarts, start_pos, tree_mask, max_seqlen, max_kvlen, cache,
            num_heads, head_dim, num_kv_heads, num_layer, layer_idx, cache_layout, scale, float(logit_cap))
    if not is_tracing():
        out = host.tree(*args)
        if out is not None:          # None: not the regular case
            return out if type(out) is not int else check(out)
    if exporting() or wants_grad(query, current_key, current_value, cache):
        return TreeCacheAttention.apply(*args)
    return _tree(*args)
