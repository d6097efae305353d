"""Rotary positions on packed heads, alone or behind an RMS norm of every query and key head.

The reference's decoder rotates queries and keys in a Python loop over the sequences
(torch_function/dynamic_batching/RotaryPositionEmbedding.py:58-77, called between the fused
projection and multi_head_cache_attention); here it is one launch for all heads of all tokens.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import Optional, Tuple

import torch

from ..._cabi import lib, check, DTYPE_CODE, ROTARY_ARGS
from ._common import exporting, heads, host, index, is_tracing, on_device, raw_stream, same_device, wants_grad


@functools.lru_cache(maxsize=64)
def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling_type: str = "", scaling_factor: float = 1.0,
                       original_max_position: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """-> (ctypes array of rotary_dim/2 doubles: angle per position of each pair, factor on cosine and sine).

    scaling_type "": f_i = theta^(-2i/rotary_dim).  "linear": f_i / s.  "ntk": theta * s^(r/(r-2)) in the place of theta,
    which stretches the slowest pair by s and leaves the fastest alone.  "yarn": pairs that turn more than beta_fast times
    over original_max_position stay, those that turn less than beta_slow times are divided by s, a ramp between
    that is linear in the number of turns, as the method is published (a ramp that is linear in the pair's index, between the two
    pairs that turn so often, gives other frequencies in the middle); cosine and sine take the factor 0.1 ln s + 1."""
    r, s = rotary_dim, float(scaling_factor)
    if r <= 0 or r % 2 or r > 256:
        raise ValueError(f"rotary_dim must be even, positive and at most 256, not {r}")
    if not theta > 0 or not math.isfinite(theta):
        raise ValueError(f"theta must be positive and finite, not {theta}")
    if scaling_type not in ("", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling_type {scaling_type!r}: '', 'linear', 'ntk' and 'yarn' are covered")
    if scaling_type and not (s >= 1.0 and math.isfinite(s)):
        raise ValueError(f"scaling_factor must be at least 1, not {scaling_factor}")
    factor = 1.0
    if scaling_type == "ntk":
        if r <= 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        theta = theta * s ** (r / (r - 2.0))
    f = [theta ** (-2.0 * i / r) for i in range(r // 2)]
    if scaling_type == "linear":
        f = [x / s for x in f]
    elif scaling_type == "yarn":
        if original_max_position <= 0 or not beta_fast > beta_slow:
            raise ValueError("yarn scaling needs original_max_position and beta_fast > beta_slow")
        for i, x in enumerate(f):
            turns = original_max_position * x / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - beta_slow) / (beta_fast - beta_slow)))
            f[i] = x * (keep + (1.0 - keep) / s)
        factor = 0.1 * math.log(s) + 1.0
    return (C.c_double * (r // 2))(*f), factor


@functools.lru_cache(maxsize=64)
def _table(*args):
    table, factor = rotary_frequencies(*args)
    return table, C.addressof(table), factor


def _launch(name, query, key, q_weight, k_weight, eps, seqstarts, start_pos, position_ids, rotary_dim, theta,
            interleaved, scaling_type, scaling_factor, original_max_position):
    dev = query.get_device()
    for t in (query, key, q_weight, k_weight, seqstarts, start_pos, position_ids):
        if t is not None and (dev < 0 or t.get_device() != dev):
            same_device(name, dev, query=query, key=key, query_norm_weight=q_weight, key_norm_weight=k_weight,
                        seqstarts=seqstarts, start_pos=start_pos, position_ids=position_ids)
    if query.dim() != 3:
        raise ValueError(f"{name}: `query` must be [tokens, num_heads, head_dim], not {tuple(query.shape)}")
    T, Hq, D = query.shape
    dtype = query.dtype
    code = DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"{name}: dtype {dtype} is not supported (float16, bfloat16, float32)")
    q = heads(name, "query", query, Hq, D, dtype)
    s0, s1, _ = q.stride()
    k, Hkv, k0, k1 = None, 0, 0, 0
    if key is not None:
        if key.dim() != 3 or key.shape[0] != T:
            raise ValueError(f"{name}: `key` must be [{T}, num_kv_heads, {D}], not {tuple(key.shape)}")
        Hkv = key.shape[1]
        k = heads(name, "key", key, Hkv, D, dtype)
        k0, k1, _ = k.stride()
    qw = kw = 0
    if q_weight is not None:
        for label, w in (("query_norm_weight", q_weight), ("key_norm_weight", k_weight)):
            if w.shape != (D,) or w.dtype is not dtype:
                raise ValueError(f"{name}: `{label}` must be [{D}] in the query's dtype")
        q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    B = ss = sp = ids = 0
    if position_ids is not None:
        position_ids = index(name, "position_ids", position_ids, T)
        ids = position_ids.data_ptr()
    else:
        if seqstarts is None or start_pos is None:
            raise ValueError(f"{name}: positions come from `position_ids` or from `seqstarts` and `start_pos`")
        B = seqstarts.numel() - 1
        seqstarts, start_pos = index(name, "seqstarts", seqstarts, max(B, 1) + 1), index(name, "start_pos", start_pos, B)
        ss, sp = seqstarts.data_ptr(), start_pos.data_ptr()
    r = rotary_dim or D
    if r > D:
        raise ValueError(f"{name}: rotary_dim {r} is above head_dim {D}")
    _, table, factor = _table(r, theta, scaling_type, scaling_factor, original_max_position)
    qo = q.new_empty((T, Hq, D))
    ko = None if k is None else k.new_empty((T, Hkv, D))
    if T == 0 or Hq == 0:
        if ko is not None and ko.numel():
            raise ValueError(f"{name}: there are no query heads")
        return qo, ko
    if Hkv == 0:
        kw = 0
    with on_device(dev):
        check(lib.pmx_rotary_embedding(ROTARY_ARGS.pack(
            q.data_ptr(), k.data_ptr() if Hkv else 0, qw, kw, qo.data_ptr(), ko.data_ptr() if Hkv else 0, ss, sp, ids, table,
            T, B, Hq, Hkv, D, s0, s1, k0, k1, r, 1 if interleaved else 0, code, eps, factor), raw_stream(dev)))
    return qo, ko


class RotaryPositionEmbedding(torch.autograd.Function):
    """opmx.dynamic_batching::RotaryPositionEmbedding; no backward."""

    @staticmethod
    def symbolic(g, query, key, seqstarts, start_pos, position_ids, rotary_dim: int = 0, theta: float = 10000.0,
                 interleaved: bool = False, scaling_type: str = "", scaling_factor: float = 1.0,
                 original_max_position: int = 0):
        args = [query] + [t for t in (key, seqstarts, start_pos, position_ids) if t is not None]
        out = g.op("opmx.dynamic_batching::RotaryPositionEmbedding", *args, rotary_dim_i=rotary_dim, theta_f=theta,
                   interleaved_i=interleaved, scaling_type_s=scaling_type, scaling_factor_f=scaling_factor,
                   original_max_position_i=original_max_position, bypass_key_i=key is None,
                   position_ids_i=position_ids is not None, outputs=1 if key is None else 2)
        return out.setTypeAs(query) if key is None else (out[0].setTypeAs(query), out[1].setTypeAs(key))

    @staticmethod
    def forward(ctx, query, key, seqstarts, start_pos, position_ids, rotary_dim: int = 0, theta: float = 10000.0,
                interleaved: bool = False, scaling_type: str = "", scaling_factor: float = 1.0,
                original_max_position: int = 0):
        if torch.onnx.is_in_onnx_export():
            return query if key is None else (query, key)
        q, k = _launch("rotary_position_embedding", query, key, None, None, 0.0, seqstarts, start_pos, position_ids,
                       rotary_dim, theta, interleaved, scaling_type, scaling_factor, original_max_position)
        return q if key is None else (q, k)


class QkNormRotaryEmbedding(torch.autograd.Function):
    """opmx.dynamic_batching::QkNormRotaryEmbedding; no backward."""

    @staticmethod
    def symbolic(g, query, key, query_norm_weight, key_norm_weight, eps, seqstarts, start_pos, position_ids,
                 rotary_dim: int = 0, theta: float = 10000.0, interleaved: bool = False, scaling_type: str = "",
                 scaling_factor: float = 1.0, original_max_position: int = 0):
        args = [query, key, query_norm_weight, key_norm_weight]
        args += [t for t in (seqstarts, start_pos, position_ids) if t is not None]
        q, k = g.op("opmx.dynamic_batching::QkNormRotaryEmbedding", *args, eps_f=eps, rotary_dim_i=rotary_dim,
                    theta_f=theta, interleaved_i=interleaved, scaling_type_s=scaling_type,
                    scaling_factor_f=scaling_factor, original_max_position_i=original_max_position,
                    position_ids_i=position_ids is not None, outputs=2)
        return q.setTypeAs(query), k.setTypeAs(key)

    @staticmethod
    def forward(ctx, query, key, query_norm_weight, key_norm_weight, eps, seqstarts, start_pos, position_ids,
                rotary_dim: int = 0, theta: float = 10000.0, interleaved: bool = False, scaling_type: str = "",
                scaling_factor: float = 1.0, original_max_position: int = 0):
        if torch.onnx.is_in_onnx_export():
            return query, key
        return _launch("qk_norm_rotary_embedding", query, key, query_norm_weight, key_norm_weight, eps, seqstarts,
                       start_pos, position_ids, rotary_dim, theta, interleaved, scaling_type, scaling_factor,
                       original_max_position)


def rotary_position_embedding(query: torch.Tensor, key: Optional[torch.Tensor], seqstarts: Optional[torch.Tensor],
                              start_pos: Optional[torch.Tensor], position_ids: Optional[torch.Tensor] = None,
                              rotary_dim: int = 0, theta: float = 10000.0, interleaved: bool = False,
                              scaling_type: str = "", scaling_factor: float = 1.0, original_max_position: int = 0
                              ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """-> (query, key) with the first `rotary_dim` (0: all) values of every head rotated by their token's position.

    query [T, num_heads, head_dim], key [T, num_kv_heads, head_dim] or None; views with unit inner stride (of a fused
    projection's output) are read in place, the results are dense.  Token t of sequence b is at position
    start_pos[b] + t - seqstarts[b], or at position_ids[t] where those are given (drafted trees: the depth).
    Tokens of no sequence are copied.  Pairs are (i, i + rotary_dim/2), or (2i, 2i+1) when `interleaved`;
    `scaling_type` as in rotary_frequencies().  float16, bfloat16, float32; one rounding of the result."""
    if not is_tracing():
        r = rotary_dim or query.shape[-1]
        _, table, factor = _table(r, theta, scaling_type, scaling_factor, original_max_position)
        out = host.rotary(query, key, None, None, 0.0, seqstarts, start_pos, position_ids, r, 1 if interleaved else 0, table,
                          factor)
        if out is not None:          # None: not the regular case
            return out if type(out) is tuple else check(out)
    args = (query, key, seqstarts, start_pos, position_ids, rotary_dim, theta, interleaved, scaling_type,
            scaling_factor, original_max_position)
    if exporting() or wants_grad(query, key):
        out = RotaryPositionEmbedding.apply(*args)
        return (out, None) if key is None else out
    return _launch("rotary_position_embedding", query, key, None, None, 0.0, *args[2:])


def qk_norm_rotary_embedding(query: torch.Tensor, key: torch.Tensor, query_norm_weight: torch.Tensor,
                             key_norm_weight: torch.Tensor, eps: float, seqstarts: Optional[torch.Tensor],
                             start_pos: Optional[torch.Tensor], position_ids: Optional[torch.Tensor] = None,
                             rotary_dim: int = 0, theta: float = 10000.0, interleaved: bool = False,
                             scaling_type: str = "", scaling_factor: float = 1.0, original_max_position: int = 0
                             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """rotary_position_embedding() of RMS-normed heads, in the same pass: every head becomes
    x * weight / sqrt(mean(x^2) + eps) over its head_dim values (weights [head_dim], one for all query heads and
    one for all key heads), then the rotation; one rounding at the end."""
    if query_norm_weight is None or key_norm_weight is None or key is None:
        raise ValueError("qk_norm_rotary_embedding: key and both norm weights are needed")
    if not is_tracing():
        r = rotary_dim or query.shape[-1]
        _, table, factor = _table(r, theta, scaling_type, scaling_factor, original_max_position)
        out = host.rotary(query, key, query_norm_weight, key_norm_weight, float(eps), seqstarts, start_pos, position_ids, r,
                          1 if interleaved else 0, table, factor)
        if out is not None:
            return out if type(out) is tuple else check(out)
    args = (query, key, query_norm_weight, key_norm_weight, float(eps), seqstarts, start_pos, position_ids, rotary_dim,
            theta, interleaved, scaling_type, scaling_factor, original_max_position)
    if exporting() or wants_grad(query, key, query_norm_weight, key_norm_weight):
        return QkNormRotaryEmbedding.apply(*args)
    return _launch("qk_norm_rotary_embedding", *args)
