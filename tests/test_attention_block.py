"""The attention block's operators without a GPU: frequencies, refusals of the operators and of the C ABI."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import attention_block as ab


@pytest.fixture(scope="module")
def DB():
    import ppl.pmx_b200.torch_function as F
    return F.dynamic_batching


@pytest.mark.parametrize("r", [2, 6, 64, 128, 256])
@pytest.mark.parametrize("kw", [{}, dict(scaling_type="linear", scaling_factor=4.0), dict(scaling_type="ntk", scaling_factor=4.0),
                                dict(scaling_type="yarn", scaling_factor=16.0, original_max_position=4096)])
def test_frequencies_match_their_definition(DB, r, kw):
    if r == 2 and kw.get("scaling_type") == "ntk":
        with pytest.raises(ValueError):
            DB.rotary_frequencies(r, 1e4, **kw)
        return
    table, factor = DB.rotary_frequencies(r, 1e4, **kw)
    want, wf = ab.frequencies(r, 1e4, kw.get("scaling_type", ""), kw.get("scaling_factor", 1.0),
                              kw.get("original_max_position", 0))
    np.testing.assert_allclose(np.array(table[:]), want, rtol=1e-13)
    assert abs(factor - wf) < 1e-15


def test_yarn_keeps_the_fast_pairs_and_stretches_the_slow_ones(DB):
    plain, _ = DB.rotary_frequencies(128, 1e4)
    yarn, factor = DB.rotary_frequencies(128, 1e4, "yarn", 8.0, 4096)
    assert yarn[0] == plain[0] and math.isclose(yarn[63], plain[63] / 8, rel_tol=1e-14)
    assert math.isclose(factor, 0.1 * math.log(8.0) + 1)
    assert all(p / 8 * (1 - 1e-12) <= y <= p for p, y in zip(plain, yarn))


@pytest.mark.parametrize("args", [(0,), (3,), (258,), (64, 0.0), (64, float("inf")), (64, 1e4, "unknown"),
                                  (64, 1e4, "linear", 0.5), (64, 1e4, "linear", float("nan")), (64, 1e4, "yarn", 2.0, 0),
                                  (64, 1e4, "yarn", 2.0, 4096, 1.0, 1.0)])
def test_frequencies_refuse(DB, args):
    with pytest.raises(ValueError):
        DB.rotary_frequencies(*args)


def test_operators_refuse_cpu_tensors(DB):
    q, i = torch.zeros(4, 2, 64), torch.arange(3)
    cache = torch.zeros(8, 1, 2, 2, 64)
    for call in (lambda: DB.rotary_position_embedding(q, q, i, i[:2]),
                 lambda: DB.qk_norm_rotary_embedding(q, q, q[0, 0], q[0, 0], 1e-6, i, i[:2]),
                 lambda: DB.prompt_attention(q, q, q, i, i, 2, 2, 2, 64),
                 lambda: DB.tree_cache_attention(q, q, q, i, i[:2], i[:2], torch.zeros(4, dtype=torch.int64), 2, 2, cache, 2, 64),
                 lambda: DB.compact_cache(cache, i[:2], i[:2], i, i[:2], 1)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_c_abi_refuses_before_it_launches():
    from ppl.pmx_b200 import _cabi
    from ppl.pmx_b200._cabi import lib
    f = (C.c_double * 128)(*([1.0] * 128))

    def caller(fn, packer, **defaults):
        def call(**kw):
            assert set(kw) <= set(defaults)
            return fn(packer.pack(*{**defaults, **kw}.values()), None)
        return call

    rotary = caller(lib.pmx_rotary_embedding, _cabi.ROTARY_ARGS, q=16, k=16, qw=0, kw=0, qo=16, ko=16, ss=16, sp=16, ids=0,
                    f=C.addressof(f), T=4, B=2, Hq=4, Hkv=2, D=64, s0=256, s1=64, s2=128, s3=64, r=64, il=0, dt=0, eps=0.0,
                    m=1.0)
    assert rotary(q=0) == -1 and rotary(qo=0) == -1 and rotary(f=0) == -1
    assert rotary(T=0) == -1 and rotary(Hq=0) == -1 and rotary(D=0) == -1
    assert rotary(k=0) == -1 and rotary(Hkv=0) == -1 and rotary(ko=0) == -1
    assert rotary(ss=0) == -1 and rotary(sp=0) == -1 and rotary(B=0) == -1
    assert rotary(r=63) == -1 and rotary(r=66) == -1 and rotary(r=0) == -1 and rotary(r=258, D=512) == -2
    assert rotary(qw=16) == -1 and rotary(kw=16) == -1 and rotary(dt=7) == -2

    prompt = caller(lib.pmx_prompt_attention, _cabi.PROMPT_ATTENTION_ARGS, q=16, k=16, v=16, ss=16, ks=16, pre=0, sl=0, out=16,
                    ws=0, Tq=4, Tk=4096, B=1, Hq=4, Hkv=2, D=64, q0=256, q1=64, k0=128, k1=64, v0=128, v1=64, ms=4, mk=4096,
                    causal=1, dt=0, wb=0, scale=1.0, cap=0.0)
    for name in ("q", "k", "v", "ss", "ks", "out"):
        assert prompt(**{name: 0}) == -1
    for name in ("Tq", "Tk", "B", "Hq", "Hkv", "D", "ms", "mk"):
        assert prompt(**{name: 0}) == -1, name
    assert prompt(Hq=3) == -1 and prompt(D=257) == -2 and prompt(dt=5) == -2 and prompt(B=1 << 21) == -2
    assert prompt(scale=0.0) == -1 and prompt(scale=float("inf")) == -1 and prompt(scale=float("nan")) == -1
    assert prompt(cap=-1.0) == -1 and prompt(cap=float("inf")) == -1
    assert prompt() == -4 and prompt(ws=16, wb=64) == -4                # few rows, many keys: a split, and so a workspace
    assert prompt(ws=8, wb=1 << 30) == -3
    assert lib.pmx_attention_workspace_bytes(4, 1, 4, 2, 64, 4, 100, 0) == 0
    assert lib.pmx_attention_workspace_bytes(4, 1, 4, 2, 64, 4, 4096, 2) == 0           # 32-bit tensors: the plain kernel

    tree = caller(lib.pmx_tree_cache_attention, _cabi.TREE_ATTENTION_ARGS, q=16, k=16, v=16, cache=16, ss=16, cs=16, sp=16,
                  mask=16, out=16, ws=0, Tq=4, B=1, Hq=4, Hkv=2, D=64, q0=256, q1=64, k0=128, k1=64, v0=128, v1=64, rows=9, lo=0,
                  rs=256, kvs=128, hs=64, ms=4, mk=4096, dt=0, wb=0, scale=1.0, cap=0.0)
    for name in ("q", "k", "v", "cache", "ss", "cs", "sp", "mask", "out"):
        assert tree(**{name: 0}) == -1
    assert tree(ms=65) == -2 and tree(rows=0) == -1 and tree(mk=0) == -1 and tree(Hq=5) == -1 and tree() == -4

    compact = caller(lib.pmx_compact_cache, _cabi.COMPACT_CACHE_ARGS, cache=16, cs=16, sp=16, ast=16, ai=16, B=1, n=4, most=4,
                     layers=1, heads=1, D=64, rows=8, rs=128, ls=1024, kvs=64, hs=64, dt=0)
    for name in ("cache", "cs", "sp", "ast", "ai"):
        assert compact(**{name: 0}) == -1
    for name in ("B", "n", "most", "layers", "heads", "D", "rows"):
        assert compact(**{name: 0}) == -1
    assert compact(most=65) == -2 and compact(B=70000) == -2 and compact(dt=3) == -2
    for fn in (lib.pmx_rotary_embedding, lib.pmx_prompt_attention, lib.pmx_tree_cache_attention, lib.pmx_compact_cache):
        assert fn(None, None) == -1


def test_packed_arguments_match_the_header():
    """The structs of include/pmx_moe.h, member by member: 8-byte members in the packers' order."""
    import os
    import re
    from ppl.pmx_b200 import _cabi
    text = open(os.path.join(os.path.dirname(_cabi.PKG), "..", "include", "pmx_moe.h")).read()
    for name, packer in (("rotary", _cabi.ROTARY_ARGS), ("prompt_attention", _cabi.PROMPT_ATTENTION_ARGS),
                         ("tree_attention", _cabi.TREE_ATTENTION_ARGS), ("compact_cache", _cabi.COMPACT_CACHE_ARGS)):
        body = re.search(r"typedef struct pmx_%s_args \{(.*?)\} pmx_%s_args;" % (name, name), text, re.S).group(1)
        kinds = ""
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";")[:-1]:
            # pointers, 64-bit integers, doubles
            assert "*" in decl or "int64_t" in decl or "double" in decl, decl
            kinds += ("d" if "double" in decl and "*" not in decl else "q") * (decl.count(",") + 1)
        q, d = kinds.count("q"), kinds.count("d")
        assert kinds == "q" * q + "d" * d
        assert packer.format == "=%dq" % q + ("%dd" % d if d else "") and packer.size == 8 * (q + d)


def test_export_as_custom_operators(DB):
    """Every operator exports as one node, as the operators beside it do."""
    from torch.onnx._internal.torchscript_exporter import utils as U, _globals

    class Block(torch.nn.Module):
        def forward(s, q, k, v, starts, past, ids, mask, cache, w):
            q, k = DB.qk_norm_rotary_embedding(q, k, w, w, 1e-6, starts, past)
            q, k = DB.rotary_position_embedding(q, k, starts, past, ids)
            a = DB.prompt_attention(q, k, v, starts, starts, 4, 4, 4, 64, num_kv_heads=2)
            return DB.tree_cache_attention(a, k, v, starts, past, past, mask, 4, 4, cache, 4, 64, num_kv_heads=2)

    z = torch.zeros
    args = (z(4, 4, 64), z(4, 2, 64), z(4, 2, 64), torch.tensor([0, 4]), z(1, dtype=torch.int64), torch.arange(4),
            torch.ones(4, dtype=torch.int64), z(9, 1, 2, 2, 64), z(64))
    _globals.GLOBALS.export_onnx_opset_version = 11
    _globals.GLOBALS.in_onnx_export = True
    try:
        with U.exporter_context(Block(), torch.onnx.TrainingMode.EVAL, False):
            graph, _, _ = U._model_to_graph(Block(), args, do_constant_folding=False)
    finally:
        _globals.GLOBALS.in_onnx_export = False
    kinds = [n.kind() for n in graph.nodes() if n.kind().startswith("opmx")]
    assert kinds == ["opmx.dynamic_batching::" + n for n in ("QkNormRotaryEmbedding", "RotaryPositionEmbedding",
                                                             "PromptAttention", "TreeCacheAttention")]
