"""The attention block's host side without a GPU: what asks for a derivative, what the package needs to be imported, what an
export holds, sizes of workspaces."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def DB():
    import ppl.pmx_b200.torch_function as F
    return F.dynamic_batching


def test_gradients_and_tangents_are_noticed(DB):
    import torch.autograd.forward_ad as fw
    from ppl.pmx_b200.torch_function.dynamic_batching._common import wants_grad
    x = torch.ones(3)
    assert not wants_grad(x, None) and wants_grad(None, x.clone().requires_grad_())
    with torch.no_grad():
        assert not wants_grad(x.clone().requires_grad_())
    with fw.dual_level():
        dual = fw.make_dual(x, x)
        assert wants_grad(x, dual) and not wants_grad(x)
        with torch.no_grad():
            assert wants_grad(dual)
    assert not wants_grad(dual)


@pytest.mark.parametrize("calls", ["None", "types.SimpleNamespace(built_for='torch 1.0, python 3.1')", "types.SimpleNamespace()"])
def test_the_package_does_without_the_host_calls(calls):
    """Missing, not loadable, or of another torch: a warning, and every call takes the general path."""
    code = f"""
import sys, types, warnings
sys.modules["ppl.pmx_b200._host_calls"] = {calls}
with warnings.catch_warnings(record=True) as said:
    warnings.simplefilter("always")
    import ppl.pmx_b200.torch_function as F
assert any("_host_calls.so is not used" in str(w.message) for w in said), said
import torch
DB = F.dynamic_batching
q, i = torch.zeros(4, 2, 64), torch.arange(3)
for call in (lambda: DB.rotary_position_embedding(q, q, i, i[:2]), lambda: DB.prompt_attention(q, q, q, i, i, 2, 2, 2, 64),
             lambda: DB.tree_cache_attention(q, q, q, i, i[:2], i[:2], torch.zeros(4).long(), 2, 2, torch.zeros(8, 1, 2, 2, 64), 2, 64),
             lambda: DB.compact_cache(torch.zeros(8, 1, 2, 2, 64), i[:2], i[:2], i, i[:2], 1)):
    try:
        call()
        raise SystemExit("not refused")
    except RuntimeError as e:
        assert "no CPU fallback" in str(e)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


def test_the_host_calls_are_used_here(DB):
    from ppl.pmx_b200 import _host_calls
    from ppl.pmx_b200.torch_function.dynamic_batching import _common
    assert _common.host is _host_calls


def test_a_failed_build_of_the_host_calls_leaves_none(tmp_path, monkeypatch, capsys):
    from ppl.pmx_b200 import build
    target = tmp_path / "_host_calls.so"
    target.write_bytes(b"of an earlier build")
    monkeypatch.setattr(build, "HOST", str(target))
    monkeypatch.setattr(build, "_host_command", lambda: ["false"])
    build._build_host()
    assert not target.exists()
    monkeypatch.setattr(build, "_host_command", lambda: 1 / 0)
    build._build_host()
    assert capsys.readouterr().err.count("host_calls.cpp was not built") == 2


def test_host_calls_of_another_torch_are_built_anew(monkeypatch):
    from ppl.pmx_b200 import build
    monkeypatch.setattr(build, "_stale", lambda target: False)
    now = build._built_for()
    assert not build._host_stale()
    monkeypatch.setattr(build, "_built_for", lambda: now[:-1])
    assert build._host_stale()


def test_exported_attention_keeps_its_lengths(DB):
    """max_seqlen (rows behind it are zero) and max_kvlen are inputs of the nodes, given as ints or as tensors."""
    from torch.onnx._internal.torchscript_exporter import utils as U, _globals

    class Block(torch.nn.Module):
        def forward(s, q, k, starts, past, mask, cache, most):
            a = DB.prompt_attention(q, k, k, starts, starts, 3, most, 4, 64, num_kv_heads=2, alibi_slopes=torch.ones(4))
            return DB.tree_cache_attention(a, k, k, starts, past, past, mask, most, 7, cache, 4, 64, num_kv_heads=2)

    z = torch.zeros
    args = (z(4, 4, 64), z(4, 2, 64), torch.tensor([0, 4]), z(1, dtype=torch.int64), torch.ones(4, dtype=torch.int64),
            z(9, 1, 2, 2, 64), torch.tensor([5]))
    _globals.GLOBALS.export_onnx_opset_version = 11
    _globals.GLOBALS.in_onnx_export = True
    try:
        with U.exporter_context(Block(), torch.onnx.TrainingMode.EVAL, False):
            graph, _, _ = U._model_to_graph(Block(), args, do_constant_folding=False)
    finally:
        _globals.GLOBALS.in_onnx_export = False
    prompt, tree = [n for n in graph.nodes() if n.kind().startswith("opmx")]
    most = list(graph.inputs())[6]
    constant = lambda v: v.node().t("value").tolist()        # noqa: E731
    p, t = list(prompt.inputs()), list(tree.inputs())
    assert len(p) == 8 and constant(p[5]) == [3] and p[6].debugName() == most.debugName() and prompt.i("alibi_slopes") == 1
    assert len(t) == 10 and t[7].debugName() == most.debugName() and constant(t[8]) == [7]


@pytest.mark.parametrize("tokens,sequences,heads,kv_heads,most", [(4, 1, 4, 2, 4), (64, 64, 64, 64, 1), (400, 1, 4, 2, 400),
                                                                  (5000, 100, 8, 8, 300), (6400, 6400, 8, 8, 1)])
def test_a_bound_on_the_keys_may_be_any_number(tokens, sequences, heads, kv_heads, most):
    """max_kvlen is a bound: one beyond every tensor (no bound at all) plans what the largest possible one does."""
    from ppl.pmx_b200._cabi import lib
    size = lambda n: lib.pmx_attention_workspace_bytes(tokens, sequences, heads, kv_heads, 64, most, n, 0)     # noqa: E731
    want = size(1 << 31)
    assert 0 < want < 1 << 30 or want == 0 and most > 128
    for n in ((1 << 31) + 1, 1 << 40, 1 << 57, 1 << 62, (1 << 63) - 1):
        assert size(n) == want
