"""The attention block's operators on the GPU where they are easiest to get wrong."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_block as ab
from tests.helpers import TORCH_DT, dev, host
from tests.test_attention_block_gpu import DB, UNIT, cache_of, check_attention, i64, no_wait_ran_out, prompt_case, starts, values  # noqa: F401

pytestmark = pytest.mark.gpu

KIND = {"nan": (float("nan"), torch.isnan), "inf": (float("inf"), torch.isposinf), "-inf": (float("-inf"), torch.isneginf)}


# ------------------------------------------------------------------------------- values that are not finite
def spread_columns(D):
    return sorted({1, D // 2 - 1, D // 2, D - 2})


def only_its_column(got, clean, sees, col, is_kind):
    """Rows of `sees` hold the value in column `col`, everything else is what it is without it."""
    blind = [t for t in range(len(got)) if t not in sees]
    assert is_kind(got[sees][..., col]).all()
    assert torch.equal(got[blind], clean[blind])
    rest = [c for c in range(got.shape[-1]) if c != col]
    assert torch.equal(got[..., rest], clean[..., rest])


@pytest.mark.parametrize("kind", sorted(KIND))
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("bf16", 96)])
@pytest.mark.parametrize("keys", [5, 128, 131, 256, 300, 513, 2500])
def test_bad_values_of_few_rows_reach_all_columns(DB, kind, dtype, D, keys):
    """Few rows: both softmax halves work on the same rows, on one, two and more key tiles, whole and cut into pieces."""
    rng = np.random.default_rng(keys)
    Hq, Hkv, n = 4, 2, 4
    q, k, v, ss, ks, ms, mk = prompt_case(rng, [(n, keys), (2, 40)], Hq, Hkv, D, dtype)
    x, is_kind = KIND[kind]
    tq, tk, tv = dev(q, dtype), dev(k, dtype), dev(v, dtype)
    a = (i64(ss), i64(ks), ms, mk, Hq, D)
    clean = DB.prompt_attention(tq, tk, tv, *a, num_kv_heads=Hkv)
    for j in sorted({0, keys // 2, keys - n, keys - 1}):
        for col in spread_columns(D):
            bad = tv.clone()
            bad[j, :, col] = x
            sees = [i for i in range(n) if i + keys - n >= j]
            for _ in range(4):                                  # a flag read too early is not read too early every time
                only_its_column(DB.prompt_attention(tq, tk, bad, *a, num_kv_heads=Hkv), clean, sees, col, is_kind)


@pytest.mark.parametrize("kind", sorted(KIND))
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("past", [0, 5, 128, 200, 300, 2500])
def test_bad_values_of_drafted_trees_reach_all_columns(DB, kind, dtype, D, past):
    rng = np.random.default_rng(past)
    Hq, Hkv, n = 4, 2, 6
    x, is_kind = KIND[kind]
    cache = dev(cache_of(rng, 0, past + n + 9, 1, Hkv, D, dtype), dtype)
    q, k, v = (dev(values(rng, (n, h, D), dtype), dtype) for h in (Hq, Hkv, Hkv))
    mask = [1 | 1 << i for i in range(n)]                       # every token sees the first one and itself,
    mask[5] |= 1 << 2                                           # the last one the third as well
    run = lambda v, c: DB.tree_cache_attention(q, k, v, i64([0, n]), i64([3]), i64([past]), i64(mask), n, past + n, c, Hq,  # noqa: E731
                                               D, num_kv_heads=Hkv)
    clean = run(v, cache.clone())
    for col in spread_columns(D):
        for token, sees in ((0, list(range(n))), (2, [2, 5]), (5, [5])):
            bad = v.clone()
            bad[token, :, col] = x
            for _ in range(4):
                only_its_column(run(bad, cache.clone()), clean, sees, col, is_kind)
        for j in sorted({0, past // 2, past - 1} if past else {}):
            bad = cache.clone()
            bad[3 + j, 0, 1, :, col] = x
            for _ in range(4):
                only_its_column(run(v, bad.clone()), clean, list(range(n)), col, is_kind)


# ------------------------------------------------------------------------------- hidden content under a cap, a bias, a prefix
SCORES = {"cap": dict(cap=0.7), "high_cap": dict(cap=40.0), "bias": dict(alibi=True), "prefix": dict(prefix=[33, 8]),
          "all": dict(cap=5.0, alibi=True, prefix=[33, 9])}
HIDDEN = [float("nan"), float("inf"), float("-inf"), 300.0]


def hidden_prompt(DB, dtype, Hq, Hkv, D, lens, scores, seed=5):
    """-> clean call, its reference, and run(key, value, query)"""
    rng = np.random.default_rng(seed)
    cap, prefix = scores.get("cap", 0.0), scores.get("prefix")
    q, k, v, ss, ks, ms, mk = prompt_case(rng, lens, Hq, Hkv, D, dtype, 9)
    slopes = (2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32) if scores.get("alibi") else None
    tq, tk, tv = dev(q, dtype), dev(k, dtype), dev(v, dtype)

    def run(tq=tq, tk=tk, tv=tv):
        return DB.prompt_attention(tq, tk, tv, i64(ss), i64(ks), ms, mk, Hq, D, num_kv_heads=Hkv, logit_cap=cap,
                                   alibi_slopes=None if slopes is None else torch.from_numpy(slopes).cuda(),
                                   prefix_lens=None if prefix is None else i64(prefix))
    ref = ab.prompt_attention(q, k, v, ss, ks, True, 1 / math.sqrt(D), cap, slopes, prefix)
    return run, ref, (tq, tk, tv), mk, cap


@pytest.mark.parametrize("bad", HIDDEN)
@pytest.mark.parametrize("scores", sorted(SCORES))
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [("bf16", 4, 2, 128), ("f16", 3, 1, 64), ("f16", 6, 1, 64), ("f32", 2, 1, 32)])
@pytest.mark.parametrize("n,L", [(70, 200), (70, 201), (9, 131), (9, 132)])
def test_hidden_content_with_scores_of_every_kind(DB, bad, scores, dtype, Hq, Hkv, D, n, L):
    """Hidden keys and values at odd and even places, next to visible ones: later tokens, the next sequence, behind the last."""
    lens = [(n, L), (8, 64)]
    run, ref, (tq, tk, tv), mk, cap = hidden_prompt(DB, dtype, Hq, Hkv, D, lens, SCORES[scores])
    for j in (L - n + 4, L - n + 5, L - 1, L, L + 64):
        kk, vv = tk.clone(), tv.clone()
        kk[j], vv[j] = bad, bad
        if j < L:
            sees = [i for i in range(n) if i + L - n >= j]
        else:
            sees = list(range(n, n + 8)) if j == L else []
        blind = [t for t in range(n + 8) if t not in sees]
        got = run(tk=kk, tv=vv)
        check_attention(got[blind], tuple(x[blind] for x in ref), dtype, D, mk, cap, dtype != "f32")
        if sees and not math.isfinite(bad):
            assert not torch.isfinite(got[sees]).any()


@pytest.mark.parametrize("bad", HIDDEN)
@pytest.mark.parametrize("cap", [0.0, 0.7, 40.0])
@pytest.mark.parametrize("past", [130, 131, 0])
def test_hidden_rows_and_siblings_with_a_cap(DB, bad, cap, past):
    rng = np.random.default_rng(past)
    Hq, Hkv, D, n, dtype = 6, 2, 64, 7, "f16"
    cache_np = cache_of(rng, 0, 200, 1, Hkv, D, dtype)
    q, k, v = (values(rng, (n, h, D), dtype) for h in (Hq, Hkv, Hkv))
    mask = np.array([0b1, 0b11, 0b101, 0b1001, 0b10101, 0b100011, 0b1000001], np.int64)
    ref = ab.tree_attention(q, k, v, cache_np.copy(), 0, 0, [0, n], [20], [past], mask, 1 / math.sqrt(D), cap)
    for token, sees in ((1, [1, 5]), (2, [2, 4]), (3, [3])):
        cache, kk, vv = dev(cache_np, dtype), dev(k, dtype), dev(v, dtype)
        cache[:20], cache[20 + past:] = bad, bad
        kk[token], vv[token] = bad, bad
        got = DB.tree_cache_attention(dev(q, dtype), kk, vv, i64([0, n]), i64([20]), i64([past]), i64(mask), n, past + n, cache, Hq, D,
                                      num_kv_heads=Hkv, logit_cap=cap)
        blind = [t for t in range(n) if t not in sees]
        check_attention(got[blind], tuple(x[blind] for x in ref), dtype, D, past + n, cap)


# ------------------------------------------------------------------------------- bits of a capped row
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [("f16", 4, 2, 64), ("f16", 3, 1, 64), ("f16", 12, 1, 128)])
@pytest.mark.parametrize("cap", [2.0, 300.0])
@pytest.mark.parametrize("n,L", [(70, 201), (9, 131)])
def test_bits_of_a_capped_row_do_not_depend_on_hidden_content(DB, dtype, Hq, Hkv, D, cap, n, L):
    """Neither hidden keys nor the rows of another sequence, nor what other calls left behind, change a result by a bit.  (Rows
    of the same sequence may: those that share a warp take the same form of tanh.)"""
    run, _, (tq, tk, tv), _, _ = hidden_prompt(DB, dtype, Hq, Hkv, D, [(n, L), (8, 64)], dict(cap=cap))
    clean = run()
    for x in (float("nan"), 400.0):
        for j in (L - 1, L, L + 64):
            kk = tk.clone()
            kk[j] = x
            blind = list(range(n, n + 8) if j < L else range(n if j == L else n + 8))
            assert torch.equal(run(tk=kk)[blind], clean[blind])
        for t in (0, n - 1, n, n + 8):
            qq = tq.clone()
            qq[t] = x
            blind = list(range(n, n + 8) if t < n else range(n if t == n else n + 8))
            assert torch.equal(run(tq=qq)[blind], clean[blind])
    for x in (float("nan"), 400.0, 0.0):                        # what another call leaves in the SM's memory
        filler = torch.full((4096, 4, D), x, device="cuda", dtype=TORCH_DT[dtype])
        DB.prompt_attention(filler, filler, filler, i64([0, 4096]), i64([0, 4096]), 4096, 4096, 4, D)
        got = run()
        assert torch.equal(got[:n + 8], clean[:n + 8])


# ------------------------------------------------------------------------------- compaction
@pytest.mark.parametrize("most,listed", [(3, 12), (10, 12), (16, 20), (20, 40), (64, 70), (32, 33)])
def test_compaction_moves_no_more_than_max_accept(DB, most, listed):
    rng = np.random.default_rng(most)
    cache = cache_of(rng, 1, 200, 2, 2, 16, "f16")
    picks = rng.permutation(listed)
    t = dev(cache, "f16")
    DB.compact_cache(t, i64([5, 100]), i64([3, 2]), i64([0, listed, listed + 2]), i64(list(picks) + [1, 0]), most, num_layer=2,
                     cache_layout=1)
    ab.compact_cache(cache, 1, [5, 100], [3, 2], [0, most, most + 2], list(picks[:most]) + [1, 0])
    assert np.array_equal(host(t), cache)


def test_compaction_stays_within_its_sequence(DB):
    """A negative start_pos, or a sequence in front of the cache: no row of another sequence moves or is taken."""
    rng = np.random.default_rng(4)
    cache = cache_of(rng, 0, 40, 1, 2, 16, "f16")
    t = dev(cache, "f16")
    cs, sp = [10, -6, 20, (1 << 63) - 1], [-3, 5, 4, (1 << 63) - 1]
    picks = [[1, 2, 5, 6, 4], [3, 4, 2, 0], [2, 0], [4, 5, 6]]
    DB.compact_cache(t, i64(cs), i64(sp), i64(starts([len(p) for p in picks])), i64(sum(picks, [])), 5)
    want = cache.copy()
    for c, s, p in zip(cs, sp, picks):
        for i, j in enumerate(p):
            if max(c, 0) <= c + s + i < 40 and max(c, 0) <= c + s + j < 40:
                want[c + s + i] = cache[c + s + j]
    assert np.array_equal(host(t), want)


# ------------------------------------------------------------------------------- tangents, memory, workspaces
def every_operator(DB, q, k, v, w, cache, indices):
    ss, z = i64([0, 5]).to(indices), i64([0])
    D, H = q.shape[2], q.shape[1]
    return {"rotary": lambda: DB.rotary_position_embedding(q, k, ss, z),
            "norm": lambda: DB.qk_norm_rotary_embedding(q, k, w, w, 1e-6, ss, z),
            "prompt": lambda: DB.prompt_attention(q, k, v, ss, ss, 5, 5, H, D),
            "tree": lambda: DB.tree_cache_attention(q, k, v, ss, z, z, i64([1] * 5), 5, 5, cache, H, D),
            "compact": lambda: DB.compact_cache(cache, z, z, i64([0, 2]).to(indices), i64([1, 2]), 2)}


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("indices", [torch.int64, torch.int32])
def test_a_tangent_is_refused_not_dropped(DB, which, indices):
    import torch.autograd.forward_ad as fw
    t = [torch.randn(5, 2, 64, device="cuda") for _ in range(3)] + [torch.randn(64, device="cuda"),
                                                                     torch.randn(9, 1, 2, 2, 64, device="cuda")]
    uses = {"rotary": (0, 1), "norm": (0, 1, 3), "prompt": (0, 1, 2), "tree": (0, 1, 2, 4), "compact": (4,)}
    with fw.dual_level():
        x = list(t)
        x[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        for name, call in every_operator(DB, *x, indices).items():
            if which in uses[name]:
                with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward|backward"):
                    call()
            else:
                call()
    q = t[0]
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: every_operator(DB, x, *t[1:], indices)["prompt"](), (q,), (q,))


def test_running_out_of_memory_says_so(DB):
    q = torch.zeros(1, 1, 128, device="cuda", dtype=torch.float16).expand(1 << 30, 1, 128)      # a result of 256 GB
    for ss in (i64([0, 1 << 30]), i64([0, 1 << 30]).int()):
        with pytest.raises(torch.OutOfMemoryError):
            DB.rotary_position_embedding(q, None, ss, i64([0]))


def test_workspace_is_asked_for_at_every_call(DB, monkeypatch):
    """Its size goes by the current device: no answer is kept for a call on another one."""
    from ppl.pmx_b200.torch_function.dynamic_batching import masked_attention as M
    real, asked = M.lib, []

    class Lib:
        def __getattr__(self, name):
            if name == "pmx_attention_workspace_bytes":
                asked.append(name)
            return getattr(real, name)
    monkeypatch.setattr(M, "lib", Lib())
    q = torch.ones(4, 2, 64, device="cuda", dtype=torch.float16)
    k = torch.ones(4096, 2, 64, device="cuda", dtype=torch.float16)
    for n in (1, 2):
        DB.prompt_attention(q, k, k, i64([0, 4]).int(), i64([0, 4096]), 4, 4096, 2, 64)
        assert len(asked) == n


def test_results_do_not_depend_on_the_way_through_the_host(DB, monkeypatch):
    from ppl.pmx_b200.torch_function.dynamic_batching import _common, cache_rows, masked_attention, rotary
    rng = np.random.default_rng(0)
    t = [dev(values(rng, (5, 2, 64), "f16"), "f16") for _ in range(3)] + [dev(values(rng, (64,), "f16"), "f16")]
    cache = dev(values(rng, (9, 1, 2, 2, 64), "f16"), "f16")

    def results():
        c = cache.clone()
        return [x for call in every_operator(DB, *t, c, torch.int64).values() for r in [call()]
                for x in (r if isinstance(r, tuple) else (r,))] + [c]
    want = results()
    for module in (cache_rows, masked_attention, rotary):
        monkeypatch.setattr(module, "host", _common._GeneralPath)
    assert all(torch.equal(a, b) for a, b in zip(results(), want))


@pytest.mark.parametrize("cap", [1e-3, 1e-30, 1e-38, 1e-41, 1e30])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_caps_from_nothing_to_no_cap(DB, cap, dtype):
    """Any positive cap: scores of zero among others stay zero, a cap near nothing leaves all keys alike."""
    rng = np.random.default_rng(2)
    q, k, v, ss, ks, ms, mk = prompt_case(rng, [(40, 140), (3, 9)], 2, 1, 64, dtype)
    q[1], k[3] = 0, 0
    got = DB.prompt_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), i64(ss), i64(ks), ms, mk, 2, 64, num_kv_heads=1,
                              logit_cap=cap)
    check_attention(got, ab.prompt_attention(q, k, v, ss, ks, True, 1 / 8.0, cap), dtype, 64, mk, min(cap, 30.0), dtype != "f32")


# ------------------------------------------------------------------------------- weak keys in f16
@pytest.mark.parametrize("log2", [17.25, 25.5, 30.75])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_weak_keys_beside_a_dominant_one(DB, log2, first, dtype):
    """n keys of probability 2^-log2 beside one of (nearly) 1, whose value is zero: together they are the result.
    On the way a probability takes 16 bits, scaled by 2^11 in f16: half a step of 2^-11 of it, or 2^-25 of the scaled value
    where that is below 2^-14: 2^-36 absolute."""
    T, H, D, n = 2560, 8, 64, 60000
    rng = np.random.default_rng(1)
    q = torch.zeros(T, H, D, device="cuda", dtype=TORCH_DT[dtype])
    k = torch.zeros(n + 1, H, D, device="cuda", dtype=TORCH_DT[dtype])
    v = torch.ones(n + 1, H, D, device="cuda", dtype=TORCH_DT[dtype])
    at = 0 if first else n
    q[..., 0], k[at, :, 0], v[at] = 4.0, log2 * math.log(2) / 4, 0.0
    s = 4.0 * float(k[at, 0, 0])
    w = n * math.exp(-s)
    want = w / (1 + w)
    got = DB.prompt_attention(q, k, v, i64([0, T]), i64([0, n + 1]), T, n + 1, H, D, is_causal=False, scale=1.0)
    # two roundings to 16 bits; the products' sum over n / 16 steps and the probabilities' in 32; scores of 2^-19
    tol = (2 * UNIT[dtype] + (n / 8 + n / 128) * 2.0 ** -24 + 2.0 ** -19) * want + n * 2.0 ** -36 * (dtype == "f16") + 2.0 ** -25
    assert (got.double() - want).abs().max() <= tol


@pytest.mark.parametrize("fill", [0x7F, 0xFF, 0x01])
def test_starts_that_do_not_rise_stay_inside(DB, fill):
    """Sequences that overlap or end before they begin, over keys in many pieces: what is computed then is of no use, but
    nothing outside the tensors is touched, whatever the workspace held before."""
    Hq, Hkv, D = 4, 2, 64
    q = torch.ones(8, Hq, D, device="cuda", dtype=torch.float16)
    k = torch.ones(9100, Hkv, D, device="cuda", dtype=torch.float16)
    cache = torch.ones(9200, 1, 2, Hkv, D, device="cuda", dtype=torch.float16)
    for ss in ([0, 4, 2, 6], [7, 3, 5, 1], [0, -4, 90, 8], [3, 3, 1, 1]):
        junk = [torch.full((n,), fill, device="cuda", dtype=torch.uint8) for n in (1 << 20, 8 << 20, 32 << 20)]
        del junk
        DB.prompt_attention(q, k, k, i64(ss), i64([0, 3000, 6000, 9100]), 4, 9100, Hq, D, num_kv_heads=Hkv)
        DB.tree_cache_attention(q, k[:8], k[:8], i64(ss), i64([0, 3000, 6000]), i64([2900, 2900, 3100]), i64([-1] * 8), 4, 3110, cache,
                                Hq, D, num_kv_heads=Hkv)
    torch.cuda.synchronize()


@pytest.mark.parametrize("lens", [[(3, 40), (1, 700)], [(300, 300), (2, 900)]])
@pytest.mark.parametrize("most", [1 << 31, 1 << 57, (1 << 63) - 1])
def test_lengths_without_a_bound(DB, lens, most):
    """max_seqlen and max_kvlen are bounds; one that says nothing is as good as any."""
    rng = np.random.default_rng(7)
    q, k, v, ss, ks, ms, mk = prompt_case(rng, lens, 4, 2, 64, "bf16")
    ref = ab.prompt_attention(q, k, v, ss, ks, True, 1 / 8.0)
    for a, b in ((ms, most), (most, mk), (most, most)):
        got = DB.prompt_attention(dev(q, "bf16"), dev(k, "bf16"), dev(v, "bf16"), i64(ss), i64(ks), a, b, 4, 64, num_kv_heads=2)
        check_attention(got, ref, "bf16", 64, mk, 0.0)


# ------------------------------------------------------------------------------- rows outside the cache
@pytest.mark.parametrize("dtype,D", [("f16", 64), ("f32", 48)])
def test_drafted_rows_outside_the_cache_or_before_their_sequence_are_dropped(DB, dtype, D):
    """A sequence that begins before the cache stores and sees only the rows that exist; one with a negative start_pos sees no
    row and stores none in front of its first."""
    rng = np.random.default_rng(3)
    Hq, Hkv, rows = 4, 2, 60
    cache_np = cache_of(rng, 2, rows, 1, Hkv, D, dtype)
    n = [4, 4, 3, 2, 2]
    cs, sp = [-4, 20, 50, 1 << 62, -(1 << 62)], [3, -2, 12, 1 << 62, -(1 << 62)]
    ss, T = starts(n), sum(n)
    q, k, v = (values(rng, (T, h, D), dtype) for h in (Hq, Hkv, Hkv))
    masks = np.array([(1 << (i + 1)) - 1 for m in n for i in range(m)], np.int64)
    cache = dev(cache_np, dtype)
    got = DB.tree_cache_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), i64(ss), i64(cs), i64(sp), i64(masks), 4, 20, cache,
                                  Hq, D, num_kv_heads=Hkv, cache_layout=2)
    want = cache_np.copy()
    for b, m in enumerate(n):
        for i in range(m):
            row = cs[b] + sp[b] + i
            if max(cs[b], 0) <= row < rows:
                want[0, 0, row], want[0, 1, row] = k[ss[b] + i], v[ss[b] + i]
    assert np.array_equal(host(cache), want)
    lo = [0, 20, 50, 0, 0]
    past = [0, 0, 10, 0, 0]
    ref = ab.tree_attention(q, k, v, cache_np.copy(), 2, 0, ss, lo, past, masks, 1 / math.sqrt(D))
    check_attention(got, ref, dtype, D, 20, 0.0, dtype != "f32")


def test_a_cache_without_rows_is_refused(DB):
    q = torch.ones(2, 2, 64, device="cuda", dtype=torch.float16)
    cache = torch.empty(0, 1, 2, 2, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="rows"):
        DB.tree_cache_attention(q, q, q, i64([0, 2]), i64([0]), i64([0]), i64([1, 3]), 2, 2, cache, 2, 64)


def test_a_captured_speculative_step_follows_its_inputs(DB):
    """Rotation by depth, tree attention and compaction in one graph: replays with other lengths, masks and accepted rows give
    what eager calls give, with the captured bounds."""
    rng = np.random.default_rng(11)
    B, n, Hq, Hkv, D, rows = 3, 6, 8, 2, 128, 700
    base = dev(cache_of(rng, 1, B * rows, 1, Hkv, D, "bf16"), "bf16")
    x = dev(values(rng, (B * n, Hq + 2 * Hkv, D), "bf16"), "bf16")
    ss, cs, a = i64(np.arange(B + 1) * n), i64(np.arange(B) * rows), i64([0, 2, 4, 6])
    past, ids, mask, picks = (i64(np.zeros(m)) for m in (B, B * n, B * n, 6))

    def step(cache):
        q, k = DB.rotary_position_embedding(x[:, :Hq], x[:, Hq:Hq + Hkv], None, None, ids)
        o = DB.tree_cache_attention(q, k, x[:, Hq + Hkv:], ss, cs, past, mask, n, 640, cache, Hq, D, num_kv_heads=Hkv, cache_layout=1)
        DB.compact_cache(cache, cs, past, a, picks, 2, cache_layout=1)
        return o
    static = base.clone()
    step(static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for lengths in ([0, 0, 0], [600, 1, 127], [128, 0, 512]):
        past.copy_(i64(lengths))
        ids.copy_(i64([p + d for p in lengths for d in rng.integers(0, n, n)]))
        mask.copy_(i64([(1 << i | int(rng.integers(0, 1 << i))) for _ in range(B) for i in range(n)]))
        picks.copy_(i64(rng.integers(0, n, 6)))
        static.copy_(base)
        graph.replay()
        eager = base.clone()
        want = step(eager)
        assert torch.equal(out, want) and torch.equal(static, eager)
