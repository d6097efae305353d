"""The attention block's operators on the GPU against their definitions in 64 bits (oracle/attention_block.py):
rotary positions, norms of the heads with the rotation, prompt attention, tree attention over the cache, cache
compaction, and a speculative step made of them."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_block as ab
from oracle import moe_oracle as orc
from tests.helpers import TORCH_DT, dev, host

pytestmark = pytest.mark.gpu

UNIT = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


@pytest.fixture(scope="module")
def DB():
    import ppl.pmx_b200.torch_function as F
    return F.dynamic_batching


@pytest.fixture(autouse=True)
def no_wait_ran_out(DB):
    yield
    DB.attention_check()


def values(rng, shape, dtype, scale=1.0):
    return orc.round_to_dtype((rng.standard_normal(shape) * scale).astype(np.float32), dtype)


def i64(a):
    return torch.tensor(np.asarray(a), dtype=torch.int64, device="cuda")


def starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


# ------------------------------------------------------------------------------------------- rotary positions
def rotary_close(got, want, x, dtype, factor, wmax=1.0):
    """One rounding of the result, and 32-bit arithmetic on the way: the angle is off by at most 2^-23 radians (its
    turn is rounded to 24 bits below one half: 2 pi 2^-26, plus half a step of the doubled value's cosine), cosine and
    sine by 2^-22, the norm's factor by D 2^-24 + 2^-22; each of the two products by 2^-24.  Pairs are at most
    sqrt(2) times the larger member; 2^-20 of the head's largest value covers them."""
    top = np.abs(x).max(-1, keepdims=True) * factor * wmax * 2
    tol = UNIT[dtype] * np.abs(want) * 1.01 + 2.0 ** -20 * top + 2.0 ** -25 * (dtype == "f16")
    bad = np.abs(host(got).astype(np.float64) - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.abs(host(got) - want).max()}"


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,r", [(8, 2, 128, 128), (4, 1, 64, 32), (3, 3, 96, 96), (5, 1, 80, 20), (2, 2, 256, 256),
                                        (1, 1, 10, 6), (6, 2, 64, 2), (12, 4, 48, 48)])
def test_rotary(DB, dtype, interleaved, Hq, Hkv, D, r):
    rng = np.random.default_rng(D + r)
    lens, past = [1, 0, 13, 4], [7, 3, 0, 123456]
    ss, T = starts(lens), sum(lens) + 3                       # three rows behind the last sequence
    q, k = values(rng, (T, Hq, D), dtype), values(rng, (T, Hkv, D), dtype)
    gq, gk = DB.rotary_position_embedding(dev(q, dtype), dev(k, dtype), i64(ss), i64(past), rotary_dim=r, theta=1e4,
                                          interleaved=interleaved)
    pos, live = ab.positions(ss, past, T)
    f, m = ab.frequencies(r, 1e4)
    for got, x in ((gq, q), (gk, k)):
        rotary_close(got, ab.rotary(x, pos, live, f, m, interleaved), x, dtype, m)
        assert np.array_equal(host(got)[~live], x[~live]) and np.array_equal(host(got)[..., r:], x[..., r:])


@pytest.mark.parametrize("scaling", [dict(scaling_type="linear", scaling_factor=4.0), dict(scaling_type="ntk", scaling_factor=8.0),
                                     dict(scaling_type="yarn", scaling_factor=16.0, original_max_position=4096)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_scaled_far_positions_by_ids(DB, scaling, norm):
    rng = np.random.default_rng(3)
    T, Hq, Hkv, D = 37, 4, 2, 128
    ids = np.concatenate([[0, 1, -5, 2 ** 31 + 11, 10 ** 6, 10 ** 9], rng.integers(0, 1 << 22, T - 6)])
    q, k = values(rng, (T, Hq, D), "f32"), values(rng, (T, Hkv, D), "f32")
    wq, wk = values(rng, D, "f32") + 1, values(rng, D, "f32") + 1
    if norm:
        got = DB.qk_norm_rotary_embedding(dev(q, "f32"), dev(k, "f32"), dev(wq, "f32"), dev(wk, "f32"), 1e-5, None, None,
                                          i64(ids), theta=1e6, **scaling)
    else:
        got = DB.rotary_position_embedding(dev(q, "f32"), dev(k, "f32"), None, None, i64(ids), theta=1e6, **scaling)
    f, m = ab.frequencies(D, 1e6, scaling["scaling_type"], scaling["scaling_factor"], scaling.get("original_max_position", 0))
    for g, x, w in ((got[0], q, wq), (got[1], k, wk)):
        want = ab.rotary(x, ids, np.ones(T, bool), f, m, False, w if norm else None, 1e-5)
        # the 32-bit turn of a position p is p f / 2 pi taken in 64 bits: off by p f 2^-53, 2^-22 at 2^31
        rotary_close(g, want, x if not norm else x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5), "f32", m,
                     np.abs(w).max() if norm else 1.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,r,T", [(8, 2, 128, 128, 1), (4, 2, 64, 32, 33), (3, 1, 96, 48, 5), (2, 1, 72, 30, 6),
                                          (2, 2, 256, 128, 9), (4, 1, 128, 128, 9000)])
def test_qk_norm_rotary_of_a_fused_projection(DB, dtype, interleaved, Hq, Hkv, D, r, T):
    """Query and key are views into the projection's rows [T, (Hq + 2 Hkv) D]."""
    rng = np.random.default_rng(T)
    rows = values(rng, (T, Hq + 2 * Hkv, D), dtype)
    rows[0, 0] = 0                                            # a head of zeros stays zero
    wq, wk = (orc.round_to_dtype(1 + 0.3 * rng.standard_normal(D).astype(np.float32), dtype) for _ in range(2))
    x = dev(rows, dtype)
    gq, gk = DB.qk_norm_rotary_embedding(x[:, :Hq], x[:, Hq:Hq + Hkv], dev(wq, dtype), dev(wk, dtype), 1e-6, i64([0, T]),
                                         i64([41]), rotary_dim=r, theta=5e5, interleaved=interleaved)
    assert gq.is_contiguous() and gk.is_contiguous()
    f, m = ab.frequencies(r, 5e5)
    pos, live = np.arange(41, 41 + T), np.ones(T, bool)
    keep = np.arange(T) if T < 100 else np.concatenate([[0, 1, 7, 8, T - 1], rng.integers(0, T, 60)])
    for got, h0, h1, w in ((gq, 0, Hq, wq), (gk, Hq, Hq + Hkv, wk)):
        part = rows[keep, h0:h1].astype(np.float64)
        normed = part / np.sqrt((part * part).mean(-1, keepdims=True) + 1e-6)
        want = ab.rotary(rows[keep, h0:h1], pos[keep], live[keep], f, m, interleaved, w, 1e-6)
        rotary_close(got[torch.from_numpy(keep).cuda()], want, normed, dtype, m, np.abs(w).max())
    # the norm alone on rows of no sequence: they are copied
    gq, _ = DB.qk_norm_rotary_embedding(x[:, :Hq], x[:, Hq:Hq + Hkv], dev(wq, dtype), dev(wk, dtype), 1e-6, i64([0, 0]),
                                        i64([41]), rotary_dim=r)
    assert torch.equal(gq, x[:, :Hq])


def test_rotary_without_key_and_odd_strides(DB):
    rng = np.random.default_rng(0)
    base = dev(values(rng, (9, 3 * 64 + 1), "f16"), "f16")
    q = base[:, 1:].unflatten(1, (3, 64))                     # rows that begin off a 16-byte boundary
    got, none = DB.rotary_position_embedding(q, None, i64([0, 9]), i64([5]))
    assert none is None
    want, _ = DB.rotary_position_embedding(q.contiguous(), None, i64([0, 9]), i64([5]))
    assert torch.equal(got, want)
    t = dev(values(rng, (3, 64, 9), "f16"), "f16").permute(2, 0, 1)                 # inner stride not one
    assert torch.equal(DB.rotary_position_embedding(t, None, i64([0, 9]), i64([5]))[0],
                       DB.rotary_position_embedding(t.contiguous(), None, i64([0, 9]), i64([5]))[0])
    empty = torch.empty(0, 3, 64, dtype=torch.float16, device="cuda")
    assert DB.rotary_position_embedding(empty, empty, i64([0, 0]), i64([5]))[1].shape == (0, 3, 64)


# ------------------------------------------------------------------------------------------- prompt attention
LENS = {"one": [(1, 1)], "short": [(5, 5), (0, 0), (17, 17), (1, 1)], "tile": [(127, 127), (128, 128), (129, 129)],
        "chunk": [(3, 300), (70, 201), (33, 33), (0, 40)], "more_queries_than_keys": [(10, 4), (6, 0), (3, 3)],
        "few_rows_long": [(1, 2500), (2, 40), (5, 1111)]}


def prompt_case(rng, lens, Hq, Hkv, D, dtype, extra=0):
    n, L = [a for a, _ in lens], [b for _, b in lens]
    T, K = sum(n) + extra, sum(L) + extra
    return (values(rng, (T, Hq, D), dtype), values(rng, (K, Hkv, D), dtype), values(rng, (K, Hkv, D), dtype), starts(n),
            starts(L), max(max(n), 1), max(max(L), 1))


def check_attention(got, ref, dtype, D, keys, cap, tensor_cores=True):
    o, A, dots, tops = ref
    tol = ab.attention_tolerance(o, A, dots, tops, UNIT[dtype], UNIT[dtype] if tensor_cores else 0.0, D, keys, cap)
    err = np.abs(host(got).astype(np.float64) - o)
    assert np.isfinite(err).all(), f"{(~np.isfinite(err)).sum()} results are not finite"
    bad = err > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {err.max()} with a bound of {tol[bad].min()}, first at {np.argwhere(bad)[0]}"


def run_prompt(DB, dtype, lens, Hq, Hkv, D, causal=True, cap=0.0, alibi=False, prefix=None, scale=None, seed=0, extra=0):
    rng = np.random.default_rng(seed + D + Hq)
    q, k, v, ss, ks, ms, mk = prompt_case(rng, lens, Hq, Hkv, D, dtype, extra)
    slopes = (2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32) if alibi else None
    got = DB.prompt_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), i64(ss), i64(ks), ms, mk, Hq, D,
                              is_causal=causal, num_kv_heads=Hkv, scale=scale, logit_cap=cap,
                              alibi_slopes=None if slopes is None else torch.from_numpy(slopes).cuda(),
                              prefix_lens=None if prefix is None else i64(prefix))
    ref = ab.prompt_attention(q, k, v, ss, ks, causal, scale or 1 / math.sqrt(D), cap, slopes, prefix)
    check_attention(got, ref, dtype, D, mk, cap)
    return got, ss


@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [("bf16", 4, 1, 128), ("f16", 2, 2, 64), ("bf16", 3, 1, 96), ("f16", 12, 2, 40),
                                            ("f32", 2, 1, 64), ("bf16", 2, 1, 33), ("f16", 2, 2, 256)])
def test_prompt_attention_lengths_and_heads(DB, lens, dtype, Hq, Hkv, D):
    if lens in ("few_rows_long", "tile") and (D in (33, 256) or dtype == "f32"):
        pytest.skip("the plain kernel has no tiles and no split")
    run_prompt(DB, dtype, LENS[lens], Hq, Hkv, D)


@pytest.mark.parametrize("options", [dict(causal=False), dict(cap=5.0), dict(alibi=True), dict(prefix=[20, 0, 300, 7]),
                                     dict(cap=30.0, alibi=True, prefix=[100, 1, 0, 40]), dict(scale=0.01), dict(scale=3.0),
                                     dict(causal=False, alibi=True), dict(causal=False, cap=9.0, prefix=[20, 0, 300, 7])])
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [("bf16", 8, 2, 128), ("f16", 2, 2, 64), ("f32", 2, 1, 32)])
def test_prompt_attention_options(DB, options, dtype, Hq, Hkv, D):
    run_prompt(DB, dtype, [(140, 140), (1, 9), (30, 350), (40, 40)], Hq, Hkv, D, **options)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 1), (7, 1), (16, 1), (64, 1), (96, 1), (130, 1), (8, 8)])
def test_prompt_attention_groups(DB, Hq, Hkv):
    run_prompt(DB, "f16", [(19, 60), (3, 3)], Hq, Hkv, 64)


@pytest.mark.parametrize("dtype,Hq,Hkv,D,causal,alibi", [("bf16", 4, 2, 64, True, False), ("f16", 3, 3, 128, True, True),
                                                         ("bf16", 2, 1, 80, False, False)])
def test_prompt_attention_of_many_ragged_sequences(DB, dtype, Hq, Hkv, D, causal, alibi):
    """More sequences than a warp has lanes, empty ones among them, several rounds of items for every CTA."""
    rng = np.random.default_rng(21)
    lens = [(int(n), int(n + more)) for n, more in zip(rng.integers(0, 280, 75), rng.integers(0, 3, 75) * 50)]
    lens[0], lens[40], lens[74] = (0, 0), (0, 17), (300, 300)
    run_prompt(DB, dtype, lens, Hq, Hkv, D, causal=causal, alibi=alibi, extra=2)


@pytest.mark.parametrize("rows,Hq,Hkv,D", [(4, 2, 1, 128), (1, 1, 1, 64), (9, 6, 2, 40)])
def test_few_rows_over_keys_in_many_pieces(DB, rows, Hq, Hkv, D):
    """A long key axis is cut into more pieces than a warp has lanes, next to sequences of one piece and of none."""
    run_prompt(DB, "bf16", [(3, 60), (rows, 9100), (0, 5), (2, 2)], Hq, Hkv, D)


@pytest.mark.parametrize("cap", [0.5, 2.0, 4.0, 12.0])
def test_scores_around_the_cap(DB, cap):
    """Scores from far below the cap to far above it: tanh by either polynomial and by the exponential, in all mixtures."""
    run_prompt(DB, "f16", [(130, 130), (7, 300)], 2, 1, 64, cap=cap, scale=0.2)


@pytest.mark.parametrize("lens,most", [([(20, 20), (7, 30)], 9), ([(300, 300), (90, 200)], 150), ([(3, 2000)], 2),
                                       ([(200, 3000)], 150)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_past_max_seqlen_are_zero(DB, dtype, lens, most):
    rng = np.random.default_rng(2)
    q, k, v, ss, ks, _, mk = prompt_case(rng, lens, 2, 1, 64, dtype)
    args = (dev(q, dtype), dev(k, dtype), dev(v, dtype), i64(ss), i64(ks))
    torch.full((1 << 20,), float("nan"), device="cuda")               # freed: what the results' memory may hold
    got = DB.prompt_attention(*args, most, mk, 2, 64, num_kv_heads=1)
    o, A, dots, tops = ab.prompt_attention(q, k, v, ss, ks, True, 1 / 8.0, 0.0, None, None)
    keep = np.concatenate([np.arange(s, min(s + most, e)) for s, e in zip(ss[:-1], ss[1:])])
    rest = np.setdiff1d(np.arange(len(q)), keep)
    check_attention(got[torch.from_numpy(keep).cuda()], (o[keep], A[keep], dots[keep], tops[keep]), dtype, 64, mk, 0.0)
    assert len(rest) and not got[torch.from_numpy(rest).cuda()].any()


@pytest.mark.parametrize("lens", [[(300, 300)], [(2, 1500)], [(600, 600), (1, 700)]])
def test_rows_of_no_sequence_are_zero(DB, lens):
    got, ss = run_prompt(DB, "bf16", lens, 4, 2, 128, extra=5)
    assert not got[int(ss[-1]):].any()


BAD = [float("nan"), float("inf"), float("-inf"), "lowest"]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("f32", 32)])
@pytest.mark.parametrize("where", ["later_token", "other_sequence", "behind"])
def test_what_a_token_may_not_see_does_not_reach_it(DB, bad, dtype, D, where):
    """Values that are not finite, or the type's lowest, in later positions, in the next sequence, behind the last."""
    Hq, Hkv = 4, 2
    rng = np.random.default_rng(5)
    lens = [(70, 200), (150, 150)]
    q, k, v, ss, ks, ms, mk = prompt_case(rng, lens, Hq, Hkv, D, dtype, 9)
    x = torch.finfo(TORCH_DT[dtype]).min if bad == "lowest" else bad
    tq, tk, tv = dev(q, dtype), dev(k, dtype), dev(v, dtype)
    run = lambda: DB.prompt_attention(tq, tk, tv, i64(ss), i64(ks), ms, mk, Hq, D, num_kv_heads=Hkv)  # noqa: E731
    clean = run()
    if where == "later_token":            # position 170 of the first sequence: its query 40 is the first to see it
        sees, blind = torch.arange(40, 70), torch.cat([torch.arange(0, 40), torch.arange(70, 229)])
        tk[170], tv[170] = x, x
    elif where == "other_sequence":       # the first row of the second sequence, behind the first's last key
        sees, blind = torch.arange(70, 220), torch.cat([torch.arange(0, 70), torch.arange(220, 229)])
        tk[200], tv[200] = x, x
    else:
        sees, blind = torch.arange(0), torch.arange(0, 229)
        tk[350:], tv[350:] = x, x
        tq[220:] = x
    got = run()
    assert torch.equal(got[blind.cuda()], clean[blind.cuda()])
    if bad != "lowest" and len(sees):
        assert not torch.isfinite(got[sees.cuda()]).any()


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64)])
def test_values_that_are_not_finite_reach_those_who_see_them(DB, dtype, D):
    """Only the values hold them: the columns that hold one say so, from the first token that sees it on."""
    rng = np.random.default_rng(6)
    q, k, v, ss, ks, ms, mk = prompt_case(rng, [(150, 150)], 2, 1, D, dtype)
    v[20, 0, 3], v[140, 0, 5], v[130, 0, 7], v[141, 0, 7], v[149, 0, 11] = np.nan, np.inf, -np.inf, np.inf, -np.inf
    got = host(DB.prompt_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), i64(ss), i64(ks), ms, mk, 2, D,
                                   num_kv_heads=1))
    for col, first, seen in ((3, 20, np.isnan), (5, 140, np.isposinf), (11, 149, np.isneginf)):
        assert np.isfinite(got[:first, :, col]).all() and seen(got[first:, :, col]).all()
    assert np.isfinite(got[:130, :, 7]).all() and np.isneginf(got[130:141, :, 7]).all() and np.isnan(got[141:, :, 7]).all()
    rest = np.setdiff1d(np.arange(D), [3, 5, 7, 11])
    assert np.isfinite(got[:, :, rest]).all()


def test_prompt_attention_views_streams_and_graphs(DB):
    rng = np.random.default_rng(9)
    T, Hq, Hkv, D = 200, 8, 2, 128
    rows = dev(values(rng, (T, Hq + 2 * Hkv, D), "bf16"), "bf16")
    q, k, v = rows[:, :Hq], rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:]
    ss = i64([0, 90, 200])
    args = (ss, ss, 110, 110, Hq, D)
    want = DB.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), *args, num_kv_heads=Hkv)
    assert torch.equal(DB.prompt_attention(q, k, v, *args, num_kv_heads=Hkv), want)
    wide = torch.zeros(T, Hkv, D + 1, device="cuda", dtype=torch.bfloat16)
    wide[..., 1:] = k                                          # rows off a 16-byte boundary
    assert torch.equal(DB.prompt_attention(q, wide[..., 1:], v, *args, num_kv_heads=Hkv), want)
    kk, vv = (x.unsqueeze(2).expand(T, Hkv, Hq // Hkv, D).flatten(1, 2) for x in (k, v))
    assert torch.equal(DB.prompt_attention(q, kk, vv, *args), want)          # one key head a query head
    one = k[:, :1].expand(T, Hkv, D)                           # stride zero over the heads
    assert torch.equal(DB.prompt_attention(q, one, one, *args, num_kv_heads=Hkv),
                       DB.prompt_attention(q, one.contiguous(), one.contiguous(), *args, num_kv_heads=Hkv))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = DB.prompt_attention(q, k, v, *args, num_kv_heads=Hkv)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    q2 = q.contiguous()
    with torch.cuda.graph(graph):
        out = DB.prompt_attention(q2, k, v, *args, num_kv_heads=Hkv)
    q2.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, DB.prompt_attention(torch.zeros_like(q), k, v, *args, num_kv_heads=Hkv))
    assert torch.equal(want, DB.prompt_attention(q, k, v, ss.int(), ss.int(), torch.tensor([110]), torch.tensor(110), Hq, D,
                                                 num_kv_heads=Hkv))


def test_prompt_attention_refuses(DB):
    q = torch.zeros(6, 4, 64, device="cuda", dtype=torch.float16)
    k = torch.zeros(6, 2, 64, device="cuda", dtype=torch.float16)
    ss = i64([0, 6])
    ok = dict(query=q, key=k, value=k, seqstarts=ss, kvstarts=ss, max_seqlen=6, max_kvlen=6, num_heads=4, head_dim=64,
              num_kv_heads=2)
    DB.prompt_attention(**ok)
    for change, kind in ((dict(num_heads=8), ValueError), (dict(num_kv_heads=4), ValueError), (dict(num_kv_heads=3), ValueError),
                         (dict(key=k.float()), TypeError), (dict(value=k[:5]), ValueError), (dict(kvstarts=i64([0, 3, 6])), ValueError),
                         (dict(seqstarts=i64([0])), ValueError), (dict(seqstarts=ss.float(), kvstarts=ss), TypeError),
                         (dict(max_seqlen=0), ValueError), (dict(max_kvlen=-1), ValueError), (dict(scale=0.0), ValueError),
                         (dict(scale=float("nan")), ValueError), (dict(logit_cap=-2.0), ValueError),
                         (dict(alibi_slopes=torch.ones(3, device="cuda")), ValueError), (dict(prefix_lens=i64([1, 2])), ValueError),
                         (dict(kvstarts=ss.cpu()), RuntimeError),
                         (dict(query=q.double(), key=k.double(), value=k.double()), TypeError), (dict(query=q.view(24, 64)), ValueError)):
        with pytest.raises(kind):
            DB.prompt_attention(**{**ok, **change})
    assert DB.prompt_attention(**{**ok, "query": q[:0], "seqstarts": i64([0, 0])}).shape == (0, 4, 64)
    assert not DB.prompt_attention(**{**ok, "key": k[:0], "value": k[:0], "kvstarts": i64([0, 0])}).any()
    with pytest.raises(Exception, match="backward|derivative|grad"):
        DB.prompt_attention(**{**ok, "query": q.clone().requires_grad_()}).sum().backward()


def test_index_arrays_that_lead_outside_stay_inside(DB):
    """Starts, positions and lengths beyond the tensors are cut to them (what is computed then is of no use)."""
    q = torch.ones(6, 4, 64, device="cuda", dtype=torch.float16)
    k = torch.ones(6, 2, 64, device="cuda", dtype=torch.float16)
    for s, t in (([0, 60], [0, 60]), ([5, 2], [0, 6]), ([-9, 3], [-7, 900]), ([0, 6], [4, 1])):
        DB.prompt_attention(q, k, k, i64(s), i64(t), 6, 6, 4, 64, num_kv_heads=2)
        DB.prompt_attention(q.float(), k.float(), k.float(), i64(s), i64(t), 6, 6, 4, 64, num_kv_heads=2)
    cache = torch.ones(2, 2, 9, 2, 64, device="cuda", dtype=torch.float16)
    for c, p in ((0, 100), (8, 5), (-4, 3), (50, -1)):
        DB.tree_cache_attention(q, k, k, i64([0, 6]), i64([c]), i64([p]), i64([-1] * 6), 6, 9, cache, 4, 64, num_kv_heads=2,
                                num_layer=2, cache_layout=2)
    torch.cuda.synchronize()


# --------------------------------------------------------------------------------------------- tree attention
def random_masks(rng, lens):
    out = []
    for n in lens:
        seen = []
        for i in range(n):
            parent = int(rng.integers(-1, i)) if i else -1
            seen.append((1 << i) | (seen[parent] if parent >= 0 else 0))
        out += [m - 2 ** 64 if m >> 63 else m for m in seen]
    return np.array(out, dtype=np.int64)


def cache_of(rng, layout, rows, layers, heads, D, dtype):
    shape = {0: (rows, layers, 2, heads, D), 1: (layers, rows, 2, heads, D), 2: (layers, 2, rows, heads, D),
             3: (layers, 2, heads, rows, D)}[layout]
    return values(rng, shape, dtype)


def run_tree(DB, dtype, Hq, Hkv, D, drafted, past, layout=0, cap=0.0, scale=None, masks=None, seed=1, layers=2, layer=1):
    rng = np.random.default_rng(seed + D + layout)
    room = [p + n + 2 for n, p in zip(drafted, past)]
    order = rng.permutation(len(room))
    cs = np.zeros(len(room), np.int64)
    at = 0
    for b in order:                                            # sequences need not be in cache order
        cs[b], at = at, at + room[b]
    cache = cache_of(rng, layout, at, layers, Hkv, D, dtype)
    T = sum(drafted)
    q, k, v = values(rng, (T, Hq, D), dtype), values(rng, (T, Hkv, D), dtype), values(rng, (T, Hkv, D), dtype)
    masks = random_masks(rng, drafted) if masks is None else masks
    ss = starts(drafted)
    tc = dev(cache, dtype)
    got = DB.tree_cache_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), i64(ss), i64(cs), i64(past), i64(masks),
                                  max(drafted), max(p + n for n, p in zip(drafted, past)), tc, Hq, D, num_kv_heads=Hkv,
                                  num_layer=layers, layer_idx=layer, cache_layout=layout, scale=scale, logit_cap=cap)
    ref = ab.tree_attention(q, k, v, cache, layout, layer, ss, cs, past, masks, scale or 1 / math.sqrt(D), cap)
    assert np.array_equal(host(tc), cache), "only the new rows of the layer change, to the new keys and values"
    check_attention(got, ref, dtype, D, max(past) + 64, cap)
    return got


@pytest.mark.parametrize("layout", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype,Hq,Hkv,D,drafted,past", [
    ("bf16", 8, 2, 128, [5, 1, 16, 7], [700, 0, 128, 1]), ("f16", 4, 4, 64, [64, 33, 2], [50, 127, 1000]),
    ("bf16", 6, 2, 96, [8, 8], [256, 255]), ("f16", 32, 4, 128, [64, 40], [300, 3]), ("f32", 4, 2, 64, [4, 9], [33, 0]),
    ("bf16", 2, 1, 40, [3], [5]), ("f16", 2, 1, 100, [3, 5], [40, 7])])
def test_tree_attention(DB, layout, dtype, Hq, Hkv, D, drafted, past):
    run_tree(DB, dtype, Hq, Hkv, D, drafted, past, layout)


@pytest.mark.parametrize("kw", [dict(cap=4.0), dict(scale=0.5), dict(cap=30.0, scale=0.02)])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 48)])
def test_tree_attention_scores(DB, kw, dtype, D):
    run_tree(DB, dtype, 4, 2, D, [6, 20], [300, 17], 3, **kw)


@pytest.mark.parametrize("past", [[0, 0, 0], [0, 200, 0]])
def test_tree_tokens_that_see_nothing_are_zero(DB, past):
    masks = np.array([0, 3, 0, 0, 7, 0, 0, 0, 4], np.int64)   # three tokens a sequence; some see no drafted token
    got = run_tree(DB, "bf16", 4, 1, 128, [3, 3, 3], past, 1, masks=masks)
    assert not got[0].any() and not got[7].any() and got[8].any()


def test_tree_of_one_token_is_a_decode_step(DB):
    rng = np.random.default_rng(4)
    B, Hq, Hkv, D, past = 5, 8, 2, 128, [300, 0, 17, 128, 65]
    cap = 310
    cache = dev(cache_of(rng, 0, B * cap, 1, Hkv, D, "f16"), "f16")
    q, k, v = (dev(values(rng, (B, h, D), "f16"), "f16") for h in (Hq, Hkv, Hkv))
    cs, sp = i64(np.arange(B) * cap), i64(past)
    c2 = cache.clone()
    got = DB.tree_cache_attention(q, k, v, i64(np.arange(B + 1)), cs, sp, i64([1] * B), 1, 301, cache, Hq, D, num_kv_heads=Hkv)
    want = DB.multi_head_cache_attention(q, k, v, i64(np.arange(B + 1)), i64(starts(np.array(past) + 1)), cs, sp,
                                         torch.tensor([B]), torch.tensor([1]), torch.tensor([301]), c2, None, None, Hq, D,
                                         True, False, Hkv)
    assert torch.equal(cache, c2)
    # both round probabilities and result once: four half steps of values that are at most 1 here, and their sums
    assert (got.float() - want.float()).abs().max() <= 4 * UNIT["f16"] * float(want.float().abs().max() + 1)


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dtype,D,n", [("bf16", 128, 6), ("f16", 64, 40), ("f32", 48, 6)])
def test_hidden_rows_of_the_cache_and_of_siblings_do_not_reach_a_token(DB, bad, dtype, D, n):
    rng = np.random.default_rng(8)
    Hq, Hkv, past, rows = 4, 2, 131, 600
    x = torch.finfo(TORCH_DT[dtype]).min if bad == "lowest" else bad
    cache = dev(cache_of(rng, 0, rows, 1, Hkv, D, dtype), dtype)
    q, k, v = (dev(values(rng, (n + 3, h, D), dtype), dtype) for h in (Hq, Hkv, Hkv))
    mask = [1 << i for i in range(n)]                         # every token sees itself alone
    mask[n - 1] |= 1 << 2                                     # the last one also the third
    run = lambda c: DB.tree_cache_attention(q, k, v, i64([0, n]), i64([40]), i64([past]), i64(mask + [0] * 3), n,  # noqa: E731
                                            past + n, c, Hq, D, num_kv_heads=Hkv)
    clean = run(cache.clone())
    cache[:40], cache[40 + past:] = x, x                      # before the sequence's first row, behind its last
    k[2], v[2] = x, x
    k[n:], v[n:], q[n:] = x, x, x                             # rows behind the last sequence
    got = run(cache)
    keep = [i for i in range(n) if i not in (2, n - 1)]
    assert torch.equal(got[keep], clean[keep]) and not got[n:].any()
    if bad != "lowest":
        assert not torch.isfinite(got[2]).any() and not torch.isfinite(got[n - 1]).any()


def test_tree_attention_refuses(DB):
    q = torch.zeros(6, 4, 64, device="cuda", dtype=torch.float16)
    k = torch.zeros(6, 2, 64, device="cuda", dtype=torch.float16)
    cache = torch.zeros(20, 3, 2, 2, 64, device="cuda", dtype=torch.float16)
    ok = dict(query=q, current_key=k, current_value=k, seqstarts=i64([0, 6]), cachestarts=i64([0]), start_pos=i64([4]),
              tree_mask=i64([63] * 6), max_seqlen=6, max_kvlen=10, cache=cache, num_heads=4, head_dim=64, num_kv_heads=2,
              num_layer=3, layer_idx=1)
    from ppl.pmx_b200._cabi import PmxError
    DB.tree_cache_attention(**ok)
    for change, kind in ((dict(max_seqlen=65), PmxError), (dict(tree_mask=i64([1] * 5)), ValueError), (dict(cache_layout=3), ValueError),
                         (dict(cache=cache.float()), TypeError), (dict(layer_idx=3), ValueError), (dict(num_layer=2), ValueError),
                         (dict(cache=cache[..., :32].contiguous()), ValueError), (dict(cache=cache[:, :, :, :1].contiguous()), ValueError),
                         (dict(cache=cache.transpose(0, 1)), ValueError), (dict(cache=cache.cpu()), RuntimeError),
                         (dict(current_key=k[:5]), ValueError), (dict(cachestarts=i64([0, 1])), ValueError)):
        with pytest.raises(kind):
            DB.tree_cache_attention(**{**ok, **change})


# -------------------------------------------------------------------------------------------- cache compaction
@pytest.mark.parametrize("layout", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype,heads,D", [("f16", 2, 128), ("bf16", 1, 36), ("f32", 3, 8), ("f16", 1, 33), ("bf16", 2, 2)])
@pytest.mark.parametrize("most", [3, 12, 30, 64])
def test_compact_cache(DB, layout, dtype, heads, D, most):
    rng = np.random.default_rng(most)
    past, drafted = [9, 0, 30, 4], [most, most, 1, most + 2]
    cs = starts([p + n + 1 for p, n in zip(past, drafted)])
    cache = cache_of(rng, layout, int(cs[-1]), 3, heads, D, dtype)
    picks = [sorted(rng.choice(most, max(1, most // 2), replace=False)), list(rng.permutation(most)), [], [1] * (most - 1) + [-3]]
    a, idx = starts([len(p) for p in picks]), np.concatenate([np.asarray(p, np.int64) for p in picks])
    t = dev(cache, dtype)
    got = DB.compact_cache(t, i64(cs[:-1]), i64(past), i64(a), i64(idx), most, num_layer=3, cache_layout=layout)
    assert got is t
    ab.compact_cache(cache, layout, cs[:-1], past, a, idx)
    assert np.array_equal(host(got), cache)


def test_compact_cache_stays_inside_and_refuses(DB):
    cache = torch.arange(8 * 2 * 2 * 16, device="cuda", dtype=torch.float32).view(8, 2, 2, 1, 16)
    before = cache.clone()
    DB.compact_cache(cache, i64([6]), i64([1]), i64([0, 3]), i64([5, 9, 1 << 40]), 3, num_layer=2)      # all rows outside
    DB.compact_cache(cache, i64([1 << 50]), i64([1]), i64([0, 3]), i64([0, 1, 1]), 3, num_layer=2)
    DB.compact_cache(cache, i64([0]), i64([1]), i64([0, 300]), i64([1, 2, 3]), 3, num_layer=2)           # more than there are
    assert torch.equal(cache, before)
    assert DB.compact_cache(cache, i64([0]), i64([1]), i64([0, 0]), i64([]), 3, num_layer=2) is cache
    for args, kind in (((cache, i64([0, 1]), i64([1]), i64([0, 1]), i64([1]), 1, 2), ValueError),
                       ((cache, i64([0]), i64([1]), i64([0]), i64([1]), 1, 2), ValueError),
                       ((cache, i64([0]), i64([1]), i64([0, 1]), i64([1]), 65, 2), ValueError),
                       ((cache, i64([0]), i64([1]), i64([0, 1]), i64([1]), 0, 2), ValueError),
                       ((cache, i64([0]), i64([1]), i64([0, 1]), i64([1]), 1, 3), ValueError),
                       ((cache[:, :1], i64([0]), i64([1]), i64([0, 1]), i64([1]), 1, 1), ValueError),
                       ((cache.double(), i64([0]), i64([1]), i64([0, 1]), i64([1]), 1, 2), TypeError),
                       ((cache, i64([0]), i64([1]), i64([0, 1]), i64([1]).float(), 1, 2), TypeError)):
        with pytest.raises(kind):
            DB.compact_cache(*args)


# ------------------------------------------------------------------------------------------------ all together
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompt_then_a_speculative_step_equals_the_long_prompt(DB, dtype):
    """A prompt, then a drafted tree of which one path is accepted, then a decode step: every accepted token's
    result is what one prompt over the whole text gives, and so is the cache."""
    rng = np.random.default_rng(2)
    Hq, Hkv, D, B = 8, 2, 128, 2
    L, n = [150, 40], [7, 4]
    path = [[0, 2, 5], [0, 3]]                                # accepted drafted tokens of each sequence
    parents = [[-1, 0, 0, 1, 2, 2, 5], [-1, 0, 0, 0]]
    wq, wk = (torch.ones(D, device="cuda", dtype=TORCH_DT[dtype]) for _ in range(2))
    prompt = [dev(values(rng, (l, Hq + 2 * Hkv, D), dtype), dtype) for l in L]
    draft = [dev(values(rng, (m, Hq + 2 * Hkv, D), dtype), dtype) for m in n]
    last = [dev(values(rng, (1, Hq + 2 * Hkv, D), dtype), dtype) for _ in range(B)]
    rot = lambda x, ss, sp, ids=None: DB.qk_norm_rotary_embedding(x[:, :Hq], x[:, Hq:Hq + Hkv], wq, wk, 1e-6, ss, sp, ids)  # noqa: E731
    # all at once
    text = [torch.cat([p, d[pa], la]) for p, d, pa, la in zip(prompt, draft, path, last)]
    ss = i64(starts([len(t) for t in text]))
    rows = torch.cat(text)
    q, k = rot(rows, ss, i64([0] * B))
    want = DB.prompt_attention(q, k, rows[:, Hq + Hkv:], ss, ss, 200, 200, Hq, D, num_kv_heads=Hkv)
    # step by step
    cap = 200
    cache = torch.zeros(B * cap, 1, 2, Hkv, D, device="cuda", dtype=TORCH_DT[dtype])
    cs = i64(np.arange(B) * cap)
    rows, s0 = torch.cat(prompt), i64(starts(L))
    q, k = rot(rows, s0, i64([0] * B))
    first = DB.prompt_attention(q, k, rows[:, Hq + Hkv:], s0, s0, max(L), max(L), Hq, D, num_kv_heads=Hkv)
    for b in range(B):
        cache[b * cap:b * cap + L[b], 0, 0], cache[b * cap:b * cap + L[b], 0, 1] = k[s0[b]:s0[b + 1]], rows[s0[b]:s0[b + 1], Hq + Hkv:]
    masks, depth = [], []
    for ps in parents:
        seen, deep = [], []
        for i, p in enumerate(ps):
            seen.append((1 << i) | (seen[p] if p >= 0 else 0))
            deep.append(deep[p] + 1 if p >= 0 else 0)
        masks += seen
        depth.append(deep)
    rows, s1 = torch.cat(draft), i64(starts(n))
    ids = i64([L[b] + d for b in range(B) for d in depth[b]])
    q, k = rot(rows, None, None, ids)
    second = DB.tree_cache_attention(q, k, rows[:, Hq + Hkv:], s1, cs, i64(L), i64(masks), max(n), max(L) + max(n), cache, Hq, D,
                                     num_kv_heads=Hkv)
    DB.compact_cache(cache, cs, i64(L), i64(starts([len(p) for p in path])), i64(sum(path, [])), 3)
    past = [l + len(p) for l, p in zip(L, path)]
    rows = torch.cat(last)
    q, k = rot(rows, i64([0, 1, 2]), i64(past))
    third = DB.multi_head_cache_attention(q, k, rows[:, Hq + Hkv:], i64([0, 1, 2]), i64(starts([p + 1 for p in past])), cs,
                                          i64(past), torch.tensor([B]), torch.tensor([1]), torch.tensor([max(past) + 1]),
                                          cache, None, None, Hq, D, True, False, Hkv)
    got = torch.cat([torch.cat([first[s0[b]:s0[b + 1]], second[s1[b]:s1[b + 1]][path[b]], third[b:b + 1]]) for b in range(B)])
    # two results of the same sums, each with its probabilities and its result rounded once (values up to ~4)
    assert (got.float() - want.float()).abs().max() <= 4 * UNIT[dtype] * float(want.float().abs().max())


def test_calls_that_need_converting_give_the_same_as_regular_ones(DB):
    """Regular calls take a short way through the host (host_calls.cpp); index arrays of 32 bits, lengths as tensors,
    strided arrays and parameters take the general one."""
    rng = np.random.default_rng(12)
    T, Hq, Hkv, D = 40, 4, 2, 64
    x = dev(values(rng, (T, Hq + 2 * Hkv, D), "bf16"), "bf16")
    q, k, v, w = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], torch.ones(D, device="cuda", dtype=torch.bfloat16)
    ss, sp = i64([0, 15, 40]), i64([3, 0])
    wide = torch.stack([ss, ss], 1)[:, 0]                       # the same values with a stride
    one = lambda n: torch.tensor([n])                           # noqa: E731
    eq = lambda a, b: all(torch.equal(m, n) for m, n in zip(a, b))  # noqa: E731
    want = DB.rotary_position_embedding(q, k, ss, sp)
    assert eq(DB.rotary_position_embedding(q, k, ss.int(), sp), want) and eq(DB.rotary_position_embedding(q, k, wide, sp.int()), want)
    want = DB.qk_norm_rotary_embedding(q, k, w, w, 1e-6, ss, sp)
    assert eq(DB.qk_norm_rotary_embedding(q, k, torch.nn.Parameter(w, False), w, 1e-6, ss, sp.int()), want)
    args = dict(num_kv_heads=Hkv, logit_cap=20.0, prefix_lens=i64([4, 9]), alibi_slopes=torch.full((Hq,), 0.25, device="cuda"))
    want = DB.prompt_attention(q, k, v, ss, ss, 25, 25, Hq, D, **args)
    assert torch.equal(DB.prompt_attention(q, k, v, wide, ss.int(), one(25), one(25), Hq, D, **args), want)
    assert torch.equal(DB.prompt_attention(q, k, v, ss, ss, 25, 25, Hq, D, **{**args, "alibi_slopes": args["alibi_slopes"].double()}), want)
    caches = [dev(cache_of(np.random.default_rng(3), 1, 90, 2, Hkv, D, "bf16"), "bf16") for _ in range(2)]
    mask = i64([-1] * T)
    outs = [DB.tree_cache_attention(q, k, v, s, i64([0, 40]), sp, mask, m, n, c, Hq, D, num_kv_heads=Hkv, num_layer=2, layer_idx=1,
                                    cache_layout=1) for c, s, m, n in zip(caches, (ss, ss.int()), (25, one(25)), (40, one(40)))]
    assert eq(outs, outs[::-1]) and torch.equal(*caches)
    for c, s, m in zip(caches, (i64([0, 2, 5]), i64([0, 2, 5]).int()), (3, one(3))):
        DB.compact_cache(c, i64([0, 40]), sp, s, i64([1, 4, 3, 0, 24]), m, num_layer=2, cache_layout=1)
    assert torch.equal(*caches)
    with torch.no_grad():                                       # a gradient that nobody asks for
        assert eq(DB.rotary_position_embedding(q.clone().requires_grad_(), k, ss, sp), DB.rotary_position_embedding(q, k, ss, sp))
    with pytest.raises(Exception, match="backward|derivative|grad"):
        DB.rotary_position_embedding(q.clone().requires_grad_(), k, ss, sp)[0].sum().backward()


def test_graphs_and_streams_side_by_side(DB):
    """Two captured calls with workspaces of their own, replayed in turn with other inputs, and eager calls on two streams."""
    rng = np.random.default_rng(31)
    Hq, Hkv, D = 8, 2, 128
    q = [dev(values(rng, (4, Hq, D), "bf16"), "bf16") for _ in range(4)]
    k = dev(values(rng, (3000, Hkv, D), "bf16"), "bf16")
    call = lambda x, keys: DB.prompt_attention(x, k[:keys], k[:keys], i64([0, 4]), i64([0, keys]), 4, keys, Hq, D,  # noqa: E731
                                               num_kv_heads=Hkv)
    want = [[call(x, keys) for keys in (3000, 1700)] for x in q]
    ss, ends, static = i64([0, 4]), {n: i64([0, n]) for n in (3000, 1700)}, q[0].clone()
    graphs, outs = [], []
    for keys in (3000, 1700):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(DB.prompt_attention(static, k[:keys], k[:keys], ss, ends[keys], 4, keys, Hq, D, num_kv_heads=Hkv))
        graphs.append(graph)
    for i, x in enumerate(q):
        static.copy_(x)
        for g in ((0, 1), (1, 0))[i % 2]:
            graphs[g].replay()
            assert torch.equal(outs[g], want[i][g])
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for n, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[n].append(call(q[n], 3000))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[n][0]) for n in range(2) for x in got[n])


def test_tree_attention_drops_what_is_behind_max_seqlen_and_outside_the_cache(DB):
    """Rows of a sequence behind its first max_seqlen are zero and not stored; rows beyond the cache's end are not stored."""
    rng = np.random.default_rng(32)
    Hq, Hkv, D, rows = 4, 2, 64, 40
    cache_np = values(rng, (rows, 1, 2, Hkv, D), "f16")
    q, k, v = (values(rng, (12, h, D), "f16") for h in (Hq, Hkv, Hkv))
    masks = np.array([(1 << (i % 6 + 1)) - 1 for i in range(12)], dtype=np.int64)
    cache = dev(cache_np, "f16")
    got = DB.tree_cache_attention(dev(q, "f16"), dev(k, "f16"), dev(v, "f16"), i64([0, 6, 12]), i64([0, 20]), i64([5, 18]),
                                  i64(masks), 4, 30, cache, Hq, D, num_kv_heads=Hkv)
    keep = np.array([0, 1, 2, 3, 6, 7, 8, 9])
    want = cache_np.copy()
    ref = ab.tree_attention(q[keep], k[keep], v[keep], want, 0, 0, [0, 4, 8], [0, 20], [5, 18], masks[keep], 1 / 8.0)
    check_attention(got[torch.from_numpy(keep).cuda()], ref, "f16", D, 30, 0.0)
    assert not got[torch.tensor([4, 5, 10, 11], device="cuda")].any()
    assert np.array_equal(host(cache), want)
