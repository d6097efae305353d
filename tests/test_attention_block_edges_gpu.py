"""The attention block's operators on the GPU where they are easiest to get wrong."""
import numpy as np
import pytest
import torch

from tests.helpers import dev
from tests.test_attention_block_gpu import DB, cache_of, i64, no_wait_ran_out, prompt_case, values  # noqa: F401

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
