"""The operators of a decoder's attention block for prompts and for drafted tokens, as measured work.

`listed()` and `draw()` give the cases, `prepare()` their inputs, `run()` one pass (the plain torch form, or the
framework's operators where `own` is true), `exact()` the results in 64 bits, `work()` the bytes and operations
that a pass cannot do without.  Head counts are those of a 32 / 8 head decoder and its tensor-parallel shards.
"""
import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 sequences on a tensor-parallel rank: latency
        rotary("rotary_decode", "bf16", 64, 1, 8, 2, 128, 128, 1000, spread=1),
        # ragged prompts, interleaved pairs on part of the head, far positions under linear scaling
        rotary("rotary_prompt_part", "f16", 7, 2048, 32, 8, 128, 64, 200000, interleaved=True, scaling="linear", spread=2),
        # decode step: norms of the heads and the rotation, read out of the fused projection's rows
        qk_norm("qk_norm_decode", "bf16", 256, 1, 32, 8, 128, 128, 4000, spread=3),
        # long prompts through the same
        qk_norm("qk_norm_prompt", "bf16", 4, 6000, 32, 8, 128, 128, 0, scaling="yarn", spread=4),
        # a few short prompts on a shard: latency
        prompt("prompt_short", "bf16", 4, 61, 61, 8, 2, 128, spread=5),
        # ragged prompts, capped scores, an image or instruction prefix that sees itself whole
        prompt("prompt_ragged_cap_prefix", "f16", 8, 1501, 1501, 16, 8, 64, cap=30.0, prefix=200, spread=6),
        # a chunk of each prompt against what is there already, distance bias
        prompt("prompt_chunk_alibi", "bf16", 2, 512, 6000, 32, 8, 128, alibi=True, spread=7),
        # one long prompt
        prompt("prompt_long", "bf16", 1, 8192, 8192, 32, 8, 128, spread=8),
        # a handful of drafted tokens of two users on a shard: latency
        tree("tree_small", "f16", 2, 8, 700, 8, 2, 128, 2, 0, spread=9),
        # a full serving batch with drafted trees
        tree("tree_batch", "bf16", 32, 16, 4096, 32, 8, 128, 2, 3, spread=10),
        # after verification: accepted rows of a few sequences, and of a full batch
        compact("compact_small", "bf16", 4, 8, 500, 2, 128, 4, 0, spread=11),
        compact("compact_batch", "f16", 32, 32, 300, 8, 128, 32, 3, spread=12),
    ]


def rotary(name, dtype, batch, seqlen, heads, kv_heads, dim, rotary_dim, past, interleaved=False, scaling="", spread=0):
    return dict(name=name, op="rotary", dtype=dtype, batch=batch, seqlen=seqlen, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary_dim=rotary_dim, past=past, interleaved=interleaved, scaling=scaling, spread=spread)


def qk_norm(name, *a, **k):
    return dict(rotary(name, *a, **k), op="qk_norm")


def prompt(name, dtype, batch, seqlen, kvlen, heads, kv_heads, dim, causal=True, cap=0.0, prefix=0, alibi=False, spread=0):
    return dict(name=name, op="prompt", dtype=dtype, batch=batch, seqlen=seqlen, kvlen=kvlen, heads=heads,
                kv_heads=kv_heads, dim=dim, causal=causal, cap=cap, prefix=prefix, alibi=alibi, spread=spread)


def tree(name, dtype, batch, drafted, past, heads, kv_heads, dim, layers, layout, cap=0.0, spread=0):
    return dict(name=name, op="tree", dtype=dtype, batch=batch, drafted=drafted, past=past, heads=heads,
                kv_heads=kv_heads, dim=dim, layers=layers, layout=layout, cap=cap, spread=spread)


def compact(name, dtype, batch, drafted, past, kv_heads, dim, layers, layout, spread=0):
    return dict(name=name, op="compact", dtype=dtype, batch=batch, drafted=drafted, past=past, kv_heads=kv_heads,
                dim=dim, layers=layers, layout=layout, spread=spread)


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "prompt", "prompt", "tree", "tree", "compact"])
    dtype = rng.choice(["bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    dim = rng.choice([64, 64, 96, 128, 128, 128])
    spread = rng.randrange(1 << 30)
    if op in ("rotary", "qk_norm"):
        if rng.random() < 0.2:
            dtype = "f32"
        part = rng.choice([dim, dim, dim // 2])
        batch = log_int(rng, 1, 64)
        seqlen = log_int(rng, 1, 16384 // batch)
        make = rotary if op == "rotary" else qk_norm
        c = make("", dtype, batch, seqlen, heads, kv_heads, dim, part, log_int(rng, 1, 400000),
                 interleaved=rng.random() < 0.4, scaling=rng.choice(["", "linear", "ntk", "yarn"]), spread=spread)
    elif op == "prompt":
        kvlen = log_int(rng, 1, 6000)
        seqlen = kvlen if rng.random() < 0.6 else log_int(rng, 1, kvlen)
        room = (8192 * 8192 * 32) // (heads * seqlen * kvlen + 1) // 2
        batch = log_int(rng, 1, max(1, min(16, room, 24576 // kvlen)))
        c = prompt("", dtype, batch, seqlen, kvlen, heads, kv_heads, dim, causal=rng.random() < 0.85,
                   cap=rng.choice([0.0, 0.0, 20.0, 50.0]), prefix=rng.choice([0, 0, log_int(rng, 1, kvlen)]),
                   alibi=rng.random() < 0.3, spread=spread)
    elif op == "tree":
        past = log_int(rng, 1, 16384)
        batch = log_int(rng, 1, max(1, min(48, 120000 // (past + 64))))
        c = tree("", dtype, batch, log_int(rng, 1, 64), past, heads, kv_heads, dim, rng.choice([1, 2]),
                 rng.randrange(4), cap=rng.choice([0.0, 0.0, 30.0]), spread=spread)
    else:
        batch = log_int(rng, 1, 48)
        c = compact("", dtype, batch, log_int(rng, 1, 32), log_int(rng, 1, 1000), kv_heads, dim, log_int(rng, 1, 16),
                    rng.randrange(4), spread=spread)
    del c["name"]
    return c


def lengths(case):
    """Per sequence: (new tokens, tokens before them or keys in all).  The first sequence has the case's full lengths,
    the others are ragged."""
    rng = random.Random(case["spread"])
    op, out = case["op"], []
    for b in range(case["batch"]):
        part = 1.0 if b == 0 else rng.uniform(0.4, 1.0)
        if op in ("rotary", "qk_norm"):
            n, past = max(1, round(case["seqlen"] * part)), rng.randint(0, case["past"])
        elif op == "prompt":
            past = max(1, round(case["kvlen"] * part))
            n = min(past, max(1, round(case["seqlen"] * (part if case["seqlen"] == case["kvlen"] else 1.0))))
        else:
            n, past = max(1, round(case["drafted"] * part)), round(case["past"] * part)
        out.append((n, past))
    return out


def accepted(case):
    """compact: which of the drafted rows of each sequence are accepted (about half, as verification leaves)."""
    rng = random.Random(case["spread"] + 1)
    return [sorted(rng.sample(range(n), max(1, min(n, round(n * rng.uniform(0.3, 0.7)))))) for n, _ in lengths(case)]


def work(case):
    e, lens = SIZE[case["dtype"]], lengths(case)
    new, dim = sum(n for n, _ in lens), case["dim"]
    if case["op"] in ("rotary", "qk_norm"):
        values = new * (case["heads"] + case["kv_heads"]) * dim
        return {"bytes": 2 * values * e + 8 * 2 * len(lens), "flops": values * (10 if case["op"] == "qk_norm" else 6)}
    if case["op"] == "prompt":
        pairs = 0
        for n, kv in lens:
            if not case["causal"]:
                pairs += n * kv
                continue
            pre, first = min(case["prefix"], kv), kv - n + 1      # row i sees max(first + i, pre) keys
            low = min(n, max(0, pre - first))
            pairs += low * pre + sum((first + low, first + n - 1)) * (n - low) // 2
        keys = sum(kv for _, kv in lens)
        return {"bytes": e * dim * (2 * new * case["heads"] + 2 * keys * case["kv_heads"]),
                "flops": 4 * dim * case["heads"] * pairs}
    if case["op"] == "tree":
        keys = sum(past for _, past in lens)
        return {"bytes": e * dim * (2 * new * case["heads"] + (2 * keys + 4 * new) * case["kv_heads"]) + 8 * new,
                "flops": 4 * dim * case["heads"] * sum(n * (past + n / 2) for n, past in lens)}
    moved = sum(i != j for picks in accepted(case) for i, j in enumerate(picks))
    return {"bytes": 2 * moved * case["layers"] * 2 * case["kv_heads"] * dim * e + 8 * sum(map(len, accepted(case))),
            "flops": 0}


# ----------------------------------------------------------------------------------------------- inputs
def starts(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return torch.tensor(out, dtype=torch.int64, device="cuda")


def ints(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def cache_shape(case, rows):
    layers, heads, dim = case["layers"], case["kv_heads"], case["dim"]
    return [(rows, layers, 2, heads, dim), (layers, rows, 2, heads, dim), (layers, 2, rows, heads, dim),
            (layers, 2, heads, rows, dim)][case["layout"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dt, lens = DT[case["dtype"]], lengths(case)
    new, dim = sum(n for n, _ in lens), case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if case["dtype"] == "f32" else dt)

    s = dict(case=case, seqstarts=starts([n for n, _ in lens]), max_seqlen=max(n for n, _ in lens))
    if case["op"] in ("rotary", "qk_norm"):
        heads, kv = case["heads"], case["kv_heads"]
        rows = normal(new, heads + 2 * kv, dim)                       # the fused projection's output
        s.update(q=rows[:, :heads], k=rows[:, heads:heads + kv], start_pos=ints([past for _, past in lens]))
        if case["op"] == "qk_norm":
            s.update(q_weight=(1 + 0.2 * normal(dim).float()).to(dt), k_weight=(1 + 0.2 * normal(dim).float()).to(dt))
        return s
    if case["op"] == "prompt":
        keys = sum(kv for _, kv in lens)
        s.update(q=normal(new, case["heads"], dim), k=normal(keys, case["kv_heads"], dim),
                 v=normal(keys, case["kv_heads"], dim), kvstarts=starts([kv for _, kv in lens]),
                 max_kvlen=max(kv for _, kv in lens), prefix=None, slopes=None)
        if case["prefix"]:
            s["prefix"] = ints([min(case["prefix"], kv) for _, kv in lens])
        if case["alibi"]:
            h = case["heads"]
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
        return s
    room = [past + n + 3 for n, past in lens]
    cachestarts, at = [], 0
    for r in room:
        cachestarts.append(at)
        at += r
    s.update(cache=normal(*cache_shape(case, at)), cachestarts=ints(cachestarts), start_pos=ints([p for _, p in lens]))
    if case["op"] == "compact":
        picks = accepted(case)
        s.update(accept_starts=starts([len(p) for p in picks]), accept_index=ints([i for p in picks for i in p]),
                 max_accept=max(map(len, picks)))
        return s
    mask = []
    for n, _ in lens:
        seen = []
        for i in range(n):                                            # a tree: every token sees itself and its ancestors
            parent = rng.randint(-1, i - 1) if rng.random() < 0.3 else i - 1
            seen.append((1 << i) | (seen[parent] if parent >= 0 else 0))
        mask += [m - (1 << 64) if m >> 63 else m for m in seen]
    s.update(q=normal(new, case["heads"], dim), k=normal(new, case["kv_heads"], dim), v=normal(new, case["kv_heads"], dim),
             tree_mask=ints(mask), max_kvlen=max(past + n for n, past in lens))
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotary": own_rotary, "qk_norm": own_qk_norm, "prompt": own_prompt, "tree": own_tree,
                "compact": own_compact}[op](s)
    return {"rotary": plain_rotary, "qk_norm": plain_rotary, "prompt": plain_prompt, "tree": plain_tree,
            "compact": plain_compact}[op](s)


def scaling_args(c):
    if not c["scaling"]:
        return {}
    return dict(scaling_type=c["scaling"], scaling_factor=8.0, original_max_position=8192)


def own_rotary(s):
    from ppl.pmx_b200.torch_function import dynamic_batching as DB
    c = s["case"]
    return DB.rotary_position_embedding(s["q"], s["k"], s["seqstarts"], s["start_pos"], rotary_dim=c["rotary_dim"],
                                        theta=1e6, interleaved=c["interleaved"], **scaling_args(c))


def own_qk_norm(s):
    from ppl.pmx_b200.torch_function import dynamic_batching as DB
    c = s["case"]
    return DB.qk_norm_rotary_embedding(s["q"], s["k"], s["q_weight"], s["k_weight"], 1e-6, s["seqstarts"],
                                       s["start_pos"], rotary_dim=c["rotary_dim"], theta=1e6,
                                       interleaved=c["interleaved"], **scaling_args(c))


def own_prompt(s):
    from ppl.pmx_b200.torch_function import dynamic_batching as DB
    c = s["case"]
    return DB.prompt_attention(s["q"], s["k"], s["v"], s["seqstarts"], s["kvstarts"], s["max_seqlen"], s["max_kvlen"],
                               c["heads"], c["dim"], is_causal=c["causal"], num_kv_heads=c["kv_heads"],
                               logit_cap=c["cap"], alibi_slopes=s["slopes"], prefix_lens=s["prefix"])


def own_tree(s):
    from ppl.pmx_b200.torch_function import dynamic_batching as DB
    c = s["case"]
    out = DB.tree_cache_attention(s["q"], s["k"], s["v"], s["seqstarts"], s["cachestarts"], s["start_pos"],
                                  s["tree_mask"], s["max_seqlen"], s["max_kvlen"], s["cache"], c["heads"], c["dim"],
                                  num_kv_heads=c["kv_heads"], num_layer=c["layers"], layer_idx=c["layers"] - 1,
                                  cache_layout=c["layout"], logit_cap=c["cap"])
    return [out, s["cache"]]


def own_compact(s):
    from ppl.pmx_b200.torch_function import dynamic_batching as DB
    c = s["case"]
    return DB.compact_cache(s["cache"], s["cachestarts"], s["start_pos"], s["accept_starts"], s["accept_index"],
                            s["max_accept"], num_layer=c["layers"], cache_layout=c["layout"])


# plain forms: elementary torch operations in 32 bits, sequences padded to the longest
def frequencies(c):
    """Angle per position of each rotated pair in 64 bits, and the factor on cosine and sine."""
    r, theta = c["rotary_dim"], 1e6
    i = torch.arange(0, r, 2, dtype=torch.float64, device="cuda")
    f = theta ** (-i / r)
    if c["scaling"] == "linear":
        return f / 8.0, 1.0
    if c["scaling"] == "ntk":
        return (theta * 8.0 ** (r / (r - 2))) ** (-i / r), 1.0
    if c["scaling"] == "yarn":
        keep = ((8192 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * (keep + (1 - keep) / 8.0), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def owner(seqstarts, total):
    """The sequence of each packed token, and its place in it."""
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(seqstarts, t, right=True) - 1
    return b, t - seqstarts[b]


def plain_rotary(s):
    c, r = s["case"], s["case"]["rotary_dim"]
    b, i = owner(s["seqstarts"], s["q"].shape[0])
    f, factor = frequencies(c)
    angle = (s["start_pos"][b] + i).double()[:, None, None] * f
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()

    def one(x, weight):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
        z = y.clone()
        if c["interleaved"]:
            z[..., 0:r:2] = y[..., 0:r:2] * cos - y[..., 1:r:2] * sin
            z[..., 1:r:2] = y[..., 1:r:2] * cos + y[..., 0:r:2] * sin
        else:
            h = r // 2
            z[..., :h] = y[..., :h] * cos - y[..., h:r] * sin
            z[..., h:r] = y[..., h:r] * cos + y[..., :h] * sin
        return z.to(x.dtype)

    return [one(s["q"], s.get("q_weight")), one(s["k"], s.get("k_weight"))]


def padded(x, first, longest):
    """[sequences, longest, heads, dim] in 32 bits of packed rows that begin at `first`."""
    at = (first[:, None] + torch.arange(longest, device="cuda")).clamp(max=x.shape[0] - 1)
    return x[at].float()


def attend(q, k, v, seen, cap, bias):
    """q [B, S, Hq, D], k and v [B, L, Hkv, D], seen [B, S, L]; bias [B, Hq, S, L] or None."""
    B, S, heads, D = q.shape
    L, kv = k.shape[1], k.shape[2]
    q = q.view(B, S, kv, heads // kv, D).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, D)
    score = (q @ k.permute(0, 2, 3, 1)).view(B, heads, S, L) * (1.0 / math.sqrt(D))
    if cap:
        score = cap * torch.tanh(score / cap)
    if bias is not None:
        score = score + bias
    score = score.masked_fill(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1)
    out = (p.view(B, kv, -1, L) @ v.permute(0, 2, 1, 3)).view(B, heads, S, D)
    out = out / torch.where(total == 0, 1.0, total)[..., None]
    return out.permute(0, 2, 1, 3)                                      # [B, S, Hq, D]


def plain_prompt(s):
    c = s["case"]
    S, L = s["max_seqlen"], s["max_kvlen"]
    q = padded(s["q"], s["seqstarts"][:-1], S)
    k, v = (padded(s[x], s["kvstarts"][:-1], L) for x in "kv")
    n, kv = s["seqstarts"].diff(), s["kvstarts"].diff()
    at = torch.arange(S, device="cuda") + (kv - n)[:, None]              # [B, S]: the query's place among the keys
    j = torch.arange(L, device="cuda")
    seen = (j < kv[:, None])[:, None].expand(-1, S, -1)
    if c["causal"]:
        limit = at + 1
        if s["prefix"] is not None:
            limit = torch.maximum(limit, s["prefix"][:, None])
        seen = seen & (j < limit[..., None])
    bias = None
    if s["slopes"] is not None:
        bias = -s["slopes"][:, None, None] * (at[:, None, :, None] - j).abs().float()
    out = attend(q, k, v, seen, c["cap"], bias)
    b, i = owner(s["seqstarts"], s["q"].shape[0])
    return out[b, i].to(s["q"].dtype)


def rows_first(case, cache):
    """The cache as a view [rows, layers, 2, heads, dim], whatever its layout."""
    return cache.permute([(0, 1, 2, 3, 4), (1, 0, 2, 3, 4), (2, 0, 1, 3, 4), (3, 0, 1, 2, 4)][case["layout"]])


def plain_tree(s):
    c = s["case"]
    cache = rows_first(c, s["cache"])[:, c["layers"] - 1]                # [rows, 2, heads, dim]
    b, i = owner(s["seqstarts"], s["q"].shape[0])
    cache[s["cachestarts"][b] + s["start_pos"][b] + i] = torch.stack([s["k"], s["v"]], 1)
    S, L = s["max_seqlen"], s["max_kvlen"]
    q = padded(s["q"], s["seqstarts"][:-1], S)
    kv = (s["cachestarts"][:, None] + torch.arange(L, device="cuda")).clamp(max=cache.shape[0] - 1)
    k, v = cache[:, 0][kv].float(), cache[:, 1][kv].float()
    past, j = s["start_pos"][:, None], torch.arange(L, device="cuda")
    mask = s["tree_mask"][(s["seqstarts"][:-1, None] + torch.arange(S, device="cuda")).clamp(max=s["q"].shape[0] - 1)]
    bit = (j - past).clamp(0, 63)                                        # [B, L]
    drafted = (mask[..., None] >> bit[:, None]) & 1                      # [B, S, L]
    within = (j >= past) & (j < past + s["seqstarts"].diff()[:, None])
    seen = (j < past)[:, None] | (within[:, None] & (drafted == 1))
    out = attend(q, k, v, seen, c["cap"], None)
    return [out[b, i].to(s["q"].dtype), s["cache"]]


def plain_compact(s):
    cache = rows_first(s["case"], s["cache"])
    b, i = owner(s["accept_starts"], s["accept_index"].shape[0])
    base = s["cachestarts"][b] + s["start_pos"][b]
    cache[base + i] = cache[base + s["accept_index"]]
    return s["cache"]


# ---------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s, lens = prepare(case, seed), lengths(case)
    if case["op"] in ("rotary", "qk_norm"):
        return exact_rotary(case, s, lens)
    if case["op"] == "prompt":
        return exact_prompt(case, s, lens)
    first = s["cachestarts"].tolist()
    if case["op"] == "compact":
        rows = rows_first(case, s["cache"])
        for (_, past), picks, f in zip(lens, accepted(case), first):
            rows[f + past:f + past + len(picks)] = rows[[f + past + p for p in picks]].clone()
        return s["cache"]
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    layer = rows_first(case, s["cache"])[:, case["layers"] - 1]
    masks = s["tree_mask"].tolist()
    for (n, past), f in zip(lens, first):
        layer[f + past:f + past + n, 0], layer[f + past:f + past + n, 1] = s["k"][at:at + n], s["v"][at:at + n]
        seen = torch.ones(n, past + n, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                seen[i, past + j] = bool(masks[at + i] >> j & 1)
        kv = layer[f:f + past + n].double()
        out[at:at + n] = exact_heads(s["q"][at:at + n].double(), kv[:, 0], kv[:, 1], seen.cuda(), case["cap"], None, None)
        at += n
    return [out, s["cache"]]


def exact_rotary(case, s, lens):
    r, theta = case["rotary_dim"], 1e6
    if case["scaling"] == "ntk":
        theta *= 8.0 ** (r / (r - 2.0))
    freq = [theta ** (-2.0 * i / r) for i in range(r // 2)]
    if case["scaling"] == "linear":
        freq = [f / 8.0 for f in freq]
    factor = 1.0
    if case["scaling"] == "yarn":
        ramp = [min(1.0, max(0.0, (8192.0 * f / (2.0 * math.pi) - 1.0) / 31.0)) for f in freq]
        freq = [f * g + f / 8.0 * (1.0 - g) for f, g in zip(freq, ramp)]
        factor = 1.0 + 0.1 * math.log(8.0)
    pos = torch.cat([torch.arange(past, past + n, dtype=torch.float64, device="cuda") for n, past in lens])
    turn = torch.polar(torch.full((len(pos), r // 2), factor, dtype=torch.float64, device="cuda"),
                       pos[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda"))[:, None]
    outs = []
    for x, w in ((s["q"], s.get("q_weight")), (s["k"], s.get("k_weight"))):
        y = x.double()
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        part = y[..., :r]
        pairs = part.unflatten(-1, (r // 2, 2)) if case["interleaved"] else part.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        outs.append(torch.cat([z, y[..., r:]], -1))
    return outs


def exact_prompt(case, s, lens):
    out, at, at_kv = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0, 0
    for n, kv in lens:
        row = torch.arange(kv - n, kv, device="cuda")[:, None]
        col = torch.arange(kv, device="cuda")[None]
        seen = torch.ones(n, kv, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = (col <= row) | (col < min(case["prefix"], kv))
        slopes = s["slopes"].double() if s["slopes"] is not None else None
        out[at:at + n] = exact_heads(s["q"][at:at + n].double(), s["k"][at_kv:at_kv + kv].double(),
                                     s["v"][at_kv:at_kv + kv].double(), seen, case["cap"], slopes, (row - col).abs())
        at, at_kv = at + n, at_kv + kv
    return out


def exact_heads(q, k, v, seen, cap, slopes, far):
    """One sequence, a head at a time: q [n, Hq, D], k and v [kv, Hkv, D], seen [n, kv]."""
    out, group = torch.empty_like(q), q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        score = q[:, h] @ k[:, h // group].T / math.sqrt(q.shape[2])
        if cap:
            score = torch.tanh(score / cap) * cap
        if slopes is not None:
            score = score - slopes[h] * far
        score[~seen] = -math.inf
        out[:, h] = torch.nan_to_num(torch.softmax(score, -1)) @ v[:, h // group]
    return out
