"""Cases of the operators for packed rows: several sequences of different lengths that share one row axis.

    sdpa_packed           attention of a step's rows to a paged cache and to each other: whole prompts
                          (causal), single tokens, and trees of drafted tokens
    rope_packed           rotary position encoding, each row at a position of its own
    cache_append_packed   chosen rows of a step's keys and values written behind their sequences' pages
    token_logprobs        log probabilities of given tokens, the entropy and the most likely tokens

`run` takes what `prepare` made: tensors in the tiled layout of the framework (16 x 16 tiles, planes
padded to whole tiles).  Where `own` is false it computes them in elementary torch operations, where it
is true it calls the framework.  Sizes are those of TinyLlama (32 query and 4 KV heads of 64 features,
a vocabulary of 32000), of the 32 / 8 / 128 heads and larger vocabularies that are common beside it,
and generic ones.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TILE = 16


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a decode step of sixteen chats of a small model, contexts of a few hundred tokens: latency
        dict(name="token_short", op="sdpa", type="bf16", seqs=16, rows_lo=1, rows_hi=1, ctx_lo=1, ctx_hi=509,
             q_heads=32, kv_heads=4, features=64, page=32, tree=False, tail=0),
        # a decode step of a loaded server: long ragged contexts, bound by reading the cache
        dict(name="token_long", op="sdpa", type="f16", seqs=32, rows_lo=1, rows_hi=1, ctx_lo=700, ctx_hi=15001,
             q_heads=32, kv_heads=8, features=128, page=64, tree=False, tail=0),
        # the verification of drafted trees, eight chats at once
        dict(name="tree_verify", op="sdpa", type="bf16", seqs=8, rows_lo=17, rows_hi=61, ctx_lo=300, ctx_hi=8003,
             q_heads=32, kv_heads=8, features=128, page=64, tree=True, tail=3),
        # prompts of different lengths packed, some of them behind a shared cached beginning
        dict(name="prompts_packed", op="sdpa", type="bf16", seqs=24, rows_lo=0, rows_hi=1201, ctx_lo=0, ctx_hi=400,
             q_heads=32, kv_heads=4, features=64, page=32, tree=False, tail=5),
        # one long prompt
        dict(name="prompt_long", op="sdpa", type="bf16", seqs=1, rows_lo=8191, rows_hi=8191, ctx_lo=0, ctx_hi=0,
             q_heads=32, kv_heads=8, features=128, page=64, tree=False, tail=1),
        # queries of a decode step
        dict(name="rope_step", op="rope", type="bf16", heads=32, rows=16, features=64, far=30000, skip=0),
        # queries of a long packed prompt in 32 bits, far positions, padding rows
        dict(name="rope_prompt", op="rope", type="f32", heads=32, rows=6001, features=128, far=200000, skip=9),
        # the accepted tokens of eight drafted trees go to the cache
        dict(name="append_accepted", op="append", type="bf16", seqs=8, rows_lo=1, rows_hi=7, spare=40, ctx_lo=300,
             ctx_hi=8003, kv_heads=8, features=128, page=64),
        # the keys and values of packed prompts go to the cache
        dict(name="append_prompts", op="append", type="f16", seqs=24, rows_lo=0, rows_hi=1201, spare=0, ctx_lo=0,
             ctx_hi=400, kv_heads=8, features=128, page=32),
        # the next token of sixteen chats: log probability of the token and the likeliest five
        dict(name="logprobs_step", op="logprobs", type="bf16", rows=16, vocabulary=32000, given=1, top=5),
        # a tree's nodes with their children's tokens
        dict(name="logprobs_tree", op="logprobs", type="f32", rows=333, vocabulary=50257, given=4, top=8),
        # the scoring of prompts with a large vocabulary
        dict(name="logprobs_score", op="logprobs", type="bf16", rows=2047, vocabulary=128256, given=1, top=20),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["token", "tree", "prompt", "rope", "append", "logprobs", "logprobs"])
    if op in ("token", "tree", "prompt"):
        kv, group = rng.choice([(1, 8), (2, 3), (4, 1), (4, 8), (8, 4), (8, 1), (2, 16), (3, 5)])
        case = dict(op="sdpa", type=rng.choice(["bf16", "f16"]), q_heads=kv * group, kv_heads=kv,
                    features=rng.choice([32, 64, 64, 80, 96, 128, 128]), page=rng.choice([16, 32, 48, 64, 128]),
                    tree=op == "tree", tail=rng.choice([0, 0, 1, 7]))
        if op == "token":
            hi = _spread(rng, 20, 15000)
            case.update(seqs=_spread(rng, 1, 64 if hi < 6000 else 24), rows_lo=1, rows_hi=1, ctx_lo=rng.randint(0, 9), ctx_hi=hi)
        elif op == "tree":
            hi = _spread(rng, 2, 100)
            case.update(seqs=_spread(rng, 1, 16), rows_lo=1, rows_hi=hi, ctx_lo=rng.randint(0, 9), ctx_hi=_spread(rng, 20, 8000))
        else:
            hi = _spread(rng, 30, 4000)
            case.update(seqs=_spread(rng, 1, max(1, min(32, 20000000 // (hi * hi)))), rows_lo=rng.choice([0, 1, hi // 3]),
                        rows_hi=hi, ctx_lo=0, ctx_hi=rng.choice([0, 0, _spread(rng, 1, 900)]))
        return case
    if op == "rope":
        return dict(op="rope", type=rng.choice(["bf16", "f16", "f32"]), heads=rng.choice([1, 2, 4, 8, 12, 32]),
                    rows=_spread(rng, 1, 6000), features=rng.choice([32, 64, 80, 96, 128]),
                    far=_spread(rng, 100, 500000), skip=rng.choice([0, 0, 1, 9]))
    if op == "append":
        return dict(op="append", type=rng.choice(["bf16", "f16", "f32"]), seqs=_spread(rng, 1, 48), rows_lo=rng.choice([0, 1]),
                    rows_hi=_spread(rng, 1, 600), spare=rng.choice([0, 5, 40]), ctx_lo=0, ctx_hi=_spread(rng, 1, 2000),
                    kv_heads=rng.choice([1, 2, 3, 4, 8]), features=rng.choice([32, 64, 80, 96, 128]),
                    page=rng.choice([16, 32, 48, 64, 128]))
    vocabulary = _spread(rng, 300, 150000)
    return dict(op="logprobs", type=rng.choice(["bf16", "f16", "f32"]), rows=_spread(rng, 1, max(1, min(2000, 100000000 // vocabulary))),
                vocabulary=vocabulary, given=rng.choice([1, 1, 2, 5]), top=rng.choice([0, 1, 3, 8, 20, 32]))


def _lengths(case):
    """Rows and cached tokens of each sequence: fixed by the case, the longest of both among them."""
    rng = random.Random(case["seqs"] * 7919 + case["rows_hi"] * 31 + case["ctx_hi"])
    rows = [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    rows[-1], ctx[0] = case["rows_hi"], case["ctx_hi"]
    if case["seqs"] > 2:
        rows[0], ctx[1] = case["rows_lo"], case["ctx_lo"]
    return rows, ctx


# ---------------------------------------------------------------------------
# the tiled layout
# ---------------------------------------------------------------------------

def _up(n, m=TILE):
    return (n + m - 1) // m * m


def tiled(x):
    """[..., R, C] -> [..., R/16, C/16, 16, 16], zeros in the padding."""
    r, c = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, _up(c) - c, 0, _up(r) - r))
    return x.reshape(*x.shape[:-2], _up(r) // TILE, TILE, _up(c) // TILE, TILE).transpose(-3, -2).contiguous()


def untiled(t, r, c):
    """[..., R/16, C/16, 16, 16] -> [..., R, C]"""
    t = t.transpose(-3, -2)
    return t.reshape(*t.shape[:-4], t.shape[-4] * TILE, t.shape[-2] * TILE)[..., :r, :c]


def _row(values):
    return tiled(torch.tensor([values], dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, dims, dtype, scale=1.0):
    return (torch.randn(dims, generator=gen, device="cuda") * scale).to(dtype)


def _prepare_cache(case, gen, rows, ctx, dtype):
    """A pool with a page for every page of every sequence and a few more, in a shuffled order."""
    page = case["page"]
    slots = max(1, max(-(-(c + r) // page) for c, r in zip(ctx, rows)))
    pages = sum(-(-(c + r) // page) for c, r in zip(ctx, rows)) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table = []
    for c, r in zip(ctx, rows):
        n = -(-(c + r) // page)
        table.append([order.pop() for _ in range(n)] + [0] * (slots - n))
    dims = (pages, case["kv_heads"], page, case["features"])
    return dict(k_pages=tiled(_normal(gen, dims, dtype)), v_pages=tiled(_normal(gen, dims, dtype)),
                table=tiled(torch.tensor(table, dtype=torch.int32, device="cuda")), lengths=_row(ctx),
                slots=slots, pages=pages)


def _starts(rows):
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    return starts


def _prepare_sdpa(case, gen, seed):
    rows, ctx = _lengths(case)
    dtype, starts = TYPES[case["type"]], _starts(rows)
    total = max(1, starts[-1] + case["tail"])
    s = dict(case=case, total=total, max_rows=max(1, max(rows)), longest=max(ctx))
    s.update(_prepare_cache(case, gen, [0] * len(rows), ctx, dtype))
    s["q"] = tiled(_normal(gen, (case["q_heads"], total, case["features"]), dtype, 1.5))
    s["k"] = tiled(_normal(gen, (case["kv_heads"], total, case["features"]), dtype))
    s["v"] = tiled(_normal(gen, (case["kv_heads"], total, case["features"]), dtype))
    s["starts"] = _row(starts)
    s["out"] = torch.zeros_like(tiled(torch.zeros(total, case["q_heads"] * case["features"], dtype=dtype, device="cuda")))
    s["tree"] = None
    if case["tree"]:
        # every drafted token continues one of the few before it or the context itself
        rng, words, masks = random.Random(seed), -(-s["max_rows"] // 32), []
        for n in rows:
            seen = []
            for j in range(n):
                parent = rng.randint(max(-1, j - 5), j - 1)
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << j)
            masks += seen
        masks += [0] * (total - len(masks))
        flat = [[(m >> 32 * w) & 0xFFFFFFFF for w in range(words)] for m in masks]
        s["tree"] = tiled(torch.tensor([[x - (1 << 32) if x >> 31 else x for x in m] for m in flat], dtype=torch.int32, device="cuda"))
        s["words"] = words
    return s


def _prepare_rope(case, gen, seed):
    dims = (case["heads"], case["rows"], case["features"])
    x = tiled(_normal(gen, dims, TYPES[case["type"]]))
    positions = torch.randint(0, case["far"], (1, case["rows"]), generator=gen, device="cuda", dtype=torch.int32)
    if case["skip"] and case["skip"] < case["rows"]:
        positions[0, -case["skip"]:] = -1   # padding rows
    return dict(case=case, x=x, positions=tiled(positions), out=torch.zeros_like(x), theta=10000.0)


def _prepare_append(case, gen, seed):
    rows, ctx = _lengths(case)
    dtype, starts = TYPES[case["type"]], _starts(rows)
    listed_rows, total = starts[-1], starts[-1] + case["spare"]
    s = dict(case=case, total=total, listed_rows=listed_rows)
    s.update(_prepare_cache(case, gen, rows, ctx, dtype))
    dims = (case["kv_heads"], total, case["features"])
    s["k"], s["v"] = tiled(_normal(gen, dims, dtype)), tiled(_normal(gen, dims, dtype))
    s["starts"], s["rows"] = _row(starts), None
    if case["spare"]:   # some of the step's rows, in their order
        s["rows"] = _row(sorted(random.Random(seed).sample(range(total), listed_rows)))
    return s


def _prepare_logprobs(case, gen, seed):
    rows, vocabulary = case["rows"], case["vocabulary"]
    logits = torch.randn((rows, vocabulary), generator=gen, device="cuda") * 3
    logits[:, vocabulary - vocabulary // 200:] = -math.inf     # entries that no tokenizer gives out
    s = dict(case=case, logits=tiled(logits.to(TYPES[case["type"]])))
    tokens = torch.randint(0, vocabulary, (rows, case["given"]), generator=gen, device="cuda", dtype=torch.int32)
    if case["given"] > 1:
        tokens[::3, -1] = -1                                   # a node with fewer children
    s["tokens"] = tiled(tokens)
    for name, columns, dtype in (("logprobs", case["given"], torch.float32), ("entropy", 1, torch.float32),
                                 ("top_ids", case["top"], torch.int32), ("top_logprobs", case["top"], torch.float32)):
        s[name] = tiled(torch.zeros((rows, columns), dtype=dtype, device="cuda")) if columns else None
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return {"sdpa": _prepare_sdpa, "rope": _prepare_rope, "append": _prepare_append,
            "logprobs": _prepare_logprobs}[case["op"]](case, gen, seed)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _indices(s):
    """Rows of every sequence [S, max_rows] on the packed axis, and which of them there are."""
    n = s["case"]["seqs"]
    starts = untiled(s["starts"], 1, n + 1)[0].long()
    lengths = untiled(s["lengths"], 1, n)[0].long()
    at = starts[:-1, None] + torch.arange(s["max_rows"], device="cuda")
    return at, at < starts[1:, None], lengths


def _plain_sdpa(s):
    c, dtype = s["case"], s["q"].dtype
    S, Hq, Hkv, D, T, R, P = c["seqs"], c["q_heads"], c["kv_heads"], c["features"], s["total"], s["max_rows"], c["page"]
    at, there, lengths = _indices(s)
    safe = at.clamp(max=T - 1)
    pick = lambda x: untiled(x, T, D).float()[:, safe].transpose(0, 1)                       # [S, H, R, D]
    table = untiled(s["table"], S, s["slots"]).long()
    cached = lambda x: untiled(x, P, D)[table].float().transpose(1, 2).reshape(S, Hkv, s["slots"] * P, D)[:, :, :s["longest"]]
    q = pick(s["q"]).reshape(S, Hkv, Hq // Hkv * R, D)
    k = torch.cat([cached(s["k_pages"]), pick(s["k"])], 2)
    v = torch.cat([cached(s["v_pages"]), pick(s["v"])], 2)
    ctx = (torch.arange(s["longest"], device="cuda") < lengths[:, None])[:, None, :].expand(S, R, s["longest"])
    j = torch.arange(R, device="cuda")
    if c["tree"]:
        words = untiled(s["tree"], T, s["words"])[safe]                                      # [S, R, W]
        new = (words[:, :, j // 32] >> (j % 32) & 1) != 0
    else:
        new = (j[None, :] <= j[:, None]).expand(S, R, R)
    sees = torch.cat([ctx, new & there[:, None, :]], 2) & there[:, :, None]                  # [S, R, keys]
    scores = (q @ k.transpose(-1, -2)) / math.sqrt(D)
    scores = scores.reshape(S, Hkv, Hq // Hkv, R, -1).masked_fill(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    rows = (p.reshape(S, Hkv, Hq // Hkv * R, -1) @ v).reshape(S, Hq, R, D).permute(0, 2, 1, 3).reshape(S * R, Hq * D)
    out = torch.zeros((T + 1, Hq * D), device="cuda", dtype=dtype)                           # row T: rows that are not there
    out[torch.where(there, at, T).reshape(-1)] = rows.to(dtype)
    return tiled(out[:T])


def _plain_rope(s):
    c = s["case"]
    T, D = c["rows"], c["features"]
    x = untiled(s["x"], T, D).float()
    positions = untiled(s["positions"], 1, T)[0]
    frequency = torch.pow(torch.tensor(s["theta"], dtype=torch.float64, device="cuda"),
                          -2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
    angle = positions.double()[:, None] * frequency
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    out = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(s["x"].dtype)
    return tiled(torch.where((positions >= 0)[None, :, None], out, 0))


def _plain_append(s):
    c = s["case"]
    S, D, P, T, E = c["seqs"], c["features"], c["page"], s["total"], s["listed_rows"]
    starts = untiled(s["starts"], 1, S + 1)[0].long()
    lengths = untiled(s["lengths"], 1, S)[0].long()
    entry = torch.arange(E, device="cuda")
    sequence = (entry[:, None] >= starts[None, 1:]).sum(1)
    source = entry if s["rows"] is None else untiled(s["rows"], 1, E)[0].long()
    position = lengths[sequence] + entry - starts[sequence]
    page = untiled(s["table"], S, s["slots"]).long()[sequence, position // P]
    row = position % P
    got = {}
    for name, new in (("k_pages", "k"), ("v_pages", "v")):
        x = untiled(s[new], T, D)[:, source].transpose(0, 1).reshape(E, -1, D // TILE, TILE)
        s[name][page, :, row // TILE, :, row % TILE, :] = x
        got[name] = s[name]
    return got


def _plain_logprobs(s):
    c = s["case"]
    R, V = c["rows"], c["vocabulary"]
    x = untiled(s["logits"], R, V).float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    whole = top + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, (x - top) * e, 0.0).sum(-1, keepdim=True) / total
    tokens = untiled(s["tokens"], R, c["given"]).long()
    given = torch.gather(x, 1, tokens.clamp(min=0)) - whole
    given = torch.where(tokens >= 0, given, -math.inf)
    got = {"logprobs": tiled(given), "entropy": tiled(entropy)}
    if c["top"]:
        values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        got["top_ids"] = tiled(ids[:, :c["top"]].int())
        got["top_logprobs"] = tiled(values[:, :c["top"]] - whole)
    return got


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _view(iomx, x, dims):
    """A view of the framework over a tensor in the tiled layout."""
    if x is None:
        return None
    kinds = {torch.bfloat16: iomx.DT_BF16, torch.float16: iomx.DT_F16, torch.float32: iomx.DT_F32, torch.int32: iomx.DT_I32}
    return iomx.DeviceTensor.at(x.data_ptr(), kinds[x.dtype], dims).view()


def _workspace(iomx, s, query):
    status, nbytes, _ = query
    iomx.check(status, "workspace")
    s["workspace"] = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    return iomx.Buffer.at(s["workspace"].data_ptr(), s["workspace"].numel())


def _views(iomx, s):
    """The views and the workspace that a program makes once for its buffers."""
    c, h = s["case"], {}
    if c["op"] in ("sdpa", "append"):
        kv = (c["kv_heads"], s["total"], c["features"])
        pool = (s["pages"], c["kv_heads"], c["page"], c["features"])
        for name, dims in (("k", kv), ("v", kv), ("k_pages", pool), ("v_pages", pool), ("table", (c["seqs"], s["slots"])),
                           ("starts", (1, c["seqs"] + 1)), ("lengths", (1, c["seqs"]))):
            h[name] = _view(iomx, s[name], dims)
    if c["op"] == "sdpa":
        h["q"] = _view(iomx, s["q"], (c["q_heads"], s["total"], c["features"]))
        h["out"] = _view(iomx, s["out"], (s["total"], c["q_heads"] * c["features"]))
        h["tree"] = _view(iomx, s["tree"], (s["total"], s.get("words", 1)))
        h["max_rows"] = s["max_rows"]
        h["workspace"] = _workspace(iomx, s, iomx.sdpa_packed_workspace(**h))
    elif c["op"] == "append":
        h["rows"] = _view(iomx, s["rows"], (1, s["listed_rows"]))
    elif c["op"] == "rope":
        dims = (c["heads"], c["rows"], c["features"])
        h.update(x=_view(iomx, s["x"], dims), out=_view(iomx, s["out"], dims),
                 positions=_view(iomx, s["positions"], (1, c["rows"])), theta=s["theta"])
    else:
        h["logits"] = _view(iomx, s["logits"], (c["rows"], c["vocabulary"]))
        for name, columns in (("tokens", c["given"]), ("logprobs", c["given"]), ("entropy", 1), ("top_ids", c["top"]), ("top_logprobs", c["top"])):
            h[name] = _view(iomx, s[name], (c["rows"], columns))
        h["workspace"] = _workspace(iomx, s, iomx.token_logprobs_workspace(**h))
    return h


def _own(s):
    from iom_amd import iomx
    if "views" not in s:
        s["views"] = _views(iomx, s)
    h, op = s["views"], s["case"]["op"]
    stream = iomx.Stream.at(torch.cuda.current_stream().cuda_stream)
    if op == "sdpa":
        iomx.check(iomx.sdpa_packed(stream=stream, **h), "sdpa_packed")
        return s["out"]
    if op == "rope":
        iomx.check(iomx.rope_packed(stream=stream, **h), "rope_packed")
        return s["out"]
    if op == "append":
        iomx.check(iomx.cache_append_packed(stream=stream, **h), "cache_append_packed")
        return {name: s[name] for name in ("k_pages", "v_pages")}
    iomx.check(iomx.token_logprobs(stream=stream, **h), "token_logprobs")
    return {name: s[name] for name in ("logprobs", "entropy", "top_ids", "top_logprobs") if s[name] is not None}


def run(state):
    if own:
        return _own(state)
    return {"sdpa": _plain_sdpa, "rope": _plain_rope, "append": _plain_append,
            "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    size = torch.finfo(TYPES[case["type"]]).bits // 8
    if case["op"] == "rope":
        n = case["heads"] * max(1, case["rows"] - case["skip"]) * case["features"]
        return {"bytes": 2 * n * size + 4 * case["rows"], "flops": 3 * n}
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocabulary"]
        return {"bytes": n * size + case["rows"] * (8 * case["given"] + 4 + 8 * case["top"]), "flops": 6 * n}
    rows, ctx = _lengths(case)
    head = case["kv_heads"] * case["features"] * size
    if case["op"] == "append":
        return {"bytes": 4 * max(1, sum(rows)) * head, "flops": 0}
    wide = case["q_heads"] * case["features"]
    read = sum(c for c, r in zip(ctx, rows) if r)
    pairs = sum(r * c + r * (r + 1) // 2 for c, r in zip(ctx, rows))
    return {"bytes": 2 * (read + sum(rows)) * head + 2 * sum(rows) * wide * size, "flops": 4 * pairs * wide}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _matrix(t, rows, columns):
    """Rows of a tiled plane (or of several), by gathering each element's slot."""
    r = torch.arange(rows, device=t.device)[:, None]
    c = torch.arange(columns, device=t.device)[None, :]
    wide = t.shape[-3]
    slot = ((r // TILE) * wide + c // TILE) * TILE * TILE + (r % TILE) * TILE + c % TILE
    return t.reshape(*t.shape[:-4], -1)[..., slot]


def _planes(x):
    """The reverse of _matrix, zeros in the padding."""
    rows, columns = x.shape[-2:]
    r = torch.arange(rows, device=x.device)[:, None]
    c = torch.arange(columns, device=x.device)[None, :]
    high, wide = -(-rows // TILE), -(-columns // TILE)
    slot = ((r // TILE) * wide + c // TILE) * TILE * TILE + (r % TILE) * TILE + c % TILE
    t = torch.zeros((*x.shape[:-2], high * wide * TILE * TILE), dtype=x.dtype, device=x.device)
    t[..., slot] = x
    return t.reshape(*x.shape[:-2], high, wide, TILE, TILE)


def _exact_sdpa(s):
    c = s["case"]
    D, P, group = c["features"], c["page"], c["q_heads"] // c["kv_heads"]
    rows, ctx = _lengths(c)
    q, k, v = (_matrix(s[name], s["total"], D) for name in ("q", "k", "v"))
    table = _matrix(s["table"], c["seqs"], s["slots"]).tolist()
    words = _matrix(s["tree"], s["total"], s["words"]).long() if c["tree"] else None
    out = torch.zeros((s["total"], c["q_heads"] * D), dtype=torch.float64, device="cuda")
    first = 0
    for n, have, pages in zip(rows, ctx, table):
        used = pages[:-(-have // P)]
        for h in range(c["kv_heads"] if n else 0):
            cached = [torch.cat([_matrix(s[name][page, h], P, D) for page in used] + [new[h, :0]])[:have]
                      for name, new in (("k_pages", k), ("v_pages", v))]
            kk = torch.cat([cached[0], k[h, first:first + n]]).double()
            vv = torch.cat([cached[1], v[h, first:first + n]]).double()
            sees = torch.ones((n, have + n), dtype=torch.bool, device="cuda")
            i = torch.arange(n, device="cuda")
            if c["tree"]:
                sees[:, have:] = torch.bitwise_right_shift(words[first:first + n][:, i // 32], i % 32).remainder(2) == 1
            else:
                sees[:, have:] = i[:, None] >= i[None, :]
            hidden = torch.zeros(sees.shape, dtype=torch.float64, device="cuda").masked_fill(~sees, -math.inf)
            for g in range(h * group, (h + 1) * group):
                weights = torch.softmax(q[g, first:first + n].double() @ kk.T / D ** 0.5 + hidden, -1)
                out[first:first + n, g * D:(g + 1) * D] = weights @ vv
        first += n
    return _planes(out)


def _exact_rope(s):
    c = s["case"]
    half = c["features"] // 2
    x = torch.complex(*(t.double() for t in _matrix(s["x"], c["rows"], c["features"]).split(half, -1)))
    positions = _matrix(s["positions"], 1, c["rows"])[0]
    rate = torch.tensor([s["theta"] ** (-j / half) for j in range(half)], dtype=torch.float64, device="cuda")
    turned = x * torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(positions.double(), rate))
    turned = torch.cat([turned.real, turned.imag], -1)
    turned[:, positions < 0] = 0
    return _planes(turned)


def _exact_append(s):
    c = s["case"]
    rows, ctx = _lengths(c)
    table = _matrix(s["table"], c["seqs"], s["slots"]).tolist()
    chosen = list(range(s["total"])) if s["rows"] is None else _matrix(s["rows"], 1, s["listed_rows"])[0].tolist()
    place = []
    for n, have, pages in zip(rows, ctx, table):
        place += [pages[(have + i) // c["page"]] * c["page"] + (have + i) % c["page"] for i in range(n)]
    chosen = torch.tensor(chosen[:len(place)], dtype=torch.long, device="cuda")
    place = torch.tensor(place, dtype=torch.long, device="cuda")
    got = {}
    for name, new in (("k_pages", "k"), ("v_pages", "v")):
        pool = _matrix(s[name], c["page"], c["features"]).double().transpose(0, 1).reshape(c["kv_heads"], -1, c["features"])
        pool[:, place] = _matrix(s[new], s["total"], c["features"]).double()[:, chosen]
        got[name] = _planes(pool.reshape(c["kv_heads"], s["pages"], c["page"], c["features"]).transpose(0, 1))
    return got


def _exact_logprobs(s):
    c = s["case"]
    x = _matrix(s["logits"], c["rows"], c["vocabulary"]).double()
    logs = x - torch.logsumexp(x, -1, keepdim=True)
    tokens = _matrix(s["tokens"], c["rows"], c["given"]).long()
    more = torch.cat([logs, torch.full((c["rows"], 1), -math.inf, dtype=torch.float64, device="cuda")], 1)
    got = {"logprobs": _planes(torch.gather(more, 1, tokens % (c["vocabulary"] + 1))),
           "entropy": _planes(-torch.special.xlogy(logs.exp(), logs.exp()).sum(-1, keepdim=True))}
    if c["top"]:
        ids = []
        for row in logs.split(64):     # the largest, and of equal ones those with the lowest index
            order = torch.argsort(-row, dim=-1, stable=True)[:, :c["top"]]
            ids.append(order)
        ids = torch.cat(ids)
        got["top_ids"] = _planes(ids.int())
        got["top_logprobs"] = _planes(torch.gather(logs, 1, ids))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"sdpa": _exact_sdpa, "rope": _exact_rope, "append": _exact_append, "logprobs": _exact_logprobs}[case["op"]](s)
