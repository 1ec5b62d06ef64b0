"""What is measured of the operators of a step that verifies drafted tokens, through the framework's public entry points.

Every sequence of such a step brings a tree of drafted tokens (or a chain of them), a row each: row 0 is its last certain token, every other
row has an earlier one for its parent. Four kinds of case, each over the range of sizes that `draw` spans:

  norms      norms of query and key heads, rotary positions and the append to the page pool in one pass (`norm_rotary_append`)
  attention  attention of the rows over their sequence's pages and the rows that they follow (`tree_attention`)
  logits     penalties for repeated tokens, biases and grammar masks (`adjust_logits`)
  drafts     the rows' positions and masks, the accepted path, and its keys and values moved together (`map_drafts`, `accept_drafts`,
             `keep_accepted`)

The plain forms are elementary torch operations in 32 bits (angles in 64); `exact` restates the operators in 64 bits.
"""
from __future__ import annotations

import math
import random
import zlib

import torch

own = False

DEV = "cuda"
PAGE = 16
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
# (query heads, key/value heads, head size): the two benchmark models of `bench.py`, one without shared heads, one with a single
# key/value head, and heads of 64
HEADS = ((32, 8, 128), (64, 8, 128), (16, 16, 128), (16, 1, 128), (32, 8, 64))
BASE = 500000.0
EPS = 1e-6


def listed():
    return [
        # a decode step's heads
        dict(name="norms decode", kind="norms", rows=32, heads=32, kv_heads=8, dim=128, rot=128, layout="interleaved", far=8192, offset=0.0,
             padded=0, dtype="float16"),
        # 64 requests with 32 drafted tokens each, the last rows of the bucket empty
        dict(name="norms drafts", kind="norms", rows=2048, heads=32, kv_heads=8, dim=128, rot=128, layout="half", far=8192, offset=1.0,
             padded=47, dtype="bfloat16"),
        # a pass over prompts with far positions, a quarter of every head turned
        dict(name="norms prompt", kind="norms", rows=16384, heads=64, kv_heads=8, dim=128, rot=32, layout="half", far=1000000, offset=0.0,
             padded=0, dtype="float16"),
        # two short requests with a few drafts each
        dict(name="attention pair", kind="attention", heads=32, kv_heads=8, dim=128, dtype="float16", sequences=2, ctx_min=200, ctx_max=333,
             nodes_min=7, nodes_max=8, chain=False, padded=0, lens=4),
        # a server's batch, trees of 12 to 16 tokens, in a bucket of 512 rows
        dict(name="attention batch", kind="attention", heads=32, kv_heads=8, dim=128, dtype="float16", sequences=32, ctx_min=256, ctx_max=4096,
             nodes_min=12, nodes_max=16, chain=False, padded=3, lens=5),
        # wide trees on a model with many heads
        dict(name="attention wide", kind="attention", heads=64, kv_heads=8, dim=128, dtype="bfloat16", sequences=16, ctx_min=1000, ctx_max=8192,
             nodes_min=40, nodes_max=64, chain=False, padded=0, lens=6),
        # chains of a certain token and up to four drafts behind long documents
        dict(name="attention documents", kind="attention", heads=32, kv_heads=8, dim=128, dtype="float16", sequences=4, ctx_min=90000, ctx_max=131072,
             nodes_min=2, nodes_max=5, chain=True, padded=0, lens=7),
        # the next token of one request that has said a few hundred
        dict(name="logits one", kind="logits", rows=1, sequences=1, vocab=128256, dtype="float16", history=777, penalties=True, bias=5, grammar=False,
             drafts=False),
        # constrained requests over an odd vocabulary
        dict(name="logits grammar", kind="logits", rows=64, sequences=64, vocab=50001, dtype="float32", history=0, penalties=False, bias=100, grammar=True,
             drafts=False),
        # the logits of every drafted token of a batch: what a row follows counts as said
        dict(name="logits drafts", kind="logits", rows=512, sequences=32, vocab=128256, dtype="bfloat16", history=4096, penalties=True, bias=20,
             grammar=True, drafts=True),
        # a few requests with small trees
        dict(name="drafts few", kind="drafts", sequences=4, nodes_min=6, nodes_max=8, layers=4, kv_heads=8, dim=128, dtype="float16", lens=8),
        # many requests with large trees, all layers of a model
        dict(name="drafts many", kind="drafts", sequences=128, nodes_min=33, nodes_max=64, layers=32, kv_heads=8, dim=128, dtype="float16", lens=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _within(case):
    """No more of anything than the largest listed case of the kind."""
    cost, most = work(case), [work(c) for c in listed() if c["kind"] == case["kind"]]
    return all(cost[key] <= max(m[key] for m in most) for key in cost)


def draw(rng):
    """Kinds in the shares that the listed cases have; sizes over their whole range."""
    kind = rng.choice(["norms"] * 3 + ["attention"] * 4 + ["logits"] * 3 + ["drafts"] * 2)
    while True:
        if kind == "norms":
            heads, kv_heads, dim = rng.choice(HEADS)
            rows = _log(rng, 1, 16384)
            case = dict(kind=kind, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, dim // 4]),
                        layout=rng.choice(["interleaved", "half"]), far=_log(rng, 1000, 1000000), offset=rng.choice([0.0, 1.0]),
                        padded=rng.choice([0, rows // 9]), dtype=rng.choice(list(DTYPES)))
        elif kind == "attention":
            heads, kv_heads, dim = rng.choice(HEADS)
            ctx, nodes = _log(rng, 1, 131072), _log(rng, 1, 128)
            case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["float16", "bfloat16"]), sequences=_log(rng, 1, 256),
                        ctx_min=rng.choice([0, ctx // 2, ctx]), ctx_max=ctx, nodes_min=rng.choice([0, (nodes + 1) // 2, nodes]), nodes_max=nodes,
                        chain=rng.random() < 0.3, padded=rng.choice([0, 5]), lens=rng.randrange(1 << 30))
        elif kind == "logits":
            vocab = rng.choice([32768, 128256, 50001, _log(rng, 1000, 131072)])
            sequences, drafts = _log(rng, 1, 128), rng.random() < 0.5
            case = dict(kind=kind, rows=min(512, sequences * rng.choice([2, 5, 16])) if drafts else sequences, sequences=sequences, vocab=vocab,
                        dtype=rng.choice(list(DTYPES)), history=rng.choice([0, _log(rng, 1, 16384)]), penalties=rng.random() < 0.8,
                        bias=rng.choice([0, 0, _log(rng, 1, 300)]), grammar=rng.random() < 0.5, drafts=drafts)
            if not (case["penalties"] or case["bias"] or case["grammar"]):
                case["grammar"] = True
        else:
            nodes = _log(rng, 1, 64)
            case = dict(kind=kind, sequences=_log(rng, 1, 128), nodes_min=rng.choice([0, (nodes + 1) // 2, nodes]), nodes_max=nodes,
                        layers=_log(rng, 1, 32), kv_heads=rng.choice([1, 8]), dim=rng.choice([64, 128]), dtype=rng.choice(list(DTYPES)),
                        lens=rng.randrange(1 << 30))
        if _within(case):
            return case


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _gen(seed, name):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(name.encode()) ^ (seed * 7919 & 0x7FFFFFFF))


def _randn(seed, name, *shape):
    return torch.randn(shape, device=DEV, generator=_gen(seed, name))


def _randint(seed, name, low, high, *shape):
    return torch.randint(low, high, shape, device=DEV, generator=_gen(seed, name))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def _starts(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _lens(case):
    """(tokens in front, rows) of every sequence; one sequence at least has a row."""
    rng = random.Random(case["lens"])
    lo, hi = case.get("ctx_min", 1), case.get("ctx_max", 4 * PAGE)
    ctx = [rng.randint(lo, hi) for _ in range(case["sequences"])]
    nodes = [rng.randint(case["nodes_min"], case["nodes_max"]) for _ in range(case["sequences"])]
    return ctx, nodes if any(nodes) else [case["nodes_max"]] * len(nodes)


def _trees(seed, nodes):
    """Parents of every row (numbers inside its sequence): small trees by growing, rows of a depth side by side."""
    rng = random.Random(seed * 31 + 7)
    trees = []
    for n in nodes:
        loose = [-1] + [rng.randrange(max(0, i - 8), i) for i in range(1, n)]
        depth = [0] * n
        for i in range(1, n):
            depth[i] = depth[loose[i]] + 1
        order = sorted(range(n), key=lambda i: (depth[i], i))
        place = {old: new for new, old in enumerate(order)}
        trees.append([-1 if loose[old] < 0 else place[loose[old]] for old in order])
    return trees


def _ancestors(parents):
    """Of every row the rows that it sees: those that it follows, and itself."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else []) + [i])
    return seen


def _words(rows_seen, words):
    """Lists of visible rows as 32-bit words."""
    lines = []
    for seen in rows_seen:
        bits = sum(1 << j for j in seen)
        lines.append([(bits >> 32 * w & 0xFFFFFFFF) - (bits >> 32 * w + 31 & 1) * (1 << 32) for w in range(words)])
    return lines


def prepare(case, seed):
    state = {"case": case}
    kind = case["kind"]
    if kind == "norms":
        rows, heads, kv_heads, dim, dtype = case["rows"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        qkv = (_randn(seed, "qkv", rows, (heads + 2 * kv_heads) * dim) * (0.2 + 3.0 * torch.rand(rows, 1, device=DEV, generator=_gen(seed, "size")))).to(dtype)
        slots_total = _pages(rows) + 2
        slots = torch.randperm(slots_total * PAGE, device=DEV, generator=_gen(seed, "slots"))[:rows].to(torch.int32)
        if case["padded"]:
            slots[rows - case["padded"]:] = -1
        state.update(q=qkv[:, : heads * dim].view(rows, heads, dim), k=qkv[:, heads * dim: (heads + kv_heads) * dim].view(rows, kv_heads, dim),
                     v=qkv[:, (heads + kv_heads) * dim:].view(rows, kv_heads, dim), slots=slots,
                     q_weight=(1.0 - case["offset"] + 0.2 * _randn(seed, "q weight", dim)).to(dtype),
                     k_weight=(1.0 - case["offset"] + 0.2 * _randn(seed, "k weight", dim)).to(dtype),
                     freq=(BASE ** (-2.0 * torch.arange(case["rot"] // 2, dtype=torch.float64) / case["rot"])).to(DEV),
                     positions=_randint(seed, "positions", 0, case["far"], rows).to(torch.int32),
                     k_cache=torch.zeros(slots_total, kv_heads, PAGE, dim, dtype=dtype, device=DEV),
                     v_cache=torch.zeros(slots_total, kv_heads, PAGE, dim, dtype=dtype, device=DEV),
                     q_out=torch.zeros(rows, heads, dim, dtype=dtype, device=DEV))
        if own:
            from cacheir_b200 import serving_ops
            state["rule"] = serving_ops.rotary_rule(case["rot"], BASE, layout=case["layout"], device=DEV)
    elif kind == "attention":
        heads, kv_heads, dim, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        ctx, nodes = _lens(case)
        lens = [c + n for c, n in zip(ctx, nodes)]
        rows, starts = sum(nodes) + case["padded"], _starts(nodes)
        count = torch.tensor([_pages(n) for n in lens], device=DEV)
        total, width = sum(_pages(n) for n in lens) + 3, max(_pages(n) for n in lens) + 1
        order = torch.randperm(total, device=DEV, generator=_gen(seed, "pages")).to(torch.int32)
        place = torch.arange(width, device=DEV)
        first = torch.cumsum(count, 0) - count
        table = torch.where(place[None, :] < count[:, None], order[(first[:, None] + place[None, :]).clamp(max=total - 1)], 0).to(torch.int32)
        words = (max(nodes) + 31) // 32
        visible = None
        if not case["chain"]:
            lines = [line for tree in _trees(seed, nodes) for line in _words(_ancestors(tree), words)]
            visible = _i32(lines + [[0] * words] * case["padded"])
        q = (_randn(seed, "q", rows, (heads + 2 * kv_heads) * dim) * 1.5).to(dtype)[:, : heads * dim].view(rows, heads, dim)
        state.update(q=q, keys=_randn(seed, "keys", total, kv_heads, PAGE, dim).to(dtype), values=_randn(seed, "values", total, kv_heads, PAGE, dim).to(dtype),
                     table=table, seq_lens=_i32(lens), cu_rows=_i32(starts), visible=visible, ctx=ctx, nodes=nodes, starts=starts,
                     out=torch.zeros(rows, heads, dim, dtype=dtype, device=DEV))
        if own:
            from cacheir_b200 import draft_ops
            state["workspace"] = torch.empty(draft_ops.tree_attention_workspace_bytes(rows, heads, dim), dtype=torch.uint8, device=DEV)
    elif kind == "logits":
        rows, sequences, vocab, size = case["rows"], case["sequences"], case["vocab"], case["history"]
        nodes = [rows // sequences + (b < rows % sequences) for b in range(sequences)]
        starts = _starts(nodes)
        state.update(logits=(_randn(seed, "logits", rows, vocab) * 2.5).to(DTYPES[case["dtype"]]), starts=starts, nodes=nodes, cu_rows=_i32(starts),
                     row_seq=_i32([b for b, n in enumerate(nodes) for _ in range(n)]),
                     out=torch.zeros(rows, vocab, dtype=DTYPES[case["dtype"]], device=DEV))
        if case["penalties"]:
            # a text says few words often: squares of uniform numbers
            uniform = torch.rand(sequences, max(size, 1), device=DEV, generator=_gen(seed, "said"))
            lens = _randint(seed, "lens", size // 2, size + 1, sequences)
            state.update(said=(uniform ** 3 * (vocab - 1)).to(torch.int32), said_lens=lens.to(torch.int32),
                         prompt_lens=(lens.float() * torch.rand(sequences, device=DEV, generator=_gen(seed, "prompts"))).to(torch.int32),
                         repetition=1.0 + 0.5 * torch.rand(sequences, device=DEV, generator=_gen(seed, "repetition")),
                         frequency=0.4 * _randn(seed, "frequency", sequences), presence=0.4 * _randn(seed, "presence", sequences))
        if case["bias"]:
            ids = torch.stack([torch.randperm(vocab, device=DEV, generator=_gen(seed * 131 + b, "bias"))[: case["bias"]] for b in range(sequences)])
            state.update(bias_ids=ids.to(torch.int32), bias_values=3.0 * _randn(seed, "bias values", sequences, ids.shape[1]))
        if case["grammar"]:
            state["allowed"] = _randint(seed, "allowed", -(1 << 31), 1 << 31, rows, (vocab + 31) // 32).to(torch.int32)
        if case["drafts"]:
            words = (max(nodes) + 31) // 32
            trees = [_ancestors(tree) for tree in _trees(seed, nodes)]
            state.update(draft_ids=(torch.rand(rows, device=DEV, generator=_gen(seed, "drafted")) ** 3 * (vocab - 1)).to(torch.int64), trees=trees,
                         visible=_i32([line for seen in trees for line in _words(seen, words)]))
    else:
        ctx, nodes = _lens(case)
        rows, starts, dtype = sum(nodes), _starts(nodes), DTYPES[case["dtype"]]
        trees, rng = _trees(seed, nodes), random.Random(seed * 17 + 3)
        words = (max(nodes) + 31) // 32
        draft_ids, chosen = [rng.randrange(50000) for _ in range(rows)], [rng.randrange(50000) for _ in range(rows)]
        longest = 1
        for tree, lo in zip(trees, starts):
            if not tree:
                continue
            path = _ancestors(tree)[rng.randrange(len(tree))]
            # a move may not write where another one reads, so that a pass can be made again
            while any(at != i and at < len(path) for i, at in enumerate(path)):
                path = path[:-1]
            for at, then in zip(path, path[1:]):
                chosen[lo + at] = draft_ids[lo + then]
            longest = max(longest, len(path) + 1)
        count = [_pages(c + n) - c // PAGE for c, n in zip(ctx, nodes)]      # the pages that the rows are in
        first = _starts(count)
        pages = torch.randperm(first[-1] + 3, generator=torch.Generator().manual_seed(seed)).tolist()
        slots = [pages[f + (c + i) // PAGE - c // PAGE] * PAGE + (c + i) % PAGE for c, n, f in zip(ctx, nodes, first) for i in range(n)]
        keys, values = (_randn(seed, name, case["layers"], first[-1] + 3, case["kv_heads"], PAGE, case["dim"]).to(dtype) for name in ("keys", "values"))
        state.update(parents=_i32([p for tree in trees for p in tree]), draft_ids=torch.tensor(draft_ids, device=DEV), chosen=torch.tensor(chosen, device=DEV),
                     seq_lens=_i32([c + n for c, n in zip(ctx, nodes)]), cu_rows=_i32(starts), slots=_i32(slots), nodes=nodes, starts=starts, trees=trees,
                     words=words, row_seq=_i32([b for b, n in enumerate(nodes) for _ in range(n)]), most=max(nodes), depth=max(nodes), longest=longest,
                     keys=keys, values=values, pools=list(zip(keys, values)))
        if own:
            from cacheir_b200 import draft_ops, serving_ops
            state["tokens"] = serving_ops.TokenMap(positions=torch.zeros_like(state["slots"]), row_seq=state["row_seq"], slots=state["slots"],
                                                   cu_rows=state["cu_rows"], status=_i32([0]))
            state["tree"] = draft_ops.draft_tree(rows, words, DEV)
            state["accepted"] = draft_ops.accepted_drafts(case["sequences"], state["depth"], DEV)
            state["handle"] = draft_ops.page_pools([pool for layer in state["pools"] for pool in layer])
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    return {"norms": _run_norms, "attention": _run_attention, "logits": _run_logits, "drafts": _run_drafts}[kind](state)


def _rotate(x, cos, sin, rot, layout):
    """x [rows, heads, dim] float; cos, sin [rows, 1, rot / 2]."""
    out = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if layout == "interleaved" else (x[..., : rot // 2], x[..., rot // 2: rot])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    if layout == "interleaved":
        out[..., 0:rot:2], out[..., 1:rot:2] = ra, rb
    else:
        out[..., : rot // 2], out[..., rot // 2: rot] = ra, rb
    return out


def _run_norms(s):
    case = s["case"]
    if own:
        from cacheir_b200 import draft_ops
        draft_ops.norm_rotary_append(s["q"], s["k"], s["v"], s["rule"], s["positions"], s["q_weight"], s["k_weight"], eps=EPS, offset=case["offset"],
                                     slots=s["slots"], k_cache=s["k_cache"], v_cache=s["v_cache"], q_out=s["q_out"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    rows = case["rows"] - case["padded"]
    angle = s["positions"][:rows].double()[:, None] * s["freq"]
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    turned = []
    for name in ("q", "k"):
        x = s[name][:rows].float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (s[name + "_weight"].float() + case["offset"])
        turned.append(_rotate(x, cos, sin, case["rot"], case["layout"]).to(s[name].dtype))
    s["q_out"][:rows] = turned[0]
    slot = s["slots"][:rows].long()
    s["k_cache"][slot // PAGE, :, slot % PAGE] = turned[1]
    s["v_cache"][slot // PAGE, :, slot % PAGE] = s["v"][:rows]
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_attention(s):
    if own:
        from cacheir_b200 import draft_ops
        return draft_ops.tree_attention(s["q"], s["keys"], s["values"], s["table"], s["seq_lens"], s["cu_rows"], s["visible"], out=s["out"],
                                        workspace=s["workspace"])
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, scale = heads // kv_heads, dim ** -0.5
    for b, (c, n, lo) in enumerate(zip(s["ctx"], s["nodes"], s["starts"])):
        if n == 0:
            continue
        q = s["q"][lo: lo + n].float().view(n, kv_heads, group, dim).transpose(0, 1).reshape(kv_heads, n * group, dim) * scale
        pages = s["table"][b, : _pages(c + n)].long()
        k, v = (s[name][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, : c + n].float() for name in ("keys", "values"))
        scores = torch.matmul(q, k.transpose(1, 2)).view(kv_heads, n, group, c + n)
        place = torch.arange(n, device=DEV)
        if s["visible"] is None:
            seen = place[None, :] <= place[:, None]
        else:
            seen = (s["visible"][lo: lo + n][:, place // 32] >> (place % 32)[None, :] & 1) != 0
        scores[..., c:] = scores[..., c:].masked_fill(~seen[None, :, None, :], -math.inf)
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        weights = (weights / weights.sum(-1, keepdim=True)).view(kv_heads, n * group, c + n)
        s["out"][lo: lo + n] = torch.matmul(weights, v).view(kv_heads, n, group, dim).transpose(0, 1).reshape(n, heads, dim).to(s["out"].dtype)
    return s["out"]


def _run_logits(s):
    case = s["case"]
    if own:
        from cacheir_b200 import draft_ops
        history = draft_ops.TokenHistory(s["said"], s["said_lens"], s["prompt_lens"]) if case["penalties"] else None
        drafts = draft_ops.DraftedTokens(s["draft_ids"], s["visible"], s["cu_rows"]) if case["drafts"] else None
        return draft_ops.adjust_logits(s["logits"], row_seq=s["row_seq"], history=history, drafts=drafts, repetition=s.get("repetition"),
                                       frequency=s.get("frequency"), presence=s.get("presence"), bias_ids=s.get("bias_ids"),
                                       bias_values=s.get("bias_values"), allowed=s.get("allowed"), out=s["out"])
    rows, vocab, row_seq = case["rows"], case["vocab"], s["row_seq"].long()
    x = s["logits"].float()
    if case["penalties"]:
        place = torch.arange(s["said"].shape[1], device=DEV)[None, :]
        in_prompt = (place < s["prompt_lens"][:, None]).int()
        in_answer = (place < s["said_lens"][:, None]).int() - in_prompt
        said = s["said"].long()
        prompt, answer = (torch.zeros(case["sequences"], vocab, dtype=torch.int32, device=DEV).scatter_add_(1, said, w) for w in (in_prompt, in_answer))
        count, known = answer[row_seq], prompt[row_seq] > 0
        if case["drafts"]:
            most = max(s["nodes"])
            at = torch.arange(most, device=DEV)
            seen = (s["visible"][:, at // 32] >> (at % 32)[None, :] & 1)
            ids = s["draft_ids"][(s["cu_rows"].long()[row_seq][:, None] + at[None, :]).clamp(max=rows - 1)]
            count = count.scatter_add(1, ids, seen.int())
        known = known | (count > 0)
        rep = s["repetition"][row_seq][:, None]
        x = torch.where(known, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][row_seq][:, None] * count - s["presence"][row_seq][:, None] * (count > 0)
    if case["bias"]:
        x = x.scatter_add(1, s["bias_ids"].long()[row_seq], s["bias_values"][row_seq])
    if case["grammar"]:
        at = torch.arange(vocab, device=DEV)
        x = x.masked_fill((s["allowed"][:, at // 32] >> (at % 32)[None, :] & 1) == 0, -math.inf)
    s["out"].copy_(x)
    return s["out"]


def _run_drafts(s):
    case = s["case"]
    if own:
        from cacheir_b200 import draft_ops
        tree = draft_ops.map_drafts(s["parents"], s["seq_lens"], s["tokens"], s["tree"])
        accepted = draft_ops.accept_drafts(s["chosen"], s["draft_ids"], s["parents"], s["seq_lens"], s["tokens"], s["accepted"])
        draft_ops.keep_accepted(accepted, s["tokens"], s["handle"])
        return {"positions": tree.positions, "visible": tree.visible, "counts": accepted.counts, "rows": accepted.rows, "next_ids": accepted.next_ids,
                "keep_lens": accepted.keep_lens, "keys": s["keys"], "values": s["values"]}
    cu, row_seq, most, depth = s["cu_rows"].long(), s["row_seq"].long(), s["most"], s["depth"]
    nodes = cu[1:] - cu[:-1]
    at = torch.arange(most, device=DEV)
    flat = (cu[:-1, None] + at[None, :]).clamp(max=len(row_seq) - 1)             # [sequences, most]
    real = at[None, :] < nodes[:, None]
    parents = torch.where(real, s["parents"].long()[flat], -1)
    # rows seen, and from them depths: a step up for every row at once
    seen = (at[None, :, None] == at[None, None, :]).expand(len(nodes), most, most).clone()
    up = parents
    for _ in range(most):
        seen |= (up[:, :, None] == at[None, None, :])
        up = torch.where(up >= 0, torch.gather(parents, 1, up.clamp(min=0)), -1)
    place = torch.arange(len(row_seq), device=DEV) - cu[row_seq]
    lines = seen[row_seq, place]
    positions = (s["seq_lens"].long() - nodes)[row_seq] + lines.sum(-1) - 1
    bits = torch.zeros(len(row_seq), s["words"], dtype=torch.int64, device=DEV)
    bits.scatter_add_(1, (at // 32)[None, :].expand(len(row_seq), most), lines.long() << (at % 32)[None, :])
    visible = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    # the accepted path, a step down for every sequence at once
    ids, chosen = s["draft_ids"][flat], s["chosen"][flat]
    alive = nodes > 0
    path = torch.full((len(nodes), depth), -1, dtype=torch.int64, device=DEV)
    path[:, 0] = torch.where(alive, cu[:-1], -1)
    counts, now = alive.long(), torch.zeros_like(nodes)
    next_ids = torch.where(alive, chosen[:, 0], -1)
    for i in range(1, min(depth, s["longest"])):
        match = real & (parents == now[:, None]) & (ids == next_ids[:, None]) & alive[:, None]
        alive = match.any(-1)
        now = torch.where(alive, match.int().argmax(-1), now)
        path[:, i] = torch.where(alive, cu[:-1] + now, -1)
        counts += alive
        next_ids = torch.where(alive, torch.gather(chosen, 1, now[:, None])[:, 0], next_ids)
    seq, step = (path >= 0).nonzero(as_tuple=True)
    source, target = s["slots"][path[seq, step]].long(), s["slots"][cu[seq] + step].long()
    for pool in (s["keys"], s["values"]):
        pool[:, target // PAGE, :, target % PAGE] = pool[:, source // PAGE, :, source % PAGE]
    return {"positions": positions.to(torch.int32), "visible": visible, "counts": counts.to(torch.int32), "rows": path.to(torch.int32), "next_ids": next_ids,
            "keep_lens": (s["seq_lens"].long() - nodes + counts).to(torch.int32), "keys": s["keys"], "values": s["values"]}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "float32" else 2
    if kind == "norms":
        rows, heads = case["rows"] - case["padded"], case["heads"] + case["kv_heads"]
        return {"bytes": 2 * size * rows * (heads + case["kv_heads"]) * case["dim"] + 8 * case["rows"], "flops": rows * heads * (4 * case["dim"] + 3 * case["rot"])}
    if kind == "attention":
        ctx, nodes = _lens(case)
        keys, pairs = sum(c + n for c, n in zip(ctx, nodes) if n), sum(n * (c + n) for c, n in zip(ctx, nodes))
        mask = 0 if case["chain"] else 4 * sum(nodes) * ((max(nodes) + 31) // 32)
        return {"bytes": 2 * size * keys * case["kv_heads"] * case["dim"] + 2 * size * sum(nodes) * case["heads"] * case["dim"] + 4 * keys // PAGE + mask,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if kind == "logits":
        values = case["rows"] * case["vocab"]
        return {"bytes": 2 * size * values + case["sequences"] * (4 * case["history"] * case["penalties"] + 8 * case["bias"]) + values // 8 * case["grammar"],
                "flops": 2 * values}
    ctx, nodes = _lens(case)
    # rows' parents, tokens, picks in, positions and masks out; about one row in 25 moves
    return {"bytes": sum(nodes) * (4 + 8 + 8 + 4 + 4 * ((max(nodes) + 31) // 32)) + 2 * 2 * size * case["layers"] * (sum(nodes) // 25) * case["kv_heads"] * case["dim"],
            "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"norms": _exact_norms, "attention": _exact_attention, "logits": _exact_logits, "drafts": _exact_drafts}[case["kind"]](case, s)


def _exact_norms(case, s):
    live = case["rows"] - case["padded"]
    q, k_cache, v_cache = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
    angle = s["positions"][:live].double()[:, None] * s["freq"][None, :]
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]      # complex numbers

    def turned(x, weight):
        x = x[:live].double()
        x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / case["dim"] + EPS) * (weight.double() + case["offset"])
        head, rest, half = x[..., : case["rot"]], x[..., case["rot"]:], case["rot"] // 2
        pairs = head.unflatten(-1, (half, 2)) if case["layout"] == "interleaved" else head.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat([z.flatten(-2) if case["layout"] == "interleaved" else z.transpose(-1, -2).flatten(-2), rest], dim=-1)
    q[:live] = turned(s["q"], s["q_weight"])
    flat = s["slots"][:live].long()
    for cache, rows in ((k_cache, turned(s["k"], s["k_weight"])), (v_cache, s["v"][:live].double())):
        lines = cache.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"]).clone()
        lines[flat] = rows
        cache.copy_(lines.view(cache.shape[0], PAGE, case["kv_heads"], case["dim"]).transpose(1, 2))
    return {"q": q, "k_cache": k_cache, "v_cache": v_cache}


def _exact_attention(case, s):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    out = s["out"].double()
    words = None if s["visible"] is None else s["visible"].tolist()
    for b, (c, n, lo) in enumerate(zip(s["ctx"], s["nodes"], s["starts"])):
        if n == 0:
            continue
        place = torch.arange(c + n, device=DEV)
        lines = s["table"][b].long()[place // PAGE], place % PAGE
        hidden = torch.tensor([[t >= c and not (t - c <= i if words is None else words[lo + i][(t - c) // 32] >> (t - c) % 32 & 1) for t in range(max(c, 0), c + n)]
                               for i in range(n)], device=DEV)
        for h in range(kv_heads):
            k, v = (s[name][lines[0], h, lines[1]].double() for name in ("keys", "values"))                 # [c + n, dim]
            q = s["q"][lo: lo + n, h * (heads // kv_heads): (h + 1) * (heads // kv_heads)].double()
            scores = torch.einsum("ngd,td->ngt", q, k) / math.sqrt(dim)
            scores[..., c:].masked_fill_(hidden[:, None, :], -math.inf)
            out[lo: lo + n, h * (heads // kv_heads): (h + 1) * (heads // kv_heads)] = torch.einsum("ngt,td->ngd", torch.softmax(scores, dim=-1), v)
    return out


def _exact_logits(case, s):
    vocab, lines = case["vocab"], []
    for b, (n, lo) in enumerate(zip(s["nodes"], s["starts"])):
        if case["penalties"]:
            size, first = int(s["said_lens"][b]), int(s["prompt_lens"][b])
            prompt = torch.bincount(s["said"][b, :first], minlength=vocab)
            answer = torch.bincount(s["said"][b, first:size], minlength=vocab)
            rep, freq, pres = (float(s[name][b]) for name in ("repetition", "frequency", "presence"))
        for i in range(n):
            x = s["logits"][lo + i].double()
            if case["penalties"]:
                count = answer
                if case["drafts"]:
                    count = answer + torch.bincount(s["draft_ids"][[lo + j for j in s["trees"][b][i]]], minlength=vocab)
                known = ((prompt > 0) | (count > 0)).double()
                x = x * torch.where(x > 0, 1.0 / rep, rep) * known + x * (1.0 - known)
                x = x - freq * count.double() - pres * count.clamp(max=1).double()
            if case["bias"]:
                x[s["bias_ids"][b].long()] += s["bias_values"][b].double()
            if case["grammar"]:
                bits = (s["allowed"][lo + i][:, None] >> torch.arange(32, device=DEV)[None, :] & 1).flatten()[:vocab]
                x[bits == 0] = -math.inf
            lines.append(x)
    return torch.stack(lines)


def _exact_drafts(case, s):
    """The same by walking the sequences one by one on the host."""
    ids, chosen, slots, lens = (s[name].tolist() for name in ("draft_ids", "chosen", "slots", "seq_lens"))
    positions, visible, counts, rows, next_ids, keep, moves = [], [], [], [], [], [], []
    for tree, lo, length in zip(s["trees"], s["starts"], lens):
        front = length - len(tree)
        seen = _ancestors(tree)
        positions += [front + len(line) - 1 for line in seen]
        visible += _words(seen, s["words"])
        path, pick = [], -1
        at = 0 if tree else None
        while at is not None:
            path.append(at)
            pick = chosen[lo + at]
            at = next((j for j, p in enumerate(tree) if p == at and ids[lo + j] == pick), None)
        moves += [(slots[lo + j], slots[lo + i]) for i, j in enumerate(path)]
        counts.append(len(path))
        rows.append([lo + j for j in path] + [-1] * (s["depth"] - len(path)))
        next_ids.append(pick)
        keep.append(front + len(path))
    pools = []
    for pool in (s["keys"], s["values"]):
        lines = pool.double().transpose(2, 3).reshape(case["layers"], -1, case["kv_heads"], case["dim"])
        lines[:, [to for _, to in moves]] = lines[:, [at for at, _ in moves]]
        pools.append(lines.view(case["layers"], -1, PAGE, case["kv_heads"], case["dim"]).transpose(2, 3))
    return {"positions": _i32(positions), "visible": _i32(visible), "counts": _i32(counts), "rows": _i32(rows),
            "next_ids": torch.tensor(next_ids, device=DEV), "keep_lens": _i32(keep), "keys": pools[0], "values": pools[1]}
