"""What is measured of the operators of batches whose requests share prompts, through the framework's public entry points.

Four kinds of case, in the order in which a step uses them, each over the range of sizes that `draw` spans:

  tables     pages for new tokens, the map from rows to page slots, and taking tokens back (`extend_page_tables`, `shrink_page_tables`)
  rotary     rotary positions and the append to the page pool by slot (`rotary_append`)
  attention  decode attention of groups of requests with a common prefix (`shared_prefix_attention`)
  logprobs   log probabilities of given tokens with entropy and top alternatives (`token_logprobs`)

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
YARN = (16.0, 8192.0, 32.0, 1.0)            # stretched by 16 from 8192 positions; pairs of 32 and of 1 turns bound the ramp


def listed():
    return [
        # a decode step of a running batch: a page boundary now and then, nothing but latency
        dict(name="tables decode step", kind="tables", sequences=32, ctx_min=1, ctx_max=4096, new_min=1, new_max=1, rows=32, lens=1),
        # prompts of many new requests in one pass
        dict(name="tables prompts", kind="tables", sequences=1024, ctx_min=0, ctx_max=2000, new_min=0, new_max=255, rows=140001, lens=3),
        # a decode step's heads
        dict(name="rotary decode", kind="rotary", rows=32, heads=32, kv_heads=8, dim=128, rot=128, layout="interleaved", yarn=False, far=8192,
             padded=0, dtype="float16"),
        # a prompt of odd length in a padded bucket, half of every head rotated
        dict(name="rotary prompt", kind="rotary", rows=2048, heads=32, kv_heads=8, dim=128, rot=64, layout="half", yarn=False, far=8192,
             padded=47, dtype="bfloat16"),
        # a pass over prompts with far positions, frequencies stretched
        dict(name="rotary far", kind="rotary", rows=16384, heads=64, kv_heads=8, dim=128, rot=128, layout="half", yarn=True, far=1000000,
             padded=0, dtype="float16"),
        # two answers to one short question
        dict(name="attention pair", kind="attention", heads=32, kv_heads=8, dim=128, dtype="float16", groups="2x333", tail_min=1, tail_max=40, lens=4),
        # a server whose requests open with the same instructions, as many as its decode batch
        dict(name="attention instructions", kind="attention", heads=32, kv_heads=8, dim=128, dtype="float16", groups="32x2048", tail_min=16,
             tail_max=512, lens=5),
        # eight samples of each of sixteen prompts of ragged lengths
        dict(name="attention samples", kind="attention", heads=64, kv_heads=8, dim=128, dtype="bfloat16",
             groups=",".join(f"8x{n}" for n in (517, 4000, 1024, 33, 2999, 1500, 777, 3500, 16, 2048, 1333, 250, 4095, 640, 1999, 900)),
             tail_min=1, tail_max=700, lens=6),
        # many questions about one long document
        dict(name="attention document", kind="attention", heads=32, kv_heads=8, dim=128, dtype="float16", groups="64x32768", tail_min=32,
             tail_max=256, lens=7),
        # the sampled token of one request, with alternatives
        dict(name="logprobs one", kind="logprobs", rows=1, vocab=128256, dtype="float16", top=5, masked=False, temperature=1.0),
        # a batch of constrained requests over an odd vocabulary, many alternatives
        dict(name="logprobs batch", kind="logprobs", rows=64, vocab=50001, dtype="float32", top=20, masked=True, temperature=0.7),
        # scoring a prompt: every position's logits
        dict(name="logprobs prompt", kind="logprobs", rows=2048, vocab=128256, dtype="bfloat16", top=0, masked=False, temperature=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Kinds in the shares that the listed cases have; sizes over their whole range."""
    kind = rng.choice(["tables"] * 3 + ["rotary"] * 3 + ["attention"] * 4 + ["logprobs"] * 2)
    if kind == "tables":
        sequences, top = _log(rng, 1, 1024), _log(rng, 1, 255)
        ctx = _log(rng, 1, 20000 if sequences <= 128 else 2000)
        low = rng.choice([0, 1, -top])
        # (a lowest count of new tokens below zero: as many sequences again that get none)
        return dict(kind=kind, sequences=sequences, ctx_min=rng.choice([0, ctx // 2]), ctx_max=ctx, new_min=min(low, top), new_max=top,
                    rows=min(140001, sequences * top + rng.choice([0, 1, 100])), lens=rng.randrange(1 << 30))
    if kind == "rotary":
        heads, kv_heads, dim = rng.choice(HEADS)
        rows = _log(rng, 1, 16384 * 64 * 128 // (heads * dim) if heads * dim > 8192 else 16384)
        return dict(kind=kind, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, dim // 4]),
                    layout=rng.choice(["interleaved", "half"]), yarn=rng.random() < 0.5, far=_log(rng, 1000, 1000000),
                    padded=rng.choice([0, rows // 9]), dtype=rng.choice(["float16", "bfloat16"] if rows > 4096 else ["float16", "bfloat16", "float32"]))
    if kind == "attention":
        heads, kv_heads, dim = rng.choice(HEADS)
        while True:
            parts = []
            for _ in range(rng.choice([1, 1, 1, 2, _log(rng, 2, 16)])):
                parts.append((_log(rng, 1, 64), _log(rng, 16, 32768)))
            tail = _log(rng, 1, 1024)
            case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["float16", "bfloat16"]),
                        groups=",".join(f"{n}x{p}" for n, p in parts), tail_min=rng.choice([0, 1, max(1, tail // 2)]), tail_max=tail,
                        lens=rng.randrange(1 << 30))
            cost = work(case)
            most = work(next(c for c in listed() if c["name"] == "attention document"))
            if cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]:
                return case
    vocab = rng.choice([32768, 128256, 50001, _log(rng, 1000, 131072)])
    dtype = rng.choice(list(DTYPES))
    rows = _log(rng, 1, 2048 if dtype != "float32" else 1024)
    return dict(kind=kind, rows=min(rows, 2048 * 128256 // vocab), vocab=min(vocab, 128256), dtype=dtype, top=rng.choice([0, 1, 5, 20, 32]) if rows <= 256 else rng.choice([0, 0, 1, 5]),
                masked=rng.random() < 0.3, temperature=rng.choice([1.0, 1.0, 0.7]))


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
    return (max(tokens, 0) + PAGE - 1) // PAGE


def _table_lens(case):
    """(tokens held, new tokens) of every sequence; no more new ones than there are rows for."""
    rng = random.Random(case["lens"])
    held = [rng.randint(case["ctx_min"], case["ctx_max"]) for _ in range(case["sequences"])]
    new, room = [], case["rows"]
    for _ in held:
        n = max(0, min(rng.randint(case["new_min"], case["new_max"]), room))
        new.append(n)
        room -= n
    return held, new


def _attention_lens(case):
    """(rows, common tokens) of every group, and the tokens of every row behind them."""
    rng = random.Random(case["lens"])
    groups = [tuple(int(v) for v in part.split("x")) for part in case["groups"].split(",")]
    tails = [[rng.randint(case["tail_min"], case["tail_max"]) for _ in range(n)] for n, _ in groups]
    return groups, tails


def _frequencies(case):
    """Angle per position of every pair, and what cosine and sine are multiplied by."""
    dims = case["rot"]
    freq = BASE ** (-2.0 * torch.arange(dims // 2, dtype=torch.float64) / dims)
    if not case["yarn"]:
        return freq, 1.0
    factor, original, fast, slow = YARN
    pair = [dims * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(BASE)) for turns in (fast, slow)]
    lo, hi = max(math.floor(pair[0]), 0.0), min(math.ceil(pair[1]), dims - 1.0)
    ramp = ((torch.arange(dims // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return freq / factor * ramp + freq * (1.0 - ramp), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    state = {"case": case}
    kind = case["kind"]
    if kind == "tables":
        held, new = _table_lens(case)
        width = max(_pages(h + n) for h, n in zip(held, new)) + 1
        used, most = sum(_pages(h) for h in held), sum(_pages(h + n) for h, n in zip(held, new))
        ids = torch.randperm(most + 64, device=DEV, generator=_gen(seed, "ids")).to(torch.int32)
        count = torch.tensor([_pages(h) for h in held], device=DEV)
        place = torch.arange(width, device=DEV)
        first = torch.cumsum(count, 0) - count
        table = torch.where(place[None, :] < count[:, None], ids[(first[:, None] + place[None, :]).clamp(max=most + 63)], 0).to(torch.int32)
        free = torch.zeros(most + 128, dtype=torch.int32, device=DEV)
        free[: most + 64 - used] = ids[used:]
        state.update(table=table, seq_lens=_i32(held), keep=_i32(held), new_lens=_i32(new), free=free, count=_i32([most + 64 - used]),
                     total=sum(new), new_pages=most - used)
        if own:
            from cacheir_b200 import serving_ops
            state["tokens"] = serving_ops.token_map(case["rows"], case["sequences"], DEV)
        else:
            rows = case["rows"]
            state.update(positions=torch.empty(rows, dtype=torch.int32, device=DEV), row_seq=torch.empty(rows, dtype=torch.int32, device=DEV),
                         slots=torch.empty(rows, dtype=torch.int32, device=DEV))
    elif kind == "rotary":
        rows, heads, kv_heads, dim, dtype = case["rows"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        qkv = _randn(seed, "qkv", rows, (heads + 2 * kv_heads) * dim).to(dtype)
        slots_total = (rows + PAGE - 1) // PAGE + 2
        slots = torch.randperm(slots_total * PAGE, device=DEV, generator=_gen(seed, "slots"))[:rows].to(torch.int32)
        if case["padded"]:
            slots[rows - case["padded"]:] = -1
        freq, factor = _frequencies(case)
        state.update(q=qkv[:, : heads * dim].view(rows, heads, dim), k=qkv[:, heads * dim: (heads + kv_heads) * dim].view(rows, kv_heads, dim),
                     v=qkv[:, (heads + kv_heads) * dim:].view(rows, kv_heads, dim), slots=slots, freq=freq.to(DEV), factor=factor,
                     positions=_randint(seed, "positions", 0, case["far"], rows).to(torch.int32),
                     k_cache=torch.zeros(slots_total, kv_heads, PAGE, dim, dtype=dtype, device=DEV),
                     v_cache=torch.zeros(slots_total, kv_heads, PAGE, dim, dtype=dtype, device=DEV),
                     q_out=torch.zeros(rows, heads, dim, dtype=dtype, device=DEV))
        if own:
            from cacheir_b200 import serving_ops
            yarn = YARN if case["yarn"] else None
            state["rule"] = serving_ops.rotary_rule(case["rot"], BASE, layout=case["layout"], yarn=yarn, device=DEV)
    elif kind == "attention":
        heads, kv_heads, dim, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        groups, tails = _attention_lens(case)
        lens = [p + t for (_, p), tail in zip(groups, tails) for t in tail]
        width = max(_pages(n) for n in lens) + 1
        shared = [p // PAGE for _, p in groups]            # whole pages are shared, the page that a prefix ends in is each row's own
        total = sum(shared) + sum(_pages(p + t) - s for (_, p), tail, s in zip(groups, tails, shared) for t in tail) + 3
        order = torch.randperm(total, device=DEV, generator=_gen(seed, "pages")).to(torch.int32)
        table = torch.zeros(len(lens), width, dtype=torch.int32, device=DEV)
        pools = [_randn(seed, name, total, kv_heads, PAGE, dim).to(dtype) for name in ("keys", "values")]
        used = row = 0
        for (n, p), tail, s in zip(groups, tails, shared):
            prefix, used = order[used: used + s], used + s
            first = None
            for t in tail:
                mine = _pages(p + t) - s
                table[row, :s] = prefix
                table[row, s: s + mine] = order[used: used + mine]
                if p % PAGE:                                # the tokens behind the last whole page are the same in every row
                    if first is None:
                        first = order[used].long()
                    else:
                        for pool in pools:
                            pool[order[used].long(), :, : p % PAGE] = pool[first, :, : p % PAGE]
                used += mine
                row += 1
        starts = [0]
        for n, _ in groups:
            starts.append(starts[-1] + n)
        q = _randn(seed, "q", len(lens), (heads + 2 * kv_heads) * dim)[:, : heads * dim].to(dtype).view(len(lens), heads, dim) * 1.5
        state.update(q=q, keys=pools[0], values=pools[1], table=table, seq_lens=_i32(lens), lens=lens, parts=groups, starts=starts,
                     out=torch.empty(len(lens), heads, dim, dtype=dtype, device=DEV))
        if own:
            from cacheir_b200 import serving_ops
            prefix_table = table[torch.tensor(starts[:-1], device=DEV)].contiguous()
            state["groups"] = serving_ops.PrefixGroups(rows=_i32(starts), table=prefix_table, lens=_i32([p for _, p in groups]))
            need = serving_ops.shared_prefix_workspace_bytes(len(lens), heads, dim)
            state["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = _randn(seed, "logits", rows, vocab)
        logits.mul_(2.5)
        tokens = _randint(seed, "tokens", 0, vocab, rows)
        # most tokens that are asked for are likely ones
        likely = _randint(seed, "likely", 0, 4, rows) > 0
        logits[torch.arange(rows, device=DEV), tokens] += likely * (8.0 + 2.0 * _randn(seed, "lift", rows))
        if case["masked"]:
            logits.masked_fill_(torch.rand(rows, vocab, device=DEV, generator=_gen(seed, "mask")) < 0.4, -math.inf)
        state.update(logits=logits.to(DTYPES[case["dtype"]]), tokens=tokens)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    return {"tables": _run_tables, "rotary": _run_rotary, "attention": _run_attention, "logprobs": _run_logprobs}[kind](state)


def _run_tables(s):
    """A step's new tokens get their pages, and all of them are taken back (what a speculative step does with refused drafts)."""
    if own:
        from cacheir_b200 import serving_ops
        t = serving_ops.extend_page_tables(s["table"], s["seq_lens"], s["new_lens"], s["free"], s["count"], s["tokens"], page_size=PAGE)
        serving_ops.shrink_page_tables(s["table"], s["seq_lens"], s["keep"], s["free"], s["count"], t.status, page_size=PAGE)
        return {"positions": t.positions, "row_seq": t.row_seq, "slots": t.slots, "cu_rows": t.cu_rows, "table": s["table"],
                "seq_lens": s["seq_lens"], "free": s["free"], "count": s["count"]}
    table, lens, new, free, count = s["table"], s["seq_lens"], s["new_lens"], s["free"], s["count"]
    total, pages = s["total"], s["new_pages"]
    before, after = (lens + PAGE - 1) // PAGE, (lens + new + PAGE - 1) // PAGE
    need = after - before
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), need, output_size=pages)
    nth = torch.arange(pages, device=DEV)
    page = free[(count - 1 - nth).long()]
    table[seq, before[seq] + nth - (torch.cumsum(need, 0) - need)[seq]] = page
    ends = torch.cumsum(new, 0)
    cu_rows = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    row_seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), new, output_size=total)
    positions = lens[row_seq] + torch.arange(total, device=DEV) - cu_rows[row_seq]
    s["row_seq"].fill_(-1)
    s["positions"].fill_(0)
    s["slots"].fill_(-1)
    s["row_seq"][:total] = row_seq.to(torch.int32)
    s["positions"][:total] = positions.to(torch.int32)
    s["slots"][:total] = table[row_seq, positions // PAGE] * PAGE + (positions % PAGE).to(torch.int32)
    lens += new
    count -= pages
    # taking back: the pages behind the kept tokens return, the first one on top
    keep = torch.minimum(lens, s["keep"])
    first, gone = (keep + PAGE - 1) // PAGE, (lens + PAGE - 1) // PAGE - (keep + PAGE - 1) // PAGE
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), gone, output_size=pages)
    back = table[seq, first[seq] + nth - (torch.cumsum(gone, 0) - gone)[seq]]
    free[(count + pages - 1 - nth).long()] = back
    count += pages
    lens.copy_(keep)
    return {"positions": s["positions"], "row_seq": s["row_seq"], "slots": s["slots"], "cu_rows": cu_rows, "table": table, "seq_lens": lens,
            "free": free, "count": count}


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


def _run_rotary(s):
    if own:
        from cacheir_b200 import serving_ops
        serving_ops.rotary_append(s["q"], s["k"], s["v"], s["rule"], s["positions"], slots=s["slots"], k_cache=s["k_cache"], v_cache=s["v_cache"],
                                  q_out=s["q_out"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    case = s["case"]
    rows = case["rows"] - case["padded"]
    angle = s["positions"][:rows].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    q, k = (_rotate(s[name][:rows].float(), cos, sin, case["rot"], case["layout"]).to(s[name].dtype) for name in ("q", "k"))
    s["q_out"][:rows] = q
    slot = s["slots"][:rows].long()
    s["k_cache"][slot // PAGE, :, slot % PAGE] = k
    s["v_cache"][slot // PAGE, :, slot % PAGE] = s["v"][:rows]
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_attention(s):
    if own:
        from cacheir_b200 import serving_ops
        return serving_ops.shared_prefix_attention(s["q"], s["keys"], s["values"], s["table"], s["seq_lens"], s["groups"], out=s["out"],
                                                   workspace=s["workspace"])
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, scale = heads // kv_heads, dim ** -0.5
    for (n, p), lo in zip(s["parts"], s["starts"]):
        q = s["q"][lo: lo + n].float().view(n, kv_heads, group, dim).transpose(0, 1) * scale          # [kv heads, n, group, dim]
        pages = s["table"][lo, : _pages(p)].long()
        k, v = (s[name][pages].float().transpose(0, 1).reshape(kv_heads, -1, dim)[:, :p] for name in ("keys", "values"))
        common = torch.matmul(q.reshape(kv_heads, n * group, dim), k.transpose(1, 2)).view(kv_heads, n, group, p)
        lens = s["seq_lens"][lo: lo + n]
        most = max(s["lens"][lo: lo + n]) - p
        place = p + torch.arange(most, device=DEV)
        at = s["table"][lo: lo + n][:, (place // PAGE).long()].long()                                       # [n, most]
        kt, vt = (s[name][at, :, (place % PAGE)[None, :]].float().permute(2, 0, 1, 3) for name in ("keys", "values"))     # [kv heads, n, most, dim]
        rest = torch.matmul(q, kt.transpose(2, 3)).masked_fill((place[None, :] >= lens[:, None])[None, :, None, :], -math.inf)
        scores = torch.cat([common, rest], dim=-1)
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        weights = weights / weights.sum(-1, keepdim=True)
        out = torch.matmul(weights[..., :p].reshape(kv_heads, n * group, p), v).view(kv_heads, n, group, dim)
        out = out + torch.matmul(weights[..., p:], vt)
        s["out"][lo: lo + n] = out.transpose(0, 1).reshape(n, heads, dim).to(s["out"].dtype)
    return s["out"]


def _run_logprobs(s):
    case = s["case"]
    if own:
        from cacheir_b200 import serving_ops
        r = serving_ops.token_logprobs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        return {**out, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if case["top"] else out
    x = s["logits"].float()
    if case["temperature"] != 1.0:
        x = x / case["temperature"]
    x = x - x.amax(-1, keepdim=True)
    weight = torch.exp(x)
    total = weight.sum(-1, keepdim=True)
    log_total = torch.log(total)
    out = {"logprobs": (torch.gather(x, 1, s["tokens"][:, None]) - log_total)[:, 0],
           "entropy": (log_total - torch.where(weight > 0, weight * x, 0.0).sum(-1, keepdim=True) / total)[:, 0]}
    if case["top"]:
        # ties go to the lowest index: the value's bits as an ordered integer, the index behind them
        bits = (s["logits"].float() + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = bits * (1 << 32) + ((1 << 32) - 1 - torch.arange(case["vocab"], device=DEV))
        ids = (1 << 32) - 1 - (torch.topk(key, case["top"], dim=-1).values & ((1 << 32) - 1))
        out.update(top_ids=ids, top_logprobs=torch.gather(x, 1, ids) - log_total)
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "tables":
        held, new = _table_lens(case)
        pages = sum(_pages(h + n) - _pages(h) for h, n in zip(held, new))
        # lengths in and out twice, kept lengths, row starts; page ids out of the stack into the tables and back; three numbers per row
        return {"bytes": 4 * (7 * len(held) + 4 * pages + 3 * case["rows"]), "flops": 0}
    if kind == "rotary":
        size = 4 if case["dtype"] == "float32" else 2
        rows = case["rows"] - case["padded"]
        values = rows * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * size * values + 8 * case["rows"], "flops": 3 * rows * (case["heads"] + case["kv_heads"]) * case["rot"]}
    if kind == "attention":
        groups, tails = _attention_lens(case)
        keys = sum(p for _, p in groups) + sum(map(sum, tails))
        pairs = sum(n * p for n, p in groups) + sum(map(sum, tails))
        rows = sum(n for n, _ in groups)
        return {"bytes": 2 * 2 * keys * case["kv_heads"] * case["dim"] + 2 * 2 * rows * case["heads"] * case["dim"] + 4 * keys // PAGE,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["rows"] * (size * case["vocab"] + 16 + 12 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "tables":
        return _exact_tables(case, s)
    if kind == "rotary":
        live = case["rows"] - case["padded"]
        q, k_cache, v_cache = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
        angle = s["positions"][:live].double()[:, None] * s["freq"][None, :]
        turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None, :]      # complex numbers

        def turned(x):
            x = x[:live].double()
            head, rest, half = x[..., : case["rot"]], x[..., case["rot"]:], case["rot"] // 2
            pairs = head.unflatten(-1, (half, 2)) if case["layout"] == "interleaved" else head.unflatten(-1, (2, half)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            head = z.flatten(-2) if case["layout"] == "interleaved" else z.transpose(-1, -2).flatten(-2)
            return torch.cat([head, rest], dim=-1)
        q[:live] = turned(s["q"])
        flat = s["slots"][:live].long()
        for cache, rows in ((k_cache, turned(s["k"])), (v_cache, s["v"][:live].double())):
            lines = cache.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"]).clone()
            lines[flat] = rows
            cache.copy_(lines.view(cache.shape[0], PAGE, case["kv_heads"], case["dim"]).transpose(1, 2))
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    if kind == "attention":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        out = torch.zeros(len(s["lens"]), heads, dim, dtype=torch.float64, device=DEV)
        for row, length in enumerate(s["lens"]):
            if length == 0:
                continue
            place = torch.arange(length, device=DEV)
            lines = s["table"][row].long()[place // PAGE], place % PAGE
            k, v = (s[name][lines[0], :, lines[1]].double() for name in ("keys", "values"))                 # [length, kv heads, dim]
            q = s["q"][row].double().view(kv_heads, heads // kv_heads, dim)
            p = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(dim), dim=-1)
            out[row] = torch.einsum("hgt,thd->hgd", p, v).reshape(heads, dim)
        return out
    logp, entropy, ids, top = [], [], [], []
    for lo in range(0, case["rows"], 128):
        x = s["logits"][lo: lo + 128].double() / case["temperature"]
        lp = x - torch.logsumexp(x, dim=-1, keepdim=True)
        logp.append(lp.gather(1, s["tokens"][lo: lo + 128, None])[:, 0])
        entropy.append(-(torch.exp(lp) * torch.where(lp == -math.inf, 0.0, lp)).sum(-1))
        if case["top"]:
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
            ids.append(order)
            top.append(lp.gather(1, order))
    out = {"logprobs": torch.cat(logp), "entropy": torch.cat(entropy)}
    return {**out, "top_ids": torch.cat(ids), "top_logprobs": torch.cat(top)} if case["top"] else out


def _exact_tables(case, s):
    """The same by walking the sequences one by one on the host."""
    table, free = s["table"].tolist(), s["free"].tolist()
    held, new = _table_lens(case)
    count, cu, positions, row_seq, slots = int(s["count"]), [0], [], [], []
    start = count
    for b, (h, n) in enumerate(zip(held, new)):
        for t in range(h, h + n):
            if t % PAGE == 0:
                count -= 1
                table[b][t // PAGE] = free[count]
            positions.append(t)
            row_seq.append(b)
            slots.append(table[b][t // PAGE] * PAGE + t % PAGE)
        cu.append(len(positions))
    behind = case["rows"] - len(positions)
    return {"positions": _i32(positions + [0] * behind), "row_seq": _i32(row_seq + [-1] * behind), "slots": _i32(slots + [-1] * behind),
            "cu_rows": _i32(cu), "table": _i32(table), "seq_lens": _i32(held), "free": _i32(free), "count": _i32([start])}
