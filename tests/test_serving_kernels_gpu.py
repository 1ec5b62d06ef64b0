"""Operators of batches that share prompts against plain statements of them in 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # a rounding, relative to the value


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    from cacheir_b200 import _lib

    yield
    assert _lib.load_group("serving").cacheir_b200_serving_device_status(1) == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, device=DEV, generator=_gen(seed)).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- page tables -----------------------------------------------------------------------------------------------------
class Book:
    """The page walk on the host, token by token."""

    def __init__(self, lens, width, page, spare, seed):
        rng = random.Random(seed)
        pages = [(n + page - 1) // page for n in lens]
        ids = list(range(sum(pages) + spare))
        rng.shuffle(ids)
        self.page, self.lens, self.width = page, list(lens), width
        self.table, at = [], 0
        for n in pages:
            self.table.append(ids[at: at + n] + [0] * (width - n))
            at += n
        self.free = ids[at:]
        self.room = len(ids) + 7

    def tensors(self):
        free = self.free + [0] * (self.room - len(self.free))
        return _i32(self.table), _i32(self.lens), _i32(free), _i32([len(self.free)])

    def extend(self, new):
        rows, cu = [], [0]
        for b, n in enumerate(new):
            for _ in range(max(0, n)):
                pos = self.lens[b]
                if pos % self.page == 0:
                    self.table[b][pos // self.page] = self.free.pop()
                rows.append((pos, b, self.table[b][pos // self.page] * self.page + pos % self.page))
                self.lens[b] += 1
            cu.append(len(rows))
        return rows, cu

    def shrink(self, keep, held):
        back = []
        for b, n in enumerate(keep):
            n = min(max(n, 0), self.lens[b])
            first = max((n + self.page - 1) // self.page, held[b])
            back += self.table[b][first: (self.lens[b] + self.page - 1) // self.page]
            self.lens[b] = n
        self.free += back[::-1]


def _same_book(book, table, lens, free, count):
    assert lens.tolist() == book.lens and int(count) == len(book.free)
    assert free[: len(book.free)].tolist() == book.free
    assert table.tolist() == book.table


@pytest.mark.parametrize("lens,new,page,rows", [
    ([0], [1], 16, 1), ([15], [1], 16, 1), ([16], [1], 16, 4), ([0, 0, 0], [0, 0, 0], 16, 5), ([7, 0, 33, 16], [0, 40, -3, 17], 16, 57),
    ([5, 9, 1], [300, 1, 2], 1, 303), ([5, 100, 64], [11, 0, 700], 64, 800), ([3] * 40, list(range(40)), 5, 780),
    ([i * 37 % 501 for i in range(1500)], [i * 13 % 4 for i in range(1500)], 16, 2250), ([0, 12], [9000, 31], 16, 9100),
    ([i % 33 for i in range(16384)], [1] * 16384, 16, 16390), ([2000] * 3, [5000, 0, 4999], 16, 9999)])
def test_page_tables_follow_the_walk_token_by_token(lens, new, page, rows):
    from cacheir_b200 import serving_ops as S

    width = max((n + max(m, 0) + page - 1) // page for n, m in zip(lens, new)) + 1
    book = Book(lens, width, page, sum((max(m, 0) + page - 1) // page + 1 for m in new), 1)
    table, seq_lens, free, count = book.tensors()
    tokens = S.token_map(rows, len(lens), DEV)
    for t in (tokens.positions, tokens.row_seq, tokens.slots, tokens.cu_rows):
        t.fill_(77)                                       # what an earlier step left
    before = [t.clone() for t in (table, seq_lens, free, count)]
    S.extend_page_tables(table, seq_lens, _i32(new), free, count, tokens, page_size=page)
    want, cu = book.extend(new)
    behind = rows - len(want)
    assert tokens.cu_rows.tolist() == cu and int(tokens.status) == 0
    assert tokens.positions.tolist() == [r[0] for r in want] + [0] * behind
    assert tokens.row_seq.tolist() == [r[1] for r in want] + [-1] * behind
    assert tokens.slots.tolist() == [r[2] for r in want] + [-1] * behind
    _same_book(book, table, seq_lens, free, count)
    # all taken back: the stack is as it was, and the same step again gives the same pages
    slots, taken = tokens.slots.clone(), table.clone()
    S.shrink_page_tables(table, seq_lens, before[1], free, count, tokens.status, page_size=page)
    assert torch.equal(seq_lens, before[1].clamp(min=0)) and torch.equal(free, before[2]) and torch.equal(count, before[3])
    S.extend_page_tables(table, seq_lens, _i32(new), free, count, tokens, page_size=page)
    assert torch.equal(tokens.slots, slots) and torch.equal(table, taken) and int(tokens.status) == 0


@pytest.mark.parametrize("seed", range(6))
def test_page_tables_over_many_steps(seed):
    """Random steps: sequences grow, shrink, end and start over, some of their first pages belonging to others."""
    from cacheir_b200 import serving_ops as S

    rng = random.Random(seed)
    n, page = rng.choice([1, 3, 50, 1100]), rng.choice([1, 7, 16])
    book = Book([rng.randint(0, 40) for _ in range(n)], 100, page, 60 * n, seed)
    held = [rng.randint(0, 2) for _ in range(n)]
    table, seq_lens, free, count = book.tensors()
    tokens, held_pages = S.token_map(n * 12, n, DEV), _i32(held)
    book.lens = [max(length, page * h) for length, h in zip(book.lens, held)]              # (a row holds the pages that it shares)
    seq_lens.copy_(_i32(book.lens))
    for step in range(12):
        new = [rng.choice([0, 1, 1, rng.randint(0, 12)]) if length < 80 else 0 for length in book.lens]
        S.extend_page_tables(table, seq_lens, _i32(new), free, count, tokens, page_size=page)
        rows, cu = book.extend(new)
        assert tokens.slots[: len(rows)].tolist() == [r[2] for r in rows] and tokens.cu_rows.tolist() == cu
        keep = [rng.choice([0 if h == 0 else h * page, length, length - 1, length + 5, length // 2]) for length, h in zip(book.lens, held)]
        keep = [max(k, h * page) for k, h in zip(keep, held)]
        S.shrink_page_tables(table, seq_lens, _i32(keep), free, count, tokens.status, page_size=page, held_pages=held_pages)
        book.shrink(keep, held)
        assert int(tokens.status) == 0
        _same_book(book, table, seq_lens, free, count)
    keep = [0] * n                                        # everybody ends: shared pages stay with their owners
    S.shrink_page_tables(table, seq_lens, _i32(keep), free, count, tokens.status, page_size=page, held_pages=held_pages)
    book.shrink(keep, held)
    _same_book(book, table, seq_lens, free, count)


def test_page_tables_refuse_as_a_whole():
    from cacheir_b200 import serving_ops as S

    book = Book([30, 5, 16], 4, 16, 3, 0)
    table, seq_lens, free, count = book.tensors()
    tokens = S.token_map(64, 3, DEV)
    state = lambda: [t.clone() for t in (table, seq_lens, free, count)]
    before = state()

    def refused(new, status, tokens=tokens, count=count):
        tokens.status.zero_()
        tokens.slots.fill_(5)
        S.extend_page_tables(table, seq_lens, _i32(new), free, count, tokens, page_size=16)
        assert int(tokens.status) == status
        assert tokens.slots.tolist() == [-1] * tokens.slots.numel() and tokens.cu_rows.tolist() == [0, 0, 0, 0] and tokens.row_seq.max() == -1
        assert all(torch.equal(a, b) for a, b in zip(before[:3], (table, seq_lens, free)))
    refused([30, 30, 1], 2)                               # 2 + 2 + 1 pages of 3
    refused([3, 3, 59], -2)                               # 75 tokens in a table of 64
    refused([2 ** 31 - 1, 0, 0], -2)
    refused([0, 5, 0], -1, tokens=S.token_map(4, 3, DEV))
    refused([1, 0, 0], -3, count=_i32([-1]))
    refused([1, 0, 0], -3, count=_i32([free.numel() + 1]))
    # the first reason stays, later calls work all the same
    S.extend_page_tables(table, seq_lens, _i32([9999, 0, 0]), free, count, tokens, page_size=16)
    S.extend_page_tables(table, seq_lens, _i32([2, 0, 0]), free, count, tokens, page_size=16)
    assert int(tokens.status) == -3 and seq_lens.tolist() == [32, 5, 16] and tokens.cu_rows.tolist() == [0, 2, 2, 2]
    # a stack that could not take the pages, a length beyond the table
    status = _i32([0])
    small = free[: int(count)].contiguous()
    S.shrink_page_tables(table, seq_lens, _i32([0, 0, 0]), small, count, status, page_size=16)
    assert int(status) == -3 and seq_lens.tolist() == [32, 5, 16] and int(count) == 3
    seq_lens[1] = 65
    status.zero_()
    S.shrink_page_tables(table, seq_lens, _i32([0, 0, 0]), free, count, status, page_size=16)
    assert int(status) == -2 and int(count) == 3


def test_page_tables_captured_and_replayed():
    """A decode step in a graph: 40 replays without the host, against the walk."""
    from cacheir_b200 import serving_ops as S

    book = Book([3, 0, 31, 16], 8, 16, 40, 3)
    table, seq_lens, free, count = book.tensors()
    tokens, ones = S.token_map(6, 4, DEV), _i32([1, 1, 1, 0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            S.extend_page_tables(table, seq_lens, ones, free, count, tokens, page_size=16)
    for _ in range(40):
        graph.replay()
        rows, _ = book.extend([1, 1, 1, 0])
    torch.cuda.synchronize()
    assert tokens.slots.tolist() == [r[2] for r in rows] + [-1] * 3
    _same_book(book, table, seq_lens, free, count)


# ---- rotary positions ------------------------------------------------------------------------------------------------
def _rotated(x, angle, rot, layout, factor):
    """x [rows, heads, dim] in double as complex numbers times e^(i angle)."""
    x = x.double()
    half = rot // 2
    first, second = (x[..., 0:rot:2], x[..., 1:rot:2]) if layout == "interleaved" else (x[..., :half], x[..., half:rot])
    z = torch.complex(first, second) * torch.polar(torch.full_like(angle, factor), angle)[:, None, :]
    out = x.clone()
    if layout == "interleaved":
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        out[..., :half], out[..., half:rot] = z.real, z.imag
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,rot,page,yarn", [
    (1, 4, 2, 128, 128, 16, False), (33, 8, 1, 128, 64, 16, True), (7, 3, 3, 96, 32, 5, False), (5, 2, 1, 64, 22, 16, False), (4, 1, 1, 7, 4, 3, False),
    (300, 4, 4, 64, 64, 16, True), (2, 5, 1, 1024, 1024, 2, False), (3, 2, 2, 2, 2, 1, False), (593, 32, 8, 128, 128, 16, True), (1200, 4, 2, 64, 32, 16, False),
    (3001, 3, 1, 96, 96, 16, False)])
def test_rotary_append_against_complex_numbers(dtype, layout, rows, heads, kv_heads, dim, rot, page, yarn):
    from cacheir_b200 import serving_ops as S
    from cacheir_b200.ragged import rotary_frequencies, yarn_frequencies

    setting = (16.0, 8192.0, 32.0, 1.0)
    rule = S.rotary_rule(rot, 500000.0, layout=layout, yarn=setting if yarn else None, device=DEV)
    freq, factor = yarn_frequencies(rot, 500000.0, *setting) if yarn else (rotary_frequencies(rot, 500000.0), 1.0)
    qkv = _randn(1, rows, (heads + 2 * kv_heads) * dim + 3 * 8, dtype=dtype)               # rows wider than their heads
    q = qkv[:, : heads * dim].unflatten(1, (heads, dim))
    k = qkv[:, heads * dim: (heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    v = qkv[:, (heads + kv_heads) * dim: (heads + 2 * kv_heads) * dim].unflatten(1, (kv_heads, dim))
    positions = torch.randint(0, 2 ** 31 - 1, (rows,), device=DEV, generator=_gen(2)).to(torch.int32)
    positions[::3] = torch.arange(0, rows, 3, device=DEV, dtype=torch.int32)
    pages = (rows + page - 1) // page + 2
    slots = torch.randperm(pages * page, device=DEV, generator=_gen(3))[:rows].to(torch.int32)
    if rows > 3:
        slots[1], slots[3] = -1, pages * page                                               # padding, and a slot behind the pool
    live = (slots >= 0) & (slots < pages * page)
    k_cache, v_cache = (torch.full((pages, kv_heads, page, dim), 9.0, device=DEV, dtype=dtype) for _ in range(2))
    q_out = torch.full((rows, heads, dim), 7.0, device=DEV, dtype=dtype)
    S.rotary_append(q, k, v, rule, positions, slots=slots, k_cache=k_cache, v_cache=v_cache, q_out=q_out)
    angle = positions.double()[:, None] * torch.from_numpy(freq).to(DEV)[None, :]

    def check(got, x, rows=slice(None)):
        want = _rotated(x, angle, rot, layout, factor)[rows]
        # sine and cosine are good to 2^-22 (argument, function, factor), products and sum add three roundings
        size = x.double().abs().amax(-1, keepdim=True)[rows] * 2 * factor
        assert bool(((got.double() - want).abs() <= HALF[dtype] * want.abs() + 2.0 ** -21 * size).all())
    check(q_out[live], q, live)
    assert bool((q_out[~live] == 7.0).all())
    line = slots[live].long()
    check(k_cache.transpose(1, 2).reshape(-1, kv_heads, dim)[line], k, live)
    assert torch.equal(v_cache.transpose(1, 2).reshape(-1, kv_heads, dim)[line], v[live])
    untouched = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    untouched[line] = False
    for cache in (k_cache, v_cache):
        assert bool((cache.transpose(1, 2).reshape(-1, kv_heads, dim)[untouched] == 9.0).all())
    # without pools, q and k in place: the bits of the rows above, every row
    saved = q_out[live].clone(), k_cache.transpose(1, 2).reshape(-1, kv_heads, dim)[line].clone()
    kept, k_before = v.clone(), k.clone()
    check_q = q.clone()
    S.rotary_append(q, k, None, rule, positions)
    assert torch.equal(q[live], saved[0]) and torch.equal(k[live], saved[1]) and torch.equal(v, kept)
    check(q, check_q)
    check(k, k_before)


def test_rotary_append_matches_rope_append_near_the_start():
    """Positions below 64, whole heads, interleaved: the older kernel's angles are 32-bit, off by up to 64 * 2^-23."""
    from cacheir_b200 import ops
    from cacheir_b200 import serving_ops as S

    rows, heads, kv_heads, dim = 40, 8, 2, 128
    qkv = _randn(5, rows, (heads + 2 * kv_heads) * dim, dtype=torch.float16)
    positions, table = torch.arange(rows, device=DEV, dtype=torch.int32), torch.arange(rows, device=DEV, dtype=torch.int32)[:, None].repeat(1, 8).contiguous()
    pools = [torch.zeros(rows, kv_heads, 16, dim, device=DEV, dtype=torch.float16) for _ in range(4)]
    heads_of = lambda t, lo, n: t[:, lo * dim: (lo + n) * dim].unflatten(1, (n, dim))
    S.rotary_append(heads_of(qkv, 0, heads), heads_of(qkv, heads, kv_heads), heads_of(qkv, heads + kv_heads, kv_heads), S.rotary_rule(dim, 10000.0, device=DEV),
                    positions, slots=table[:, 0].contiguous() * 16 + positions % 16, k_cache=pools[0], v_cache=pools[1], q_out=(q := torch.empty(rows, heads, dim, device=DEV, dtype=torch.float16)))
    ops.rope_append(qkv, positions, table, pools[2], pools[3], q_dim=heads * dim, k_dim=kv_heads * dim, head_dim=dim, theta=10000.0)
    assert torch.equal(pools[1], pools[3])
    bound = lambda x: 2 * HALF[torch.float16] * x.abs() + 2.0 ** -15
    for a, b in ((q, heads_of(qkv, 0, heads)), (pools[0], pools[2])):
        assert bool(((a.float() - b.float()).abs() <= bound(b.float())).all())


# ---- attention over common prefixes ----------------------------------------------------------------------------------
def _paged(seed, groups, tails, heads, kv_heads, dim, page, dtype, spare=2, scale=1.0):
    """A batch whose groups alias their whole common pages and hold the same tokens in the page that the prefix ends in."""
    rng = random.Random(seed)
    lens = [max(0, p + t) for (_, p), tail in zip(groups, tails) for t in tail]
    pages = lambda n: (max(n, 0) + page - 1) // page
    shared = [p // page for _, p in groups]
    total = sum(pages(p) for _, p in groups) + sum(pages(max(n, 1)) + 1 for n in lens) + spare
    ids = list(range(total))
    rng.shuffle(ids)
    keys, values = (_randn(seed + i, total, kv_heads, page, dim, dtype=dtype) for i in (1, 2))
    width = max(max((pages(n) for n in lens), default=1), 1) + 1
    table, prefix_table = [], []
    for (n, p), tail, s in zip(groups, tails, shared):
        common = [ids.pop() for _ in range(pages(p))]
        prefix_table.append(common)
        for t in tail:
            mine = [ids.pop() for _ in range(max(0, pages(p + t) - s))]
            if mine and p % page:
                for pool in (keys, values):
                    pool[mine[0], :, : p % page] = pool[common[-1], :, : p % page]
            row = common[:s] + mine
            table.append((row + [total - 1] * width)[:width])
    wide = max(max(map(len, prefix_table)), 1)
    prefix_table = [(c + [0] * wide)[:wide] for c in prefix_table]
    q = _randn(seed + 3, len(lens), heads * dim + 16, dtype=dtype)[:, : heads * dim].unflatten(1, (heads, dim)) * scale
    starts = [0]
    for n, _ in groups:
        starts.append(starts[-1] + n)
    return q, keys, values, _i32(table), _i32(lens), starts, _i32(prefix_table), [p for _, p in groups]


def _attend(q, keys, values, table, lens, scale, owner, prefix_table, prefix_lens):
    """Row by row in 64 bits, keys below a group's prefix through the group's pages; and sum p |v|, what errors are relative to."""
    rows, heads, dim = q.shape
    kv_heads, page = keys.shape[1], keys.shape[2]
    out, size = (torch.zeros(rows, heads, dim, dtype=torch.float64, device=DEV) for _ in range(2))
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        t = torch.arange(n, device=DEV)
        ids = table[b].long()[torch.div(t, page, rounding_mode="floor").clamp(max=table.shape[1] - 1)]
        if owner[b] >= 0:
            below = t < prefix_lens[owner[b]]
            ids = torch.where(below, prefix_table[owner[b]].long()[torch.div(t, page, rounding_mode="floor").clamp(max=prefix_table.shape[1] - 1)], ids)
        k, v = (pool[ids, :, t % page].double() for pool in (keys, values))
        s = torch.einsum("hgd,thd->hgt", q[b].double().view(kv_heads, -1, dim), k) * scale
        p = torch.softmax(s, dim=-1)
        out[b] = torch.einsum("hgt,thd->hgd", p, v).reshape(heads, dim)
        size[b] = torch.einsum("hgt,thd->hgd", p, v.abs()).reshape(heads, dim)
    return out, size


def _owners(starts, rows):
    return [next((g for g in range(len(starts) - 1) if starts[g] <= b < starts[g + 1]), -1) for b in range(rows)]


def _check_attention(got, want, size, dtype):
    """The result's rounding; half a step of every weight p that is rounded before it meets v; and in 32 bits the scores (up to 512 products
    of size up to about 30 in all, in units of log 2, twice for the denominator), exponentials, sums: 2^-11 in 16 bits, 2^-16 in 32."""
    arithmetic = 2.0 ** -16 if dtype == torch.float32 else HALF[dtype] + 2.0 ** -11
    gap = (got.double() - want).abs()
    assert bool((gap <= HALF[dtype] * want.abs() + arithmetic * size + 1e-30).all()), float((gap / (size + 1e-30)).max())


SHAPES = [
    # groups (rows, common tokens), own tokens of every row, heads, kv heads, head size, page
    ([(2, 333)], [[1, 40]], 32, 8, 128, 16),
    ([(3, 64)], [[0, 5, 130]], 8, 2, 128, 16),
    ([(1, 48), (4, 16), (2, 0), (5, 129)], [[3], [1, 2, 3, 4], [7, 0], [0, 0, 1, 15, 16]], 8, 2, 64, 16),
    ([(40, 260)], [[i * 7 % 50 for i in range(40)]], 32, 8, 128, 16),
    ([(70, 130)], [[i % 3 for i in range(70)]], 8, 2, 128, 16),
    ([(17, 1000), (1, 2000), (9, 31)], [[i * 11 % 90 for i in range(17)], [500], [i for i in range(9)]], 16, 1, 128, 16),
    ([(6, 200)], [[1, 2, 3, 300, 5, 6]], 20, 1, 64, 16),
    ([(5, 77)], [[9, 8, 7, 6, 5]], 6, 6, 80, 16),
    ([(5, 77)], [[9, 8, 7, 6, 5]], 4, 2, 128, 32),
    ([(4, 50)], [[9, 8, 7, 60]], 4, 2, 64, 7),
    ([(3, 20)], [[9, 1, 2]], 6, 2, 33, 16),
    ([(2, 40)], [[3, 4]], 2, 1, 512, 16),
    ([(300, 150)], [[i % 20 for i in range(300)]], 8, 8, 64, 16),
    ([(2, 5000), (33, 700), (1, 1)], [[700, 0], [i * 3 % 64 for i in range(33)], [0]], 8, 2, 128, 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_shared_prefix_attention_against_64_bits(dtype, shape):
    from cacheir_b200 import serving_ops as S

    groups, tails, heads, kv_heads, dim, page = SHAPES[shape]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(shape, groups, tails, heads, kv_heads, dim, page, dtype)
    given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
    got = S.shared_prefix_attention(q, keys, values, table, lens, given)
    want, size = _attend(q, keys, values, table, lens, dim ** -0.5, _owners(starts, len(lens)), prefix_table, prefix_lens)
    _check_attention(got, want, size, dtype)
    again = S.shared_prefix_attention(q, keys, values, table, lens, given)
    assert torch.equal(got, again)
    # nothing shared: the batch as rows of their own
    _check_attention(S.shared_prefix_attention(q, keys, values, table, lens, None), want, size, dtype)


MANY = [
    # as SHAPES; more groups than a warp (32) and than a block (64) lays out by itself, several items for every block, tiles of one and of two
    # groups of 128 query rows in turn, heads per key/value head that do not divide 128, long common parts in many pieces, long own parts
    ([(1 + i % 3, 20 + 37 * i) for i in range(36)], [[j for j in range(1 + i % 3)] for i in range(36)], 8, 2, 128, 16),
    ([(2, 40 + i % 5 * 130) for i in range(70)], [[i % 7, 0] for i in range(70)], 8, 2, 64, 32),
    ([(i % 4, 300 if i % 5 else 0) for i in range(130)], [[i % 19 + 1] * (i % 4) for i in range(130)], 4, 4, 128, 16),
    ([(8, 1000)] * 8, [[3] * 8] * 8, 64, 8, 128, 16),
    ([(20 if i % 2 else 3, 500 - 9 * i) for i in range(40)], [[i % 30 for j in range(20 if i % 2 else 3)] for i in range(40)], 64, 4, 128, 16),
    ([(90, 700), (30, 260), (7, 1400)] * 6, [[i % 40 for i in range(90)], [i for i in range(30)], [0] * 7] * 6, 36, 12, 64, 16),
    ([(64, 9000)], [[i % 9 for i in range(64)]], 8, 2, 128, 16),
    ([(2, 6000), (1, 900)], [[5, 3000], [2100]], 16, 4, 128, 16),
    ([(3, 31)] * 11, [[1, 700, 33]] * 11, 48, 12, 128, 48),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", range(len(MANY)))
def test_shared_prefix_attention_of_many_groups_and_pieces(dtype, shape):
    from cacheir_b200 import serving_ops as S

    groups, tails, heads, kv_heads, dim, page = MANY[shape]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(shape + 50, groups, tails, heads, kv_heads, dim, page, dtype)
    given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
    got = S.shared_prefix_attention(q, keys, values, table, lens, given)
    want, size = _attend(q, keys, values, table, lens, dim ** -0.5, _owners(starts, len(lens)), prefix_table, prefix_lens)
    _check_attention(got, want, size, dtype)
    assert torch.equal(got, S.shared_prefix_attention(q, keys, values, table, lens, given))


@pytest.mark.parametrize("dtype,dim,page", [(torch.float16, 128, 16), (torch.bfloat16, 64, 16), (torch.float32, 64, 16), (torch.bfloat16, 80, 16)])
def test_shared_prefix_attention_with_infinite_scores_and_values_that_are_no_numbers(dtype, dim, page):
    from cacheir_b200 import serving_ops as S

    # a whole tile of keys and single ones, common and own, with a score of -inf: they have no weight
    groups, tails = [(3, 200), (2, 300)], [[40, 0, 9], [17, 90]]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(5, groups, tails, 8, 2, dim, page, dtype)
    q[..., 0] = 1.0
    for ids, tokens in ((prefix_table[0], range(128)), (prefix_table[1], (0, 5, 299)), (table[0], (*range(200, 216), 230)), (table[4], (389,))):
        for t in tokens:
            keys[ids[t // page], :, t % page, 0] = float("-inf")
    for b in range(3):           # (own copies of the page that the prefix ends in hold what it holds)
        keys[table[b, 192 // page], :, : 200 % page] = keys[prefix_table[0, 192 // page], :, : 200 % page]
    for b in (3, 4):
        keys[table[b, 288 // page], :, : 300 % page] = keys[prefix_table[1, 288 // page], :, : 300 % page]
    given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
    want, size = _attend(q, keys, values, table, lens, dim ** -0.5, _owners(starts, 5), prefix_table, prefix_lens)
    for g in (given, None):
        _check_attention(S.shared_prefix_attention(q, keys, values, table, lens, g), want, size, dtype)
    # a row with a NaN among its keys is NaN in every head that sees it, the others are as before; a row of no tokens is 0 whatever its group holds
    keys[table[3, 305 // page], 1, 305 % page, 3] = float("nan")
    lens[1] = 0
    values[prefix_table[0, 0], 0, 3] = float("nan")
    values[prefix_table[0, 1], 1, 3] = float("inf")
    for g in (given, None):
        got = S.shared_prefix_attention(q, keys, values, table, lens, g)
        assert bool(got[3, 4:].isnan().all()) and bool((got[1] == 0).all())
        _check_attention(got[3:, :4], want[3:, :4], size[3:, :4], dtype)
        _check_attention(got[4], want[4], size[4], dtype)
    keys[prefix_table[1, 0], 0, 0, 1] = float("nan")
    keys[prefix_table[1, 0], 0, 0, 0] = 0.0
    got = S.shared_prefix_attention(q, keys, values, table, lens, given)
    assert bool(got[3:, :4].isnan().all()) and bool(got[4, 4:].isfinite().all())


@pytest.mark.parametrize("dtype,dim,page", [(torch.float16, 128, 16), (torch.bfloat16, 64, 16), (torch.float32, 64, 16), (torch.float16, 128, 8)])
def test_shared_prefix_attention_edges(dtype, dim, page):
    """Rows outside every group, empty groups, rows that end inside their prefix or are empty, prefixes cut by their table, foreign page ids
    and NaN where nobody may look."""
    from cacheir_b200 import serving_ops as S

    heads, kv_heads = 8, 2
    groups, tails = [(3, 0), (6, 100), (2, 40)], [[5, 90, 0], [0, 1, -100, -60, -99, 70], [2, 300]]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(3, groups, tails, heads, kv_heads, dim, page, dtype)
    for pool in (keys, values):
        used = torch.zeros(pool.shape[0] * page, dtype=torch.bool, device=DEV)
        for b, n in enumerate(lens.tolist()):
            t = torch.arange(n, device=DEV)
            used[table[b].long()[t // page] * page + t % page] = True
        for g, n in enumerate(prefix_lens):
            t = torch.arange(n, device=DEV)
            used[prefix_table[g].long()[t // page] * page + t % page] = True
        pool.transpose(1, 2)[~used.view(-1, page)] = float("nan")
    # entries that must not matter: below the prefix in a row's own table, behind its length, behind a prefix
    for b in range(len(lens)):
        g = _owners(starts, len(lens))[b]
        table[b, : prefix_lens[g] // page] = 1 << 30
        table[b, (int(lens[b]) + page - 1) // page:] = -5
    for g, n in enumerate(prefix_lens):
        prefix_table[g, (n + page - 1) // page:] = 1 << 29
    # group 0 has no prefix, one is empty, the last two rows belong to no group
    rows = _i32([0, 3, 3, 9])
    order = [0, 0, 1]
    given = S.PrefixGroups(rows, prefix_table[order].contiguous(), _i32([0, 5, 100]))
    owner = [0] * 3 + [2] * 6 + [-1] * 2
    table[9:11, : prefix_lens[2] // page] = prefix_table[2, : prefix_lens[2] // page]      # (so theirs are read from the row)
    out = torch.full((11, heads * dim + 8), 3.0, device=DEV, dtype=dtype)
    view = out[:, : heads * dim].unflatten(1, (heads, dim))
    S.shared_prefix_attention(q, keys, values, table, lens, given, out=view)
    want, size = _attend(q, keys, values, table.clamp(0, keys.shape[0] - 1), lens, dim ** -0.5, owner, prefix_table[order].clamp(0, keys.shape[0] - 1), [0, 5, 100])
    assert bool((out[:, heads * dim:] == 3.0).all())
    _check_attention(view, want, size, dtype)
    assert bool((view[2] == 0).all()) and bool((view[5] == 0).all())                         # rows of length 0
    # a prefix that its table cannot hold counts as long as the table: the rest comes from the rows' own pages
    short = S.PrefixGroups(_i32([9, 11]), prefix_table[2:, : 1].contiguous(), _i32([10 ** 9]))
    got = S.shared_prefix_attention(q, keys, values, table, lens.clamp(min=-3), S.PrefixGroups(short.rows, short.table, short.lens))[9:]
    _check_attention(got, want[9:], size[9:], dtype)


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 128), (torch.bfloat16, 128), (torch.float32, 64)])
def test_shared_prefix_attention_with_sharp_and_growing_scores(dtype, dim):
    """Scores that rise along the context by hundreds, one key that takes everything, and equal ones."""
    from cacheir_b200 import serving_ops as S

    heads, kv_heads, page = 8, 2, 16
    groups, tails = [(20, 700)], [[i * 5 % 60 for i in range(20)]]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(9, groups, tails, heads, kv_heads, dim, page, dtype)
    given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
    keys.zero_()
    q[..., 0] = 16.0
    ids = prefix_table[0].long()
    ramp = torch.arange(ids.numel() * page, device=DEV).view(-1, page) / 16.0
    for case in ("rising", "falling", "one", "equal"):
        keys.zero_()
        if case == "rising":
            keys[ids, :, :, 0] = ramp[:, None].to(dtype)
        elif case == "falling":
            keys[ids, :, :, 0] = (40.0 - ramp)[:, None].to(dtype)
        elif case == "one":
            keys[ids[20], :, 3, 0] = 60.0
        want, size = _attend(q, keys, values, table, lens, 0.5, [0] * 20, prefix_table, prefix_lens)
        got = S.shared_prefix_attention(q, keys, values, table, lens, given, softmax_scale=0.5)
        # the products are exact here, their sum is a score of up to 500, rounded to 2^-15 of log 2
        slack = 2.0 ** -14 * size
        assert bool(((got.double() - want).abs() <= HALF[dtype] * (want.abs() + size) + slack + 1e-30).all()), case


def test_shared_prefix_attention_agrees_with_decode_attention():
    """The same batch through `paged_attention_decode_batch`, which reads every row's pages by itself; and as one group or many."""
    from cacheir_b200 import ops
    from cacheir_b200 import serving_ops as S

    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(4, [(24, 512)], [[i * 9 % 100 + 1 for i in range(24)]], 32, 8, 128, 16, torch.float16)
    given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
    plain = ops.paged_attention_decode_batch(q, keys, values, table, lens)
    want, size = _attend(q, keys, values, table, lens, 128 ** -0.5, [-1] * 24, prefix_table, prefix_lens)
    _check_attention(plain, want, size, torch.float16)
    _check_attention(S.shared_prefix_attention(q, keys, values, table, lens, given), want, size, torch.float16)
    many = S.PrefixGroups(_i32(list(range(25))), prefix_table.expand(24, -1).contiguous(), _i32([512 - i for i in range(24)]))
    _check_attention(S.shared_prefix_attention(q, keys, values, table, lens, many), want, size, torch.float16)


def test_shared_prefix_attention_in_a_graph_follows_its_inputs():
    """Captured once; groups, lengths and pages change between replays. Two graphs of their own workspaces beside one another."""
    from cacheir_b200 import serving_ops as S

    batches = [_paged(20 + i, [(8, p), (4, 64)], [[j + t for j in range(8)], [t] * 4], 8, 2, 128, 16, torch.float16, spare=90 - i) for i, (p, t) in enumerate([(160, 3), (33, 30)])]
    width = max(b[3].shape[1] for b in batches)
    wide = max(b[6].shape[1] for b in batches)
    pools = max(b[1].shape[0] for b in batches)
    pad = lambda t, n: torch.nn.functional.pad(t, (0, n - t.shape[1]))
    live = [torch.zeros(12, 8, 128, device=DEV, dtype=torch.float16), *(torch.zeros(pools, 2, 16, 128, device=DEV, dtype=torch.float16) for _ in range(2)),
            torch.zeros(12, width, device=DEV, dtype=torch.int32), torch.zeros(12, device=DEV, dtype=torch.int32)]
    given = S.PrefixGroups(_i32([0, 8, 12]), torch.zeros(2, wide, device=DEV, dtype=torch.int32), _i32([0, 0]))
    graphs = []
    for _ in range(2):
        out = torch.empty_like(live[0])
        workspace = torch.empty(S.shared_prefix_workspace_bytes(12, 8, 128), device=DEV, dtype=torch.uint8)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(graph, stream=stream):
                S.shared_prefix_attention(*live, given, out=out, workspace=workspace)
        graphs.append((graph, out, stream, workspace))
    torch.cuda.synchronize()
    for q, keys, values, table, lens, starts, prefix_table, prefix_lens in batches:
        live[0].copy_(q)
        live[1][: keys.shape[0]], live[2][: values.shape[0]] = keys, values
        live[3].copy_(pad(table, width))
        live[4].copy_(lens)
        given.table.copy_(pad(prefix_table, wide))
        given.lens.copy_(_i32(prefix_lens))
        torch.cuda.synchronize()
        for graph, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want, size = _attend(q, keys, values, table, lens, 128 ** -0.5, _owners(starts, 12), prefix_table, prefix_lens)
        for _, out, _, _ in graphs:
            _check_attention(out, want, size, torch.float16)


# ---- log probabilities -----------------------------------------------------------------------------------------------
def _logprobs(logits, tokens, top, temperature):
    x = logits.double() / temperature
    x = x - x.amax(-1, keepdim=True)                       # (first: at a value of 1e38 the logarithm of a sum would be lost in 64 bits too)
    lp = x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    lp = torch.where(lp < -torch.finfo(torch.float32).max, -math.inf, lp)                  # what a float32 cannot hold
    entropy = -(torch.exp(lp) * torch.where(lp == -math.inf, 0.0, lp)).sum(-1)
    order = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, tokens.clamp(0, logits.shape[1] - 1)[:, None])[:, 0], entropy, order, lp.gather(1, order)


def _check_logprobs(got, logits, tokens, top, temperature):
    logp, entropy, ids, top_logp = _logprobs(logits, tokens, top, temperature)
    # chains of up to 512 additions of positive terms, exponentials good to 2^-21, and the result's own rounding
    chain = 512 * 2.0 ** -24 + 2.0 ** -20
    near = lambda a, b: bool(((a.double() - b).abs() <= chain + 2.0 ** -22 * b.abs())[b.isfinite()].all()) and torch.equal(a.isfinite(), b.isfinite())
    assert near(got.logprobs, logp)
    assert bool(((got.entropy.double() - entropy).abs() <= 2 * chain * (1 + entropy)).all())
    if top:
        assert torch.equal(got.top_ids, ids)
        assert near(got.top_logprobs, top_logp)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top,temperature", [
    (1, 1, 1, 1.0), (1, 128256, 5, 1.0), (3, 7, 7, 0.5), (64, 32000, 20, 0.7), (5, 50001, 32, 1.0), (300, 1000, 0, 1.0), (17, 8193, 1, 2.5), (2, 33, 32, 1.0),
    (150, 40000, 3, 1.0), (1, 131072, 32, 1.0), (700, 4096, 2, 1.0)])
def test_token_logprobs_against_64_bits(dtype, rows, vocab, top, temperature):
    from cacheir_b200 import serving_ops as S

    logits = (_randn(rows, rows, vocab) * 3.0).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=_gen(1))
    _check_logprobs(S.token_logprobs(logits, tokens, top=top, temperature=temperature), logits, tokens, top, temperature)
    got = S.token_logprobs(logits, None, top=top)
    assert got.logprobs is None and bool(got.entropy.isfinite().all()) and (got.top_ids is None) == (top == 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_token_logprobs_masks_ties_and_values_that_are_no_numbers(dtype):
    from cacheir_b200 import serving_ops as S

    vocab, inf, nan = 2050, math.inf, math.nan
    logits = torch.zeros(12, vocab, device=DEV, dtype=dtype)
    logits[1, :] = -inf
    logits[2, :] = -inf
    logits[2, 1999] = -40.0                                # one token is left
    logits[3, ::2] = -inf
    logits[4, 100:110] = 3.0                               # equal ones by rising index
    logits[5, 7], logits[5, 9] = 0.0, -0.0                 # which are equal too
    logits[6, 5] = nan
    logits[7, 6] = inf
    logits[8, :] = torch.finfo(dtype).min                  # the type's lowest value is a value
    logits[9, :], logits[9, 44] = torch.finfo(dtype).min, 10.0
    logits[10, :], logits[10, 3], logits[10, 2] = -inf, torch.finfo(dtype).max, -torch.finfo(dtype).max
    logits[11, :] = torch.arange(vocab, device=DEV) % 5
    tokens = torch.tensor([0, 5, 1999, 0, 105, 9, 1, 6, 2049, 44, 3, 4], device=DEV)
    top = 20
    got = S.token_logprobs(logits, tokens, top=top)
    plain = [0, 2, 3, 4, 5, 8, 9, 10, 11]
    at = torch.tensor(plain, device=DEV)
    picked = S.TokenLogprobs(got.logprobs[at], got.entropy[at], got.top_ids[at], got.top_logprobs[at])
    _check_logprobs(picked, logits[at], tokens[at], top, 1.0)
    assert got.top_ids[0].tolist() == list(range(top)) and got.top_ids[1].tolist() == list(range(top)) and got.top_ids[5].tolist() == list(range(top))
    assert got.top_ids[4].tolist() == list(range(100, 110)) + list(range(10))
    assert float(got.logprobs[2]) == 0.0 and float(got.entropy[2]) == 0.0 and got.top_ids[2].tolist() == [1999] + list(range(19))
    assert float(got.logprobs[1]) == -inf and float(got.entropy[1]) == 0.0 and bool((got.top_logprobs[1] == -inf).all())
    for row, first in ((6, 5), (7, 6)):
        assert math.isnan(got.logprobs[row]) and math.isnan(got.entropy[row]) and bool(got.top_logprobs[row].isnan().all())
        assert got.top_ids[row].tolist() == [first] + list(range(first)) + list(range(first + 1, top))
    assert float(got.logprobs[3]) == pytest.approx(-math.log(vocab / 2 if vocab % 2 == 0 else vocab // 2), abs=1e-5) if tokens[3] % 2 else float(got.logprobs[3]) == -inf
    # rows without a token, and tokens that are none
    odd = S.token_logprobs(logits[:3], torch.tensor([-1, vocab, -100], device=DEV)).logprobs
    assert float(odd[0]) == 0.0 and math.isnan(odd[1]) and float(odd[2]) == 0.0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_token_logprobs_of_strided_rows_and_every_offset(dtype):
    """Rows of a wider buffer that start at any alignment, values behind the row's end that would win."""
    from cacheir_b200 import serving_ops as S

    wide = (_randn(3, 9, 5013) * 3.0).to(dtype)
    wide[:, 4500:] = 60.0
    for lo, vocab in ((0, 4500), (1, 4499), (3, 4001), (8, 4096), (5, 17)):
        logits = wide[:, lo: lo + vocab]
        tokens = torch.randint(0, vocab, (9,), device=DEV, generator=_gen(lo))
        _check_logprobs(S.token_logprobs(logits, tokens, top=9), logits, tokens, 9, 1.0)


def test_token_logprobs_ordered_values_that_keep_beating_the_best():
    """Rising, falling and constant rows: every element, or none, enters a list of the largest so far."""
    from cacheir_b200 import serving_ops as S

    vocab = 30011
    rise = torch.arange(vocab, device=DEV, dtype=torch.float32) / 1000.0
    logits = torch.stack([rise, rise.flip(0), torch.zeros_like(rise), -rise])
    tokens = torch.tensor([0, 1, 2, 3], device=DEV)
    _check_logprobs(S.token_logprobs(logits, tokens, top=32), logits, tokens, 32, 1.0)
    _check_logprobs(S.token_logprobs(logits.half(), tokens, top=32), logits.half(), tokens, 32, 1.0)


# ---- together --------------------------------------------------------------------------------------------------------
def test_a_batch_of_samples_of_one_prompt_step_by_step():
    """What a server does with several samples of a prompt: their new tokens get slots, heads are turned and appended, attention reads the
    prompt once, the sampled tokens are scored; against the same steps in 64 bits over contiguous histories. Then everybody ends and
    the stack of free pages is full again."""
    from cacheir_b200 import serving_ops as S
    from cacheir_b200.ragged import rotary_frequencies

    batch, heads, kv_heads, dim, page, vocab, prompt = 5, 8, 2, 64, 16, 999, 37
    dtype = torch.float16
    shared = prompt // page                                # two pages are common, five tokens behind them each row's own
    pools = [torch.zeros(40, kv_heads, page, dim, device=DEV, dtype=dtype) for _ in range(2)]
    free = _i32(list(range(40))[::-1])
    count = _i32([40])
    rule, freq = S.rotary_rule(dim, 10000.0, layout="half", device=DEV), torch.from_numpy(rotary_frequencies(dim, 10000.0)).to(DEV)
    # the prompt as a sequence of its own
    prompt_table, prompt_len, tokens = torch.zeros(1, 8, device=DEV, dtype=torch.int32), _i32([0]), S.token_map(64, 1, DEV)
    S.extend_page_tables(prompt_table, prompt_len, _i32([shared * page]), free, count, tokens, page_size=page)
    k0, v0 = (_randn(i, prompt, kv_heads, dim, dtype=dtype) for i in (1, 2))
    pad = lambda t: torch.cat([t, torch.zeros(64 - t.shape[0], *t.shape[1:], device=DEV, dtype=t.dtype)])
    S.rotary_append(torch.zeros(64, heads, dim, device=DEV, dtype=dtype), pad(k0[: shared * page]), pad(v0[: shared * page]), rule, tokens.positions,
                    slots=tokens.slots, k_cache=pools[0], v_cache=pools[1])
    # the rows alias its pages
    table = torch.zeros(batch, 8, device=DEV, dtype=torch.int32)
    table[:, :shared] = prompt_table[:, :shared]
    lens, held = _i32([shared * page] * batch), _i32([shared] * batch)
    groups = S.PrefixGroups(_i32([0, batch]), prompt_table, _i32([shared * page]))
    history = [[(k0[t], v0[t]) for t in range(shared * page)] for _ in range(batch)]
    steps = [[prompt - shared * page] * batch] + [[1] * batch for _ in range(14)] + [[1, 0, 2, 1, 0]] * 3
    tokens = S.token_map(32, batch, DEV)
    for step, new in enumerate(steps):
        rows = sum(new)
        S.extend_page_tables(table, lens, _i32(new), free, count, tokens, page_size=page)
        q, k, v = (_randn(100 * step + i, 32, h, dim, dtype=dtype) for i, h in enumerate((heads, kv_heads, kv_heads)))
        turned = torch.zeros_like(q)
        S.rotary_append(q, k, v, rule, tokens.positions, slots=tokens.slots, k_cache=pools[0], v_cache=pools[1], q_out=turned)
        row = 0
        last = [None] * batch
        for b, n in enumerate(new):
            for i in range(n):
                history[b].append((k[row], v[row]))
                last[b] = row
                row += 1
        asked = torch.tensor([r if r is not None else 0 for r in last], device=DEV)
        got = S.shared_prefix_attention(turned[asked], pools[0], pools[1], table, lens, groups)
        for b in range(batch):
            if last[b] is None:
                continue
            n = len(history[b])
            angle = torch.arange(n, device=DEV).double()[:, None] * freq
            keys = _rotated(torch.stack([h[0] for h in history[b]]), angle, dim, "half", 1.0)
            query = _rotated(q[last[b]][None], angle[-1:], dim, "half", 1.0)[0].view(kv_heads, -1, dim)
            p = torch.softmax(torch.einsum("hgd,thd->hgt", query, keys) * dim ** -0.5, dim=-1)
            vals = torch.stack([h[1] for h in history[b]]).double()
            want = torch.einsum("hgt,thd->hgd", p, vals).reshape(heads, dim)
            size = torch.einsum("hgt,thd->hgd", p, vals.abs()).reshape(heads, dim)
            # keys and queries are rounded after their turn: scores of up to 64 such products, 2^-10 * |q| |k| / 8 below 2^-7 in all
            assert bool(((got[b].double() - want).abs() <= HALF[dtype] * want.abs() + (HALF[dtype] + 2.0 ** -6) * size).all())
        logits = _randn(step, batch, vocab)
        sampled = torch.randint(0, vocab, (batch,), device=DEV, generator=_gen(step))
        _check_logprobs(S.token_logprobs(logits, sampled, top=5), logits, sampled, 5, 1.0)
        assert int(tokens.status) == 0 and lens.tolist() == [len(h) for h in history]
    S.shrink_page_tables(table, lens, _i32([0] * batch), free, count, tokens.status, page_size=page, held_pages=held)
    S.shrink_page_tables(prompt_table, prompt_len, _i32([0]), free, count, tokens.status, page_size=page)
    assert int(count) == 40 and sorted(free.tolist()) == list(range(40)) and int(tokens.status) == 0


def test_calls_on_another_stream_and_of_no_rows():
    from cacheir_b200 import serving_ops as S

    logits, ids = _randn(1, 4, 100), torch.zeros(4, dtype=torch.int64, device=DEV)
    want = S.token_logprobs(logits, ids, top=3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = S.token_logprobs(logits, ids, top=3)
    stream.synchronize()
    assert torch.equal(got.logprobs, want.logprobs) and torch.equal(got.top_ids, want.top_ids)
    none = S.token_logprobs(logits[:0], ids[:0], top=3)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 3)
    pool = torch.zeros(2, 2, 16, 64, device=DEV)
    empty = S.shared_prefix_attention(torch.zeros(0, 4, 64, device=DEV), pool, pool, torch.zeros(0, 3, device=DEV, dtype=torch.int32), _i32([]), None)
    assert empty.shape == (0, 4, 64)
    S.rotary_append(torch.zeros(0, 4, 64, device=DEV), torch.zeros(0, 2, 64, device=DEV), None, S.rotary_rule(64, 1e4, device=DEV), _i32([]))


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 48)])
def test_a_whole_step_captured_and_replayed_beside_the_same_steps_called(dtype, dim):
    """Pages, slots, append, attention, scores and the way back as one graph on a stream of its own; the same bits as calls of the same state."""
    from cacheir_b200 import serving_ops as S

    batch, heads, kv_heads, page, vocab, shared = 6, 8, 2, 16, 1003, 3
    rule = S.rotary_rule(dim, 10000.0, layout="interleaved", scaling=(8.0, 1.0, 4.0, 8192.0), device=DEV)
    qkv = torch.zeros(24, (heads + 2 * kv_heads) * dim, device=DEV, dtype=dtype)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1))
    logits, sampled = torch.zeros(batch, vocab, device=DEV, dtype=dtype), torch.zeros(batch, device=DEV, dtype=torch.int64)
    new, keep = (torch.zeros(batch, device=DEV, dtype=torch.int32) for _ in range(2))
    held = _i32([shared] * 4 + [0, 0])
    groups = S.PrefixGroups(_i32([0, 4]), _i32([[60, 61, 62]]), _i32([shared * page]))

    def state():
        pools = [_randn(i, 64, kv_heads, page, dim, dtype=dtype) for i in (1, 2)]
        table = torch.zeros(batch, 12, device=DEV, dtype=torch.int32)
        table[:4, :shared] = groups.table
        return dict(pools=pools, table=table, lens=_i32([shared * page] * 4 + [0, 0]), free=_i32(list(range(60))), count=_i32([60]),
                    tokens=S.token_map(24, batch, DEV), turned=torch.zeros(24, heads, dim, device=DEV, dtype=dtype),
                    workspace=torch.zeros(S.shared_prefix_workspace_bytes(batch, heads, dim), device=DEV, dtype=torch.uint8))

    def step(s):
        S.extend_page_tables(s["table"], s["lens"], new, s["free"], s["count"], s["tokens"], page_size=page)
        S.rotary_append(q, k, v, rule, s["tokens"].positions, slots=s["tokens"].slots, k_cache=s["pools"][0], v_cache=s["pools"][1], q_out=s["turned"])
        out = S.shared_prefix_attention(s["turned"][:batch], *s["pools"], s["table"], s["lens"], groups, workspace=s["workspace"])
        scores = S.token_logprobs(logits, sampled, top=4)
        S.shrink_page_tables(s["table"], s["lens"], keep, s["free"], s["count"], s["tokens"].status, page_size=page, held_pages=held)
        return out, scores

    called, captured = state(), state()
    step(state())                                    # (everything has been launched once before it is captured)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        out, scores = step(captured)
    torch.cuda.synchronize()
    rng = random.Random(4)
    for i in range(12):
        lens = called["lens"].tolist()
        add = [rng.randrange(0, 5) for _ in range(batch)]
        qkv.copy_(_randn(100 + i, *qkv.shape, dtype=dtype))
        logits.copy_(_randn(200 + i, batch, vocab, dtype=dtype))
        sampled.copy_(torch.tensor([rng.randrange(-1, vocab + 1) for _ in range(batch)]))
        new.copy_(_i32(add))
        keep.copy_(_i32([n + a - rng.randrange(0, 3) if n + a > 50 else n + a for n, a in zip(lens, add)]))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        want, want_scores = step(called)             # (beside it)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in ((scores.logprobs, want_scores.logprobs), (scores.entropy, want_scores.entropy), (scores.top_logprobs, want_scores.top_logprobs)):
            assert bool(((a == b) | (a.isnan() & b.isnan())).all())
        assert torch.equal(scores.top_ids, want_scores.top_ids)
        for name in ("table", "lens", "free", "count"):
            assert torch.equal(captured[name], called[name]), name
        assert all(torch.equal(a, b) for a, b in zip(captured["pools"], called["pools"]))
        assert int(called["tokens"].status) == 0 and int(captured["tokens"].status) == 0


def test_two_threads_with_streams_and_head_sizes_of_their_own():
    """Calls of both kinds of kernels from two threads at once: each gets the bits that it gets alone."""
    import threading

    from cacheir_b200 import serving_ops as S

    shapes = [[(512, torch.float32), (128, torch.float16), (64, torch.float32)], [(80, torch.float32), (64, torch.bfloat16), (256, torch.float32)]]
    plans = []
    for side, kinds in enumerate(shapes):
        calls = []
        for i, (dim, dtype) in enumerate(kinds):
            q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(60 + 3 * side + i, [(3, 90), (2, 33)], [[4, 0, 20], [1, 50]], 8, 2, dim, 16, dtype)
            given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
            workspace = torch.empty(S.shared_prefix_workspace_bytes(5, 8, dim), device=DEV, dtype=torch.uint8)
            args = (q, keys, values, table, lens, given)
            calls.append((args, workspace, S.shared_prefix_attention(*args, workspace=workspace)))
        plans.append((torch.cuda.Stream(), calls))
    torch.cuda.synchronize()
    wrong = []

    def work(stream, calls):
        try:
            with torch.cuda.stream(stream):
                for _ in range(60):
                    for args, workspace, want in calls:
                        if not torch.equal(S.shared_prefix_attention(*args, workspace=workspace), want):
                            wrong.append(want.shape)
        except Exception as error:                           # (a thread's exception would be lost)
            wrong.append(error)
    threads = [threading.Thread(target=work, args=plan) for plan in plans]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("groups", [[(i % 5, i * 7 % 40) for i in range(2110)], [(4220, 19)]])
def test_general_attention_of_more_tiles_than_a_narrow_grid_takes(groups):
    """64 heads on one key/value head, thousands of rows of a few tokens: 67 thousand tiles and more."""
    from cacheir_b200 import serving_ops as S

    tails = [[(i + j) % 6 for j in range(n)] for i, (n, _) in enumerate(groups)]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(70, groups, tails, 64, 1, 16, 8, torch.float32)
    rows = len(lens)
    assert rows * 64 // 8 * 2 > 65535
    owner = [g for g, (n, _) in enumerate(groups) for _ in range(n)]
    got = S.shared_prefix_attention(q, keys, values, table, lens, S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens)))
    want, size = _attend(q, keys, values, table, lens, 0.25, owner, prefix_table, prefix_lens)
    _check_attention(got, want, size, torch.float32)
    # rows before the first group and behind the last one belong to none: the same keys out of their own pages
    part = S.PrefixGroups(_i32([starts[1] if len(groups) > 1 else 700, starts[-2] if len(groups) > 1 else 4000]), prefix_table[1:2] if len(groups) > 1 else prefix_table,
                          _i32([0 if len(groups) > 1 else 16]))
    mine = table.clone()
    for b in range(rows):
        shared = prefix_lens[owner[b]] // 8
        mine[b, :shared] = prefix_table[owner[b], :shared]
    _check_attention(S.shared_prefix_attention(q, keys, values, mine, lens, part), want, size, torch.float32)


@pytest.mark.parametrize("dtype,dim,page", [(torch.float16, 128, 16), (torch.bfloat16, 64, 48), (torch.bfloat16, 128, 16), (torch.float32, 64, 16)])
@pytest.mark.parametrize("more", [0, 40, 70])
def test_rows_that_end_inside_their_prefix_see_nothing_behind_their_end(dtype, dim, page, more):
    """Others of the group go on to tokens whose keys and values are no numbers, or infinite. More groups than a warp and than a block lays out by itself."""
    from cacheir_b200 import serving_ops as S

    groups = [(70, 300), (3, 1000)] + [(1, 17)] * more
    ends = [1, 15, 16, 17, 127, 128, 129, 140, 141, 142]
    tails = [[(ends[i % 10] if i % 10 else i // 10) - 300 for i in range(68)] + [0, 9], [-999, -700, 40]] + [[i % 3] for i in range(more)]
    q, keys, values, table, lens, starts, prefix_table, prefix_lens = _paged(80 + more, groups, tails, 8, 2, dim, page, dtype)
    owner = _owners(starts, len(lens))
    want, size = _attend(q, keys, values, table, lens, dim ** -0.5, owner, prefix_table, prefix_lens)
    given = S.PrefixGroups(_i32(starts), prefix_table, _i32(prefix_lens))
    _check_attention(S.shared_prefix_attention(q, keys, values, table, lens, given), want, size, dtype)
    for t, k, v in ((142, math.nan, math.nan), (143, math.inf, -math.inf), (299, 1.0, math.inf), (200, math.nan, 1.0)):
        keys[prefix_table[0, t // page], :, t % page] = k
        values[prefix_table[0, t // page], :, t % page] = v
    keys[prefix_table[1, 300 // page], :, 300 % page] = math.nan
    values[prefix_table[1, 300 // page], :, 300 % page] = math.nan
    # (a row's own table is not read below the prefix)
    for b in range(73):
        table[b, : prefix_lens[owner[b]] // page] = -7
    got = S.shared_prefix_attention(q, keys, values, table, lens, given)
    live = torch.tensor([b not in (68, 69, 72) for b in range(len(lens))], device=DEV)
    _check_attention(got[live], want[live], size[live], dtype)
    assert bool(got[[68, 69, 72]].isnan().all())
    assert torch.equal(got[live], S.shared_prefix_attention(q, keys, values, table, lens, given)[live])


def test_rotary_append_of_two_rows_to_one_slot_leaves_values_of_either():
    """Which of them stays is open, value by value; nothing else of the pool is touched and every row's q is its own."""
    from cacheir_b200 import serving_ops as S

    rule = S.rotary_rule(64, 10000.0, layout="half", device=DEV)
    q, k, v = (_randn(i, 300, heads, 64, dtype=torch.float16) for i, heads in ((1, 4), (2, 2), (3, 2)))
    positions = torch.arange(300, device=DEV, dtype=torch.int32)
    alone_q, alone_k = torch.empty_like(q), torch.empty_like(k)
    S.rotary_append(q, k, None, rule, positions, q_out=alone_q, k_out=alone_k)
    pools = [torch.full((4, 2, 16, 64), 9.0, device=DEV, dtype=torch.float16) for _ in range(2)]
    out = torch.empty_like(q)
    slots = torch.where(positions % 3 == 0, 37, 5).to(torch.int32)
    S.rotary_append(q, k, v, rule, positions, slots=slots, k_cache=pools[0], v_cache=pools[1], q_out=out)
    assert torch.equal(out, alone_q)
    for pool, rows in zip(pools, (alone_k, v)):
        lines = pool.transpose(1, 2).reshape(64, 2, 64)
        for slot in (5, 37):
            assert bool((lines[slot] == rows[slots == slot]).any(0).all())
        rest = torch.ones(64, dtype=torch.bool, device=DEV)
        rest[[5, 37]] = False
        assert bool((lines[rest] == 9.0).all())


def test_pools_and_logits_of_more_than_two_to_the_31_values():
    """What lies behind 2^31 values (and 2^32 bytes) is found: appended to, attended to by both kinds of kernels, scored."""
    from cacheir_b200 import serving_ops as S

    heads, kv_heads, dim, dtype = 16, 8, 128, torch.float16
    slots = 2 ** 31 // (kv_heads * 16 * dim) + 4000
    pools = [torch.empty(slots, kv_heads, 16, dim, device=DEV, dtype=dtype) for _ in range(2)]
    assert pools[0].numel() > 2 ** 31
    ids = [slots - 1, 3, slots - 3000, 131072, slots - 17, 131071, slots // 2, 70000, slots - 2]
    for i, pool in enumerate(pools):
        for page in ids:
            pool[page] = _randn(page % 1000 + i, kv_heads, 16, dim, dtype=dtype)
    # appends to both ends of the pool
    rule = S.rotary_rule(dim, 10000.0, layout="half", device=DEV)
    q, k, v = (_randn(i, 4, h, dim, dtype=dtype) for i, h in ((1, heads), (2, kv_heads), (3, kv_heads)))
    where, offset = [slots - 1, 3, 131072, slots - 17], [15, 0, 7, 2]
    turned, turned_k = torch.empty_like(q), torch.empty_like(k)
    S.rotary_append(q, k, None, rule, _i32([5, 6, 7, 8]), q_out=turned, k_out=turned_k)
    S.rotary_append(q, k, v, rule, _i32([5, 6, 7, 8]), slots=_i32([p * 16 + o for p, o in zip(where, offset)]), k_cache=pools[0], v_cache=pools[1], q_out=q)
    assert torch.equal(q, turned)
    for row, (p, o) in enumerate(zip(where, offset)):
        assert torch.equal(pools[0][p, :, o], turned_k[row]) and torch.equal(pools[1][p, :, o], v[row])
    table = _i32([ids[:3] + [ids[3], ids[4]], ids[:3] + [ids[5], 0], ids[:3] + [ids[6], ids[7]], [ids[8], ids[7], ids[5], 0, 0]])
    lens, given = _i32([80, 50, 65, 33]), S.PrefixGroups(_i32([0, 3]), _i32([ids[:3]]), _i32([48]))
    want, size = _attend(q, *pools, table, lens, dim ** -0.5, [0, 0, 0, -1], given.table, [48])
    for groups in (given, None):
        _check_attention(S.shared_prefix_attention(q, *pools, table, lens, groups), want, size, dtype)
    # the same memory as pages of eight tokens, for the general kernels
    small = [pool.view(2 * slots, kv_heads, 8, dim) for pool in pools]
    halves = lambda t: torch.stack([2 * t, 2 * t + 1], dim=-1).flatten(-2).to(torch.int32).contiguous()
    given = S.PrefixGroups(given.rows, halves(given.table), given.lens)
    want, size = _attend(q, *small, halves(table), lens, dim ** -0.5, [0, 0, 0, -1], given.table, [48])
    for groups in (given, None):
        _check_attention(S.shared_prefix_attention(q, *small, halves(table), lens, groups), want, size, dtype)
    del pools, small, pool
    logits = torch.empty(17000, 128256, device=DEV, dtype=torch.bfloat16)
    assert logits.numel() > 2 ** 31
    rows = [0, 8371, 8372, 16742, 16744, 16999]              # on both sides of 2^30 and 2^31 values
    for r in rows:
        logits[r] = _randn(r, 128256, dtype=torch.bfloat16) * 3.0
    tokens = torch.arange(17000, device=DEV) * 7 % 128256
    got, at = S.token_logprobs(logits, tokens, top=3), torch.tensor(rows, device=DEV)
    picked = S.TokenLogprobs(got.logprobs[at], got.entropy[at], got.top_ids[at], got.top_logprobs[at])
    _check_logprobs(picked, logits[at], tokens[at], 3, 1.0)
