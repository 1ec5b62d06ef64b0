"""Kernels of steps that verify drafted tokens against plain implementations in 64 bits."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _close(got, want, bound, what=""):
    """|got - want| <= bound everywhere; not-a-number and infinities in the same places."""
    got = got.double()
    same = torch.isnan(got) == torch.isnan(want)
    assert bool(same.all()), f"{what}: NaN in other places ({int((~same).sum())})"
    off = torch.where(got == want, 0.0, (got - want).abs())
    bad = torch.nan_to_num(off, nan=0.0, posinf=math.inf) > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} values off, worst by {float((off / bound)[bad].max()):.3g} bounds"


def _trees(rng, nodes, shape):
    """Parents of every sequence's rows."""
    if shape == "chain":
        return [[i - 1 for i in range(n)] for n in nodes]
    if shape == "star":
        return [[-1] + [0] * (n - 1) if n else [] for n in nodes]
    return [[-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)] if n else [] for n in nodes]


def _seen(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else []) + [i])
    return seen


def _words(lists, words):
    lines = []
    for seen in lists:
        bits = sum(1 << j for j in seen if j < 32 * words)
        lines.append([(bits >> 32 * w & 0xFFFFFFFF) - (bits >> 32 * w + 31 & 1) * (1 << 32) for w in range(words)])
    return lines


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


# ---- attention ---------------------------------------------------------------------------------------------------------
class Case:
    """A batch in a shuffled pool; `lists`: of every row the rows of its sequence that it sees (None: a chain without a mask)."""

    def __init__(self, *, heads=8, kv_heads=2, dim=128, page=16, dtype=F16, ctx=(40,), nodes=(5,), lists="tree", behind=0, padded=0, words=None, seed=0, wide_q=0, scale=1.5):
        rng, gen = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed + 1)
        randn = lambda *shape: torch.randn(shape, device=DEV, generator=gen)
        self.heads, self.kv_heads, self.dim, self.page, self.nodes, self.ctx = heads, kv_heads, dim, page, list(nodes), list(ctx)
        self.lens = [c + n for c, n in zip(ctx, nodes)]
        self.starts = _starts(nodes)
        rows = self.starts[-1] + behind + padded
        self.before = 0
        if lists is not None and isinstance(lists, str):
            lists = [line for tree in _trees(rng, nodes, lists) for line in _seen(tree)]
        self.lists = lists
        self.words = words or max(1, (max(nodes) + 31) // 32)
        pages = [(n + page - 1) // page for n in self.lens]
        total, width = sum(pages) + 2, max(max(pages), 1) + 1
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        table, used = [[total + 7 if i % 2 else -3 for i in range(width)] for _ in pages], 0           # (entries behind the end are no pages)
        for b, n in enumerate(pages):
            table[b][:n] = order[used: used + n]
            used += n
        self.table, self.seq_lens, self.cu_rows = _i32(table), _i32(self.lens), _i32(self.starts)
        self.visible = None if lists is None else _i32(_words(lists, self.words) + [[-1] * self.words] * (rows - self.starts[-1]))
        self.q = (randn(rows, (heads + wide_q) * dim) * scale).to(dtype)[:, : heads * dim].view(rows, heads, dim)
        self.keys, self.values = (randn(total, kv_heads, page, dim).to(dtype) for _ in range(2))
        self.out = torch.full((rows, heads, dim), 7.0, dtype=dtype, device=DEV)

    def place(self, b, t):
        """Where token t of sequence b lies: (page, offset)."""
        return int(self.table[b, t // self.page]), t % self.page

    def spoil_behind(self):
        """What stands behind the sequences' ends in their last pages is no number."""
        for b, n in enumerate(self.lens):
            if n % self.page:
                at = int(self.table[b, n // self.page])
                for pool in (self.keys, self.values):
                    pool[at, :, n % self.page:] = math.nan

    def call(self, **more):
        from cacheir_b200 import draft_ops
        return draft_ops.tree_attention(self.q, self.keys, self.values, self.table, self.seq_lens, self.cu_rows, self.visible, out=self.out, **more)

    def want(self):
        """(result in 64 bits, how far off it may be)"""
        result, bound = self.out.double().clone(), torch.zeros(self.out.shape, dtype=torch.float64, device=DEV)
        group, eps = self.heads // self.kv_heads, 0.0 if self.out.dtype is F32 else _half_step(self.out.dtype)
        for b, (n, lo, length) in enumerate(zip(self.nodes, self.starts, self.lens)):
            if n == 0:
                continue
            t = torch.arange(length, device=DEV)
            ids = self.table[b].long()[t // self.page]
            inside = (ids >= 0) & (ids < self.keys.shape[0])
            k, v = (torch.where(inside[:, None, None], pool[ids.clamp(0, self.keys.shape[0] - 1), :, t % self.page].double(), 0.0) for pool in (self.keys, self.values))
            for i in range(n):
                seen = torch.ones(length, dtype=torch.bool, device=DEV)
                mine = range(i + 1) if self.lists is None else [j for j in self.lists[lo + i] if j < 32 * self.words]
                seen[max(length - n, 0):] = False
                seen[[length - n + j for j in mine if 0 <= length - n + j < length and j < n]] = True
                q = self.q[lo + i].double().view(self.kv_heads, group, self.dim)
                ks, vs = k[seen], v[seen]                                                  # [keys, kv_heads, dim]
                if ks.shape[0] == 0:
                    result[lo + i] = 0.0
                    continue
                scores = torch.einsum("hgd,thd->hgt", q, ks) / math.sqrt(self.dim)
                p = torch.softmax(scores, dim=-1)
                p = torch.where((scores == -math.inf).all(-1, keepdim=True), 0.0, p)
                live = torch.where(p[..., None] > 0, vs.permute(1, 0, 2)[:, None], 0.0) if not bool(torch.isfinite(vs).all()) else vs.permute(1, 0, 2)[:, None]
                o = (p[..., None] * live).sum(-2)
                weight = (p[..., None] * live.abs()).sum(-2)
                size = torch.where(torch.isfinite(scores), torch.einsum("hgd,thd->hgt", q.abs(), ks.abs()) / math.sqrt(self.dim), 0.0).amax(-1)
                # output and probabilities rounded to the element type; scores: `dim` products added in 32 bits, scaled, an exponential of 2 steps;
                # sums over the keys in 32 bits
                slack = 2 * (self.dim * 2.0 ** -24 * size + 2.0 ** -20) + (8 + ks.shape[0]) * 2.0 ** -24
                far = eps * (o.abs() + weight) * (1 + 2.0 ** -7) + slack[..., None] * weight + 2.0 ** -24
                if self.out.dtype is F32:
                    far = far + 2.0 ** -24 * o.abs()
                result[lo + i] = o.view(self.heads, self.dim)
                bound[lo + i] = far.view(self.heads, self.dim)
        return result, torch.nan_to_num(bound, nan=0.0, posinf=0.0)

    def check(self, **more):
        want, bound = self.want()
        got = self.call(**more)
        _close(got, want, bound, f"{self.lens} {self.nodes}")
        return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 2, 128), (8, 8, 64), (16, 1, 128), (6, 2, 64), (10, 2, 128), (4, 2, 96), (3, 1, 33), (2, 1, 512)])
def test_trees_of_all_heads_and_types(dtype, heads, kv_heads, dim):
    Case(heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, ctx=(0, 37, 300), nodes=(7, 1, 33), lists="tree", seed=dim).check()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim", [1, 63, 65, 127, 129, 192, 200, 256, 257, 320, 511])
def test_heads_of_any_size(dtype, dim):
    Case(heads=6, kv_heads=2, dim=dim, dtype=dtype, ctx=(70, 0, 513), nodes=(9, 3, 40), seed=dim).check()


@pytest.mark.parametrize("page", [16, 32, 128, 8, 5, 48])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_page_sizes(page, dtype):
    case = Case(page=page, dtype=dtype, ctx=(0, 1, 130, 257), nodes=(3, 16, 17, 5), seed=page)
    case.spoil_behind()
    case.check()


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 127, 128, 129, 143, 144, 145, 255, 256, 257, 1000])
def test_lengths_around_the_ends_of_pages_and_tiles(length, dim):
    """Rows end at the length, whatever the number of them; what stands behind may hold anything."""
    nodes = [1, min(length, 2), min(length, 16), min(length, 31), min(length, 40)]
    case = Case(dim=dim, ctx=[length - n for n in nodes], nodes=nodes, dtype=BF16, seed=length)
    case.spoil_behind()
    case.check()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 100, 128, 200])
@pytest.mark.parametrize("lists", ["tree", None, "star"])
def test_numbers_of_rows(n, lists):
    """Rows of one tile of queries, two, and several; 32 bits of a word and more."""
    Case(ctx=(70, 3, 513), nodes=(n, max(1, n // 2), 1), lists=lists, dtype=F16, seed=n).check()


@pytest.mark.parametrize("heads, kv_heads", [(64, 1), (48, 2), (7, 1), (80, 1)])
def test_many_and_odd_heads_per_key_value_head(heads, kv_heads):
    Case(heads=heads, kv_heads=kv_heads, ctx=(200, 90), nodes=(9, 3), dtype=BF16).check()


def test_one_row_each_is_the_decode_attention():
    from cacheir_b200 import ops
    case = Case(ctx=(99, 0, 700), nodes=(1, 1, 1), lists=None)
    got = case.check()
    table = case.table.clamp(0, case.keys.shape[0] - 1)
    plain = ops.paged_attention_decode_batch(case.q, case.keys, case.values, table, case.seq_lens)
    assert float((got.float() - plain.float()).norm() / plain.float().norm()) < 2e-3


def test_sequences_without_rows_and_rows_without_sequences():
    """Rows behind the last sequence stay as they were; a sequence may have no rows, or all of its tokens as rows."""
    case = Case(ctx=(50, 20, 0, 9, 0), nodes=(0, 6, 4, 0, 0), padded=3, seed=4)
    got = case.check()
    assert bool((got[10:] == 7.0).all())


def test_random_masks_and_rows_that_see_nothing():
    rng = random.Random(5)
    nodes = (20, 33, 5, 64)
    lists = [sorted(rng.sample(range(n), rng.randrange(0, n + 1))) if rng.random() < 0.7 else [] for n in nodes for _ in range(n)]
    got = Case(ctx=(0, 0, 30, 0), nodes=nodes, lists=lists, dtype=BF16, seed=5).check()
    empty = [i for i, seen in enumerate(lists) if not seen and not 53 <= i < 58]
    assert empty and bool((got[empty] == 0).all())


def test_bits_behind_a_sequence_s_rows_are_not_looked_at():
    case = Case(ctx=(40, 11), nodes=(5, 9), words=3)
    want, bound = case.want()
    for lo, n in zip(case.starts, case.nodes):
        case.visible[lo: lo + n, 0] |= ~((1 << n) - 1)
        case.visible[lo: lo + n, 1:] = -1
    _close(case.call(), want, bound)


def test_rows_behind_the_masks_bits_are_seen_by_none():
    case = Case(ctx=(40,), nodes=(50,), lists="chain", words=1)
    case.check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ctx, nodes, heads", [(0, 9, 8), (100, 40, 8), (120, 20, 64), (1000, 33, 4), (2000, 130, 4)])
@pytest.mark.parametrize("lists", ["tree", None])
def test_what_a_row_does_not_see_may_hold_anything(dtype, ctx, nodes, heads, lists):
    """Infinities and NaN in a row's key and value reach the rows that follow it and no others."""
    case = Case(heads=heads, kv_heads=2 if heads > 4 else 1, ctx=(ctx, 17), nodes=(nodes, 4), dtype=dtype, lists=lists, seed=nodes)
    case.spoil_behind()
    bad = [nodes - 1, nodes // 2 + 1]
    kinds = [(math.nan, math.nan), (1.0, math.inf)]
    for j, (k, v) in zip(bad, kinds):
        page, offset = case.place(0, ctx + j)
        case.keys[page, :, offset] = k
        case.values[page, 0, offset, ::3] = v
    want, bound = case.want()
    # where a visible value is infinite or no number, so is the result; elsewhere nothing has changed
    got = case.call()
    plain = torch.isfinite(want)
    assert bool((torch.isfinite(got.double()) == plain).all())
    _close(torch.where(plain, got.double(), 0.0), torch.where(plain, want, 0.0), bound)
    assert bool(torch.isnan(want).any()) and bool(plain.any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads, dim, ctx, nodes", [(8, 128, 5, 300), (8, 64, 2000, 120), (64, 128, 900, 40), (3, 64, 0, 33), (16, 128, 3000, 70)])
@pytest.mark.parametrize("lists", ["tree", None])
def test_many_values_that_are_no_numbers(dtype, heads, dim, ctx, nodes, lists):
    """Infinities of either sign and NaN in many rows' values, some of whose keys have scores of -inf and so no weight."""
    kv_heads = 1 if heads == 3 else 2
    case = Case(heads=heads, kv_heads=kv_heads, dim=dim, ctx=(ctx, 30), nodes=(nodes, 9), dtype=dtype, lists=lists, seed=heads)
    case.q[:] = case.q.abs()
    rng = random.Random(nodes)
    for j in rng.sample(range(nodes), nodes // 3):
        page, offset = case.place(0, ctx + j)
        for kind in (math.inf, -math.inf, math.nan):
            if rng.random() < 0.5:
                case.values[page, rng.randrange(kv_heads), offset, rng.randrange(dim)] = kind
        if rng.random() < 0.3:
            case.keys[page, :, offset] = -math.inf
    want, bound = case.want()
    got = case.call()
    assert bool(torch.isnan(want).any()) and bool((want == math.inf).any()) and bool((want == -math.inf).any())
    _close(got, want, bound)


def test_one_infinite_value_takes_little_time():
    """Rows look for it together (one by one the call took a hundred times as long, and waits of very long chains would have run out)."""
    case = Case(dim=128, ctx=(100,), nodes=(6000,), lists=None, dtype=BF16)

    def shortest():
        times = []
        for _ in range(6):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            case.call()
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    plain = shortest()
    page, offset = case.place(0, 6099)
    case.values[page, :, offset, 5] = math.inf
    assert shortest() < 20 * plain
    assert bool((case.out[5999, :, 5] == math.inf).all()) and int(torch.isfinite(case.out).logical_not().sum()) == 8


def test_scores_of_minus_infinity_and_nan():
    case = Case(ctx=(300, 300), nodes=(4, 4), dtype=BF16)
    case.q[:] = case.q.abs()
    page, offset = case.place(0, 130)
    case.keys[page, :, offset] = -math.inf                       # a score of -inf for every row: no weight
    page, offset = case.place(1, 299)
    case.keys[page, 0, offset] = math.nan
    want, bound = case.want()
    got = case.call()
    assert bool(torch.isnan(want[4:, :4]).all()) and bool(torch.isnan(got[4:, :4]).all())
    keep = torch.isfinite(want)
    _close(torch.where(keep, got.double(), 0.0), torch.where(keep, want, 0.0), bound)
    assert bool(torch.isfinite(got[:4]).all())


def test_page_ids_outside_the_pool_read_as_zeros():
    case = Case(ctx=(60,), nodes=(4,))
    case.table[0, 1] = case.keys.shape[0]
    case.table[0, 2] = -1
    case.check()


def test_more_rows_than_tokens_and_tables_that_are_too_short():
    """Tokens that are not there are seen by nobody."""
    case = Case(ctx=(-3, 30), nodes=(8, 4), dtype=BF16)
    case.check()
    case = Case(ctx=(60, 20), nodes=(10, 4))
    case.table = case.table[:, :4].contiguous()                  # 64 tokens of 70
    got = case.call()
    assert bool(torch.isfinite(got).all())
    assert bool((got[4:10] != 7.0).any())


@pytest.mark.parametrize("sequences", [3, 400, 1500])
def test_many_sequences(sequences):
    rng = random.Random(sequences)
    ctx, nodes = [rng.choice([0, 5, 40, 130]) for _ in range(sequences)], [rng.choice([0, 1, 2, 5]) for _ in range(sequences)]
    if sequences > 1000:
        ctx, nodes = [c if b % 50 == 0 else 3 for b, c in enumerate(ctx)], [n if b % 10 == 0 else b % 2 for b, n in enumerate(nodes)]
    Case(heads=4, kv_heads=2, dim=64, ctx=ctx, nodes=nodes, seed=sequences).check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads, kv_heads", [(32, 8), (64, 4)])
def test_blocks_with_many_items_of_many_tiles(dim, heads, kv_heads):
    """Items of one group of query rows and of two, in turn, and no wait of a kernel has given up."""
    from cacheir_b200 import _lib
    rng = random.Random(dim + heads)
    ctx, nodes = [rng.choice([0, 100, 800, 1500]) for _ in range(60)], [rng.choice([0, 1, 3, 17, 40]) for _ in range(60)]
    Case(heads=heads, kv_heads=kv_heads, dim=dim, ctx=ctx, nodes=nodes, dtype=BF16, seed=dim).check()
    assert _lib.load_group("drafts").cacheir_b200_drafts_device_status(0) == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("most", [60, 300, 900])
def test_blocks_with_many_short_items(dim, most):
    """Items of one tile, of two and of three, of one half of the rows and of both, one after the other in every block."""
    from cacheir_b200 import _lib
    rng = random.Random(dim + most)
    ctx, nodes = [rng.choice([0, 3, 90, 150, most]) for _ in range(200)], [rng.choice([0, 1, 2, 20]) for _ in range(200)]
    Case(heads=32, kv_heads=4, dim=dim, ctx=ctx, nodes=nodes, lists=None, dtype=F16, seed=dim).check()
    assert _lib.load_group("drafts").cacheir_b200_drafts_device_status(0) == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_one_group_of_warps_far_behind_the_other(dim):
    """Chains whose later rows, which are one group's, go through many tokens for one that is no number, among hundreds of sequences of one tile, which are all the
    other group's: more than there are places for items in shared memory."""
    from cacheir_b200 import _lib
    ctx, nodes = [], []
    for part in range(3):
        ctx += [900] + [3 + part] * 150
        nodes += [200 + part] + [1] * 150
    case = Case(heads=32, kv_heads=8, dim=dim, ctx=ctx, nodes=nodes, lists=None, dtype=BF16, seed=dim)
    for b in range(0, len(nodes), 151):
        page, offset = case.place(b, ctx[b] + nodes[b] - 1)
        case.values[page, :, offset, ::5] = math.inf
    want, bound = case.want()
    got = case.call()
    plain = torch.isfinite(want)
    assert bool((torch.isfinite(got.double()) == plain).all()) and not bool(plain.all())
    _close(torch.where(plain, got.double(), 0.0), torch.where(plain, want, 0.0), bound)
    assert _lib.load_group("drafts").cacheir_b200_drafts_device_status(0) == 0


@pytest.mark.parametrize("lists", ["tree", None])
def test_long_context_in_many_pieces(lists):
    got = Case(heads=4, kv_heads=1, ctx=(40000, 77), nodes=(6, 3), lists=lists, dtype=BF16, wide_q=2).check()
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads, nodes", [(1, 1), (3, 1), (1, 5), (4, 2), (3, 4), (16, 1), (5, 5), (32, 1), (11, 3), (32, 3)])
def test_few_rows_in_many_pieces(heads, nodes, dim):
    """Pieces are joined by lanes that share them out; one of them holds nothing but keys without weight, another a value that is no number, for the last row alone."""
    case = Case(heads=heads, kv_heads=1, dim=dim, ctx=(30000, 9000), nodes=(nodes, nodes), lists=None, dtype=BF16, seed=heads)
    case.q[:] = case.q.abs()
    for t in range(5000, 6000):
        page, offset = case.place(0, t)
        case.keys[page, :, offset] = -math.inf
    page, offset = case.place(1, 9000 + nodes - 1)
    case.values[page, :, offset] = math.nan
    want, bound = case.want()
    got = case.call()
    last = slice(2 * nodes - 1, 2 * nodes)
    assert bool(torch.isnan(got[last]).all())
    _close(got[: 2 * nodes - 1], want[: 2 * nodes - 1], bound[: 2 * nodes - 1])
    assert torch.equal(got[: 2 * nodes - 1], case.call()[: 2 * nodes - 1])


def test_a_long_chain_of_rows():
    """A prompt's rows over its own cache: no mask, more rows than words have bits."""
    Case(heads=4, kv_heads=2, dim=64, ctx=(100,), nodes=(1100,), lists=None).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_are_not_cut_and_need_no_scratch(dtype):
    from cacheir_b200 import draft_ops
    case = Case(heads=8, kv_heads=2, dim=512, ctx=(20, 7, 0, 4), nodes=(1500, 600, 0, 40), padded=2, lists=None, dtype=dtype, seed=3)
    assert draft_ops.tree_attention_workspace_bytes(case.q.shape[0], 8, 512) == 0
    case.values[case.place(1, 606)[0], :, case.place(1, 606)[1], 9] = math.inf       # (of the last row alone)
    want, bound = case.want()
    got = case.call()
    _close(got, want, bound)
    assert bool((got[2140:] == 7.0).all()) and int((got == math.inf).sum()) == 8


def test_strides_alignment_and_workspaces():
    from cacheir_b200 import draft_ops
    case = Case(ctx=(200, 31), nodes=(7, 12), wide_q=4, dtype=BF16)
    want, bound = case.want()
    need = draft_ops.tree_attention_workspace_bytes(19, 8, 128)
    first = case.call(workspace=torch.empty(need, dtype=torch.uint8, device=DEV)).clone()
    _close(first, want, bound)
    assert torch.equal(case.call().view(torch.int16), first.view(torch.int16)), "the same bits again"
    room = torch.empty(19 * 8 * 128 + 1, dtype=BF16, device=DEV)       # rows that begin anywhere
    room[1:] = case.q.reshape(-1)
    case.q, case.out = room[1:].view(19, 8, 128), torch.empty(19 * 8 * 128 + 1, dtype=BF16, device=DEV)[1:].view(19, 8, 128)
    _close(case.call(), want, bound)
    case.q = case.q.clone()
    case.out = torch.empty(19, 9 * 128, dtype=BF16, device=DEV)[:, 64: 64 + 8 * 128].view(19, 8, 128)
    _close(case.call(), want, bound)


def test_softmax_scale():
    case = Case(ctx=(50,), nodes=(5,), dtype=BF16)
    q = case.q.clone()
    case.q = q * 2
    want = case.call().clone()
    case.q = q
    assert float((case.call(softmax_scale=2 / math.sqrt(128)).float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())


def test_large_scores_move_the_reference():
    """Scores that grow along the keys by more than a factor of 2^14 at a time."""
    case = Case(ctx=(1500, 700), nodes=(3, 30), dtype=BF16, scale=0.0)
    case.q[:] = 0.0
    case.q[..., 0] = 40.0
    for b, n in enumerate(case.lens):
        for t in range(n):
            page, offset = case.place(b, t)
            case.keys[page, :, offset, 0] = (t * 37 % 400 if b else t) / 8.0
    case.check()


def test_another_stream_and_a_captured_call():
    from cacheir_b200 import draft_ops
    case = Case(ctx=(600, 90, 0), nodes=(9, 3, 4), dtype=F16)
    want, bound = case.want()
    workspace = torch.empty(draft_ops.tree_attention_workspace_bytes(16, 8, 128), dtype=torch.uint8, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        case.call(workspace=workspace)
    stream.synchronize()
    _close(case.out, want, bound)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.call(workspace=workspace)
    case.out.fill_(7.0)
    graph.replay()
    _close(case.out, want, bound)
    # the same graph for other lengths, rows and masks
    other = Case(ctx=(123, 400, 77), nodes=(2, 5, 8), dtype=F16, padded=1, seed=9)
    for name in ("keys", "values"):
        pool = getattr(other, name)
        grown = torch.zeros_like(case.keys) if pool.shape[0] < case.keys.shape[0] else pool
        grown[: pool.shape[0]] = pool
        assert grown.shape == case.keys.shape, "the first batch has more pages"
        getattr(case, name).copy_(grown)
        setattr(other, name, grown)
    table = torch.zeros_like(case.table)
    table[:, : other.table.shape[1]] = other.table
    case.table.copy_(table)
    for name in ("seq_lens", "cu_rows", "visible", "q"):
        getattr(case, name).copy_(getattr(other, name))
    other.out = case.out
    case.out.fill_(7.0)
    want, bound = other.want()
    graph.replay()
    _close(case.out, want, bound)
    torch.cuda.synchronize()


def test_first_use_inside_two_graphs_and_overlapping_calls():
    """Calls on two streams at once, each with a workspace of its own."""
    from cacheir_b200 import draft_ops
    cases = [Case(ctx=(3000, 200), nodes=(6, 9), seed=s, dtype=BF16) for s in (1, 2)]
    wants = [c.want() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    spaces = [torch.empty(draft_ops.tree_attention_workspace_bytes(15, 8, 128), dtype=torch.uint8, device=DEV) for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for case, stream, space in zip(cases, streams, spaces):
            with torch.cuda.stream(stream):
                case.call(workspace=space)
    torch.cuda.synchronize()
    for case, (want, bound) in zip(cases, wants):
        _close(case.out, want, bound)


# ---- norms, rotary positions, append -----------------------------------------------------------------------------------
def _norm_want(x, weight, offset, eps, rule_freq, positions, rot, layout):
    """(values in 64 bits, magnitudes that errors are relative to)"""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * (weight.double() + offset)
    angle = positions.double()[:, None] * rule_freq[None, :]
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    out, size = y.clone(), y.abs()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if layout == "interleaved" else (y[..., : rot // 2], y[..., rot // 2: rot])
    first, second = a * cos - b * sin, a * sin + b * cos
    both = a.abs() + b.abs()
    if layout == "interleaved":
        out[..., 0:rot:2], out[..., 1:rot:2], size[..., 0:rot:2], size[..., 1:rot:2] = first, second, both, both
    else:
        out[..., : rot // 2], out[..., rot // 2: rot], size[..., : rot // 2], size[..., rot // 2: rot] = first, second, both, both
    return out, size


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim, rot", [(128, 128), (64, 64), (128, 32), (256, 128), (96, 96), (80, 20), (33, 2), (7, 6), (1024, 1024), (512, 64)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_normed_heads_and_append(dtype, dim, rot, layout):
    from cacheir_b200 import draft_ops, serving_ops
    rows, heads, kv_heads, page = 37, 3, 2, 16
    gen = torch.Generator(device=DEV).manual_seed(dim * 3 + rot)
    fused = (torch.randn(rows, (heads + 2 * kv_heads) * dim, device=DEV, generator=gen) * torch.logspace(-2, 2, rows, device=DEV)[:, None]).to(dtype)
    fused[5] = 0.0
    q, k, v = (fused[:, lo * dim: hi * dim].view(rows, -1, dim) for lo, hi in ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    weights = [(1 + 0.3 * torch.randn(dim, device=DEV, generator=gen)) for _ in range(2)]
    kind = dim % 3
    weights = [w.to(dtype) for w in weights] if kind == 0 else weights if kind == 1 else [weights[0].to(dtype), None]
    offset = 1.0 if kind == 1 else 0.0
    rule = serving_ops.rotary_rule(rot, 10000.0, layout=layout)
    freq = (10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).to(DEV)
    positions = torch.randint(0, 100000, (rows,), device=DEV, generator=gen).to(torch.int32)
    slots = torch.randperm(4 * page, device=DEV, generator=gen)[:rows].to(torch.int32)
    slots[7], slots[30] = -1, 4 * page + 3
    pools = [torch.full((4, kv_heads, page, dim), 5.0, dtype=dtype, device=DEV) for _ in range(2)]
    q_out, k_out = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    eps = 1e-5
    draft_ops.norm_rotary_append(q, k, v, rule, positions, weights[0], weights[1], eps=eps, offset=offset, slots=slots, k_cache=pools[0], v_cache=pools[1],
                                 q_out=q_out, k_out=k_out)
    # a rounding; mean, root, weight and angle in 32 bits: dim / 32 + 16 steps at most of the pair's size
    steps = (dim / 32 + 16) * 2.0 ** -24
    live = [r for r in range(rows) if r not in (7, 30)]
    for out, x, w in ((q_out, q, weights[0]), (k_out, k, weights[1])):
        want, size = _norm_want(x, w, offset, eps, freq, positions, rot, layout)
        bound = _half_step(dtype) * (want.abs() + steps * size) + steps * size + (2.0 ** -25 if dtype is F16 else 0.0)
        _close(out[live], want[live], bound[live], str(dtype))
        assert bool((out[[7, 30]] == 9.0).all()), "rows outside the pool are left out"
    flat = slots[live].long()
    assert torch.equal(pools[0][flat // page, :, flat % page], k_out[live]) and torch.equal(pools[1][flat // page, :, flat % page], v[live])
    rest = torch.ones(4 * page, dtype=torch.bool, device=DEV)
    rest[flat] = False
    rest = rest.nonzero()[:, 0]
    assert all(bool((pool[rest // page, :, rest % page] == 5.0).all()) for pool in pools)
    # in place, without an append
    again = fused.clone()
    q2, k2 = again[:, : heads * dim].view(rows, heads, dim), again[:, heads * dim: (heads + kv_heads) * dim].view(rows, kv_heads, dim)
    draft_ops.norm_rotary_append(q2, k2, None, rule, positions, weights[0], weights[1], eps=eps, offset=offset)
    assert torch.equal(q2[live], q_out[live]) and torch.equal(k2[live], k_out[live])
    assert torch.equal(again[:, (heads + kv_heads) * dim:], fused[:, (heads + kv_heads) * dim:])


@pytest.mark.parametrize("rows, heads, kv_heads", [(1, 32, 8), (700, 5, 1), (5000, 7, 3)])
def test_normed_heads_of_few_and_many_rows(rows, heads, kv_heads):
    from cacheir_b200 import draft_ops, serving_ops
    gen = torch.Generator(device=DEV).manual_seed(rows)
    q, k = (torch.randn(rows, h, 64, device=DEV, generator=gen).to(BF16) for h in (heads, kv_heads))
    rule, freq = serving_ops.rotary_rule(64, 5e5, layout="half"), (5e5 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    positions = torch.randint(0, 2 ** 31 - 1, (rows,), device=DEV, generator=gen).to(torch.int32)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    draft_ops.norm_rotary_append(q, k, None, rule, positions, None, None, eps=0.0, q_out=q_out, k_out=k_out)
    for out, x in ((q_out, q), (k_out, k)):
        assert bool(torch.isfinite(out).all())
        length = torch.linalg.vector_norm(out.double(), dim=-1)
        assert float((length - 8.0).abs().max()) <= 8.0 * 2.0 ** -8, "turns keep a normed head's length"


@pytest.mark.parametrize("rows, heads, kv_heads, dim, rot", [(33, 32, 8, 128, 128), (700, 32, 8, 128, 128), (5000, 32, 8, 128, 128), (33, 64, 8, 128, 32), (700, 64, 8, 128, 32), (5000, 64, 8, 128, 128),
                                                             (700, 40, 5, 64, 64), (700, 20, 4, 256, 64), (33, 25, 5, 80, 20), (700, 11, 1, 33, 32), (5000, 9, 3, 96, 96)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_normed_heads_of_many_a_lane(rows, heads, kv_heads, dim, rot, layout, dtype):
    """More heads than a block has lanes for at a time: several heads a lane, queries, keys and values among them, with weights that differ."""
    from cacheir_b200 import draft_ops, serving_ops
    page, gen = 16, torch.Generator(device=DEV).manual_seed(rows + heads)
    fused = (torch.randn(rows, (heads + 2 * kv_heads) * dim, device=DEV, generator=gen) * 3).to(dtype)
    q, k, v = (fused[:, lo * dim: hi * dim].view(rows, -1, dim) for lo, hi in ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    weights = [(1 + 0.3 * torch.randn(dim, device=DEV, generator=gen)).to(dtype if rows != 700 else F32), (2 + 0.3 * torch.randn(dim, device=DEV, generator=gen)).to(dtype if rows != 700 else F32)]
    if rows == 33:
        weights[0 if heads == 32 else 1] = None
    offset, eps = (1.0 if rows == 700 else 0.0), 1e-5
    rule = serving_ops.rotary_rule(rot, 10000.0, layout=layout)
    freq = (10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).to(DEV)
    positions = torch.randint(0, 100000, (rows,), device=DEV, generator=gen).to(torch.int32)
    pages = rows // page + 2
    slots = torch.randperm(pages * page, device=DEV, generator=gen)[:rows].to(torch.int32)
    slots[rows // 2] = -1
    pools = [torch.full((pages, kv_heads, page, dim), 5.0, dtype=dtype, device=DEV) for _ in range(2)]
    q_out, k_out = torch.full((rows, heads, dim), 9.0, dtype=dtype, device=DEV), torch.full((rows, kv_heads, dim), 9.0, dtype=dtype, device=DEV)
    draft_ops.norm_rotary_append(q, k, v, rule, positions, weights[0], weights[1], eps=eps, offset=offset, slots=slots, k_cache=pools[0], v_cache=pools[1],
                                 q_out=q_out, k_out=k_out)
    steps = (dim / 32 + 16) * 2.0 ** -24                           # (as above)
    live = torch.ones(rows, dtype=torch.bool, device=DEV)
    live[rows // 2] = False
    for out, x, w in ((q_out, q, weights[0]), (k_out, k, weights[1])):
        want, size = _norm_want(x, w, offset, eps, freq, positions, rot, layout)
        bound = _half_step(dtype) * (want.abs() + steps * size) + steps * size
        _close(out[live], want[live], bound[live], str(dtype))
        assert bool((out[~live] == 9.0).all())
    flat = slots[live].long()
    assert torch.equal(pools[0][flat // page, :, flat % page], k_out[live]) and torch.equal(pools[1][flat // page, :, flat % page], v[live])
    rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    rest[flat] = False
    rest = rest.nonzero()[:, 0]
    assert all(bool((pool[rest // page, :, rest % page] == 5.0).all()) for pool in pools)


def test_norms_without_weights_are_the_rotary_append_of_normed_heads():
    from cacheir_b200 import draft_ops, serving_ops
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, k = torch.randn(50, 4, 128, device=DEV, generator=gen), torch.randn(50, 2, 128, device=DEV, generator=gen)
    rule, positions = serving_ops.rotary_rule(128, 1e4, yarn=(16.0, 8192.0, 32.0, 1.0)), torch.randint(0, 9999, (50,), device=DEV, generator=gen).to(torch.int32)
    normed = [x / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6).float() for x in (q, k)]
    serving_ops.rotary_append(*normed, None, rule, positions)
    draft_ops.norm_rotary_append(q, k, None, rule, positions, None, None)
    for got, want in zip((q, k), normed):
        assert float((got - want).abs().max()) <= 24 * 2.0 ** -24 * 2 * float(want.abs().max())


# ---- logits --------------------------------------------------------------------------------------------------------------
def _logits_case(rows, sequences, vocab, dtype, seed, *, width=0, biases=0, grammar=False, drafts=False, wide=0):
    from cacheir_b200 import draft_ops
    rng, gen = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.rand(shape, device=DEV, generator=gen)
    nodes = [rows // sequences + (b < rows % sequences) for b in range(sequences)]
    more = {}
    row_seq = [b for b, n in enumerate(nodes) for _ in range(n)]
    if drafts or rows != sequences:
        more["row_seq"] = _i32(row_seq)
    logits = ((rand(rows, vocab + wide) - 0.5) * 20).to(dtype)[:, :vocab]
    logits[0, : min(3, vocab)] = torch.tensor([-math.inf, 0.0, -0.0], device=DEV).to(dtype)[: min(3, vocab)]
    if width:
        tokens = (rand(sequences, width) ** 2 * (vocab + 2)).to(torch.int32) - 1                     # (some outside the vocabulary)
        lens = _i32([rng.randrange(0, width + 3) - 1 for _ in range(sequences)])
        more["history"] = draft_ops.TokenHistory(tokens, lens, _i32([rng.randrange(-1, width + 2) for _ in range(sequences)]) if seed % 2 else None)
    if width or drafts:
        more.update(repetition=0.8 + rand(sequences), frequency=rand(sequences) - 0.5, presence=rand(sequences) - 0.5)
    if biases:
        ids = (rand(sequences, biases) * (vocab + 1)).to(torch.int32) - 1
        if biases > 2:
            ids[:, 0] = ids[:, biases - 1]                                                            # (a token twice: the last counts)
        more.update(bias_ids=ids, bias_values=10 * rand(sequences, biases) - 5)
    if grammar:
        more["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), device=DEV, generator=gen).to(torch.int32)
        more["allowed"][rows // 2] = 0
    if drafts:
        trees = [_seen(tree) for tree in _trees(rng, nodes, "tree")]
        words = max(1, (max(nodes) + 31) // 32)
        ids = torch.tensor([rng.choice([-1, vocab, 2 ** 40, rng.randrange(vocab), vocab - 1]) if i % 4 else vocab // 2 for i in range(rows)], device=DEV)
        more["drafts"] = draft_ops.DraftedTokens(ids, _i32([line for seen in trees for line in _words(seen, words)]), _i32(_starts(nodes)))
        more["_trees"] = trees
    return logits, row_seq, more


def _logits_want(logits, row_seq, more):
    rows, vocab = logits.shape
    out, size = logits.double().clone(), logits.double().abs()
    history, drafts = more.get("history"), more.get("drafts")
    base = {}
    for r, b in enumerate(row_seq):
        base.setdefault(b, r)
        count, prompt = torch.zeros(vocab, dtype=torch.float64), set()
        if history is not None:
            n = min(int(history.lens[b]), history.tokens.shape[1])
            first = 0 if history.prompt_lens is None else int(history.prompt_lens[b])
            for i, t in enumerate(history.tokens[b, : max(n, 0)].tolist()):
                if 0 <= t < vocab:
                    if i < first:
                        prompt.add(t)
                    else:
                        count[t] += 1
        if drafts is not None:
            for j in more["_trees"][b][r - base[b]]:
                t = int(drafts.ids[base[b] + j])
                if 0 <= t < vocab:
                    count[t] += 1
        known = count > 0
        if prompt:
            known[list(prompt)] = True
        count, known = count.to(DEV), known.to(DEV)
        x = out[r]
        if "repetition" in more:
            rep = more["repetition"][b].double()
            x = torch.where(known, torch.where(x > 0, x / rep, x * rep), x)
            size[r] = torch.maximum(size[r], x.abs())
            freq, pres = more["frequency"][b].double(), more["presence"][b].double()
            x = x - freq * count - pres * (count > 0)
            size[r] += (freq * count).abs() + pres.abs() * (count > 0)
        if "bias_ids" in more:
            bias = torch.zeros(vocab, dtype=torch.float64)
            for t, value in zip(more["bias_ids"][b].tolist(), more["bias_values"][b].tolist()):
                if 0 <= t < vocab:
                    bias[t] = value
            x = x + bias.to(DEV)
            size[r] += bias.abs().to(DEV)
        if "allowed" in more:
            at = torch.arange(vocab, device=DEV)
            x = torch.where((more["allowed"][r][at // 32] >> (at % 32) & 1) != 0, x, -math.inf)
        out[r] = x
    return out, size


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows, sequences, vocab", [(1, 1, 128256), (5, 5, 50001), (12, 3, 1000), (40, 40, 31), (3, 3, 1), (64, 2, 9999), (300, 20, 2049)])
@pytest.mark.parametrize("kind", ["all", "penalties", "grammar", "bias", "drafts"])
def test_adjusted_logits(dtype, rows, sequences, vocab, kind):
    from cacheir_b200 import draft_ops
    logits, row_seq, more = _logits_case(rows, sequences, vocab, dtype, rows + vocab, width=700 if kind in ("all", "penalties") else 0,
                                         biases=7 if kind in ("all", "bias") else 0, grammar=kind in ("all", "grammar"), drafts=kind in ("all", "drafts"), wide=vocab % 5)
    want, size = _logits_want(logits, row_seq, more)
    # four operations in 32 bits, each within half a step of the largest value on the way, and the rounding of the output
    size = torch.nan_to_num(size, posinf=0.0)
    bound = lambda t: 8 * 2.0 ** -24 * size + _half_step(t) * (size if t is F32 else torch.nan_to_num(want, neginf=0.0).abs() + 8 * 2.0 ** -24 * size) + 2.0 ** -25
    call = {k: v for k, v in more.items() if not k.startswith("_")}
    before = logits.clone()
    out = torch.full((rows, vocab), 3.0, dtype=dtype, device=DEV)
    assert draft_ops.adjust_logits(logits, out=out, **call) is out
    assert torch.equal(logits, before)
    _close(out, want, bound(dtype), kind)
    wide = torch.full((rows, vocab), 3.0, dtype=F32, device=DEV)
    draft_ops.adjust_logits(logits, out=wide, **call)
    _close(wide, want, bound(F32), kind + " to float32")
    draft_ops.adjust_logits(logits, **call)
    assert torch.equal(logits, out), "in place: the same values"


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows, sequences", [(130, 7), (200, 9), (512, 21), (520, 100)])
@pytest.mark.parametrize("kind", ["all", "drafts", "grammar"])
def test_adjusted_logits_of_blocks_with_several_rows(dtype, rows, sequences, kind):
    """Blocks of 2, 4 and 8 rows, whose sequence changes inside them or which have a row of no sequence: rows that share a count, and a count that begins again."""
    from cacheir_b200 import draft_ops
    vocab = 33001
    logits, row_seq, more = _logits_case(rows, sequences, vocab, dtype, rows, width=200 if kind == "all" else 0, biases=30 if kind == "all" else 0, grammar=kind != "drafts",
                                         drafts=kind != "grammar", wide=rows % 3)
    want, size = _logits_want(logits, row_seq, more)
    nobody = [3, 64, rows // 2 + 1, rows - 2]
    if kind == "grammar":
        more["row_seq"] = _i32(row_seq)
    more["row_seq"][nobody] = -1
    live = [r for r in range(rows) if r not in nobody]
    want, size = want[live], torch.nan_to_num(size[live], posinf=0.0)
    # (the bound of the test above)
    bound = 8 * 2.0 ** -24 * size + _half_step(dtype) * (size if dtype is F32 else torch.nan_to_num(want, neginf=0.0).abs() + 8 * 2.0 ** -24 * size) + 2.0 ** -25
    call = {k: v for k, v in more.items() if not k.startswith("_")}
    before = logits.clone()
    out = torch.full((rows, vocab), 3.0, dtype=dtype, device=DEV)
    draft_ops.adjust_logits(logits, out=out, **call)
    assert torch.equal(logits, before) and bool((out[nobody] == 3.0).all())
    _close(out[live], want, bound, kind)
    draft_ops.adjust_logits(logits, **call)
    assert torch.equal(logits[live], out[live]) and torch.equal(logits[nobody], before[nobody])


def test_adjusted_logits_of_more_rows_than_a_grid_has():
    from cacheir_b200 import draft_ops
    gen = torch.Generator(device=DEV).manual_seed(1)
    rows, vocab, sequences = 70001, 45, 5
    logits = torch.randn(rows, vocab, device=DEV, generator=gen)
    row_seq = torch.randint(0, sequences, (rows,), device=DEV, generator=gen).to(torch.int32)
    tokens = torch.randint(0, vocab, (sequences, 9), device=DEV, generator=gen).to(torch.int32)
    presence = torch.arange(1, sequences + 1, device=DEV).float() / 4
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, 2), device=DEV, generator=gen).to(torch.int32)
    said = torch.zeros(sequences, vocab, dtype=torch.bool, device=DEV).scatter_(1, tokens.long(), True)
    want = torch.where(said, -presence[:, None], 0.0)[row_seq.long()] + logits
    at = torch.arange(vocab, device=DEV)
    want = torch.where((allowed[:, at // 32] >> (at % 32) & 1) != 0, want, -math.inf)
    draft_ops.adjust_logits(logits, row_seq=row_seq, history=draft_ops.TokenHistory(tokens, _i32([9] * sequences)), presence=presence, allowed=allowed)
    assert torch.equal(logits, want)


def test_logits_rows_of_no_sequence_are_left_alone():
    from cacheir_b200 import draft_ops
    logits, row_seq, more = _logits_case(9, 3, 777, BF16, 4, width=50, grammar=True)
    more["row_seq"] = _i32([0, 0, -1, 1, 1, 3, 2, 2, -5])
    out = torch.full_like(logits, 3.0)
    draft_ops.adjust_logits(logits, out=out, **more)
    assert bool((out[[2, 5, 8]] == 3.0).all()) and not bool((out[[0, 1, 3, 4, 6, 7]] == 3.0).all(-1).any())
    only = torch.full_like(logits, 3.0)
    draft_ops.adjust_logits(logits, row_seq=more["row_seq"].clamp(max=2), allowed=more["allowed"], out=only)
    assert bool((only[[2, 8]] == 3.0).all())


def test_logits_keep_nan_and_masks_win():
    from cacheir_b200 import draft_ops
    logits = torch.tensor([[math.nan, math.nan, math.inf, 1.0]], device=DEV)
    history = draft_ops.TokenHistory(_i32([[0, 1, 2, 3]]), _i32([4]))
    out = draft_ops.adjust_logits(logits, history=history, repetition=torch.tensor([2.0], device=DEV), allowed=_i32([[0b1101]]))
    assert bool(torch.isnan(out[0, 0])) and float(out[0, 1]) == -math.inf and float(out[0, 2]) == math.inf and float(out[0, 3]) == 0.5


def test_logits_on_another_stream_and_captured():
    from cacheir_b200 import draft_ops
    logits, row_seq, more = _logits_case(20, 4, 5000, BF16, 7, width=100, biases=4, grammar=True, drafts=True)
    trees = more.pop("_trees")
    out = torch.zeros_like(logits)
    draft_ops.adjust_logits(logits, out=out, **more)
    first = out.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            draft_ops.adjust_logits(logits, out=out, **more)
    out.zero_()
    graph.replay()
    assert torch.equal(out, first) and trees
    logits.copy_(logits.flip(1))
    graph.replay()
    want = torch.zeros_like(out)
    draft_ops.adjust_logits(logits, out=want, **more)
    assert torch.equal(out, want)


@pytest.mark.parametrize("row_0", ["in the history", "among the drafts", "of the prompt"])
def test_drafted_tokens_are_penalized_like_said_ones(row_0):
    """A row's logits are those of a sequence whose history ends with the tokens that the row follows, row 0's among them."""
    from cacheir_b200 import draft_ops
    rng, gen = random.Random(6), torch.Generator(device=DEV).manual_seed(6)
    nodes, vocab, width = (6, 1, 40, 9), 301, 80
    trees = [_seen(tree) for tree in _trees(rng, nodes, "tree")]
    prompts = [[rng.randrange(vocab) for _ in range(rng.randrange(1, 12))] for _ in nodes]
    answers = [[] if row_0 == "of the prompt" else [rng.randrange(40) for _ in range(rng.randrange(1, 20))] for _ in nodes]
    ids, lines, firsts = [], [], []
    for seen, prompt, answer in zip(trees, prompts, answers):
        certain = prompt + answer                                     # (row 0 is the last of them)
        own = [certain[-1]] + [rng.randrange(40) for _ in seen[1:]]
        lines += [certain + [own[j] for j in row[1:]] for row in seen]
        firsts += [len(prompt)] * len(seen)
        ids += [own[0] if row_0 == "among the drafts" else -1] + own[1:]
    logits = torch.randn(len(ids), vocab, device=DEV, generator=gen) * 4
    rand = lambda: torch.rand(len(nodes), device=DEV, generator=gen)
    penalties = dict(repetition=0.8 + rand(), frequency=rand() - 0.2, presence=rand() - 0.2)
    row_seq = _i32([b for b, n in enumerate(nodes) for _ in range(n)])
    padded = lambda line: line + [7] * (width - len(line))
    want = draft_ops.adjust_logits(logits.clone(), history=draft_ops.TokenHistory(_i32([padded(line) for line in lines]), _i32([len(line) for line in lines]), _i32(firsts)),
                                   **{name: value[row_seq.long()].contiguous() for name, value in penalties.items()})
    said = [prompt + answer[: -1 if row_0 == "among the drafts" else None] for prompt, answer in zip(prompts, answers)]
    history = draft_ops.TokenHistory(_i32([padded(line) for line in said]), _i32([len(line) for line in said]), _i32([len(prompt) for prompt in prompts]))
    visible = _i32([line for seen in trees for line in _words(seen, 2)])
    got = draft_ops.adjust_logits(logits.clone(), row_seq=row_seq, history=history, **penalties,
                                  drafts=draft_ops.DraftedTokens(torch.tensor(ids, device=DEV), visible, _i32(_starts(nodes))))
    assert torch.equal(got, want) and not torch.equal(got, logits)


# ---- drafts ----------------------------------------------------------------------------------------------------------------
def _walk(parents, ids, chosen, depth):
    path, pick = [], -1
    at = 0 if parents else None
    while at is not None and len(path) < depth:
        path.append(at)
        pick = chosen[at]
        at = next((j for j in range(at + 1, len(parents)) if parents[j] == at and ids[j] == pick), None)
    return path, pick


@pytest.mark.parametrize("nodes, words", [((1,), 1), ((8, 0, 3), 1), ((33, 32, 31, 1), 2), ((200, 5, 64, 0, 129), 7), ((1100, 40), 32), ((3,) * 300, 1)])
@pytest.mark.parametrize("shape", ["tree", "chain", "star"])
def test_positions_masks_and_paths(nodes, words, shape):
    from cacheir_b200 import draft_ops, serving_ops
    rng = random.Random(len(nodes) * 7 + words)
    trees, starts = _trees(rng, nodes, shape), _starts(nodes)
    rows, padded = starts[-1], 5
    front = [rng.randrange(0, 100) for _ in nodes]
    tokens = serving_ops.token_map(rows + padded, len(nodes), DEV)
    tokens.cu_rows.copy_(_i32(starts))
    parents = [p for tree in trees for p in tree] + [3] * padded
    if rows > 6:
        odd = starts[nodes.index(max(nodes))] + 2                   # what is no earlier row counts as none
        parents[odd] = 77777
        trees[nodes.index(max(nodes))][2] = -1
    seq_lens = _i32([f + n for f, n in zip(front, nodes)])
    tree = draft_ops.draft_tree(rows + padded, words, DEV)
    tree.positions.fill_(9)
    tree.visible.fill_(9)
    assert draft_ops.map_drafts(_i32(parents), seq_lens, tokens, tree) is tree
    seen = [_seen(t) for t in trees]
    assert tree.positions.tolist() == [f + len(line) - 1 for f, lists in zip(front, seen) for line in lists] + [0] * padded
    assert tree.visible.tolist() == [line for lists in seen for line in _words(lists, words)] + [[0] * words] * padded
    assert int(tree.status) == (max(nodes) if max(nodes) > 32 * words else 0)

    ids = [rng.randrange(4) for _ in parents]
    chosen = [rng.randrange(4) for _ in parents]
    for depth in (1, 3, max(nodes)):
        accepted = draft_ops.accepted_drafts(len(nodes), depth, DEV)
        accepted.rows.fill_(5)
        draft_ops.accept_drafts(torch.tensor(chosen, device=DEV), torch.tensor(ids, device=DEV), _i32(parents), seq_lens, tokens, accepted)
        walks = [_walk(t, ids[lo: lo + len(t)], chosen[lo: lo + len(t)], depth) for t, lo in zip(trees, starts)]
        assert accepted.counts.tolist() == [len(path) for path, _ in walks]
        assert accepted.rows.tolist() == [[lo + j for j in path] + [-1] * (depth - len(path)) for (path, _), lo in zip(walks, starts)]
        assert accepted.next_ids.tolist() == [pick for _, pick in walks]
        assert accepted.keep_lens.tolist() == [f + len(path) for f, (path, _) in zip(front, walks)]


def test_a_tree_of_more_rows_than_bits_says_so():
    from cacheir_b200 import draft_ops, serving_ops
    tokens, tree = serving_ops.token_map(90, 2, DEV), draft_ops.draft_tree(90, 1, DEV)
    tokens.cu_rows.copy_(_i32([0, 40, 90]))
    draft_ops.map_drafts(_i32(list(range(-1, 39)) + list(range(-1, 49))), _i32([40, 50]), tokens, tree)
    assert int(tree.status) == 50
    assert tree.positions.tolist() == list(range(40)) + list(range(50)) and tree.visible[39].tolist() == [-1]


@pytest.mark.parametrize("shape", ["chain", "near", "far"])
def test_a_path_of_many_rows(shape):
    """Rows far behind the words' bits: positions and paths all the same, in a time that grows as the rows do."""
    from cacheir_b200 import draft_ops, serving_ops
    rng, n, words = random.Random(3), 30000, 3
    parents = [i - 1 if shape == "chain" else rng.randrange(max(0, i - 90) if shape == "near" else 0, i) if i else -1 for i in range(n)]
    parents[70] = 70                                               # (no earlier row)
    depths, seen = [], []
    for i, up in enumerate(parents):
        mine = 1 << i if i < 32 * words else 0
        depths.append(depths[up] + 1 if 0 <= up < i else 0)
        seen.append(mine | (seen[up] if 0 <= up < i else 0))
    tokens, tree = serving_ops.token_map(n, 1, DEV), draft_ops.draft_tree(n, words, DEV)
    tokens.cu_rows.copy_(_i32([0, n]))
    seq_lens = _i32([n + 5])
    draft_ops.map_drafts(_i32(parents), seq_lens, tokens, tree)
    assert tree.positions.tolist() == [5 + d for d in depths] and int(tree.status) == n
    want = torch.tensor([[(bits >> 32 * w) & 0xffffffff for w in range(words)] for bits in seen])
    assert torch.equal(tree.visible.long().cpu() & 0xffffffff, want)

    parents[70] = 69
    follows = {}
    for i, up in enumerate(parents):
        follows.setdefault(up, []).append(i)
    ids, chosen, path = list(range(n)), [-5] * n, [0]              # the path that always takes the last row
    while path[-1] in follows:
        path.append(follows[path[-1]][-1])
        chosen[path[-2]] = path[-1]
    accepted = draft_ops.accepted_drafts(1, n, DEV)
    draft_ops.accept_drafts(torch.tensor(chosen, device=DEV), torch.tensor(ids, device=DEV), _i32(parents), seq_lens, tokens, accepted)
    assert int(accepted.counts) == len(path) and accepted.rows[0, : len(path)].tolist() == path
    assert bool((accepted.rows[0, len(path):] == -1).all()) and int(accepted.next_ids) == -5 and int(accepted.keep_lens) == 5 + len(path)


@pytest.mark.parametrize("dtype, dim", [(F16, 128), (BF16, 64), (F32, 128), (F16, 33), (F32, 5), (BF16, 7)])
@pytest.mark.parametrize("layers", [1, 70])
def test_accepted_keys_and_values_lie_together(dtype, dim, layers):
    from cacheir_b200 import draft_ops, serving_ops
    rng = random.Random(dim)
    nodes, page, kv_heads = (12, 1, 40, 0, 5), 16, 3
    starts = _starts(nodes)
    paths = [[0, 1, 2, 5, 6, 11], [0], [0] + sorted(rng.sample(range(1, 40), 21)), [], [0, 4]]
    total = 6 * page
    slots = rng.sample(range(total), starts[-1])
    slots[starts[4] + 1] = -1                                     # (a row of nowhere: nothing comes to it)
    gen = torch.Generator(device=DEV).manual_seed(1)
    pools = [torch.randn(6, kv_heads, page, dim, device=DEV, generator=gen).to(dtype) for _ in range(2 * layers)]
    want = []
    for pool in pools:
        lines = pool.transpose(1, 2).reshape(total, kv_heads, dim).clone()
        source = lines.clone()
        for lo, path in zip(starts, paths):
            for i, j in enumerate(path):
                if slots[lo + i] >= 0 and slots[lo + j] >= 0:
                    lines[slots[lo + i]] = source[slots[lo + j]]
        want.append(lines.view(6, page, kv_heads, dim).transpose(1, 2))
    tokens = serving_ops.token_map(starts[-1], len(nodes), DEV)
    tokens.cu_rows.copy_(_i32(starts))
    tokens.slots.copy_(_i32(slots))
    accepted = draft_ops.accepted_drafts(len(nodes), 25, DEV)
    accepted.counts.copy_(_i32([len(p) for p in paths]))
    accepted.rows.copy_(_i32([[lo + j for j in p] + [-1] * (25 - len(p)) for lo, p in zip(starts, paths)]))
    draft_ops.keep_accepted(accepted, tokens, draft_ops.page_pools(pools))
    for got, line in zip(pools, want):
        assert torch.equal(got, line)


# ---- together --------------------------------------------------------------------------------------------------------------
def _step(state, sizes):
    """A whole step on one attention layer: pages, positions, append, attention, logits, path, pages back."""
    from cacheir_b200 import draft_ops, ops, serving_ops
    heads, kv_heads, dim, vocab = sizes
    s = state
    t = serving_ops.extend_page_tables(s["table"], s["lens"], s["new"], s["free"], s["count"], s["tokens"], page_size=16)
    tree = draft_ops.map_drafts(s["parents"], s["lens"], t, s["tree"])
    fused = s["embed"][s["ids"]]
    rows = fused.shape[0]
    q, k, v = (fused[:, lo * dim: hi * dim].view(rows, -1, dim) for lo, hi in ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    draft_ops.norm_rotary_append(q, k, v, s["rule"], tree.positions, s["q_weight"], s["k_weight"], slots=t.slots, k_cache=s["keys"], v_cache=s["values"], q_out=s["q"])
    draft_ops.tree_attention(s["q"], s["keys"], s["values"], s["table"], s["lens"], t.cu_rows, tree.visible, out=s["out"], workspace=s["workspace"])
    logits = (s["out"].view(rows, -1) @ s["head"]).contiguous()
    draft_ops.adjust_logits(logits, row_seq=t.row_seq, drafts=draft_ops.DraftedTokens(s["ids"], tree.visible, t.cu_rows), repetition=s["repetition"],
                            allowed=s["allowed"])
    chosen = ops.argmax_rows(logits)
    accepted = draft_ops.accept_drafts(chosen, s["ids"], s["parents"], s["lens"], t, s["accepted"])
    draft_ops.keep_accepted(accepted, t, s["handle"])
    serving_ops.shrink_page_tables(s["table"], s["lens"], accepted.keep_lens, s["free"], s["count"], t.status, page_size=16)
    return chosen


def test_a_step_with_drafts_says_what_single_tokens_say():
    """Trees of drafts, some of them right, against one token at a time; the step is captured and replayed."""
    from cacheir_b200 import draft_ops, ops, serving_ops
    heads, kv_heads, dim, vocab, sequences, most = 8, 2, 64, 97, 3, 7
    sizes = (heads, kv_heads, dim, vocab)
    gen = torch.Generator(device=DEV).manual_seed(11)
    shared = dict(embed=torch.randn(vocab, (heads + 2 * kv_heads) * dim, device=DEV, generator=gen).to(BF16), head=torch.randn(heads * dim, vocab, device=DEV, generator=gen).to(BF16),
                  rule=serving_ops.rotary_rule(dim, 1e4, layout="half"), q_weight=torch.ones(dim, dtype=BF16, device=DEV) * 2, k_weight=torch.ones(dim, dtype=BF16, device=DEV) * 2,
                  repetition=torch.full((sequences,), 1.0, device=DEV))

    def fresh(rows):
        pools = [torch.zeros(40, kv_heads, 16, dim, dtype=BF16, device=DEV) for _ in range(2)]
        return dict(shared, table=torch.zeros(sequences, 10, dtype=torch.int32, device=DEV), lens=_i32([0] * sequences), new=_i32([0] * sequences),
                    free=torch.randperm(40, device=DEV, generator=gen).to(torch.int32), count=_i32([40]), tokens=serving_ops.token_map(rows, sequences, DEV),
                    parents=_i32([-1] * rows), tree=draft_ops.draft_tree(rows, 1, DEV), ids=torch.zeros(rows, dtype=torch.int64, device=DEV), keys=pools[0], values=pools[1],
                    handle=draft_ops.page_pools(pools), q=torch.zeros(rows, heads, dim, dtype=BF16, device=DEV), out=torch.zeros(rows, heads, dim, dtype=BF16, device=DEV),
                    workspace=torch.empty(draft_ops.tree_attention_workspace_bytes(rows, heads, dim), dtype=torch.uint8, device=DEV),
                    allowed=torch.full((rows, 4), -1, dtype=torch.int32, device=DEV), accepted=draft_ops.accepted_drafts(sequences, most, DEV))

    # one token at a time
    single, said = fresh(sequences), [[1], [2], [3]]
    for _ in range(60):
        single["new"].copy_(_i32([1] * sequences))
        single["ids"].copy_(torch.tensor([line[-1] for line in said], device=DEV))
        chosen = _step(single, sizes).tolist()
        for line, token in zip(said, chosen):
            line.append(token)
    # trees: two children a row, of which one is what single tokens said (mostly)
    rng, rows = random.Random(2), sequences * most
    trees, lines = fresh(rows), [[1], [2], [3]]
    parents = [-1, 0, 0, 1, 1, 3, 3]
    graph, steps, kept = None, 0, 0
    while min(len(line) for line in lines) < 50:
        ids = []
        for line, truth in zip(lines, said):
            at = len(line) - 1
            ahead = truth[at:] + [0] * most
            right = rng.random() < 0.8
            ids += [line[-1], ahead[1] if right else 50, 51, ahead[2], 52, 53, ahead[3]]
        trees["new"].copy_(_i32([most] * sequences))
        trees["parents"].copy_(_i32(parents * sequences))
        trees["ids"].copy_(torch.tensor(ids, device=DEV))
        if graph is None and steps == 1:
            saved = {name: trees[name].clone() for name in ("table", "lens", "free", "count", "keys", "values")}
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                _step(trees, sizes)
            for name, value in saved.items():
                trees[name].copy_(value)
        if graph is not None:
            graph.replay()
        else:
            _step(trees, sizes)
        accepted = trees["accepted"]
        counts, path, following = accepted.counts.tolist(), accepted.rows.tolist(), accepted.next_ids.tolist()
        for b, line in enumerate(lines):
            line += [ids[r] for r in path[b][1: counts[b]]] + [following[b]]
        kept += sum(counts)
        steps += 1
        assert trees["lens"].tolist() == [len(line) - 1 for line in lines]
        assert int(trees["tokens"].status) == 0 and int(trees["tree"].status) == 0
    assert [line[:50] for line in lines] == [truth[:50] for truth in said]
    assert kept > 2 * steps * sequences, "drafts were accepted"
    torch.cuda.synchronize()
    graph = None


def test_a_step_with_penalties_says_what_single_tokens_say(monkeypatch):
    """The same with a history of all certain tokens, row 0's among them, and penalties: the history grows by what was accepted."""
    from cacheir_b200 import draft_ops, serving_ops
    heads, kv_heads, dim, vocab, sequences, most, width = 8, 2, 64, 97, 3, 7, 90
    sizes = (heads, kv_heads, dim, vocab)
    gen = torch.Generator(device=DEV).manual_seed(12)
    shared = dict(embed=torch.randn(vocab, (heads + 2 * kv_heads) * dim, device=DEV, generator=gen).to(BF16), head=torch.randn(heads * dim, vocab, device=DEV, generator=gen).to(BF16),
                  rule=serving_ops.rotary_rule(dim, 1e4, layout="half"), q_weight=torch.ones(dim, dtype=BF16, device=DEV) * 2, k_weight=torch.ones(dim, dtype=BF16, device=DEV) * 2,
                  repetition=torch.tensor([1.3, 1.0, 1.1], device=DEV))
    history = draft_ops.TokenHistory(torch.zeros(sequences, width, dtype=torch.int32, device=DEV), _i32([1] * sequences), _i32([1] * sequences))
    plain = draft_ops.adjust_logits

    def adjust(logits, *, drafts, **more):
        ids = drafts.ids.clone()
        ids[:: len(ids) // sequences] = -1                            # (rows 0, which the history has)
        return plain(logits, history=history, frequency=torch.tensor([0.5, 2.0, 0.0], device=DEV), presence=torch.tensor([0.0, 1.0, 3.0], device=DEV),
                     drafts=draft_ops.DraftedTokens(ids, drafts.visible, drafts.cu_rows), **more)

    monkeypatch.setattr(draft_ops, "adjust_logits", adjust)

    def run(rows, count, drafted):
        """What is said in steps of so many rows a sequence."""
        pools = [torch.zeros(40, kv_heads, 16, dim, dtype=BF16, device=DEV) for _ in range(2)]
        s = dict(shared, table=torch.zeros(sequences, 10, dtype=torch.int32, device=DEV), lens=_i32([0] * sequences), new=_i32([rows] * sequences),
                 free=torch.randperm(40, device=DEV, generator=gen).to(torch.int32), count=_i32([40]), tokens=serving_ops.token_map(rows * sequences, sequences, DEV),
                 parents=_i32(([-1, 0, 0, 1, 1, 3, 3])[:rows] * sequences), tree=draft_ops.draft_tree(rows * sequences, 1, DEV),
                 ids=torch.zeros(rows * sequences, dtype=torch.int64, device=DEV), keys=pools[0], values=pools[1], handle=draft_ops.page_pools(pools),
                 q=torch.zeros(rows * sequences, heads, dim, dtype=BF16, device=DEV), out=torch.zeros(rows * sequences, heads, dim, dtype=BF16, device=DEV),
                 workspace=torch.empty(draft_ops.tree_attention_workspace_bytes(rows * sequences, heads, dim), dtype=torch.uint8, device=DEV),
                 allowed=torch.full((rows * sequences, 4), -1, dtype=torch.int32, device=DEV), accepted=draft_ops.accepted_drafts(sequences, most, DEV))
        lines, steps = [[1], [2], [3]], 0
        while min(len(line) for line in lines) < count:
            for b, line in enumerate(lines):
                history.tokens[b, : len(line)] = _i32(line)
            history.lens.copy_(_i32([len(line) for line in lines]))
            ids = [token for b, line in enumerate(lines) for token in [line[-1]] + drafted(b, line)]
            s["ids"].copy_(torch.tensor(ids, device=DEV))
            _step(s, sizes)
            counts, path, following = s["accepted"].counts.tolist(), s["accepted"].rows.tolist(), s["accepted"].next_ids.tolist()
            for b, line in enumerate(lines):
                line += [ids[r] for r in path[b][1: counts[b]]] + [following[b]]
            steps += 1
        return lines, steps

    said, _ = run(1, 60, lambda b, line: [])
    rng = random.Random(4)

    def guess(b, line):
        ahead = said[b][len(line):] + [0] * most
        return [ahead[0] if rng.random() < 0.8 else 50, 51, ahead[1], 52, 53, ahead[2]]

    lines, steps = run(most, 50, guess)
    assert [line[:50] for line in lines] == [truth[:50] for truth in said]
    assert steps < 40, "drafts were accepted"
    assert all(len(set(line)) > 10 for line in lines), "penalties keep the lines from going round"
