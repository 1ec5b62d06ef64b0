"""Torch-tensor wrappers over the operators of batches whose requests share prompts (include/cacheir_b200_serving.h).

The operators of a step, in its order: pages and slots for new tokens (`extend_page_tables`, and back: `shrink_page_tables`), rotary
positions with the append to the page pool (`rotary_append`), decode attention that reads a common prefix once for all of its requests
(`shared_prefix_attention`), log probabilities of tokens (`token_logprobs`).

Same rules as `ops`: validate, pass device pointers on the current stream, raise on a non-zero status. All tensors of a call are on one
CUDA device, which need not be the current one; the call runs on that device's current stream.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import LogprobsArgs, PrefixArgs, RotaryArgs, TablesArgs, check
from .ops import _require_cuda, dtype_code

MAX_TOP = 32
MAX_SEQUENCES = 16384
LAYOUTS = {"interleaved": 0, "half": 1}
# the argument structs as bytes (a third of the time that their ctypes classes take to fill, half of that of as many arguments)
TABLES_BYTES = struct.Struct("@11Q5i4x")
ROTARY_BYTES = struct.Struct("@10Q5q9if")
PREFIX_BYTES = struct.Struct("@11Q2q10if4x")
LOGPROBS_BYTES = struct.Struct("@6Qqd4i")
assert [s.size for s in (TABLES_BYTES, ROTARY_BYTES, PREFIX_BYTES, LOGPROBS_BYTES)] == [
    ctypes.sizeof(c) for c in (TablesArgs, RotaryArgs, PrefixArgs, LogprobsArgs)]

_I32 = torch.int32
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_calls: dict[str, object] = {}         # entry points that have been called


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


# (As these launch kernels of a few microseconds, what they do on the host is kept to about as many: shapes and strides are taken once, the
# current device is looked up and only switched where the tensors are on another one.)
def _launch(what: str, tensors: tuple, args: bytes) -> None:
    """Calls the entry point `what` with its struct and the current stream of the device that all the tensors are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            _require_cuda(*tensors)
            raise ValueError(f"all tensors of a call must be on one device, got {sorted({str(t.device) for t in tensors if t is not None})}")
    if index < 0:
        _require_cuda(*tensors)
    call = _calls.get(what)
    if call is None:
        call = _calls[what] = getattr(_lib.load_group("serving"), "cacheir_b200_" + what)
    if index == _current_device():
        code = call(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = call(args, _raw_stream(index))
    if code:
        check(code, what)


def _check_ints(what: str, *tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and (t.dtype is not _I32 or not t.is_contiguous()):
            raise TypeError(f"{what} must be contiguous int32 tensors")


def _check_heads(name: str, t: torch.Tensor) -> tuple[int, int, int, int]:
    """(rows, heads, head size, row stride)"""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        rows, heads, dim = shape
        if heads > 0 and dim > 0 and (stride[2] == 1 or dim == 1) and (stride[1] == dim or heads == 1):
            if rows > 1 and stride[0] < heads * dim:
                raise ValueError(f"{name}: rows must not overlap")
            return rows, heads, dim, stride[0]
    raise ValueError(f"{name} must be [rows, heads, dim] with dense heads: only the row stride may differ from heads * dim")


# ---- page tables -----------------------------------------------------------------------------------------------------
@dataclass
class TokenMap:
    """The rows of a step (all int32, on the device): row r is the token at `positions[r]` of sequence `row_seq[r]`, its key and value
    go to `slots[r]` (page * page_size + offset); sequence b has the rows cu_rows[b] .. cu_rows[b + 1] - 1. Rows behind the last token:
    position 0, sequence -1, slot -1. `status` keeps the first refusal until it is set to 0 (see `extend_page_tables`)."""

    positions: torch.Tensor
    row_seq: torch.Tensor
    slots: torch.Tensor
    cu_rows: torch.Tensor
    status: torch.Tensor


def token_map(rows: int, sequences: int, device: torch.device | str) -> TokenMap:
    """Room for `rows` tokens of `sequences` sequences."""
    if rows < 1 or sequences < 1:
        raise ValueError("a token map has at least one row and one sequence")
    sizes = (rows, rows, rows, sequences + 1, 1)
    return TokenMap(*(torch.zeros(n, dtype=torch.int32, device=device) for n in sizes))


def _check_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, change: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  status: torch.Tensor, page_size: int) -> tuple[int, int]:
    _check_ints("page tables, lengths, free pages and status", page_table, seq_lens, change, free_pages, free_count, status)
    shape = page_table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError("page_table must be [sequences, max_pages]")
    sequences, max_pages = shape
    if seq_lens.numel() != sequences or change.numel() != sequences:
        raise ValueError("lengths must be [sequences]")
    if not 1 <= sequences <= MAX_SEQUENCES:
        raise ValueError(f"a call takes 1 to {MAX_SEQUENCES} sequences")
    if free_pages.numel() < 1 or free_count.numel() != 1 or status.numel() != 1:
        raise ValueError("free_pages must be a stack [capacity], free_count and status one number each")
    if page_size < 1:
        raise ValueError("page_size must be positive")
    if change.data_ptr() == seq_lens.data_ptr():
        raise ValueError("the lengths that a call changes cannot also be its other lengths")
    return sequences, max_pages


def extend_page_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                       free_count: torch.Tensor, tokens: TokenMap, *, page_size: int) -> TokenMap:
    """Room for new_lens[b] more tokens of every sequence b, and where they go.

    New pages come off the stack free_pages[: free_count] into page_table [sequences, max_pages] int32, sequence by sequence; seq_lens
    and free_count are brought up to date and `tokens` is filled. Everything stays on the device, so that a captured graph can do it.
    Nothing changes (and `tokens` has no rows, every slot -1) where the call cannot be done; tokens.status then holds, until the caller sets
    it to 0, the number of missing pages, -1 (more tokens than rows), -2 (a sequence longer than its table) or -3 (free_count outside the
    stack). Beside `kv_cache.B200PagedKVCache.extend`, which walks the same pages on the host."""
    positions, row_seq, slots, cu_rows, status = tokens.positions, tokens.row_seq, tokens.slots, tokens.cu_rows, tokens.status
    sequences, max_pages = _check_tables(page_table, seq_lens, new_lens, free_pages, free_count, status, page_size)
    _check_ints("token map", positions, row_seq, slots, cu_rows)
    rows = positions.numel()
    if row_seq.numel() != rows or slots.numel() != rows or cu_rows.numel() != sequences + 1:
        raise ValueError("the token map was made for other sizes")
    args = TABLES_BYTES.pack(page_table.data_ptr(), seq_lens.data_ptr(), new_lens.data_ptr(), 0, free_pages.data_ptr(), free_count.data_ptr(),
                             positions.data_ptr(), row_seq.data_ptr(), slots.data_ptr(), cu_rows.data_ptr(), status.data_ptr(), sequences, max_pages,
                             page_size, free_pages.numel(), rows)
    _launch("extend_page_tables", (page_table, seq_lens, new_lens, free_pages, free_count, positions, row_seq, slots, cu_rows, status), args)
    return tokens


def shrink_page_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, keep_lens: torch.Tensor, free_pages: torch.Tensor,
                       free_count: torch.Tensor, status: torch.Tensor, *, page_size: int, held_pages: torch.Tensor | None = None) -> None:
    """Sequence b keeps its first min(keep_lens[b], seq_lens[b]) tokens (0: it ends); the pages behind them return to the stack, the first
    one on top, so that extending again gives them back in their order. page_table keeps its entries. The first held_pages[b] pages of a
    row belong to somebody else (a common prefix) and never return. `status` as in `extend_page_tables` (-2, -3)."""
    sequences, max_pages = _check_tables(page_table, seq_lens, keep_lens, free_pages, free_count, status, page_size)
    if held_pages is not None:
        _check_ints("held_pages", held_pages)
        if held_pages.numel() != sequences:
            raise ValueError("held_pages must be [sequences]")
    args = TABLES_BYTES.pack(page_table.data_ptr(), seq_lens.data_ptr(), keep_lens.data_ptr(), _ptr(held_pages), free_pages.data_ptr(),
                             free_count.data_ptr(), 0, 0, 0, 0, status.data_ptr(), sequences, max_pages, page_size, free_pages.numel(), 0)
    _launch("shrink_page_tables", (page_table, seq_lens, keep_lens, free_pages, free_count, status, held_pages), args)


# ---- rotary positions ------------------------------------------------------------------------------------------------
@dataclass
class RotaryRule:
    """How heads turn: `turns` int64 [rot/2] (turns per position of every pair as a binary fraction, bits of an unsigned number), the pair
    layout, and a factor of cosine and sine."""

    turns: torch.Tensor
    layout: str
    factor: float = 1.0

    @property
    def rot(self) -> int:
        return 2 * int(self.turns.numel())


def turn_fractions(frequencies: np.ndarray) -> np.ndarray:
    """Angles per position (radians, float64) as turns: freq / 2 pi modulo 1, in units of 2^-64, as int64 bits."""
    freq = np.asarray(frequencies, dtype=np.float64)
    if freq.ndim != 1 or freq.size < 1 or not np.all(np.isfinite(freq)):
        raise ValueError("frequencies must be a row of finite numbers")
    turns = freq / (2.0 * np.pi)
    bits = [int((t - math.floor(t)) * 2.0 ** 64) & (2 ** 64 - 1) for t in turns.tolist()]
    return np.array(bits, dtype=np.uint64).view(np.int64)


def rotary_rule(rot: int, base: float, *, layout: str = "interleaved", scaling: tuple[float, float, float, float] | None = None,
                yarn: tuple[float, float, float, float] | None = None, device: torch.device | str = "cuda") -> RotaryRule:
    """The rule of frequencies base^(-2i/rot), as they are or scaled for long contexts as `ragged.rotary_frequencies` (scaling: factor,
    low, high, original) or `ragged.yarn_frequencies` (yarn: factor, original, fast, slow) do it."""
    from .ragged import rotary_frequencies, yarn_frequencies
    if layout not in LAYOUTS:
        raise ValueError(f"unknown pair layout {layout!r}: {sorted(LAYOUTS)}")
    if rot < 2 or rot % 2 or not base > 0:
        raise ValueError("rot must be an even number of at least 2 and base positive")
    if scaling is not None and yarn is not None:
        raise ValueError("one kind of scaling at a time")
    freq, factor = yarn_frequencies(rot, base, *yarn) if yarn is not None else (rotary_frequencies(rot, base, scaling), 1.0)
    return RotaryRule(torch.from_numpy(turn_fractions(freq)).to(device), layout, factor)


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, rule: RotaryRule, positions: torch.Tensor, *,
                  slots: torch.Tensor | None = None, k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                  q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> None:
    """Turns the first rule.rot values of every head of q [R, H, D] and k [R, KVH, D] to positions int32 [R] (rows may be strided views of
    a fused buffer), into q_out (default: in place) and k_out. With slots int32 [R] and the pools [slots, KVH, page, D] the turned k and v
    [R, KVH, D] are also appended: row r to page slots[r] // page, offset slots[r] % page; rows whose slot is outside the pool (padding: -1)
    are left out altogether. Rows with one slot: each value there is of one of them, any. Without slots, k_out defaults to in place; with
    them, to nowhere but the pool.

    Beside `ops.rope_append`: both pair layouts, part of a head, scaled frequencies, float32 to bfloat16, far positions exactly."""
    rows, heads, dim, q_stride = _check_heads("q", q)
    k_rows, kv_heads, k_dim, k_stride = _check_heads("k", k)
    turns, layout = rule.turns, LAYOUTS.get(rule.layout)
    rot = 2 * turns.numel()
    if k_dim != dim or k_rows != rows or rot > dim:
        raise ValueError("q and k must share their rows and their head size, of which the rule turns no more than all")
    if turns.dtype is not torch.int64 or not turns.is_contiguous() or layout is None or rot < 2:
        raise ValueError("the rule must come from rotary_rule")
    _check_ints("positions and slots", positions, slots)
    if positions.numel() != rows or (slots is not None and slots.numel() != rows):
        raise ValueError("positions and slots must have one number per row")
    dtype = q.dtype
    v_stride = q_out_stride = k_out_stride = num_slots = page_size = 0
    if slots is None:
        if k_cache is not None or v_cache is not None:
            raise ValueError("an append to the pools needs slots")
        if k_out is None:
            k_out = k
    else:
        if v is None or k_cache is None or v_cache is None:
            raise ValueError("slots need v and both pools")
        v_rows, v_heads, v_dim, v_stride = _check_heads("v", v)
        if v_rows != rows or v_heads != kv_heads or v_dim != dim:
            raise ValueError("k and v must have one shape")
        shape = k_cache.shape
        if len(shape) != 4 or v_cache.shape != shape or shape[1] != kv_heads or shape[3] != dim or shape[0] < 1 or shape[2] < 1:
            raise ValueError("the pools must be [slots, KVH, page, D]")
        num_slots, _, page_size, _ = shape
        if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
            raise ValueError("the pools must be contiguous")
        if num_slots * page_size > 2 ** 31:
            raise ValueError("slots reach pools of up to 2^31 rows")
        if v.dtype is not dtype or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
            raise TypeError("q, k, v, the outputs and the pools must have one dtype")
    if q_out is None:
        q_out, q_out_stride = q, q_stride
    else:
        out_rows, out_heads, out_dim, q_out_stride = _check_heads("q_out", q_out)
        if out_rows != rows or out_heads != heads or out_dim != dim:
            raise ValueError("outputs must have their inputs' shapes")
    if k_out is not None:
        out_rows, out_heads, out_dim, k_out_stride = _check_heads("k_out", k_out)
        if out_rows != rows or out_heads != kv_heads or out_dim != dim:
            raise ValueError("outputs must have their inputs' shapes")
    if k.dtype is not dtype or q_out.dtype is not dtype or (k_out is not None and k_out.dtype is not dtype):
        raise TypeError("q, k, v, the outputs and the pools must have one dtype")
    code = dtype_code(dtype)
    if rows == 0:
        return
    args = ROTARY_BYTES.pack(
        q.data_ptr(), k.data_ptr(), _ptr(v), q_out.data_ptr(), _ptr(k_out), _ptr(k_cache), _ptr(v_cache), positions.data_ptr(), _ptr(slots),
        turns.data_ptr(), q_stride, k_stride, v_stride, q_out_stride, k_out_stride, rows, heads, kv_heads, dim, rot, layout, num_slots, page_size,
        code, rule.factor)
    _launch("rotary_append", (q, k, q_out, positions, turns, slots, v, k_out, k_cache, v_cache), args)


# ---- attention over common prefixes ----------------------------------------------------------------------------------
@dataclass
class PrefixGroups:
    """Neighbouring rows of a batch that open with the same tokens: rows rows[g] .. rows[g + 1] - 1 share the first lens[g] tokens, which lie
    in the pages table[g] (int32 [G + 1], [G, prefix pages], [G], on the device). Any row's own page list starts with those pages
    where the rows alias them (`kv_cache.B200PagedKVCache.share_prefix`)."""

    rows: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor


def prefix_groups(caches, device: torch.device | str, *, min_tokens: int = 1) -> PrefixGroups | None:
    """The groups of a batch of `kv_cache.B200PagedKVCache`: neighbours that alias the same leading pages, with as many common tokens as all
    of a group's rows share. A row joins the group before it where they have at least `min_tokens` in common and no fewer tokens are then
    shared in all than without it. None: no two neighbours share anything."""
    starts, shared, page_size = [0], [], None
    for cache in caches:
        ids, page_size = cache.page_ids()[: cache.tokens // cache.page_size], cache.page_size       # whole pages
        if shared:
            common = 0
            for a, b in zip(shared[-1], ids):
                if a != b:
                    break
                common += 1
            rows = starts[-1] - starts[-2]
            if common * page_size >= max(1, min_tokens) and (rows == 1 or rows * common >= (rows - 1) * len(shared[-1])):
                shared[-1] = shared[-1][:common]
                starts[-1] += 1
                continue
        shared.append(ids)
        starts.append(starts[-1] + 1)
    if not shared or starts[-1] == len(shared):
        return None
    sizes = [b - a for a, b in zip(starts, starts[1:])]
    lens = [len(ids) * page_size if n > 1 else 0 for ids, n in zip(shared, sizes)]
    width = max(max((n // page_size for n in lens)), 1)
    table = [ids[:width] + [0] * (width - len(ids)) if n else [0] * width for ids, n in zip(shared, lens)]
    return PrefixGroups(*(torch.tensor(v, dtype=torch.int32, device=device) for v in (starts, table, lens)))


def shared_prefix_workspace_bytes(batch: int, heads: int, head_dim: int) -> int:
    """Scratch of `shared_prefix_attention`."""
    return int(_lib.load_group("serving").cacheir_b200_shared_prefix_workspace_bytes(int(batch), int(heads), int(head_dim)))


def shared_prefix_launches(batch: int, heads: int, kv_heads: int, head_dim: int, page_size: int, groups: int, dtype: torch.dtype) -> int:
    """Kernels that one `shared_prefix_attention` launches for these extents (aligned, dense q)."""
    return int(_lib.load_group("serving").cacheir_b200_shared_prefix_launches(int(batch), int(heads), int(kv_heads), int(head_dim), int(page_size),
                                                                             int(groups), dtype_code(dtype)))


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                            groups: PrefixGroups | None, *, out: torch.Tensor | None = None, softmax_scale: float | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """`ops.paged_attention_decode_batch` for rows that share prefixes: the keys and values of a group's common tokens are read once and
    multiplied with the queries of all of its rows. On tensor cores: float16 and bfloat16, heads of 64 and 128, pages of a multiple of 16
    tokens, up to 64 query heads per key/value head. Everything else takes general kernels that are slower than `ops.paged_attention_decode_batch`
    is on the same batch.

    q: [B, H, D] (rows may be strided views); k_cache/v_cache: [slots, KVH, page, D] contiguous, of q's dtype; page_table: int32
    [B, max_pages], every row's own page list from its first token on; seq_lens: int32 [B]. Row b attends to tokens t < seq_lens[b]:
    those below its group's prefix through groups.table, the others through page_table (whose entries below the prefix are not read). A row
    of length 0, or below, gives zeros. B up to 65535, D up to 512. `workspace`: `shared_prefix_workspace_bytes(B, H, D)` bytes of any type;
    calls that may overlap need one each (default: a fresh one)."""
    batch, heads, dim, q_stride = _check_heads("q", q)
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("expected k_cache/v_cache [slots,KVH,page,D]")
    slots, kv_heads, page_size, pool_dim = shape
    dtype = q.dtype
    if pool_dim != dim or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError("q and the KV pool must share head_dim and dtype")
    if kv_heads < 1 or heads % kv_heads or slots < 1 or page_size < 1:
        raise ValueError("the query heads must be a multiple of the pool's heads")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the KV pool must be contiguous")
    _check_ints("page_table and seq_lens", page_table, seq_lens)
    shape = page_table.shape
    if len(shape) != 2 or shape[0] != batch or shape[1] < 1 or seq_lens.numel() != batch:
        raise ValueError("page_table must be [B, max_pages] and seq_lens [B]")
    max_pages, count, prefix_pages = shape[1], 0, 0
    group_rows = prefix_table = prefix_lens = None
    if groups is not None:
        group_rows, prefix_table, prefix_lens = groups.rows, groups.table, groups.lens
        _check_ints("the prefix groups", group_rows, prefix_table, prefix_lens)
        count, shape = prefix_lens.numel(), prefix_table.shape
        if group_rows.numel() != count + 1 or len(shape) != 2 or shape[0] != count or not 1 <= count <= max(1, batch) or shape[1] < 1:
            raise ValueError("prefix groups must have rows [G + 1], table [G, prefix pages] and lens [G], G no more than the batch's rows")
        prefix_pages = shape[1]
    if out is None:
        out = torch.empty((batch, heads, dim), device=q.device, dtype=dtype)
    out_rows, out_heads, out_dim, out_stride = _check_heads("out", out)
    if out_rows != batch or out_heads != heads or out_dim != dim or out.dtype is not dtype:
        raise ValueError("out must match q's shape and dtype")
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("softmax_scale must be positive")
    code = dtype_code(dtype)
    if batch == 0:
        return out
    if workspace is None:
        workspace = torch.empty(shared_prefix_workspace_bytes(batch, heads, dim), device=q.device, dtype=torch.uint8)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    args = PREFIX_BYTES.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), _ptr(group_rows),
                      _ptr(prefix_table), _ptr(prefix_lens), workspace.data_ptr(), workspace.nbytes, q_stride, out_stride, batch, heads, kv_heads, dim,
                      page_size, slots, max_pages, count, prefix_pages, code, scale)
    _launch("shared_prefix_attention", (q, k_cache, v_cache, page_table, seq_lens, out, workspace, group_rows, prefix_table, prefix_lens), args)
    return out


# ---- log probabilities -----------------------------------------------------------------------------------------------
@dataclass
class TokenLogprobs:
    """float32 [R] log probabilities of the tokens and entropies (nats); int64 / float32 [R, top] likeliest tokens."""

    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


def check_scoring(vocab: int, top: int, temperature: float) -> None:
    """What `token_logprobs` takes."""
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {MAX_TOP} and no more than the vocabulary")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError("temperature must be 1e-6 to 1e6")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None, *, top: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of tokens int64 [R] under softmax(logits / temperature), the rows' entropies, and the `top` likeliest tokens with
    theirs (equal logits by rising index, like `ops.argmax_rows`). logits: [R, V] with dense rows (the row stride may be wider).

    -inf masks a token out; a row of nothing else has log probabilities -inf and entropy 0. NaN or +inf in a row give NaN. A token below 0
    means none (log probability 0), one of V or more gives NaN."""
    shape = logits.shape
    if len(shape) != 2:
        raise ValueError("logits must be [R, V]")
    (rows, vocab), (row_stride, stride) = shape, logits.stride()
    if vocab < 1 or (stride != 1 and vocab > 1) or (rows > 1 and row_stride < vocab):
        raise ValueError("logits must be [R, V] with dense rows that do not overlap")
    check_scoring(vocab, top, temperature)
    if tokens is not None and (tokens.dtype is not torch.int64 or tokens.numel() != rows or not tokens.is_contiguous()):
        raise ValueError("tokens must be contiguous int64 [R]")
    code, device = dtype_code(logits.dtype), logits.device
    entropy = torch.empty(rows, dtype=torch.float32, device=device)
    result = TokenLogprobs(None if tokens is None else torch.empty_like(entropy), entropy,
                           entropy.new_empty((rows, top), dtype=torch.int64) if top else None, entropy.new_empty((rows, top)) if top else None)
    args = LOGPROBS_BYTES.pack(logits.data_ptr(), _ptr(tokens), _ptr(result.logprobs), entropy.data_ptr(), _ptr(result.top_ids),
                               _ptr(result.top_logprobs), row_stride if rows > 1 else vocab, temperature, rows, vocab, top, code)
    _launch("token_logprobs", (logits, tokens), args)
    return result
