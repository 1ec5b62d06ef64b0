"""Torch-tensor wrappers over the operators of a step that verifies drafted tokens (include/cacheir_b200_drafts.h).

Every sequence of such a step brings rows, a token each: row 0 is its last certain token, every other row follows an earlier one of the same sequence
(its parent), so that the rows are a tree, or a chain. They take the places behind the sequence's tokens, and their slots come from
`serving_ops.extend_page_tables`. The operators in the order of the step: positions and masks of the rows (`map_drafts`), norms of query and key
heads with rotary positions and the append (`norm_rotary_append`; without norms `serving_ops.rotary_append`), attention under the tree's mask
(`tree_attention`), penalties, biases and grammar masks on the logits (`adjust_logits`), the accepted path (`accept_drafts`) and its keys and values
moved together (`keep_accepted`), behind which `serving_ops.shrink_page_tables` takes the other rows back.

Same rules as `ops`: validate, pass device pointers on the current stream, raise on a non-zero status. All tensors of a call are on one
CUDA device, which need not be the current one; the call runs on that device's current stream.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import AcceptArgs, DraftMapArgs, KeepArgs, LogitsArgs, NormRotaryArgs, TreeArgs
from .ops import dtype_code
from .serving_ops import ROTARY_BYTES, RotaryRule, TokenMap, _check_heads, _check_ints, _launch, _ptr, _rotary_call

MAX_WORDS = 32
MAX_SEQUENCES = 65535
# the argument structs as bytes (see `serving_ops`)
NORM_BYTES = struct.Struct("@2Qi2f4x")
TREE_BYTES = struct.Struct("@10Q2q10if4x")
LOGITS_BYTES = struct.Struct("@15Q2q8i")
MAP_BYTES = struct.Struct("@6Q3i4x")
ACCEPT_BYTES = struct.Struct("@9Q3i4x")
KEEP_BYTES = struct.Struct("@5Q9i4x")
assert [s.size for s in (TREE_BYTES, LOGITS_BYTES, MAP_BYTES, ACCEPT_BYTES, KEEP_BYTES)] == [
    ctypes.sizeof(c) for c in (TreeArgs, LogitsArgs, DraftMapArgs, AcceptArgs, KeepArgs)]
assert ROTARY_BYTES.size + NORM_BYTES.size == ctypes.sizeof(NormRotaryArgs)

_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


# ---- rows of drafted tokens ------------------------------------------------------------------------------------------
@dataclass
class DraftTree:
    """What `map_drafts` fills (int32, on the device): row r stands at `positions[r]`, and sees those rows j of its sequence whose bit j % 32 of
    visible[r, j // 32] is set. `status` becomes the number of rows of a sequence that has more than visible has bits, until it is set to 0."""

    positions: torch.Tensor
    visible: torch.Tensor
    status: torch.Tensor


def draft_tree(rows: int, words: int, device: torch.device | str) -> DraftTree:
    """Room for `rows` rows, up to 32 `words` of them per sequence."""
    if rows < 1 or not 1 <= words <= MAX_WORDS:
        raise ValueError(f"a draft tree has at least one row and 1 to {MAX_WORDS} words")
    return DraftTree(*(torch.zeros(shape, dtype=_I32, device=device) for shape in (rows, (rows, words), 1)))


def _check_rows(rows: int, tokens_cu_rows: torch.Tensor, seq_lens: torch.Tensor | None) -> int:
    sequences = tokens_cu_rows.numel() - 1
    if not 1 <= sequences <= MAX_SEQUENCES:
        raise ValueError(f"a call takes 1 to {MAX_SEQUENCES} sequences (cu_rows [sequences + 1])")
    if rows < 1:
        raise ValueError("a call takes at least one row")
    if seq_lens is not None and seq_lens.numel() != sequences:
        raise ValueError("seq_lens must be [sequences]")
    return sequences


def _check_visible(visible: torch.Tensor, rows: int) -> int:
    shape = visible.shape
    if len(shape) != 2 or shape[0] != rows or not 1 <= shape[1] <= MAX_WORDS:
        raise ValueError(f"visible must be [rows, words] with 1 to {MAX_WORDS} words")
    return shape[1]


def map_drafts(parents: torch.Tensor, seq_lens: torch.Tensor, tokens: TokenMap, tree: DraftTree) -> DraftTree:
    """Positions and masks of rows from their parents: int32 [R], a parent's number inside its sequence (row 0 of a sequence: 0), -1 for none (what is
    not an earlier row counts as none). Row i of n stands at seq_lens[b] - n + (rows that it follows), and sees the rows that it follows and itself.
    seq_lens int32 [S] counts the rows already (as after `extend_page_tables`); `tokens` says which rows are whose. Rows behind the last sequence get
    position 0 and see nothing. Fills and returns `tree`."""
    positions, visible, status, cu_rows = tree.positions, tree.visible, tree.status, tokens.cu_rows
    _check_ints("parents, lengths, row starts and the tree", parents, seq_lens, cu_rows, positions, visible, status)
    rows = parents.numel()
    sequences = _check_rows(rows, cu_rows, seq_lens)
    words = _check_visible(visible, rows)
    if positions.numel() != rows or status.numel() != 1:
        raise ValueError("the draft tree was made for other sizes")
    args = MAP_BYTES.pack(parents.data_ptr(), cu_rows.data_ptr(), seq_lens.data_ptr(), positions.data_ptr(), visible.data_ptr(), status.data_ptr(), rows,
                          sequences, words)
    _launch("map_drafts", (parents, cu_rows, seq_lens, positions, visible, status), args, "drafts")
    return tree


@dataclass
class AcceptedDrafts:
    """What `accept_drafts` fills: of sequence b the rows[b, : counts[b]] (row numbers; -1 behind them), the token that comes next (`next_ids`, int64),
    and keep_lens[b], the tokens that it has then (for `serving_ops.shrink_page_tables`). int32 [S], [S, depth], int64 [S], int32 [S]."""

    counts: torch.Tensor
    rows: torch.Tensor
    next_ids: torch.Tensor
    keep_lens: torch.Tensor


def accepted_drafts(sequences: int, depth: int, device: torch.device | str) -> AcceptedDrafts:
    """Room for paths of up to `depth` rows."""
    if not 1 <= sequences <= MAX_SEQUENCES or depth < 1:
        raise ValueError(f"accepted drafts are of 1 to {MAX_SEQUENCES} sequences and have a depth of at least 1")
    made = lambda dtype, *shape: torch.zeros(shape, dtype=dtype, device=device)
    return AcceptedDrafts(made(_I32, sequences), made(_I32, sequences, depth), made(_I64, sequences), made(_I32, sequences))


def _check_accepted(accepted: AcceptedDrafts, sequences: int) -> int:
    counts, path = accepted.counts, accepted.rows
    _check_ints("accepted drafts", counts, path, accepted.keep_lens)
    if counts.numel() != sequences or len(path.shape) != 2 or path.shape[0] != sequences or path.shape[1] < 1 or accepted.keep_lens.numel() != sequences:
        raise ValueError("the accepted drafts were made for other sizes")
    if accepted.next_ids.dtype is not _I64 or accepted.next_ids.numel() != sequences or not accepted.next_ids.is_contiguous():
        raise ValueError("next_ids must be contiguous int64 [sequences]")
    return path.shape[1]


def _check_ids(name: str, ids: torch.Tensor, rows: int) -> None:
    if ids.dtype is not _I64 or ids.numel() != rows or not ids.is_contiguous():
        raise ValueError(f"{name} must be contiguous int64 [R]")


def accept_drafts(chosen: torch.Tensor, draft_ids: torch.Tensor, parents: torch.Tensor, seq_lens: torch.Tensor, tokens: TokenMap,
                  accepted: AcceptedDrafts) -> AcceptedDrafts:
    """The path of every sequence that was picked: row 0, then, while there is one, the first row whose parent is the row arrived at and whose token
    (draft_ids int64 [R]) is the one picked there (chosen int64 [R]: `ops.argmax_rows` of the logits, or a sample of them). Up to accepted.rows.shape[1]
    rows; next_ids is what was picked at the last. A sequence without rows: count 0, next -1, and it keeps its tokens. Fills and returns `accepted`."""
    cu_rows, rows = tokens.cu_rows, parents.numel()
    _check_ints("parents, lengths and row starts", parents, seq_lens, cu_rows)
    sequences = _check_rows(rows, cu_rows, seq_lens)
    _check_ids("chosen", chosen, rows)
    _check_ids("draft_ids", draft_ids, rows)
    depth = _check_accepted(accepted, sequences)
    args = ACCEPT_BYTES.pack(chosen.data_ptr(), draft_ids.data_ptr(), parents.data_ptr(), cu_rows.data_ptr(), seq_lens.data_ptr(), accepted.counts.data_ptr(),
                             accepted.rows.data_ptr(), accepted.next_ids.data_ptr(), accepted.keep_lens.data_ptr(), rows, sequences, depth)
    _launch("accept_drafts", (chosen, draft_ids, parents, cu_rows, seq_lens, accepted.counts, accepted.rows, accepted.next_ids, accepted.keep_lens), args,
            "drafts")
    return accepted


class PagePools:
    """The pools [slots, KVH, page, D] of a model's layers, keys and values, of one shape and type, whose addresses a call passes on."""

    def __init__(self, pools):
        self.tensors = tuple(pools)
        if not self.tensors:
            raise ValueError("there are no pools")
        first = self.tensors[0]
        if len(first.shape) != 4 or min(first.shape) < 1:
            raise ValueError("the pools must be [slots, KVH, page, D]")
        for t in self.tensors:
            if t.shape != first.shape or t.dtype is not first.dtype or t.device != first.device or not t.is_contiguous():
                raise ValueError("the pools must be contiguous and of one shape, type and device")
        self.code = dtype_code(first.dtype)
        self.addresses = (ctypes.c_void_p * len(self.tensors))(*(t.data_ptr() for t in self.tensors))
        if len(set(self.addresses)) != len(self.tensors):
            raise ValueError("a pool is there twice")


def page_pools(pools) -> PagePools:
    """What `keep_accepted` takes, made once: the pools of all layers, in any order."""
    return PagePools(pools)


def keep_accepted(accepted: AcceptedDrafts, tokens: TokenMap, pools: PagePools) -> None:
    """Moves the keys and values of every sequence's accepted rows to the slots of its first rows, in all pools at once, so that its tokens lie
    together: what stood in the slot of the path's i-th row goes to that of row i. Slots outside the pools are left out."""
    cu_rows, slots = tokens.cu_rows, tokens.slots
    _check_ints("slots and row starts", cu_rows, slots)
    rows = slots.numel()
    sequences = _check_rows(rows, cu_rows, None)
    depth = _check_accepted(accepted, sequences)
    num_slots, kv_heads, page_size, dim = pools.tensors[0].shape
    args = KEEP_BYTES.pack(ctypes.addressof(pools.addresses), slots.data_ptr(), cu_rows.data_ptr(), accepted.counts.data_ptr(), accepted.rows.data_ptr(),
                           len(pools.tensors), rows, sequences, depth, num_slots, kv_heads, page_size, dim, pools.code)
    _launch("keep_accepted", (slots, cu_rows, accepted.counts, accepted.rows, pools.tensors[0]), args, "drafts")


# ---- norms, rotary positions, append -----------------------------------------------------------------------------------
def norm_rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, rule: RotaryRule, positions: torch.Tensor,
                       q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, *, eps: float = 1e-6, offset: float = 0.0,
                       slots: torch.Tensor | None = None, k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                       q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> None:
    """`serving_ops.rotary_append` of heads that are normed first: x / sqrt(mean(x^2) + eps) * (weight + offset) for every head of q and k, in the same
    pass and with one rounding. q_weight, k_weight [D] in the heads' type or float32 (None: no weight), offset 1 for weights that are kept less 1.
    v is appended as it is. All other arguments as there."""
    args, tensors = _rotary_call(q, k, v, rule, positions, slots, k_cache, v_cache, q_out, k_out)
    dim, weight = q.shape[2], k_weight if q_weight is None else q_weight
    for w in (q_weight, k_weight):
        if w is not None and (w.numel() != dim or not w.is_contiguous()):
            raise ValueError("weights must be contiguous [D]")
    weight_dtype = _F32 if weight is None else weight.dtype
    if (weight_dtype is not _F32 and weight_dtype is not q.dtype) or (k_weight is not None and k_weight.dtype is not weight_dtype):
        raise TypeError("both weights must be of the heads' type, or float32")
    if not (0.0 <= eps < math.inf and -math.inf < offset < math.inf):
        raise ValueError("eps must be finite and not negative, offset finite")
    if args:
        _launch("norm_rotary_append", (*tensors, q_weight, k_weight), args + NORM_BYTES.pack(_ptr(q_weight), _ptr(k_weight), dtype_code(weight_dtype), eps, offset),
                "drafts")


# ---- attention -----------------------------------------------------------------------------------------------------------
def tree_attention_workspace_bytes(rows: int, heads: int, head_dim: int) -> int:
    """Scratch of `tree_attention`, enough for any type and pools: 39 to 68 MB with heads of 128, however many rows there are. 0: none."""
    return int(_lib.load_group("drafts").cacheir_b200_tree_attention_workspace_bytes(int(rows), int(heads), int(head_dim)))


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, cu_rows: torch.Tensor,
                   visible: torch.Tensor | None = None, *, out: torch.Tensor | None = None, softmax_scale: float | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """`ops.paged_attention_decode_batch` for sequences that bring several rows each, the last tokens of their seq_lens: every row attends to all tokens in
    front of its sequence's rows, and to those of the rows that `visible` names.

    q: [R, H, D] (rows may be strided views); k_cache/v_cache: [slots, KVH, page, D] contiguous, of q's dtype; page_table: int32 [S, max_pages];
    seq_lens: int32 [S], the rows among them; cu_rows: int32 [S + 1], sequence b has the rows cu_rows[b] .. cu_rows[b + 1] - 1. visible: int32
    [R, words], bit j % 32 of word j // 32 for row j of the sequence (`map_drafts` makes them; any other mask will do); None: a chain, rows see those
    before them and themselves. Rows that see nothing give zeros; rows behind the last sequence are left as they were in `out`. What a row does not
    see may hold anything, NaN too. On the tensor cores (16 bits, D 64 or 128, pages of a multiple of 16) probabilities are rounded to q's type before they meet
    the values, elsewhere not; the rest is in 32 bits. D up to 512, S up to 65535, R up to 2^24. `workspace`: `tree_attention_workspace_bytes(R, H, D)` bytes of any type; calls that
    may overlap need one each (default: a fresh one)."""
    rows, heads, dim, q_stride = _check_heads("q", q)
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
    _check_ints("page_table, seq_lens, cu_rows and visible", page_table, seq_lens, cu_rows, visible)
    sequences, shape = seq_lens.numel(), page_table.shape
    if len(shape) != 2 or shape[0] != sequences or shape[1] < 1 or cu_rows.numel() != sequences + 1:
        raise ValueError("page_table must be [S, max_pages], seq_lens [S] and cu_rows [S + 1]")
    words = 0 if visible is None else _check_visible(visible, rows)
    if out is None:
        out = torch.zeros((rows, heads, dim), device=q.device, dtype=dtype)
    out_rows, out_heads, out_dim, out_stride = _check_heads("out", out)
    if out_rows != rows or out_heads != heads or out_dim != dim or out.dtype is not dtype:
        raise ValueError("out must match q's shape and dtype")
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("softmax_scale must be positive")
    code = dtype_code(dtype)
    if rows == 0 or sequences == 0:
        return out
    if workspace is None:
        workspace = torch.empty(tree_attention_workspace_bytes(rows, heads, dim), device=q.device, dtype=torch.uint8)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    args = TREE_BYTES.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), cu_rows.data_ptr(),
                           _ptr(visible), workspace.data_ptr(), workspace.nbytes, q_stride, out_stride, rows, sequences, heads, kv_heads, dim, page_size, slots,
                           shape[1], words, code, scale)
    _launch("tree_attention", (q, k_cache, v_cache, page_table, seq_lens, out, workspace, cu_rows, visible), args, "drafts")
    return out


# ---- logits ----------------------------------------------------------------------------------------------------------------
@dataclass
class TokenHistory:
    """What every sequence has said: int32 tokens [S, width], of which lens[b] count; the first prompt_lens[b] of them are the prompt (None: none). Beside
    `DraftedTokens` a token is in one of the two only: see there."""

    tokens: torch.Tensor
    lens: torch.Tensor
    prompt_lens: torch.Tensor | None = None


@dataclass
class DraftedTokens:
    """The rows' own tokens (int64 [R]) and which of them each sees (`visible` and `cu_rows` as in `tree_attention`).

    Row 0 of a sequence, its last certain token, is among what its rows see, and would count twice if the history held it too. So either history.lens ends in
    front of it, and ids has it: it counts as generated; or the history holds it and ids[row 0] is -1. The latter is what the first step behind a prompt
    needs, whose row 0 is a token of the prompt, and will do for every step. `accept_drafts` does not look at ids of rows 0."""

    ids: torch.Tensor
    visible: torch.Tensor
    cu_rows: torch.Tensor


def adjust_logits(logits: torch.Tensor, *, row_seq: torch.Tensor | None = None, history: TokenHistory | None = None, drafts: DraftedTokens | None = None,
                  repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits [R, V] as the next token is to be picked from, before `ops.argmax_rows` or `token_logprobs`. For token t of a row of sequence b

        c = times that t was generated (history behind the prompt) or is drafted in front of the row, itself included (row 0: see `DraftedTokens`)
        where c > 0 or t is in the prompt: x / repetition[b] where x > 0, else x * repetition[b]
        x - frequency[b] * c - (presence[b] where c > 0) + bias of t, and -inf where t is not allowed

    row_seq: int32 [R] (None: row r is of sequence r); rows of a sequence outside 0 .. S - 1 are left as they are in `out`. repetition (above 0),
    frequency, presence: float32 [S]. bias_ids int32, bias_values float32 [S, K]: of several entries with one token the last counts, ids outside
    the vocabulary (-1) are none. allowed: int32 [R, ceil(V / 32)], bit t % 32 of word t // 32. out: default in place (then only what changes is
    written), else rows that do not lie over those of the logits; of their type or float32. Worked out in 32 bits, rounded once. Logits and out have dense rows (the row stride may be wider)."""
    shape = logits.shape
    if len(shape) != 2:
        raise ValueError("logits must be [R, V]")
    (rows, vocab), (row_stride, stride), dtype = shape, logits.stride(), logits.dtype
    if vocab < 1 or (stride != 1 and vocab > 1) or (rows > 1 and row_stride < vocab):
        raise ValueError("logits must be [R, V] with dense rows that do not overlap")
    if out is None:
        out, out_stride = logits, row_stride
    else:
        if out.shape != shape:
            raise ValueError("out must be [R, V] with dense rows that do not overlap")
        out_stride, stride = out.stride()
        if (stride != 1 and vocab > 1) or (rows > 1 and out_stride < vocab):
            raise ValueError("out must be [R, V] with dense rows that do not overlap")
        if out.dtype is not dtype and (out.dtype is not _F32 or out.data_ptr() == logits.data_ptr()):
            raise TypeError("out must have the logits' type, or be another tensor of float32")
        if rows > 1 and out_stride != row_stride and out.data_ptr() == logits.data_ptr():
            raise ValueError("logits that are changed in place keep their row stride")
    counts = []                                                       # what the arguments say about the number of sequences
    said = said_lens = prompt_lens = draft_ids = visible = cu_rows = None
    width = words = biases = 0
    if history is not None:
        said, said_lens, prompt_lens = history.tokens, history.lens, history.prompt_lens
        _check_ints("the history", said, said_lens, prompt_lens)
        if len(said.shape) != 2:
            raise ValueError("a history must have tokens [S, width], lens [S] and prompt_lens [S]")
        count, width = said.shape
        if width < 1 or said_lens.numel() != count or (prompt_lens is not None and prompt_lens.numel() != count):
            raise ValueError("a history must have tokens [S, width], lens [S] and prompt_lens [S]")
        counts.append(count)
    if drafts is not None:
        draft_ids, visible, cu_rows = drafts.ids, drafts.visible, drafts.cu_rows
        _check_ints("the drafts' masks and row starts", visible, cu_rows)
        _check_ids("drafted tokens", draft_ids, rows)
        words = _check_visible(visible, rows)
        counts.append(cu_rows.numel() - 1)
    for t in (repetition, frequency, presence):
        if t is not None:
            if t.dtype is not _F32 or t.dim() != 1 or not t.is_contiguous():
                raise TypeError("repetition, frequency and presence must be contiguous float32 [S]")
            counts.append(t.numel())
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None or bias_ids.dim() != 2 or bias_ids.shape != bias_values.shape:
            raise ValueError("bias_ids and bias_values must both be [S, K]")
        _check_ints("bias_ids", bias_ids)
        if bias_values.dtype is not _F32 or not bias_values.is_contiguous():
            raise TypeError("bias_values must be contiguous float32")
        count, biases = bias_ids.shape
        counts.append(count)
    _check_ints("allowed and row_seq", allowed, row_seq)
    if allowed is not None and allowed.shape != (rows, (vocab + 31) // 32):
        raise ValueError("allowed must be [R, ceil(V / 32)]")
    if row_seq is not None and row_seq.numel() != rows:
        raise ValueError("row_seq must be [R]")
    # (where nothing is a sequence's own, every row that has one counts)
    sequences = counts[0] if counts else rows if row_seq is None else 2 ** 31 - 1
    if counts and (sequences < 1 or counts.count(sequences) != len(counts)):
        raise ValueError("all arguments must be of the same number of sequences, one at least")
    if rows == 0:
        return out
    if row_seq is None and sequences != rows:
        raise ValueError("without row_seq there must be as many sequences as rows")
    args = LOGITS_BYTES.pack(logits.data_ptr(), out.data_ptr(), _ptr(row_seq), _ptr(said), _ptr(said_lens), _ptr(prompt_lens), _ptr(draft_ids), _ptr(cu_rows),
                             _ptr(visible), _ptr(repetition), _ptr(frequency), _ptr(presence), _ptr(bias_ids), _ptr(bias_values), _ptr(allowed),
                             row_stride if rows > 1 else vocab, out_stride if rows > 1 else vocab, rows, sequences, vocab, width, words, biases, dtype_code(dtype),
                             dtype_code(out.dtype))
    _launch("adjust_logits", (logits, out, row_seq, said, said_lens, prompt_lens, draft_ids, cu_rows, visible, repetition, frequency, presence, bias_ids,
                              bias_values, allowed), args, "drafts")
    return out
