"""Operators of steps that verify drafted tokens, on the CPU: the library's ABI and refusals."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    from cacheir_b200 import _lib, build

    build.build(groups=("drafts",))
    return _lib.load_group("drafts")


def test_library_exports_every_declared_symbol(lib):
    from cacheir_b200 import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "cacheir_b200_drafts.h").read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(cacheir_b200_[a-z0-9_]+)\s*\(", text)))
    assert all(hasattr(lib, name) for name in declared)
    assert sorted(_lib.GROUP_SIGNATURES["drafts"]) == declared, "ctypes table and header disagree"


def test_argument_structs_have_the_compiler_s_layout(tmp_path):
    from cacheir_b200 import _lib

    lines, want = [], []
    for name, struct in (("cacheir_b200_norm_rotary_args", _lib.NormRotaryArgs), ("cacheir_b200_tree_args", _lib.TreeArgs),
                         ("cacheir_b200_logits_args", _lib.LogitsArgs), ("cacheir_b200_draft_map_args", _lib.DraftMapArgs),
                         ("cacheir_b200_accept_args", _lib.AcceptArgs), ("cacheir_b200_keep_args", _lib.KeepArgs)):
        want.append(ctypes.sizeof(struct))
        lines.append(f'std::printf("%zu ", sizeof({name}));')
        for field, _ in struct._fields_:
            want.append(getattr(struct, field).offset)
            lines.append(f'std::printf("%zu ", offsetof({name}, {field}));')
    (tmp_path / "layout.cpp").write_text('#include <cstddef>\n#include <cstdio>\n#include "cacheir_b200_drafts.h"\nint main() {\n' + "\n".join(lines) + "\n}\n")
    subprocess.run(["g++", "-I", str(ROOT / "include"), "layout.cpp", "-o", "layout"], cwd=tmp_path, check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want


def test_c_entry_points_refuse_before_they_launch(lib):
    """Codes of calls that never reach the device: missing pointers, extents, limits, scratch."""
    from cacheir_b200._lib import AcceptArgs, DraftMapArgs, KeepArgs, LogitsArgs, NormRotaryArgs, RotaryArgs, TreeArgs

    some = 4096                                               # an address that no refused call looks at
    good_rotary = dict(q=some, k=some, v=some, q_out=some, k_cache=some, v_cache=some, positions=some, slots=some, turns=some, rows=2, heads=4, kv_heads=2, dim=64,
                       rot=64, num_slots=3, page_size=16, dtype=1, factor=1.0)
    norm = lambda weight_dtype=1, eps=1e-6, **new: lib.cacheir_b200_norm_rotary_append(ctypes.byref(NormRotaryArgs(
        rotary=RotaryArgs(**{**good_rotary, **new}), q_weight=some, k_weight=some, weight_dtype=weight_dtype, eps=eps, offset=0.0)), None)
    assert norm(rows=0) == 0
    bad = [dict(q=None), dict(v=None), dict(positions=None), dict(turns=None), dict(k_cache=None), dict(heads=0), dict(rot=3), dict(rot=66), dict(layout=2),
           dict(dtype=7), dict(slots=None), dict(eps=-1.0), dict(eps=float("nan")), dict(weight_dtype=2)]
    assert [norm(**b) for b in bad] == [-1] * len(bad)
    assert norm(dim=1026) == -5

    need = lib.cacheir_b200_tree_attention_workspace_bytes(6, 4, 64)
    assert need > 0 and lib.cacheir_b200_tree_attention_workspace_bytes(0, 4, 64) == 0
    good = dict(q=some, k_cache=some, v_cache=some, out=some, page_table=some, seq_lens=some, cu_rows=some, visible=some, workspace=some, workspace_bytes=need,
                rows=6, sequences=2, heads=4, kv_heads=2, dim=64, page_size=16, num_slots=3, max_pages=4, words=1, dtype=1)
    tree = lambda **new: lib.cacheir_b200_tree_attention(ctypes.byref(TreeArgs(**{**good, **new})), None)
    assert [tree(rows=0), tree(sequences=0)] == [0, 0]
    bad = [dict(q=None), dict(out=None), dict(page_table=None), dict(cu_rows=None), dict(seq_lens=None), dict(kv_heads=3), dict(dim=0), dict(words=0), dict(dtype=3),
           dict(num_slots=0), dict(max_pages=0)]
    assert [tree(**b) for b in bad] == [-1] * len(bad)
    assert [tree(workspace=None), tree(workspace_bytes=need - 1), tree(workspace=some + 4), tree(dim=513), tree(sequences=65536), tree(words=33), tree(rows=(1 << 24) + 1),
            tree(max_pages=1 << 27)] == [-3, -3, -2, -4, -5, -5, -5, -5]

    good_logits = dict(logits=some, out=some, row_seq=some, history=some, history_lens=some, draft_ids=some, cu_rows=some, visible=some, bias_ids=some, bias_values=some,
                       rows=2, sequences=2, vocab=9, history_width=4, words=1, biases=2)
    logits = lambda **new: lib.cacheir_b200_adjust_logits(ctypes.byref(LogitsArgs(**{**good_logits, **new})), None)
    assert [logits(rows=0), logits(vocab=0)] == [0, 0]
    bad = [dict(logits=None), dict(out=None), dict(history_lens=None), dict(history_width=0), dict(cu_rows=None), dict(visible=None), dict(words=0), dict(bias_values=None),
           dict(biases=-1), dict(row_stride=8), dict(out_stride=8), dict(dtype=5), dict(dtype=0, out_dtype=1), dict(dtype=1), dict(sequences=0)]
    assert [logits(**b) for b in bad] == [-1] * len(bad)
    assert [logits(vocab=(1 << 28) + 1), logits(words=33)] == [-5, -5]

    names = ("parents", "cu_rows", "seq_lens", "positions", "visible", "status")
    maps = lambda rows=3, sequences=2, words=1, null=None: lib.cacheir_b200_map_drafts(ctypes.byref(DraftMapArgs(
        **{name: None if i == null else some for i, name in enumerate(names)}, rows=rows, sequences=sequences, words=words)), None)
    assert [maps(rows=0), maps(sequences=0)] == [0, 0]
    assert [maps(null=i) for i in range(6)] + [maps(words=0)] == [-1] * 7
    assert [maps(words=33), maps(sequences=65536)] == [-5, -5]
    names_accept = ("chosen", "draft_ids", "parents", "cu_rows", "seq_lens", "counts", "path", "next_ids", "keep_lens")
    accept = lambda rows=3, sequences=2, depth=4, null=None: lib.cacheir_b200_accept_drafts(ctypes.byref(AcceptArgs(
        **{name: None if i == null else some for i, name in enumerate(names_accept)}, rows=rows, sequences=sequences, depth=depth)), None)
    assert [accept(rows=0), accept(null=3), accept(null=8), accept(depth=0), accept(sequences=65536)] == [0, -1, -1, -1, -5]
    array = (ctypes.c_void_p * 2)(some, some)
    good_keep = dict(pools=ctypes.addressof(array), slots=some, cu_rows=some, counts=some, path=some, pool_count=2, rows=3, sequences=2, depth=4, num_slots=3, kv_heads=2,
                     page_size=16, dim=64, dtype=1)
    keep = lambda **new: lib.cacheir_b200_keep_accepted(ctypes.byref(KeepArgs(**{**good_keep, **new})), None)
    hole = (ctypes.c_void_p * 2)(some, None)
    assert [keep(pool_count=0), keep(rows=0)] == [0, 0]
    bad = [dict(pools=None), dict(pools=ctypes.addressof(hole)), dict(slots=None), dict(counts=None), dict(depth=0), dict(num_slots=0), dict(dim=0), dict(dtype=4)]
    assert [keep(**b) for b in bad] == [-1] * len(bad)
    assert [keep(sequences=65536), keep(dim=1 << 24)] == [-5, -5]
    for name in ("norm_rotary_append", "tree_attention", "adjust_logits", "map_drafts", "accept_drafts", "keep_accepted"):
        assert getattr(lib, "cacheir_b200_" + name)(None, None) == -1


def test_scratch_of_attention_does_not_grow_with_the_batch(lib):
    size = lib.cacheir_b200_tree_attention_workspace_bytes
    for dim in (1, 33, 64, 96, 128, 256, 512):
        for heads in (1, 8, 64):
            sizes = [size(rows, heads, dim) for rows in (1, 2, 63, 64, 500, 4096, 16384, 1 << 20, 1 << 24)]
            # outputs of 64 MB in pieces and two numbers beside each, or the tensor cores' two pieces a block
            assert max(sizes) <= (64 << 20) * (dim + 2) // dim
            assert sizes[-1] == (size(1 << 23, heads, dim) if dim in (64, 128) else 0)


def test_logits_that_lie_over_one_another_are_refused(lib):
    """Values that do not change are not written where out is the logits: another row stride, or rows that lie partly over one another, would leave the wrong ones. What
    lies between the rows, or apart, goes on to the next check (here: words)."""
    from cacheir_b200 import draft_ops
    from cacheir_b200._lib import LogitsArgs

    at = 1 << 20
    call = lambda out, row_stride=20, out_stride=20, rows=3, dtype=1, out_dtype=1: lib.cacheir_b200_adjust_logits(ctypes.byref(LogitsArgs(
        logits=at, out=out, draft_ids=at, cu_rows=at, visible=at, rows=rows, sequences=3, vocab=9, words=33, row_stride=row_stride, out_stride=out_stride, dtype=dtype,
        out_dtype=out_dtype)), None)
    over = [call(at, out_stride=24), call(at, row_stride=9), call(at + 16), call(at - 16), call(at + 40), call(at + 56), call(at - 40 * 2 - 2), call(at + 18, out_dtype=0),
            call(at - 34, rows=1, out_dtype=0), call(at + 18, out_stride=24), call(at + 200, row_stride=100, out_stride=9)]
    assert over == [-1] * len(over)
    # (out_stride 22: bytes 18 to 36, 62 to 80 and 106 to 124, of logits 0 to 18, 40 to 58 and 80 to 98)
    apart = [call(at), call(at, rows=1, out_stride=24), call(at + 18, rows=1, row_stride=0), call(at + 18, out_stride=22), call(at + 18), call(at + 22), call(at - 22), call(at + 2 * 40 + 18), call(at - 2 * 40 - 18), call(at - 36, rows=1, out_dtype=0),
             call(at + 20, row_stride=40, out_stride=20, out_dtype=0), call(at + 1000, out_stride=9)]
    assert apart == [-5] * len(apart)
    room = torch.zeros(200)
    with pytest.raises(ValueError, match="row stride"):
        draft_ops.adjust_logits(room[:60].view(3, 20)[:, :9], out=room[:90].view(3, 30)[:, :9], allowed=_i32(3, 1))


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_wrappers_refuse_wrong_arguments_and_cpu_tensors(lib):
    from cacheir_b200 import draft_ops as D, serving_ops as S
    from cacheir_b200._lib import CacheIRB200Error

    def refused(call, kinds, **wrong):
        with pytest.raises(kinds):
            call(**wrong)

    tokens, tree = S.token_map(5, 3, "cpu"), D.draft_tree(5, 2, "cpu")
    maps = lambda parents=_i32(5), lens=_i32(3), tokens=tokens, tree=tree: D.map_drafts(parents, lens, tokens, tree)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        maps()
    for wrong in (dict(parents=_i32(4)), dict(lens=_i32(2)), dict(tree=D.draft_tree(6, 2, "cpu")), dict(tokens=S.token_map(5, 4, "cpu")), dict(parents=_i32(0), tree=tree)):
        refused(maps, ValueError, **wrong)
    refused(maps, TypeError, parents=torch.zeros(5, dtype=torch.int64))
    for rows, words in ((0, 1), (5, 0), (5, 33)):
        with pytest.raises(ValueError):
            D.draft_tree(rows, words, "cpu")

    ids = torch.zeros(5, dtype=torch.int64)
    accepted = D.accepted_drafts(3, 4, "cpu")
    accept = lambda chosen=ids, drafted=ids, parents=_i32(5), lens=_i32(3), accepted=accepted: D.accept_drafts(chosen, drafted, parents, lens, tokens, accepted)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        accept()
    for wrong in (dict(chosen=ids[:4]), dict(drafted=ids.int()), dict(parents=_i32(4)), dict(lens=_i32(4)), dict(accepted=D.accepted_drafts(2, 4, "cpu"))):
        refused(accept, ValueError, **wrong)
    for sequences, depth in ((0, 1), (3, 0), (65536, 1)):
        with pytest.raises(ValueError):
            D.accepted_drafts(sequences, depth, "cpu")
    pool = torch.zeros(3, 2, 16, 8)
    for pools in ([], [pool, pool], [pool, torch.zeros(3, 2, 16, 4)], [pool, pool.half()], [pool.transpose(0, 1)], [pool[0]]):
        with pytest.raises(ValueError):
            D.page_pools(pools)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        D.keep_accepted(accepted, tokens, D.page_pools([pool]))

    q, k, rule = torch.zeros(5, 4, 8), torch.zeros(5, 2, 8), S.rotary_rule(8, 1e4, device="cpu")
    norm = lambda q=q, k=k, positions=_i32(5), wq=torch.ones(8), wk=torch.ones(8), eps=1e-6, offset=0.0: D.norm_rotary_append(q, k, None, rule, positions, wq, wk, eps=eps, offset=offset)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        norm()
    for wrong in (dict(wq=torch.ones(7)), dict(wk=torch.ones(16)[::2]), dict(eps=-1e-3), dict(eps=float("nan")), dict(eps=float("inf")), dict(offset=float("nan")), dict(positions=_i32(4))):
        refused(norm, ValueError, **wrong)
    refused(norm, TypeError, wq=torch.ones(8).half())
    refused(norm, TypeError, wq=torch.ones(8).half(), wk=torch.ones(8).half())

    pools = torch.zeros(6, 2, 16, 8)
    attend = lambda q=q, keys=pools, values=pools.clone(), table=_i32(3, 4), lens=_i32(3), cu=_i32(4), visible=_i32(5, 1), out=None, scale=None, workspace=None: D.tree_attention(
        q, keys, values, table, lens, cu, visible, out=out, softmax_scale=scale, workspace=workspace)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        attend()
    for wrong in (dict(keys=pools[:, :, :, :4]), dict(keys=pools.half()), dict(q=torch.zeros(5, 3, 8)), dict(table=_i32(4, 4)), dict(table=_i32(12)), dict(lens=_i32(2)), dict(cu=_i32(3)),
                  dict(visible=_i32(4, 1)), dict(visible=_i32(5, 33)), dict(visible=_i32(5)), dict(out=torch.zeros(5, 4, 4)), dict(out=torch.zeros(5, 4, 8).half()), dict(scale=0.0),
                  dict(scale=float("inf")), dict(workspace=torch.zeros(4, 4)[:, ::2]), dict(values=pools.transpose(0, 1))):
        refused(attend, ValueError, **wrong)
    refused(attend, TypeError, visible=torch.zeros(5, 1, dtype=torch.int64))

    x = torch.zeros(5, 40)
    adjust = lambda logits=x, **more: D.adjust_logits(logits, **more)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        adjust(allowed=_i32(5, 2))
    history = D.TokenHistory(_i32(3, 7), _i32(3))
    for wrong in (dict(logits=x[0]), dict(logits=x.t()), dict(allowed=_i32(5, 1)), dict(history=history), dict(history=history, row_seq=_i32(4)), dict(out=torch.zeros(5, 41)),
                  dict(history=D.TokenHistory(_i32(3, 7), _i32(2)), row_seq=_i32(5)), dict(bias_ids=_i32(5, 2)), dict(bias_ids=_i32(5, 2), bias_values=torch.zeros(5, 3)),
                  dict(history=history, row_seq=_i32(5), repetition=torch.ones(2)), dict(drafts=D.DraftedTokens(ids[:3], _i32(5, 1), _i32(4)), row_seq=_i32(5))):
        refused(adjust, ValueError, **wrong)
    for wrong in (dict(repetition=torch.ones(5).double()), dict(out=torch.zeros(5, 40).half()), dict(allowed=torch.zeros(5, 2, dtype=torch.int64)),
                  dict(bias_ids=_i32(5, 2), bias_values=torch.zeros(5, 2).half())):
        refused(adjust, TypeError, **wrong)
