"""Operators of batches that share prompts, on the CPU: the library's ABI, refusals, angle fractions, groups of a batch's caches."""
import ctypes
import math
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    from cacheir_b200 import _lib, build

    build.build(groups=("serving",))
    return _lib.load_group("serving")


def test_library_exports_every_declared_symbol(lib):
    from cacheir_b200 import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "cacheir_b200_serving.h").read_text(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(cacheir_b200_[a-z0-9_]+)\s*\(", text)))
    assert all(hasattr(lib, name) for name in declared)
    assert sorted(_lib.GROUP_SIGNATURES["serving"]) == declared, "ctypes table and header disagree"


def test_argument_structs_have_the_compiler_s_layout(tmp_path):
    from cacheir_b200 import _lib

    lines, want = [], []
    for name, struct in (("cacheir_b200_tables_args", _lib.TablesArgs), ("cacheir_b200_rotary_args", _lib.RotaryArgs),
                         ("cacheir_b200_prefix_args", _lib.PrefixArgs), ("cacheir_b200_logprobs_args", _lib.LogprobsArgs)):
        want.append(ctypes.sizeof(struct))
        lines.append(f'std::printf("%zu ", sizeof({name}));')
        for field, _ in struct._fields_:
            want.append(getattr(struct, field).offset)
            lines.append(f'std::printf("%zu ", offsetof({name}, {field}));')
    (tmp_path / "layout.cpp").write_text('#include <cstddef>\n#include <cstdio>\n#include "cacheir_b200_serving.h"\nint main() {\n' + "\n".join(lines) + "\n}\n")
    subprocess.run(["g++", "-I", str(ROOT / "include"), "layout.cpp", "-o", "layout"], cwd=tmp_path, check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want


def test_c_entry_points_refuse_before_they_launch(lib):
    """Codes of calls that never reach the device: missing pointers, extents, limits, scratch."""
    from cacheir_b200._lib import LogprobsArgs, PrefixArgs, RotaryArgs, TablesArgs

    some = 4096                                               # an address that no refused call looks at
    names = ("page_table", "seq_lens", "change", "free_pages", "free_count", "positions", "row_seq", "slots", "cu_rows", "status")
    tables = lambda n=4, pages=8, size=16, capacity=9, rows=3, null=None: lib.cacheir_b200_extend_page_tables(ctypes.byref(TablesArgs(
        **{name: None if i == null else some for i, name in enumerate(names)}, sequences=n, max_pages=pages, page_size=size, capacity=capacity, rows=rows)), None)
    assert [tables(n=0), tables(rows=0)] == [0, 0]
    assert [tables(null=i) for i in range(10)] == [-1] * 10
    assert [tables(pages=0), tables(size=0), tables(capacity=0)] == [-1] * 3
    assert [tables(n=16385), tables(pages=1 << 28)] == [-5, -5]
    shrink = lambda n=4, pages=8, size=16, capacity=9: lib.cacheir_b200_shrink_page_tables(ctypes.byref(TablesArgs(
        page_table=some, seq_lens=some, change=some, free_pages=some, free_count=some, status=some, sequences=n, max_pages=pages, page_size=size,
        capacity=capacity)), None)
    assert [shrink(n=0), shrink(pages=0), shrink(n=16385), shrink(capacity=0)] == [0, -1, -5, -1]

    good = dict(q=some, k=some, v=some, q_out=some, k_cache=some, v_cache=some, positions=some, slots=some, turns=some, rows=2, heads=4, kv_heads=2, dim=64,
                rot=64, num_slots=3, page_size=16, dtype=1, factor=1.0)
    rotary = lambda **new: lib.cacheir_b200_rotary_append(ctypes.byref(RotaryArgs(**{**good, **new})), None)
    assert rotary(rows=0) == 0
    bad = [dict(q=None), dict(k=None), dict(v=None), dict(positions=None), dict(turns=None), dict(k_cache=None), dict(heads=0), dict(rot=3), dict(rot=66), dict(rot=0),
           dict(layout=2), dict(dtype=7), dict(num_slots=0), dict(slots=None), dict(slots=None, k_cache=None, v_cache=None)]
    assert [rotary(**b) for b in bad] == [-1] * len(bad)
    assert rotary(dim=1026, rot=64) == -5

    need = lib.cacheir_b200_shared_prefix_workspace_bytes(2, 4, 64)
    assert need > 0 and lib.cacheir_b200_shared_prefix_workspace_bytes(0, 4, 64) == 0
    good = dict(q=some, k_cache=some, v_cache=some, out=some, page_table=some, seq_lens=some, group_rows=some, prefix_table=some, prefix_lens=some, workspace=some,
                workspace_bytes=need, batch=2, heads=4, kv_heads=2, dim=64, page_size=16, num_slots=3, max_pages=4, groups=1, prefix_pages=2, dtype=1)
    prefix = lambda **new: lib.cacheir_b200_shared_prefix_attention(ctypes.byref(PrefixArgs(**{**good, **new})), None)
    assert prefix(batch=0) == 0
    bad = [dict(q=None), dict(out=None), dict(page_table=None), dict(group_rows=None), dict(prefix_lens=None), dict(prefix_pages=0), dict(kv_heads=3), dict(dim=0),
           dict(groups=-1), dict(dtype=3), dict(num_slots=0)]
    assert [prefix(**b) for b in bad] == [-1] * len(bad)
    assert [prefix(workspace=None), prefix(workspace_bytes=need - 1), prefix(workspace=some + 4), prefix(dim=513), prefix(batch=65536)] == [-3, -3, -2, -4, -5]

    logprobs = lambda logits=some, stride=0, tokens=some, out=some, ids=some, rows=2, vocab=9, top=3, t=1.0, dtype=0: lib.cacheir_b200_token_logprobs(
        ctypes.byref(LogprobsArgs(logits=logits, tokens=tokens, logprobs=out, entropy=out, top_ids=ids, top_logprobs=ids, row_stride=stride, temperature=t,
                                  rows=rows, vocab=vocab, top=top, dtype=dtype)), None)
    assert [call(None, None) for call in (lib.cacheir_b200_extend_page_tables, lib.cacheir_b200_shrink_page_tables, lib.cacheir_b200_token_logprobs)] == [-1] * 3
    assert [logprobs(rows=0), logprobs(vocab=0)] == [0, 0]
    bad = [dict(logits=None), dict(tokens=None), dict(ids=None), dict(top=-1), dict(t=0.0), dict(t=float("nan")), dict(t=-1.0), dict(dtype=9), dict(stride=8)]
    assert [logprobs(**b) for b in bad] == [-1] * len(bad)
    assert [logprobs(top=10), logprobs(vocab=100, top=33)] == [-5, -5]


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_wrappers_refuse_wrong_arguments_and_cpu_tensors():
    from cacheir_b200 import serving_ops as S
    from cacheir_b200._lib import CacheIRB200Error

    tokens = S.token_map(5, 3, "cpu")
    extend = lambda table=_i32(3, 4), lens=_i32(3), new=_i32(3), free=_i32(8), count=_i32(1), tokens=tokens, page_size=16: S.extend_page_tables(
        table, lens, new, free, count, tokens, page_size=page_size)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        extend()
    with pytest.raises(TypeError):
        extend(lens=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        extend(table=_i32(4, 3).t())
    for wrong in (dict(table=_i32(12)), dict(lens=_i32(4)), dict(new=_i32(2)), dict(count=_i32(2)), dict(page_size=0), dict(tokens=S.token_map(5, 4, "cpu")), dict(free=_i32(0))):
        with pytest.raises(ValueError):
            extend(**wrong)
    lens = _i32(3)
    with pytest.raises(ValueError):
        extend(lens=lens, new=lens)
    with pytest.raises(ValueError):
        S.shrink_page_tables(_i32(3, 4), _i32(3), _i32(3), _i32(8), _i32(1), _i32(1), page_size=16, held_pages=_i32(2))
    with pytest.raises(ValueError):
        S.token_map(0, 3, "cpu")

    rule = S.rotary_rule(64, 10000.0, device="cpu")
    q, k, pool = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(5, 2, 16, 64)
    rotary = lambda q=q, k=k, v=k, rule=rule, positions=_i32(3), slots=_i32(3), k_cache=pool, v_cache=pool, **more: S.rotary_append(
        q, k, v, rule, positions, slots=slots, k_cache=k_cache, v_cache=v_cache, **more)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        rotary()
    for wrong in (dict(k=torch.zeros(3, 2, 32)), dict(v=None), dict(v=torch.zeros(3, 3, 64)), dict(positions=_i32(2)), dict(slots=None), dict(v_cache=None),
                  dict(k_cache=torch.zeros(5, 2, 16, 32)), dict(k_cache=torch.zeros(5, 16, 2, 64).transpose(1, 2)), dict(q=torch.zeros(3, 64, 4).transpose(1, 2)),
                  dict(rule=S.rotary_rule(128, 10000.0, device="cpu")), dict(q_out=torch.zeros(3, 5, 64)), dict(q=torch.zeros(1, 4, 64).expand(3, 4, 64))):
        with pytest.raises(ValueError):
            rotary(**wrong)
    with pytest.raises(TypeError):
        rotary(q=q.half())
    for wrong in (dict(rot=63), dict(rot=0), dict(base=-1.0), dict(layout="spiral"), dict(scaling=(8.0, 1.0, 4.0, 8192.0), yarn=(16.0, 8192.0, 32.0, 1.0))):
        with pytest.raises(ValueError):
            S.rotary_rule(**{"rot": 64, "base": 10000.0, "device": "cpu", **wrong})

    groups = S.PrefixGroups(_i32(2), _i32(1, 2), _i32(1))
    attend = lambda q=q, k=pool, v=pool, table=_i32(3, 4), lens=_i32(3), groups=groups, **more: S.shared_prefix_attention(q, k, v, table, lens, groups, **more)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        attend()
    for wrong in (dict(q=torch.zeros(3, 3, 64)), dict(k=torch.zeros(5, 2, 16, 32)), dict(table=_i32(2, 4)), dict(lens=_i32(4)), dict(softmax_scale=0.0),
                  dict(softmax_scale=float("inf")), dict(out=torch.zeros(3, 4, 32)), dict(groups=S.PrefixGroups(_i32(3), _i32(1, 2), _i32(1))),
                  dict(groups=S.PrefixGroups(_i32(1), _i32(0, 2), _i32(0))), dict(q=q.half()), dict(k=pool.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            attend(**wrong)

    logits, ids = torch.zeros(3, 9), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(CacheIRB200Error, match="no CPU fallback"):
        S.token_logprobs(logits, ids)
    for wrong in (dict(tokens=ids[:2]), dict(tokens=ids.int()), dict(top=10), dict(top=-1), dict(temperature=0.0), dict(temperature=float("nan")),
                  dict(logits=torch.zeros(9)), dict(logits=torch.zeros(9, 3).t()), dict(logits=torch.zeros(1, 9).expand(3, 9)), dict(logits=torch.zeros(3, 40), top=33)):
        with pytest.raises(ValueError):
            S.token_logprobs(**{"logits": logits, "tokens": ids, **wrong})
    with pytest.raises(TypeError):
        S.token_logprobs(logits.double(), ids)


def test_turn_fractions_are_the_angles_modulo_one_turn():
    """position * fraction (modulo 2^64) against the angle in arithmetic of 50 digits: a fraction is off by its last bit at most, so the angle
    of position p by p * 2^-64 turns, on top of the frequency's own rounding to a double."""
    from decimal import Decimal, getcontext

    from cacheir_b200 import serving_ops as S
    from cacheir_b200.ragged import rotary_frequencies

    getcontext().prec = 50
    two_pi = Decimal("6.2831853071795864769252867665590057683943387987502")
    freq = rotary_frequencies(128, 500000.0)
    bits = S.turn_fractions(freq).view(np.uint64)
    for i in (0, 1, 17, 63):
        for position in (1, 999, 1000003, 2 ** 31 - 1):
            got = Decimal((int(bits[i]) * position) % 2 ** 64) / 2 ** 64
            want = (Decimal(float(freq[i])) * position / two_pi) % 1
            gap = abs(got - want)
            assert min(gap, 1 - gap) <= Decimal(position) * (Decimal(2) ** -53 * Decimal(float(freq[i])) + Decimal(2) ** -63), (i, position)
    # whole turns vanish, negative frequencies wrap
    assert S.turn_fractions(np.array([0.0, 2 * math.pi, -math.pi])).view(np.uint64).tolist() == [0, 0, 2 ** 63]
    for wrong in ([], [float("nan")], [[1.0]]):
        with pytest.raises(ValueError):
            S.turn_fractions(np.array(wrong))


def test_rotary_rules_have_the_package_s_frequencies():
    from cacheir_b200 import serving_ops as S
    from cacheir_b200.ragged import rotary_frequencies, yarn_frequencies

    plain = S.rotary_rule(64, 10000.0, layout="half", device="cpu")
    assert plain.rot == 64 and plain.layout == "half" and plain.factor == 1.0
    np.testing.assert_array_equal(plain.turns.numpy(), S.turn_fractions(rotary_frequencies(64, 10000.0)))
    scaled = S.rotary_rule(64, 500000.0, scaling=(8.0, 1.0, 4.0, 8192.0), device="cpu")
    np.testing.assert_array_equal(scaled.turns.numpy(), S.turn_fractions(rotary_frequencies(64, 500000.0, (8.0, 1.0, 4.0, 8192.0))))
    yarn = S.rotary_rule(64, 500000.0, yarn=(16.0, 8192.0, 32.0, 1.0), device="cpu")
    freq, factor = yarn_frequencies(64, 500000.0, 16.0, 8192.0, 32.0, 1.0)
    assert yarn.factor == factor
    np.testing.assert_array_equal(yarn.turns.numpy(), S.turn_fractions(freq))


def test_groups_of_a_batch_are_the_pages_that_neighbours_alias():
    from cacheir_b200 import serving_ops as S
    from cacheir_b200.kv_cache import B200KVPageAllocator, B200PagedKVCache

    alloc = B200KVPageAllocator(page_size=4)

    def cache(tokens, of=None, common=0):
        c = B200PagedKVCache(alloc, 1)
        if of is not None:
            c.share_prefix(of, common)
        c.extend(tokens - c.tokens)
        return c
    a = cache(11)
    b, c = cache(14, a, 8), cache(9, a, 8)
    d = cache(6)
    e = cache(21)
    f, g = cache(18, e, 16), cache(30, e, 8)
    groups = S.prefix_groups([a, b, c, d, e, f, g], "cpu")
    assert groups.rows.tolist() == [0, 3, 4, 7]
    assert groups.lens.tolist() == [8, 0, 8]
    assert groups.table[0].tolist() == a.page_ids()[:2] and groups.table[2].tolist() == e.page_ids()[:2] and groups.table.shape == (3, 2)
    assert S.prefix_groups([a, d, e], "cpu") is None and S.prefix_groups([], "cpu") is None and S.prefix_groups([a], "cpu") is None
    # longer common parts than asked for only
    groups = S.prefix_groups([a, b, e, f], "cpu", min_tokens=12)
    assert groups.rows.tolist() == [0, 1, 2, 4] and groups.lens.tolist() == [0, 0, 16]
    assert groups.table[2].tolist() == e.page_ids()[:4]


def test_a_row_joins_a_group_only_where_no_fewer_tokens_are_shared():
    from cacheir_b200 import serving_ops as S
    from cacheir_b200.kv_cache import B200KVPageAllocator, B200PagedKVCache

    alloc = B200KVPageAllocator(page_size=4)
    first = B200PagedKVCache(alloc, 1)
    first.extend(40)

    def cache(common):
        c = B200PagedKVCache(alloc, 1)
        c.share_prefix(first, common)
        c.extend(3)
        return c
    long, short = [cache(36) for _ in range(3)], [cache(8) for _ in range(4)]
    groups = S.prefix_groups([*long, *short], "cpu")
    assert groups.rows.tolist() == [0, 3, 7] and groups.lens.tolist() == [36, 8]
    groups = S.prefix_groups([long[0], *short, long[1]], "cpu")       # (a lone row loses nothing by joining)
    assert groups.rows.tolist() == [0, 6] and groups.lens.tolist() == [8]


def test_launches_by_extents(lib):
    from cacheir_b200 import serving_ops as S

    launches = lambda groups, dtype=torch.float16, dim=128, page=16, heads=32, kv=8: S.shared_prefix_launches(4, heads, kv, dim, page, groups, dtype)
    assert [launches(0), launches(1), launches(64), launches(65)] == [2, 3, 3, 4]
    assert [launches(1, torch.float32), launches(1, dim=80), launches(1, page=24), launches(1, heads=130, kv=2)] == [2] * 4
    assert launches(1, torch.bfloat16, dim=64, page=48) == 3


def test_what_a_wait_says_is_the_same_in_all_lanes_of_a_warp():
    """Loops around waits hold votes and instructions of whole warps: a lane whose wait gave up must not leave alone while the others go on. What a
    bounded wait says is kept nowhere but where a vote has made it the warp's; elsewhere it is only waited."""
    for name in ("shared_prefix_mma.cu", "token_logprobs.cu"):
        lines = (ROOT / "cacheir_b200" / "csrc" / name).read_text().splitlines()
        kept = [line.strip() for line in lines if re.search(r"\bmbar_(try_)?wait\(", line) and "__all_sync(" not in line
                and not re.match(r"\s*(for \([^()]*\) )?mbar_wait\(", line)]
        assert not kept, (name, kept)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shared_prefixes", [False, True])
def test_a_runtime_reports_waits_of_every_library_that_it_may_call(monkeypatch, ragged, shared_prefixes):
    """`score_tokens` calls the serving library on any runtime. Each check reads and clears all words, so that the next one reports what came after it."""
    from types import SimpleNamespace

    from cacheir_b200 import _lib
    from cacheir_b200.runtime import B200DecodeRuntime

    words = {"core": 0, "ragged": 0, "serving": 0}

    def word(name):
        def read(reset):
            found = words[name]
            words[name] = 0 if reset else found
            return found
        return read
    monkeypatch.setattr(_lib, "_LIB", SimpleNamespace(cacheir_b200_device_status=word("core")))
    monkeypatch.setattr(_lib, "_GROUPS", {name: SimpleNamespace(**{f"cacheir_b200_{name}_device_status": word(name)}) for name in ("ragged", "serving")})
    if ragged:
        monkeypatch.setattr(_lib, "_LIB", None)               # (a ragged family's process may not have the core library at all)
        monkeypatch.setattr(_lib, "load", lambda: pytest.fail("the core library is not this runtime's"))
    runtime = SimpleNamespace(device=-1, _engine=SimpleNamespace(ragged=ragged, shared_prefixes=shared_prefixes))
    check = lambda: B200DecodeRuntime.check_device_status(runtime)
    check()
    for gave_up in ({"serving": 0x1001}, {"ragged" if ragged else "core": 0x302, "serving": 0x1001}):
        words.update(gave_up)
        with pytest.raises(RuntimeError, match="gave up"):
            check()
        check()
        assert not any(words.values())


def test_a_decode_step_of_one_row_shares_nothing():
    """It is lowered like that of a runtime without `shared_prefixes`: one launch of the ordinary attention, fused with the next product's activations
    where there are such."""
    from types import SimpleNamespace

    from cacheir_b200.runtime import _Engine

    def lowered(shared_prefixes, sessions):
        engine = SimpleNamespace(page_size=16, shared_prefixes=shared_prefixes, _plan=lambda key, pages, make: (key, make(pages)),
                                 plan_class=lambda engine, batch, width, **more: (batch, width, more))
        return _Engine.plan_for(engine, [SimpleNamespace(kv_cache=SimpleNamespace(tokens=20)) for _ in range(sessions)])
    assert lowered(False, 1) == lowered(True, 1) == (("decode", 1), (1, 2, {}))
    assert lowered(False, 3) == (("decode", 3), (3, 2, {}))
    assert lowered(True, 3) == (("decode", 3), (3, 2, {"shared_prefixes": True}))


def test_scores_are_refused_before_the_session_is_given_up():
    """A refused `score_tokens` leaves the session's tokens where they are and runs nothing."""
    from types import SimpleNamespace

    from cacheir_b200.runtime import B200DecodeRuntime

    runtime = SimpleNamespace(_engine=SimpleNamespace(config=SimpleNamespace(vocab_size=20)), device="cpu", run=lambda *a, **k: pytest.fail("the prompt was run"))
    for wrong in (dict(top=33), dict(top=21), dict(top=-1), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=1e7)):
        with pytest.raises(ValueError):
            B200DecodeRuntime.score_tokens(runtime, [1, 2, 3], **wrong)
    with pytest.raises(ValueError):
        B200DecodeRuntime.score_tokens(runtime, [1])
