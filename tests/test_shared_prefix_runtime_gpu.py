"""The runtime's decode steps with `shared_prefixes`, and the scores of tokens, on small models."""
import zlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    from cacheir_b200 import _lib

    yield
    assert _lib.load_group("serving").cacheir_b200_serving_device_status(1) == 0


def _runtime(dtype, heads=8, kv_heads=2, head_dim=64, quant=None, **more):
    from cacheir_b200 import B200DecodeRuntime, B200KVPageAllocator, ModelConfig, build_decoder_artifact

    cfg = ModelConfig(architecture="LlamaForCausalLM", vocab_size=512, hidden_size=heads * head_dim, intermediate_size=768, num_layers=2,
                      num_attention_heads=heads, num_key_value_heads=kv_heads, rms_norm_eps=1e-5, rope_theta=10000.0,
                      max_position_embeddings=1024, dtype=dtype)
    gen = torch.Generator(device="cuda")

    def synth(key, shape):
        if len(shape) == 1:
            return torch.ones(shape, device="cuda", dtype=torch.float32)
        gen.manual_seed(zlib.crc32(key.encode()))
        return torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen) * 0.05
    return B200DecodeRuntime(build_decoder_artifact(cfg, target="cuda", quant=quant, modes=("decode",)), dtype=dtype, tensor_source=synth,
                             kv_allocator=B200KVPageAllocator(page_size=16, initial_slots=256), max_seq_len=512, **more)


PROMPT = [int(t) for t in np.random.default_rng(1).integers(0, 512, 140)]


def _batch(rt):
    """Three requests that share 128 tokens of a prompt, a stranger between two of them, two that share 32 tokens."""
    holder = rt.fork()
    holder.prefill_tokens(PROMPT)
    sessions = []
    for common, rest in ((128, [5, 6, 7]), (128, [9]), (0, PROMPT[3:60]), (128, [1, 2]), (32, PROMPT[40:50]), (32, [77] * 20)):
        s = rt.fork()
        if common:
            s.kv_cache.share_prefix(holder.kv_cache, common)
        s.run([rest], mode="prefill", reset_kv=False)
        sessions.append(s)
    return holder, sessions


def _steps(rt, sessions, first, steps):
    out, tokens = [], first
    for _ in range(steps):
        logits = rt.run_decode_batch(sessions, tokens)[:, 0].float()
        out.append(logits.clone())
        tokens = [(t * 7 + 3) % 512 for t in tokens]           # (the same tokens whatever the logits)
    return out


@pytest.mark.parametrize("dtype,head_dim,quant,gate", [("float16", 64, None, 4e-3), ("float16", 128, "int8", 4e-3), ("float32", 64, None, 2e-5),
                                                       ("bfloat16", 128, None, 3e-2)])
def test_decode_with_shared_prefixes_is_decode(dtype, head_dim, quant, gate):
    """The same requests with and without, 40 steps over page boundaries; then one leaves, another takes its place. The gates are those of the
    whole model at these types."""
    plain, shared = (_runtime(dtype, head_dim=head_dim, quant=quant, shared_prefixes=on) for on in (False, True))
    results = []
    for rt in (plain, shared):
        holder, sessions = _batch(rt)
        steps = _steps(rt, sessions, [3, 1, 4, 1, 5, 9], 40)
        sessions[1].kv_cache.clear()
        sessions[1].kv_cache.share_prefix(holder.kv_cache, 64)
        sessions[1].run([[8, 8, 8]], mode="prefill", reset_kv=False)
        steps += _steps(rt, sessions, [2, 7, 1, 8, 2, 8], 10)
        steps += _steps(rt, sessions[3:] + sessions[:2], [2, 7, 1, 8, 2], 3)
        rt.check_device_status()
        results.append(steps)
    for a, b in zip(*results):
        assert float((a - b).norm() / a.norm()) <= gate
    counts = shared.cache_stats()["kernel_counts"]
    assert counts["b200.shared_prefix_attention"] > 0
    assert "b200.shared_prefix_attention" not in plain.cache_stats()["kernel_counts"]


def test_greedy_tokens_with_shared_prefixes():
    """On-device feedback: the tokens of the float32 model, alone and together."""
    results = []
    for on in (False, True):
        rt = _runtime("float32", shared_prefixes=on)
        _, sessions = _batch(rt)
        results.append(rt.decode_greedy_batch(sessions, [3, 1, 4, 1, 5, 9], 30).tolist())
    assert results[0] == results[1]


def test_plans_know_who_shares_what():
    rt = _runtime("float16", shared_prefixes=True)
    holder, sessions = _batch(rt)
    rt.run_decode_batch(sessions, [1] * 6)
    plan = rt._engine.plans[("decode", 6)]
    # (the fourth row has more in common with the first ones, but these are not its neighbours)
    assert plan.groups.rows.tolist() == [0, 2, 3, 6, 6, 6, 6] and plan.groups.lens.tolist() == [128, 0, 32, 0, 0, 0]
    assert plan.groups.table[0, :8].tolist() == holder.kv_cache.page_ids()[:8]
    rt.run_decode_batch(sessions[2:4] + sessions[:2] + sessions[4:], [1] * 6)
    assert plan.groups.rows.tolist() == [0, 1, 4, 6, 6, 6, 6] and plan.groups.lens.tolist() == [0, 128, 32, 0, 0, 0]
    alone = [rt.fork() for _ in range(6)]
    rt.run_prefill_batch(alone, [[1, 2, 3]] * 6)
    rt.run_decode_batch(alone, [1] * 6)
    assert plan.groups.rows.tolist() == [0] * 7
    launches = plan.launches_per_step
    assert launches > 0
    with pytest.raises(ValueError, match="shared_prefixes"):
        _runtime("float16", shared_prefixes=True, kv_dtype="int8")


@pytest.mark.parametrize("dtype,length", [("float32", 40), ("float16", 200), ("float32", 2)])
def test_scores_of_tokens(dtype, length):
    """Against the logits of the same prompt; chains of up to 512 additions and the logits' own values in 64 bits."""
    rt = _runtime(dtype)
    ids = (PROMPT * 2)[:length]
    logits = rt.run([ids], mode="prefill")[0].double()
    got = rt.score_tokens(ids, top=4, temperature=0.8)
    lp = torch.log_softmax(logits[:-1] / 0.8, dim=-1)
    want = lp.gather(1, torch.tensor(ids[1:], device="cuda")[:, None])[:, 0]
    assert got.logprobs.shape == (length - 1,) and bool(((got.logprobs.double() - want).abs() <= 4e-5).all())
    assert bool(((got.entropy.double() + (lp.exp() * lp).sum(-1)).abs() <= 1e-4).all())
    order = torch.sort(logits[:-1], dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(got.top_ids, order)
    assert rt.kv_cache.tokens == length
    with pytest.raises(ValueError):
        rt.score_tokens([1])


def test_a_session_alone_takes_the_ordinary_attention():
    """Its logits are the bits of a runtime without the option, its launches too (int8: attention writes the next product's activations)."""
    found = []
    for on in (False, True):
        rt = _runtime("float16", heads=8, kv_heads=2, head_dim=128, quant="int8", shared_prefixes=on)
        holder = rt.fork()
        holder.prefill_tokens(PROMPT)
        s = rt.fork()
        s.kv_cache.share_prefix(holder.kv_cache, 128)
        s.run([[5, 6, 7]], mode="prefill", reset_kv=False)
        logits = [rt.run_decode_batch([s], [t]).clone() for t in (3, 1, 4, 1, 5)]
        counts = {name: n for name, n in rt.cache_stats()["kernel_counts"].items() if "attention" in name}
        found.append((torch.cat(logits), counts, rt._engine.plans[("decode", 1)].launches_per_step))
    assert torch.equal(found[0][0], found[1][0]) and found[0][1:] == found[1][1:]
    assert "b200.shared_prefix_attention" not in found[1][1]
