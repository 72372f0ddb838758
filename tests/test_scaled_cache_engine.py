"""The engine on the scaled 8-bit cache: mixed steps, entries of any range."""
import pytest
import torch

from aws_k8s_ansible_provisioner_amd import ops
from aws_k8s_ansible_provisioner_amd.engine.config import SamplingParams
from test_engine_cpu import _engine

GREEDY = dict(temperature=0, ignore_eos=True)


# ------------------------------------------------------------------------------------------------ mixed steps
def test_prompts_of_a_mixed_step_are_planned_without_its_decode_rows(monkeypatch):
    """What bounds the prompts' keys is the longest sequence that a tile names, also where a longer one decodes in
    the same step."""
    seen, real = [], ops.scaled_attention_prefill

    def record(out, q, k, v, s, tables, lens, q_start, tile_seq, *a, max_len=None, **kw):
        named = int(lens[tile_seq.long().unique()].max())
        seen.append((named, max_len, int(lens.max())))
        return real(out, q, k, v, s, tables, lens, q_start, tile_seq, *a, max_len=max_len, **kw)

    monkeypatch.setattr(ops, "scaled_attention_prefill", record)
    eng = _engine("tiny-qwen3", kv_cache_dtype="fp8_scaled", max_num_batched_tokens=64)
    eng.add_request("long", None, SamplingParams(max_tokens=12, **GREEDY), prompt_ids=[7, 8, 9] * 50)
    for step in range(40):
        if step == 5:
            eng.add_request("short", None, SamplingParams(max_tokens=2, **GREEDY), prompt_ids=list(range(5, 25)))
        eng.step()
    assert any(named < longest for named, _, longest in seen)           # a mixed step was among them
    assert all(said == named for named, said, _ in seen)


# ------------------------------------------------------------------------------------------------ range
PROMPTS = [list(range(5, 45)), [7, 8, 9] * 14, [100, 101, 102]]


def loud(model, keys, values):
    """The same network with keys 2^keys and values 2^values times as large: query norms (or projections) and output
    projections take the powers back.  Every step of it is exact, so that with a cache that holds any range nothing
    else changes, to the last bit."""
    hq, hkv, D = model.hq, model.hkv, model.D
    for lw in model.layers:
        if lw.k_norm is not None:
            lw.k_norm.mul_(2.0 ** keys)
            lw.q_norm.mul_(2.0 ** -keys)
        else:
            lw.w_qkv[hq * D:(hq + hkv) * D].mul_(2.0 ** keys)
            lw.w_qkv[:hq * D].mul_(2.0 ** -keys)
        lw.w_qkv[(hq + hkv) * D:].mul_(2.0 ** values)
        lw.w_o.mul_(2.0 ** -values)


def generated(eng):
    """Tokens and their log-probabilities: prompts in chunks, decode steps, mixed steps."""
    sp = SamplingParams(max_tokens=8, logprobs=1, **GREEDY)
    plain = SamplingParams(max_tokens=8, **GREEDY)
    outs = eng.generate(None, sp, prompt_ids=PROMPTS)
    more = eng.generate(None, plain, prompt_ids=PROMPTS)          # (without log-probs: captured steps on the GPU)
    return [o.output_ids for o in outs] + [o.output_ids for o in more], torch.tensor([o.logprobs for o in outs])


def check_any_range(eng, keys, values, plain):
    """eng: on a scaled cache; plain: on the e4m3 cache of scale 1.  Neither keeps prefixes."""
    tokens, logp = generated(eng)
    fixed = generated(plain)
    for e in (eng, plain):
        loud(e.runner.model, keys, values)
    again, logp2 = generated(eng)
    assert again == tokens and torch.equal(logp2, logp)
    # entries beyond the largest code of scale 1, or none as large as its least normal one
    for s in eng.runner.kv_scales:
        for top, e in zip(s.amax((1, 2)).tolist(), (keys, values)):
            assert top > 1 if e > 0 else 2.0 ** -100 < top and 448 * top < 2.0 ** -6
    # that cache loses them
    now = generated(plain)
    assert float((now[1] - fixed[1]).abs().max()) > 0.05


@pytest.mark.parametrize("model", ["tiny-qwen3", "tiny-llama"])
@pytest.mark.parametrize("keys,values", [(12, 13), (-20, -21)])
def test_entries_of_any_range(model, keys, values):
    """Keys and values in the thousands, and below the least code of scale 1: the results of the plain network."""
    kw = dict(enable_prefix_caching=False)
    check_any_range(_engine(model, kv_cache_dtype="fp8_scaled", **kw), keys, values,
                    _engine(model, kv_cache_dtype="fp8", **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["tiny-qwen3", "tiny-llama"])
@pytest.mark.parametrize("keys,values", [(12, 13), (-20, -21)])
def test_entries_of_any_range_gpu(model, keys, values):
    from test_engine_gpu import _engine as engine

    kw = dict(enable_prefix_caching=False)
    eng = engine(model, kv_cache_dtype="fp8_scaled", **kw)
    assert eng.runner.graphs
    check_any_range(eng, keys, values, engine(model, kv_cache_dtype="fp8", **kw))
