"""The engine on the scaled 8-bit cache: mixed steps."""
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
