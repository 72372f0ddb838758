"""The engine on the scaled 8-bit cache: mixed steps, entries of any range, tensor parallelism."""
import json
import os
import subprocess
import sys

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


# ------------------------------------------------------------------------------------------------ ranks
CHILD = r"""
import json, os, sys
sys.path.insert(0, os.environ["ROOT"])
from aws_k8s_ansible_provisioner_amd.engine.config import EngineConfig, SamplingParams
from aws_k8s_ansible_provisioner_amd.parallel import tp_worker
import torch.distributed as dist
made = []
class Runner(tp_worker.ModelRunner):
    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        made.append(self)
tp_worker.ModelRunner = Runner
ecfg = EngineConfig(model=os.environ["MODEL"], device="cpu", max_model_len=256, max_num_seqs=8,
                    max_num_batched_tokens=32, block_size=32, num_gpu_blocks=96, kv_cache_dtype="fp8_scaled",
                    tensor_parallel_size=int(os.environ["WORLD_SIZE"]), shard_init="full", init_std=0.15)
eng, bc = tp_worker.make_tp_engine(ecfg, backend="gloo", log=lambda *a: None)
def run(n):
    return [o.output_ids for o in eng.generate(None, SamplingParams(max_tokens=n, temperature=0, ignore_eos=True),
                                               prompt_ids=json.loads(os.environ["PROMPTS"]))]
if eng is not None:
    if os.environ["TOKENS"] == "1":
        run(1)
    else:
        print("TOKENS " + json.dumps(run(8)), flush=True)
    bc.shutdown()
print("SCALES " + json.dumps(made[0].kv_scales[0].log2().tolist()), flush=True)
"""


def ranks(model, world, tokens):
    """A name -> value lookup of what each rank printed."""
    from test_tp_cpu import ROOT, _port

    port = _port()
    procs = [subprocess.Popen([sys.executable, "-c", CHILD], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                              text=True, env=dict(os.environ, RANK=str(r), WORLD_SIZE=str(world), LOCAL_RANK=str(r),
                                                  MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), ROOT=ROOT,
                                                  MODEL=model, PROMPTS=json.dumps(PROMPTS), TOKENS=str(tokens),
                                                  OMP_NUM_THREADS="1"))
             for r in range(world)]
    outs = [p.communicate(timeout=300) for p in procs]
    assert all(p.returncode == 0 for p in procs), [o[1][-3000:] for o in outs]
    lines = [[x.split(" ", 1) for x in o[0].splitlines() if x.startswith(("TOKENS ", "SCALES "))] for o in outs]
    return [{name: json.loads(x) for name, x in mine} for mine in lines]


MODELS = [("tiny-qwen3", 2), ("tiny-llama", 4)]           # (4 ranks: a kv head on two of them)


@pytest.mark.parametrize("model,world", MODELS)
def test_ranks_answer_as_one_process(model, world):
    from test_engine_cpu import _near_argmax

    one = _engine(model, kv_cache_dtype="fp8_scaled", shard_init="full")
    for p, got in zip(PROMPTS, ranks(model, world, 8)[0]["TOKENS"]):
        assert len(got) == 8
        _near_argmax(one, p, got, tol=0.5)                # (one process's, in test_scaled_cache)


@pytest.mark.parametrize("model,world", MODELS)
def test_ranks_keep_the_scales_of_their_heads(model, world):
    """The first layer's keys and values of the prompts are those of one process but for bf16 roundings of the
    projection, which move a page's largest entry by less than a factor of two: its scale by one power at most."""
    one = _engine(model, kv_cache_dtype="fp8_scaled", shard_init="full")
    one.generate(None, SamplingParams(max_tokens=1, **GREEDY), prompt_ids=PROMPTS)
    whole, hkv = one.runner.kv_scales[0].log2(), one.runner.model.hkv
    assert bool((whole > -100).any())
    for rank, said in enumerate(ranks(model, world, 1)):
        mine = torch.tensor(said["SCALES"])
        heads = slice(rank * hkv // world, max(rank * hkv // world + 1, (rank + 1) * hkv // world))
        assert mine.shape == whole[:, :, heads].shape
        assert bool(((mine - whole[:, :, heads]).abs() <= 1).all())


def test_pairs_of_prefill_and_decode_are_refused():
    """Also for engines of no role: what a pair moves would be codes without their scales."""
    from aws_k8s_ansible_provisioner_amd.parallel.pd_driver import PDPair

    eng = _engine("tiny-qwen3", kv_cache_dtype="fp8_scaled")
    for rank in range(2):
        with pytest.raises(ValueError, match="scales"):
            PDPair(eng, rank, 2)
