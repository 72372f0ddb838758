"""The scaled 8-bit cache on the CPU: the plain forms against 64 bits, and what is refused."""
import math

import pytest
import torch

import scaled_cache_oracle as orc
from aws_k8s_ansible_provisioner_amd import ops
from aws_k8s_ansible_provisioner_amd.ops import reference as ref

D = 128


def make(seed, H, G, T, slots, page, pages, norm=True, std=1.0):
    g = torch.Generator().manual_seed(seed)
    k, v, s = orc.cache(g, pages, G, page)
    qkv = (torch.randn(T, (H + 2 * G) * D, generator=g) * std).to(torch.bfloat16)
    w = [(1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16) if norm else None for _ in range(2)]
    pos = torch.randint(0, 500, (T,), generator=g)
    return qkv, k, v, s, pos, torch.tensor(slots, dtype=torch.int64), ref.rope_cos_sin(512, D, 1e4), w


def check_append(qkv, k0, v0, s0, pos, slots, cs, w, H, G, k, v, s, q, rope=True):
    """A cache after an append and its q rows against 64 bits."""
    eq, ek, ev = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6, rope)
    page = k.shape[2]
    old = orc.codes(k0, v0)
    now, want, new = orc.append(old * s0.double()[..., None, None], s0, ek, ev, slots)
    assert torch.equal(s.cpu().double(), now)
    got = orc.codes(k, v) * now[..., None, None]
    # a code's half step: 2^-4 of the value, below the normal codes 2^-10 of the scale; old entries keep theirs
    # unless their scale grew; what enters the rounding is fp32 (norm and rotation: some steps of 2^-24 of the
    # row's largest entry, 2^-18 of it here)
    row = want.abs().amax(-1, keepdim=True).clamp_max(1e300)
    tol = torch.maximum(want.abs() * 2 ** -4, now[..., None, None] * 2.0 ** -10) + row * 2 ** -18
    assert bool(((got - want).abs() <= tol)[new].all())
    grown = (now > s0.double())[..., None, None].expand_as(got) & ~new
    same = ~grown & ~new
    begun = torch.zeros_like(new)
    for x in slots.tolist():
        if 0 <= x < k.shape[0] * page and x % page == 0:
            begun[:, x // page] = True
    untouched = same | (begun & ~new)
    assert torch.equal(orc.codes(k, v)[untouched], old[untouched])
    keep = grown & ~begun
    assert bool(((got - want).abs() <= now[..., None, None] * 2.0 ** -10)[keep].all())
    if q is not None:
        # half a bf16 step, and fp32's before it
        off = (q.cpu().double().view_as(eq) - eq).abs()
        assert bool((off <= eq.abs() * 2 ** -8 + eq.abs().amax(-1, keepdim=True) * 2 ** -18).all())


CASES = [
    # H, G, page, pages, slots, norm
    (4, 2, 32, 6, [70], True),                                   # one token inside a page
    (2, 1, 32, 6, [64], False),                                  # the token that begins a page
    (4, 2, 32, 8, list(range(40, 111)), True),                   # a chunk over four pages, begun and new
    (2, 2, 64, 5, [-1, 64, 65, 66, -1, 5, 200, 9999, 319], False),   # gaps, padding, a slot outside
    (3, 1, 96, 4, list(range(96, 288)) + [7, 8, 9], True),
]


@pytest.mark.parametrize("H,G,page,pages,slots,norm", CASES)
def test_append_against_64_bits(H, G, page, pages, slots, norm):
    qkv, k, v, s, pos, sl, cs, w = make(1, H, G, len(slots), slots, page, pages, norm, std=3.0)
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    q = torch.empty(len(slots), H, D, dtype=torch.bfloat16)
    ops.scaled_cache_append(qkv, q, k, v, s, pos, sl, cs, *w, H, G, 1e-6)
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, H, G, k, v, s, q)


def test_scale_borders():
    """448 times a power of two is held by it; the next number above needs the next power."""
    for e in (-90, -9, 0, 5, 60):
        x = torch.tensor([448.0 * 2.0 ** e, 449.0 * 2.0 ** e, 447.0 * 2.0 ** e, 256.0 * 2.0 ** e])
        assert torch.equal(ref.cache_scale(x), torch.tensor([1.0, 2.0, 1.0, 1.0]) * 2.0 ** e)
        assert [orc.need(float(t)) for t in x] == ref.cache_scale(x).tolist()
    assert ref.cache_scale(torch.tensor([0.0, 1e-38, 3e38])).tolist() == [2.0 ** -100, 2.0 ** -100, 2.0 ** 100]


def test_rows_that_are_not_finite():
    """Infinities become the largest number, NaN 0, neither counts towards the scale."""
    qkv, k, v, s, pos, sl, cs, w = make(3, 1, 1, 2, [32, 33], 32, 3, False)
    qkv[0, 2 * D] = math.inf
    qkv[0, 2 * D + 1] = -math.inf
    qkv[1, 2 * D + 2] = math.nan
    top = float(qkv[:, 2 * D:][torch.isfinite(qkv[:, 2 * D:])].abs().max())
    ops.scaled_cache_append(qkv, torch.empty(2, 1, D, dtype=torch.bfloat16), k, v, s, pos, sl, cs, *w, 1, 1, 1e-6)
    assert float(s[1, 1, 0]) == orc.need(top)
    got = orc.codes(k, v)[1, 1, 0]
    assert got[0, 0] == 448 and got[0, 1] == -448 and got[1, 2] == 0 and torch.isfinite(got).all()


def test_portions_give_the_scales_of_one_call():
    """A page filled in portions ends with the scale that one call gives it, and with the same entries but
    for codes that a larger scale made subnormal."""
    qkv, k, v, s, pos, sl, cs, w = make(5, 2, 1, 60, list(range(32, 92)), 32, 3, True)
    qkv *= torch.linspace(0.1, 6, 60)[:, None].to(qkv.dtype)
    q = torch.empty(60, 2, D, dtype=torch.bfloat16)
    one = [t.clone() for t in (k, v, s)]
    ops.scaled_cache_append(qkv, q, *one, pos, sl, cs, *w, 2, 1, 1e-6)
    at = 0
    for n in (1, 1, 5, 20, 33):
        r = slice(at, at + n)
        ops.scaled_cache_append(qkv[r], q[r], k, v, s, pos[r], sl[r], cs, *w, 2, 1, 1e-6)
        at += n
    assert torch.equal(s, one[2])
    a, b = orc.codes(k, v), orc.codes(*one[:2])
    # rounded twice: half a step of the first rounding (at most half the second's), half one of the second
    assert bool(((a - b).abs() <= 2.0 ** -9)[torch.minimum(a.abs(), b.abs()) < 2 ** -6].all())
    assert torch.equal(a[b.abs() >= 2 ** -5], b[b.abs() >= 2 ** -5])


def attention_case(seed, H, G, page, lens, new, extra=2, bad=None):
    """Rows of sequences over a full cache; bad: {(sequence, column): table entry}."""
    g = torch.Generator().manual_seed(seed)
    count = [-(-n // page) for n in lens]
    pages = sum(count) + extra
    k, v, s = orc.cache(g, pages, G, page)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables = torch.full((len(lens), max(count + [1]) + 1), int(order[-1]), dtype=torch.int32)   # (a spare page)
    at = 0
    for b, n in enumerate(count):
        tables[b, :n] = order[at:at + n]
        at += n
    for (b, i), x in (bad or {}).items():
        tables[b, i] = x
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    q = torch.randn(start[-1], H, D, generator=g).to(torch.bfloat16)
    return q, k, v, s, tables, torch.tensor(lens, dtype=torch.int32), start


def close(out, want, bound):
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def test_decode_against_64_bits():
    lens = [1, 0, 33, 200]
    q, k, v, s, t, n, start = attention_case(7, 4, 2, 32, lens, [1] * 4, bad={(3, 1): 99, (2, 1): -1})
    out = torch.empty_like(q)
    ops.scaled_attention_decode(out, q, k, v, s, t, n, 2, 0.1)
    close(out, *orc.attention(q, orc.codes(k, v) * s.double()[..., None, None], t, lens, start, 0.1))
    assert not out[1].any()


def test_decode_rows_that_q_start_names():
    lens, rows = [33, 0, 70], torch.tensor([4, 1, 0], dtype=torch.int32)
    q, k, v, s, t, n, start = attention_case(10, 4, 2, 32, lens, [1] * 3)
    many, out = torch.zeros(6, 4, D, dtype=torch.bfloat16), torch.full((6, 4, D), 9.0, dtype=torch.bfloat16)
    many[rows.long()] = q
    ops.scaled_attention_decode(out, many, k, v, s, t, n, 2, 0.1, q_start=rows)
    close(out[rows.long()], *orc.attention(q, orc.codes(k, v) * s.double()[..., None, None], t, lens, start, 0.1))
    assert bool((out[[2, 3, 5]] == 9).all())


def test_prompt_against_64_bits():
    lens, new = [40, 64, 5], [40, 3, 5]
    q, k, v, s, t, n, start = attention_case(8, 4, 2, 64, lens, new)
    out = torch.empty_like(q)
    st = torch.tensor(start, dtype=torch.int32)
    tiles = torch.tensor([0, 1, 2], dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    ops.scaled_attention_prefill(out, q, k, v, s, t, n, st, *tiles, 2, 0.1)
    close(out, *orc.attention(q, orc.codes(k, v) * s.double()[..., None, None], t, lens, start, 0.1))


def refused(fn, *a, **kw):
    with pytest.raises(RuntimeError):
        fn(*a, **kw)


def refusals(dev):
    """Calls that every form refuses, before anything runs."""
    q, k, v, s, t, n, start = (x.to(dev) if torch.is_tensor(x) else x
                               for x in attention_case(9, 4, 2, 32, [40, 50], [1, 1]))
    out = torch.empty_like(q)

    def decode(**kw):
        a = dict(out=out, q=q, k=k, v=v, s=s, t=t, n=n, g=2, scale=0.1, parts=1, size=512)
        a.update(kw)
        return lambda: ops.scaled_attention_decode(a["out"], a["q"], a["k"], a["v"], a["s"], a["t"], a["n"],
                                                   a["g"], a["scale"], num_parts=a["parts"], part_size=a["size"])

    decode()()
    for bad in (dict(k=k.view(torch.int8)), dict(s=s[:1]), dict(s=s.double()), dict(v=v[:-1]), dict(g=1),
                dict(t=t.long()), dict(t=t[:1]), dict(n=n.long()), dict(scale=0.0), dict(scale=-1.0),
                dict(parts=0), dict(size=100), dict(size=8320), dict(k=k.transpose(0, 1)),
                dict(s=s.transpose(0, 1).contiguous().transpose(0, 1))):
        refused(decode(**bad))
    st = torch.tensor(start, dtype=torch.int32, device=dev)
    tile = torch.zeros(1, dtype=torch.int32, device=dev)
    refused(ops.scaled_attention_prefill, out, q, k, v, s, t, n, st, tile, tile, 2, 0.1, tile_rows=100)
    refused(ops.scaled_attention_prefill, out, q, k, v, s, t, n, st, tile, tile, 3, 0.1)
    qkv = torch.zeros(2, 8 * D, dtype=torch.bfloat16, device=dev)
    pos, sl = torch.zeros(2, dtype=torch.int64, device=dev), torch.tensor([3, 40], device=dev)
    cs = ref.rope_cos_sin(64, D, 1e4).to(dev)

    def app(**kw):
        a = dict(qkv=qkv, k=k, v=v, s=s, pos=pos, sl=sl, H=4, G=2, nd=0, qr=-1)
        a.update(kw)
        return lambda: ops.scaled_cache_append(a["qkv"], out, a["k"], a["v"], a["s"], a["pos"], a["sl"], cs, None,
                                               None, a["H"], a["G"], 1e-6, num_decode=a["nd"], q_rows=a["qr"])

    app()()
    for bad in (dict(G=1), dict(H=6), dict(nd=3), dict(qr=3), dict(qr=-2), dict(pos=pos.int()), dict(sl=sl.int()),
                dict(sl=sl[:1]), dict(pos=pos[:1]), dict(s=s[:, :1]), dict(v=v.view(torch.int8))):
        refused(app(**bad))
    # no kv heads
    refused(app(k=k[:, :0], v=v[:, :0], s=s[:, :, :0], H=8, G=0))
    # no blocks of 48 tokens
    refused(app(k=torch.zeros(2, 2, 48, D, dtype=torch.uint8, device=dev),
                v=torch.zeros(2, 2, 6, D, 8, dtype=torch.uint8, device=dev), s=torch.ones(2, 2, 2, device=dev)))


def test_refusals():
    refusals("cpu")


def test_rows_of_a_block_apart_are_refused():
    qkv, k, v, s, pos, sl, cs, w = make(11, 1, 1, 3, [1, 40, 2], 32, 3, False)
    q = torch.empty(3, 1, D, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="apart"):
        ops.scaled_cache_append(qkv, q, k, v, s, pos, sl, cs, *w, 1, 1, 1e-6)
    ops.check_scaled_slots(torch.tensor([-1, 30, 31, 32, -1, 64]), 32)
    for slots in ([5, 5], [6, 5], [5, 7], [5, -1, 6]):
        with pytest.raises(RuntimeError):
            ops.check_scaled_slots(torch.tensor(slots), 32)


def test_rows_outside_the_cache_are_in_no_block():
    """Two rows at one slot behind the cache, and rows apart of a block behind it: no entries, and no refusal."""
    slots = [9999, 40, 41, 9999, 10000, 9998, -5]
    qkv, k, v, s, pos, sl, cs, w = make(12, 2, 1, len(slots), slots, 32, 3, True)
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    q = torch.empty(len(slots), 2, D, dtype=torch.bfloat16)
    ops.scaled_cache_append(qkv, q, k, v, s, pos, sl, cs, *w, 2, 1, 1e-6)
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, 2, 1, k, v, s, q)
    ops.check_scaled_slots(sl, 32, 3)
    for bad in ([40, 9999, 41], [40, 40]):
        with pytest.raises(RuntimeError, match="apart"):
            ops.check_scaled_slots(torch.tensor(bad), 32, 3)


@pytest.mark.parametrize("capturing", [False, True])
def test_slots_are_not_checked_while_a_graph_is_captured(monkeypatch, capturing):
    """With AKAP_DEBUG_CHECKS=1 a GPU call copies its slots to the host, which a capture does not survive."""
    from types import SimpleNamespace as NS

    ran, checked = [], []
    monkeypatch.setattr(ops, "DEBUG_CHECKS", True)
    monkeypatch.setattr(ops, "_native", lambda x: True)
    monkeypatch.setattr(ops, "check_scaled_slots", lambda *a: checked.append(a[1:]))
    monkeypatch.setattr(ops, "torch", NS(cuda=NS(is_current_stream_capturing=lambda: capturing),
                                         ops=NS(akap=NS(scaled_cache_append=lambda *a: ran.append(a)))))
    qkv, k, v, s, pos, sl, cs, w = make(13, 1, 1, 2, [1, 2], 32, 3, False)
    ops.scaled_cache_append(qkv, qkv, k, v, s, pos, sl, cs, None, None, 1, 1, 1e-6)
    assert len(ran) == 1 and checked == ([] if capturing else [(32, 3)])


# ------------------------------------------------------------------------------------------------ engine
def test_engine_on_a_scaled_cache():
    """--kv-cache-dtype fp8_scaled: greedy tokens near the argmax of the dense reference, also where keys are far
    beyond the largest code."""
    from test_engine_cpu import _engine, _near_argmax
    from aws_k8s_ansible_provisioner_amd.engine.config import SamplingParams

    eng = _engine("tiny-qwen3", kv_cache_dtype="fp8_scaled")
    assert eng.runner.kv.dtype == torch.uint8 and len(eng.runner.kv_scales) == eng.runner.mcfg.num_layers
    prompts = [list(range(5, 45)), [7, 8, 9] * 14]
    outs = eng.generate(None, SamplingParams(max_tokens=8, temperature=0, ignore_eos=True), prompt_ids=prompts)
    for p, o in zip(prompts, outs):
        _near_argmax(eng, p, o.output_ids, tol=0.5)
    for s in eng.runner.kv_scales:
        assert bool((s > 2.0 ** -100).any()) and bool((torch.frexp(s)[0] == 0.5).all())


def test_engine_plans_prompts_by_their_longest_sequence(monkeypatch):
    """Not by what the block tables could hold."""
    from test_engine_cpu import _engine
    from aws_k8s_ansible_provisioner_amd.engine.config import SamplingParams

    seen, real = set(), ops.scaled_attention_prefill

    def record(out, q, k, v, s, tables, lens, *a, max_len=None, **kw):
        seen.add((int(lens.max()), max_len, tables.shape[1] * k.shape[2]))
        return real(out, q, k, v, s, tables, lens, *a, max_len=max_len, **kw)

    monkeypatch.setattr(ops, "scaled_attention_prefill", record)
    eng = _engine("tiny-qwen3", kv_cache_dtype="fp8_scaled")
    eng.generate(None, SamplingParams(max_tokens=2, temperature=0, ignore_eos=True),
                 prompt_ids=[list(range(5, 45)), [7, 8, 9] * 14])
    assert seen and all(longest == said < room for longest, said, room in seen)


def test_prompt_plans():
    for rows in (128, 256):
        for tiles in (1, 7, 64, 500, 5000):
            for n in (1, 500, 1000, 5000, 100000):
                waves, parts = ops.scaled_prefill_plan(tiles, rows, n)
                assert waves in (4, 8) and 32 * waves <= rows and 1 <= parts <= 16
                assert parts == 1 or n >= 896


def test_engine_refuses_roles_and_blocks():
    from aws_k8s_ansible_provisioner_amd.engine.config import EngineConfig

    for kw in (dict(kv_role="prefill"), dict(kv_role="decode"), dict(block_size=8192 + 32),
               dict(block_size=96 * 32 + 32)):
        with pytest.raises(ValueError):
            EngineConfig(kv_cache_dtype="fp8_scaled", **kw)
    EngineConfig(kv_cache_dtype="fp8_scaled", block_size=96)
    with pytest.raises(ValueError):
        EngineConfig(kv_cache_dtype="fp8_other")
