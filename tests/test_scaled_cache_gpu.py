"""The scaled 8-bit cache's kernels against 64 bits (scaled_cache_oracle), at the sizes and masks where they can
go wrong."""
import math

import pytest
import torch

import scaled_cache_oracle as orc
from aws_k8s_ansible_provisioner_amd import ops
from aws_k8s_ansible_provisioner_amd.ops import reference as ref
from test_scaled_cache import CASES, D, attention_case, check_append, close, make, refusals

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gpu(*xs):
    return [x.to(DEV) if torch.is_tensor(x) else x for x in xs]


def tiles(lens, new, G, rows):
    """The tile map as the scheduler makes it: ascending by work."""
    t = [(lens[b] - n + min(n, (r + rows + G - 1) // G), b, r) for b, n in enumerate(new)
         for r in range(0, n * G, rows)]
    t.sort(key=lambda x: x[0])
    return [torch.tensor([x[i] for x in t], dtype=torch.int32, device=DEV) for i in (1, 2)]


# ------------------------------------------------------------------------------------------------ append
def run_append(case, H, G, slots, decode=False, num_decode=0, q_rows=-1, rope=True):
    qkv, k, v, s, pos, sl, cs, w = case
    k1, v1, s1 = gpu(k.clone(), v.clone(), s.clone())
    q = torch.full((len(slots), H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(*gpu(qkv), q, k1, v1, s1, *gpu(pos, sl, cs, *w), H, G, 1e-6, rope, decode=decode,
                            num_decode=num_decode, q_rows=q_rows)
    torch.cuda.synchronize()
    return k1, v1, s1, q


@pytest.mark.parametrize("H,G,page,pages,slots,norm", CASES + [
    (16, 8, 32, 300, [33 * i + 5 for i in range(200)], True),            # decode rows, a page each
    (32, 8, 32, 40, list(range(11, 700)), False),
    (8, 4, 128, 9, list(range(130, 500)) + [1000], True),                # pages longer than a wave's rows
    (5, 1, 32, 3, [], True),
    (0, 2, 32, 4, [31, 32, 33], False),                                  # no query heads
    (2, 2, 32, 60, [32 * i + i % 29 + j for i in range(50) for j in range(3)], True),   # many short runs
    (2, 1, 32, 12, list(range(20, 43)) + list(range(90, 101)) + list(range(128, 130)), True),   # three in a span
    (2, 2, 64, 9, list(range(7, 64)) + list(range(130, 192)) + list(range(320, 384)), False),
    (1, 1, 256, 4, list(range(300, 700)), True),
    (8, 8, 32, 60, [i for b in range(7) for i in range(200 * b + 5, 200 * b + 5 + 85)], True),   # spans of 16 rows
    (8, 8, 32, 110, list(range(40, 2700)), False),                                               # of 32
    (2, 1, 64, 40, [64 * i + 60 - i % 3 + j for i in range(30) for j in range(1 + i % 4)], True),  # short runs, late
])
def test_append(H, G, page, pages, slots, norm):
    case = make(21, H, G, len(slots), slots, page, pages, norm, std=3.0)
    qkv, k, v, s, pos, sl, cs, w = case
    ops.check_scaled_slots(sl, page)
    for decode in (False, True):
        k1, v1, s1, q = run_append(case, H, G, slots, decode)
        check_append(qkv, k, v, s, pos, sl, cs, w, H, G, k1, v1, s1, q if H and slots else None)
    # values pass through no arithmetic before their rounding: the plain form's codes
    if slots:
        ref.scaled_cache_append(qkv, q.cpu(), k, v, s, pos, sl, cs, *w, H, G, 1e-6)
        assert torch.equal(v1.cpu(), v)


def test_append_some_query_rows_and_no_rotation():
    case = make(22, 4, 2, 50, list(range(20, 70)), 32, 5, True)
    qkv, k, v, s, pos, sl, cs, w = case
    k1, v1, s1, q = run_append(case, 4, 2, range(50), num_decode=1, q_rows=3, rope=False)
    check_append(qkv, k, v, s, pos, sl, cs, w, 4, 2, k1, v1, s1, None, rope=False)
    eq = orc.prepared(qkv, pos, cs, *w, 4, 2, 1e-6, False)[0]
    assert bool(((q[:3].cpu().double() - eq[:3]).abs() <= eq[:3].abs() * 2 ** -8 + 2 ** -16).all())
    assert bool((q[3:] == 7).all())


def test_append_rows_whose_squares_overflow():
    """The norm of such a row is infinite, its entries zeros; rows of zeros stay zeros."""
    qkv, k, v, s, pos, sl, cs, w = make(24, 2, 1, 3, [8, 9, 10], 32, 2, True)
    qkv[0, :3 * D] = 2.0 ** 100
    qkv[1, :3 * D] = 0
    k1, v1, s1, q = run_append((qkv, k, v, s, pos, sl, cs, w), 2, 1, range(3))
    assert not q[:2].any() and torch.isfinite(q[2].float()).all()
    assert not orc.codes(k1, v1)[0, 0, 0, 8:10].any()


def test_append_rounds_as_whole_tensors_do():
    """Norm and rotation by torch's operations in fp32 on the GPU, each rounded by itself: the same query rows and the
    same codes, but for what another order of the sum of squares could move: a few units of 2^-24 against a bf16 step of 2^-8
    or more, less than one entry in 10000."""
    T, H, G = 640, 8, 2
    qkv, k, v, s, pos, sl, cs, w = gpu(*make(25, H, G, T, list(range(T)), 32, T // 32, True)[:7], None)
    w = [torch.randn(D, device=DEV).bfloat16() for _ in range(2)]
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(qkv, q, k, v, s, pos, sl, cs, *w, H, G, 1e-6)
    x = qkv.float()[:, :(H + 2 * G) * D].view(T, -1, D)
    a = cs[pos][:, None]

    def turned(y, u):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * u.float()
        lo, hi = y[..., :64], y[..., 64:]
        return torch.cat([lo * a[..., :64] - hi * a[..., 64:], hi * a[..., :64] + lo * a[..., 64:]], -1)

    assert int((turned(x[:, :H], w[0]).bfloat16() != q).sum()) <= q.numel() // 10000
    want = turned(x[:, H:H + G], w[1])
    got = orc.codes(k.cpu(), v.cpu())[0].transpose(1, 2).reshape(T, G, D)
    scale = s[0].repeat_interleave(32, 0)[:, :, None]
    codes = (want / scale).clamp(-448, 448).to(torch.float8_e4m3fn).double().cpu()
    assert int((codes != got).sum()) <= got.numel() // 10000


def test_append_rows_that_are_not_finite():
    case = make(23, 2, 1, 5, [60, 61, 62, 63, 64], 32, 4, False)
    qkv = case[0]
    qkv[0, 2 * D:2 * D + 3] = torch.tensor([math.inf, -math.inf, math.nan])      # keys
    qkv[3, 3 * D] = math.nan                                                     # a value
    qkv[4, 3 * D:] = math.inf                                                    # a page's values, all of them
    k1, v1, s1, _ = run_append(case, 2, 1, range(5), rope=False)
    got = orc.codes(k1, v1)
    assert torch.isfinite(got).all()
    assert got[0, 1, 0, 28, :3].tolist() == [448, -448, 0]
    assert got[1, 1, 0, 31, 0] == 0
    assert float(s1[1, 2, 0]) == 2.0 ** -100 and bool((got[1, 2, 0, 0] == 448).all())
    # what the rows' pages held may be no number either
    case[2].fill_(0x7f)
    k1, v1, s1, _ = run_append(case, 2, 1, range(5), rope=False)
    assert float(s1[1, 1, 0]) >= 2.0 ** -100


def test_append_rows_outside_the_cache(monkeypatch):
    """They are in no block, also for the check of a call's slots."""
    slots = [9999, 40, 41, 9999, 10000, 9998, -5]
    case = make(26, 2, 1, len(slots), slots, 32, 3, True)
    qkv, k, v, s, pos, sl, cs, w = case
    monkeypatch.setattr(ops, "DEBUG_CHECKS", True)
    for decode in (False, True):
        k1, v1, s1, q = run_append(case, 2, 1, slots, decode)
        check_append(qkv, k, v, s, pos, sl, cs, w, 2, 1, k1, v1, s1, q)


def test_append_takes_wide_rows_and_views():
    qkv, k, v, s, pos, sl, cs, w = make(24, 4, 2, 40, list(range(64, 104)), 32, 6, True)
    wide = torch.zeros(40, 8 * D + 64, dtype=torch.bfloat16, device=DEV)
    wide[:, :8 * D] = qkv.to(DEV)
    k1, v1, s1 = gpu(k.clone(), v.clone(), s.clone())
    q = torch.empty(40, 4, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(wide, q, k1, v1, s1, *gpu(pos, sl, cs, *w), 4, 2, 1e-6)
    check_append(qkv, k, v, s, pos, sl, cs, w, 4, 2, k1, v1, s1, q)
    with pytest.raises(RuntimeError):
        ops.scaled_cache_append(wide[:, 1:], q, k1, v1, s1, *gpu(pos, sl, cs, *w), 4, 2, 1e-6)
    with pytest.raises(RuntimeError):
        ops.scaled_cache_append(wide, q.cpu(), k1, v1, s1, *gpu(pos, sl, cs, *w), 4, 2, 1e-6)


def test_refusals_gpu():
    refusals(DEV)


def test_rows_beyond_a_launch_are_refused():
    """As many rows as a grid cannot hold: one row, seen 2^26 times."""
    n = 1 << 26
    k, v = (torch.zeros(*shape, dtype=torch.uint8, device=DEV) for shape in ((1, 1, 32, D), (1, 1, 4, D, 8)))
    s = ops.scaled_cache_scales(1, 1, 1, DEV)[0]
    qkv = torch.zeros(1, 3 * D, dtype=torch.bfloat16, device=DEV).expand(n, -1)
    at, cs = torch.full((n,), -1, device=DEV), torch.zeros(4, D, device=DEV)
    q = torch.empty(0, 1, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="too many rows"):
        ops.scaled_cache_append(qkv, q, k, v, s, at, at, cs, None, None, 1, 1, 1e-6, decode=True, q_rows=0)


# ------------------------------------------------------------------------------------------------ decode
def run_decode(c, lens, H, G, parts=1, size=1024, scale=0.1, workspace=None):
    q, k, v, s, t, n, start = gpu(*c)
    out = torch.full_like(q, 9.0)
    ops.scaled_attention_decode(out, q, k, v, s, t, n, H // G, scale, workspace=workspace, num_parts=parts,
                                part_size=size)
    torch.cuda.synchronize()
    return out


def want_rows(c, lens, scale=0.1):
    q, k, v, s, t, n, start = c
    return orc.attention(q, orc.codes(k, v) * s.double()[..., None, None], t, lens, start, scale)


@pytest.mark.parametrize("H,G,page,lens,parts,size", [
    (2, 2, 32, [1], 1, 128),
    (4, 2, 32, [31, 32, 33, 0, 63, 64, 65, 127, 128, 129], 1, 512),
    (16, 1, 64, [1000, 70, 5], 8, 128),
    (5, 1, 96, [97, 400, 0, 383, 384, 385], 2, 384),
    (8, 8, 32, [700, 1], 3, 256),
    (12, 4, 32, [0, 0], 2, 128),
    (16, 1, 32, [2100, 3, 1025], 9, 256),                 # merges of one, two, .. groups of threads
    (3, 1, 32, [2100, 3, 1025], 9, 256),
    (2, 2, 32, [3000, 513], 24, 128),
    (16, 2, 32, [700, 40] * 140, 6, 128),                 # rows that fill the card
    (4, 4, 64, [9000], 128, 128),
    (14, 1, 32, [1000, 400, 0, 33, 520, 1700], 4, 512),    # eight waves, and their merge
    (1, 1, 32, [5000, 513, 257], 10, 512),
    (4, 2, 96, [385, 1, 255, 512, 129], 1, 512),
    (16, 1, 32, [1000, 400, 0, 33], 2, 512),               # too many query heads for eight
    (16, 8, 32, [300, 700] * 20, 1, 1024),                 # too many rows
])
def test_decode(H, G, page, lens, parts, size):
    c = attention_case(31, H, G, page, lens, [1] * len(lens))
    want = want_rows(c, lens)
    close(run_decode(c, lens, H, G, parts, size), *want)
    if parts > 1:
        ws = ops.decode_workspace(len(lens), G, H // G, parts, DEV)
        for _ in range(3):      # its tickets serve one step after the other
            close(run_decode(c, lens, H, G, parts, size, workspace=ws), *want)


# As long as a partition may be: 64 chunks to each of four waves (more query heads than eight take, or more rows), 32 to
# each of eight.  A sum of 64 chunks takes 8 additions in each, a product's row 32: 2^-13 of the weights' sum of
# magnitudes beside the 2^-8 of `bound`'s roundings.
LONG = 1 + 2 ** -4


@pytest.mark.parametrize("H,G,page,lens,parts,size", [
    (16, 1, 32, [8192, 8191, 8161, 8160, 4097, 65], 1, 8192),
    (2, 2, 32, [8192, 8191, 8161, 4097, 33, 0], 1, 8192),
    (16, 1, 96, [8064, 8063, 7969, 7968, 4033], 1, 8064),
    (2, 1, 96, [8064, 8063, 7969, 4033], 1, 8064),
    (16, 1, 32, [8193, 16384, 8192, 16383, 8224, 100], 2, 8192),
    (4, 2, 32, [8193, 16384, 8192, 8225], 2, 8192),
])
def test_decode_of_whole_partitions(H, G, page, lens, parts, size):
    c = attention_case(36, H, G, page, lens, [1] * len(lens))
    want, bound = want_rows(c, lens)
    close(run_decode(c, lens, H, G, parts, size), want, bound * LONG)
    if parts > 1:
        ws = ops.decode_workspace(len(lens), G, H // G, parts, DEV)
        close(run_decode(c, lens, H, G, parts, size, workspace=ws), want, bound * LONG)


def test_decode_beside_codes_that_are_no_numbers():
    """What stands behind a sequence's end, and in other pages, is never seen."""
    lens = [45, 300]
    c = attention_case(32, 4, 2, 32, lens, [1, 1])
    want = want_rows(c, lens)
    q, k, v, s, t, n, start = c
    ki, vi = orc.k_index(32), orc.v_index(32)
    for b, m in enumerate(lens):
        blk = int(t[b, m // 32])
        k.view(-1, 2, 32 * D)[blk][:, ki[m % 32:].reshape(-1)] = 0x7f
        v.view(-1, 2, 32 * D)[blk][:, vi[m % 32:].reshape(-1)] = 0xff
    k[int(t[0, -1])] = 0x7f
    v[int(t[0, -1])] = 0x7f
    for parts in (1, 3):
        close(run_decode(c, lens, 4, 2, parts, 128 * (4 - parts)), *want)


@pytest.mark.parametrize("parts", [1, 2])
def test_decode_pages_outside_the_cache(parts):
    lens = [100, 64, 20]
    c = attention_case(33, 4, 2, 32, lens, [1] * 3, bad={(0, 1): 1 << 30, (1, 0): -1, (1, 1): 10000, (2, 0): -7})
    out = run_decode(c, lens, 4, 2, parts, 128)
    close(out, *want_rows(c, lens))
    assert not out[1].any() and not out[2].any()


def test_decode_lengths_past_the_table():
    lens = [5000, 40]
    c = attention_case(34, 2, 1, 32, [90, 40], [1, 1])
    c = (*c[:5], torch.tensor(lens, dtype=torch.int32), c[6])
    close(run_decode(c, lens, 2, 1), *want_rows(c, lens))


def test_decode_extreme_scores():
    """Scores of some thousands: the maximum keeps the sums finite."""
    lens = [130, 300]
    c = attention_case(35, 4, 1, 32, lens, [1, 1])
    c = (c[0] * 40, *c[1:])
    close(run_decode(c, lens, 4, 1, 2, 256, scale=2.0), *want_rows(c, lens, 2.0))


# ------------------------------------------------------------------------------------------------ prompts
def run_prompt(c, lens, new, H, G, rows, scale=0.1, max_len=None):
    q, k, v, s, t, n, start = gpu(*c)
    out = torch.full_like(q, 9.0)
    st = torch.tensor(start, dtype=torch.int32, device=DEV)
    ops.scaled_attention_prefill(out, q, k, v, s, t, n, st, *tiles(lens, new, H // G, rows), H // G, scale,
                                 tile_rows=rows, max_len=max_len)
    torch.cuda.synchronize()
    return out


# (rows of a tile, the bound on the keys that the host states: it alone chooses waves and parts)
FORMS = [(128, None), (128, 100000), (256, None), (256, 2000), (256, 100000)]


def test_prompt_forms():
    """What FORMS stand for, for few tiles."""
    assert [ops.scaled_prefill_plan(4, r, n) for r, n in ((128, 500), (128, 100000), (256, 500), (256, 2000),
                                                          (256, 100000))] == \
        [(4, 1), (4, 16), (4, 1), (4, 4), (8, 16)]
    assert ops.scaled_prefill_plan(4096, 256, 2048) == (8, 1) and ops.scaled_prefill_plan(64, 256, 10016) == (8, 4)


@pytest.mark.parametrize("rows,max_len", FORMS)
@pytest.mark.parametrize("H,G,page,lens,new", [
    (1, 1, 32, [1], [1]),
    (4, 2, 32, [63, 64, 65, 1], [63, 64, 65, 1]),
    (16, 2, 64, [300, 129, 77], [300, 40, 1]),
    (5, 1, 96, [200, 97], [130, 97]),
    (8, 8, 32, [700], [260]),
    (20, 1, 32, [50, 2000], [50, 9]),
    (2, 1, 32, [2500, 1100, 257], [3, 200, 257]),
    (3, 1, 64, [511, 512, 513, 0], [2, 512, 1, 0]),
])
def test_prompts(H, G, page, lens, new, rows, max_len):
    c = attention_case(41, H, G, page, lens, new)
    close(run_prompt(c, lens, new, H, G, rows, max_len=max_len), *want_rows(c, lens))


def test_prompts_extreme_scores():
    """Scores of some thousands, rising along the keys: every tile moves the maximum."""
    lens, new = [700], [300]
    c = attention_case(45, 2, 1, 32, lens, new)
    c = (c[0] * 40, *c[1:])
    for rows, max_len in FORMS:
        close(run_prompt(c, lens, new, 2, 1, rows, 2.0, max_len), *want_rows(c, lens, 2.0))


@pytest.mark.parametrize("rows,max_len", FORMS)
def test_prompts_beside_codes_that_are_no_numbers(rows, max_len):
    lens, new = [45, 330], [45, 70]
    c = attention_case(42, 4, 2, 32, lens, new)
    want = want_rows(c, lens)
    q, k, v, s, t, n, start = c
    ki, vi = orc.k_index(32), orc.v_index(32)
    for b, m in enumerate(lens):
        blk = int(t[b, m // 32])
        k.view(-1, 2, 32 * D)[blk][:, ki[m % 32:].reshape(-1)] = 0x7f
        v.view(-1, 2, 32 * D)[blk][:, vi[m % 32:].reshape(-1)] = 0xff
    close(run_prompt(c, lens, new, 4, 2, rows, max_len=max_len), *want)


@pytest.mark.parametrize("rows,max_len", FORMS)
def test_prompts_pages_outside_the_cache(rows, max_len):
    lens, new = [200, 33], [150, 33]
    c = attention_case(43, 4, 2, 32, lens, new, bad={(0, 0): -1, (0, 3): 1 << 29, (0, 6): -5, (1, 0): 77777})
    out = run_prompt(c, lens, new, 4, 2, rows, max_len=max_len)
    close(out, *want_rows(c, lens))


@pytest.mark.parametrize("rows,max_len", FORMS)
def test_prompts_of_no_visible_keys(rows, max_len):
    """All pages outside the cache, or no length at all: rows of zeros."""
    lens, new = [300, 40], [100, 40]
    c = attention_case(46, 4, 2, 32, lens, new, bad={(0, i): -1 for i in range(10)})
    q, k, v, s, t, n, start = c
    n = torch.tensor([300, 0], dtype=torch.int32)
    out = run_prompt((q, k, v, s, t, n, start), [300, 40], new, 4, 2, rows, max_len=max_len)
    assert not out.any()


@pytest.mark.parametrize("waves,parts", [(4, 1), (8, 1), (4, 2), (8, 3)])
@pytest.mark.parametrize("page", [32, 96])
def test_prompts_of_many_key_tiles(waves, parts, page, monkeypatch):
    """More tiles of 64 keys in a part than the pages a wave looks up at once, even and odd ones."""
    lens, new = [4500, 2113, 33, 1985], [3, 70, 33, 1]
    c = attention_case(46, 2, 1, page, lens, new)
    monkeypatch.setattr(ops, "scaled_prefill_plan", lambda *a: (waves, parts))
    close(run_prompt(c, lens, new, 2, 1, 32 * waves), *want_rows(c, lens))


def test_prompts_leave_other_rows():
    """Sequences that no tile names (a mixed step's single tokens) keep their rows."""
    lens, new = [40, 100, 64], [1, 60, 64]
    c = attention_case(44, 4, 2, 32, lens, new)
    q, k, v, s, t, n, start = gpu(*c)
    out = torch.full_like(q, 9.0)
    ts, tr = tiles(lens, new, 2, 128)
    ts, tr = ts[ts != 0], tr[ts != 0]
    ops.scaled_attention_prefill(out, q, k, v, s, t, n, torch.tensor(start, dtype=torch.int32, device=DEV), ts, tr,
                                 2, 0.1)
    want, bound = want_rows(c, lens)
    close(out[1:], want[1:], bound[1:])
    assert bool((out[0] == 9).all())


# ------------------------------------------------------------------------------------------------ together
def step_case(seed, H, G, page, past, norm, room=0):
    """Decode rows of sequences with past[b] cached keys each, and pages for `room` tokens more: everything a
    step is called with."""
    lens = [p + 1 for p in past]
    q, k, v, s, t, n, start = attention_case(seed, H, G, page, [m + room for m in lens], [1] * len(lens))
    n = n - room
    slots = [int(t[b, p // page]) * page + p % page for b, p in enumerate(past)]
    qkv, _, _, _, _, sl, cs, w = make(seed + 1, H, G, len(lens), slots, page, 2, norm, std=2.0)
    pos = torch.tensor(past, dtype=torch.int64)
    return lens, qkv, k, v, s, t, n, pos, sl, ref.rope_cos_sin(max(lens), D, 1e4), w


@pytest.mark.parametrize("H,G,page,past,norm,parts,size", [
    (16, 8, 32, [0, 31, 32, 33, 95, 300], True, 1, 512),
    (4, 1, 64, [0, 63, 64, 127, 128, 500], False, 4, 128),
    (14, 1, 32, [700, 5], True, 3, 256),
    (5, 1, 96, [383, 384, 10], True, 2, 384),
    (4, 2, 256, [700, 255, 256, 300, 513], False, 4, 256),
    (15, 1, 32, [40, 64], True, 1, 128),                  # more query heads than one launch takes
    (14, 1, 32, [700, 5, 1500, 511, 512], True, 4, 512),
    (4, 2, 64, [1023, 511, 512, 513, 40], False, 2, 1024),
    (8, 8, 32, [280 + 7 * i for i in range(40)], True, 1, 1024),
])
def test_fused_step(H, G, page, past, norm, parts, size):
    lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(51, H, G, page, past, norm)
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    k1, v1, s1 = gpu(k, v, s)
    out = torch.empty(len(past), H, D, dtype=torch.bfloat16, device=DEV)
    ws = ops.decode_workspace(len(past), G, H // G, parts, DEV)
    ops.scaled_attention_decode_fused(out, *gpu(qkv), k1, v1, s1, *gpu(t, n, pos, sl, cs, *w), H // G, 0.1, 1e-6,
                                      workspace=ws, num_parts=parts, part_size=size)
    torch.cuda.synchronize()
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, H, G, k1, v1, s1, None)
    # attention over the codes as they are now; q is rounded to bf16 from fp32, so it may be the neighbour of the
    # rounded 64-bit one: both are allowed for by half a step more in every product
    q = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
    entries = orc.codes(k1, v1) * s1.cpu().double()[..., None, None]
    start = list(range(len(past) + 1))
    want, bound = orc.attention(q, entries, t, lens, start, 0.1)
    close(out, want, bound + q_bound(q, entries, t, lens, start, 0.1))


@pytest.mark.parametrize("size", [256, 512])            # four waves, eight
@pytest.mark.parametrize("page", [32, 64, 256])
def test_fused_step_where_the_scale_grows(page, size):
    """Every row's key and value are far louder than their page: its codes are rounded anew before they are read,
    whichever chunk of the page a wave holds already."""
    H, G = 4, 2
    past = [1, 31, 33, 63, 65, 100, 127, 129, 191, 255]
    lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(55, H, G, page, past, False)
    qkv[:, H * D:] *= 4096
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    k1, v1, s1 = gpu(k, v, s)
    out = torch.empty(len(past), H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_attention_decode_fused(out, *gpu(qkv), k1, v1, s1, *gpu(t, n, pos, sl, cs, *w), H // G, 1e-5, 1e-6,
                                      part_size=size)
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, H, G, k1, v1, s1, None)
    assert bool((s1.cpu()[:, sl // page] > s0[:, sl // page]).all())
    q = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
    entries = orc.codes(k1, v1) * s1.cpu().double()[..., None, None]
    start = list(range(len(past) + 1))
    want, bound = orc.attention(q, entries, t, lens, start, 1e-5)
    close(out, want, bound + q_bound(q, entries, t, lens, start, 1e-5))


@pytest.mark.parametrize("page,size,parts,past", [
    (32, 8192, 1, [8191, 8190, 8160, 8159, 4096]),
    (96, 8064, 1, [8063, 8062, 7968, 4032]),
    (32, 8192, 2, [8192, 16383, 8191, 16350, 8223]),
    (256, 8192, 1, [8191, 8160, 7937, 8000]),
])
@pytest.mark.parametrize("others", [0, 130])             # eight waves, and four
@pytest.mark.parametrize("loud", [1, 4096])              # (4096: each row's last page is rounded anew)
def test_fused_step_of_whole_partitions(page, size, parts, past, others, loud):
    H, G, scale = 4, 2, 0.1 / loud
    past = past + [i % 70 for i in range(others)]
    lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(58, H, G, page, past, False)
    qkv[:, H * D:] *= loud
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    k1, v1, s1 = gpu(k, v, s)
    out = torch.empty(len(past), H, D, dtype=torch.bfloat16, device=DEV)
    ws = ops.decode_workspace(len(past), G, H // G, parts, DEV)
    ops.scaled_attention_decode_fused(out, *gpu(qkv), k1, v1, s1, *gpu(t, n, pos, sl, cs, *w), H // G, scale, 1e-6,
                                      workspace=ws, num_parts=parts, part_size=size)
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, H, G, k1, v1, s1, None)
    q = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
    entries = orc.codes(k1, v1) * s1.cpu().double()[..., None, None]
    start = list(range(len(past) + 1))
    want, bound = orc.attention(q, entries, t, lens, start, scale)
    close(out, want, bound * LONG + q_bound(q, entries, t, lens, start, scale))


def test_fused_step_of_padding():
    """Rows without a slot append nothing, rows of no keys nothing either and are zero."""
    H, G, page = 8, 2, 32
    past = [40, 40, 40]
    lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(57, H, G, page, past, True)
    sl = torch.tensor([-1, 10 ** 9, int(sl[2])])
    n = torch.tensor([41, 41, 0], dtype=torch.int32)
    k1, v1, s1 = gpu(k.clone(), v.clone(), s.clone())
    out = torch.full((3, H, D), 5.0, dtype=torch.bfloat16, device=DEV)
    for parts, size in ((1, 512), (3, 128)):
        ws = ops.decode_workspace(3, G, H // G, parts, DEV)
        ops.scaled_attention_decode_fused(out, *gpu(qkv), k1, v1, s1, *gpu(t, n, pos, sl, cs, *w), H // G, 0.1,
                                          1e-6, workspace=ws, num_parts=parts, part_size=size)
        torch.cuda.synchronize()
        for a, b in ((k1, k), (v1, v), (s1, s)):
            assert torch.equal(a.cpu(), b)
        assert not out[2].any()
        q = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
        entries = orc.codes(k, v) * s.double()[..., None, None]
        want, bound = orc.attention(q[:2], entries, t, [41, 41], [0, 1, 2], 0.1)
        close(out[:2], want, bound + q_bound(q[:2], entries, t, [41, 41], [0, 1, 2], 0.1))


def test_empty_batches():
    q, k, v, s, t, n, start = gpu(*attention_case(58, 4, 2, 32, [40], [1]))
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    ops.scaled_attention_decode(q[:0], q[:0], k, v, s, t, n[:0], 2, 0.1)
    ops.scaled_attention_prefill(q[:0], q[:0], k, v, s, t, n[:0], n[:1], none, none, 2, 0.1)
    long = torch.empty(0, dtype=torch.int64, device=DEV)
    ops.scaled_attention_decode_fused(q[:0], torch.empty(0, 8 * D, dtype=torch.bfloat16, device=DEV), k, v, s, t,
                                      n[:0], long, long, ref.rope_cos_sin(16, D, 1e4).to(DEV), None, None, 2, 0.1,
                                      1e-6)
    torch.cuda.synchronize()


def q_bound(q, entries, t, lens, start, scale):
    """What rounding q to bf16 (half a step, 2^-8) can change: each score by 2^-8 sum |q k| scale =: d, each
    weight by a factor between e^-2d and e^2d."""
    off = torch.zeros_like(q)
    H, page = q.shape[1], entries.shape[3]
    for b, n in enumerate(lens):
        r = slice(start[b], start[b + 1])
        blks = t[b, :-(-n // page)].long()
        for h in range(H):
            kk, vv = (entries[j, blks, h * entries.shape[2] // H].reshape(-1, D)[:n] for j in (0, 1))
            rows = torch.arange(n - (start[b + 1] - start[b]), n)[:, None]
            seen = torch.arange(n)[None] <= rows
            z = (q[r, h] @ kk.T * scale).masked_fill(~seen, -math.inf)
            d = (q[r, h].abs() @ kk.abs().T * scale * 2 ** -8).masked_fill(~seen, 0).amax(-1, keepdim=True)
            off[r, h] = torch.softmax(z, -1) @ vv.abs() * torch.expm1(2 * d)
    return off


@pytest.mark.parametrize("rows,max_len", FORMS)
@pytest.mark.parametrize("norm", [True, False])
def test_prompt_step_prepares_its_queries(rows, max_len, norm):
    """A step of chunks: append without q, then the attention over the projection's rows."""
    H, G, page = 8, 2, 32
    lens, new = [90, 64, 3], [90, 20, 3]
    q, k, v, s, t, n, start = attention_case(61, H, G, page, lens, new)
    slots, pos = [], []
    for b, m in enumerate(new):
        for i in range(lens[b] - m, lens[b]):
            slots.append(int(t[b, i // page]) * page + i % page)
            pos.append(i)
    qkv, _, _, _, _, sl, cs, w = make(62, H, G, len(slots), slots, page, 2, norm)
    pos = torch.tensor(pos)
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    k1, v1, s1, x = gpu(k, v, s, qkv)
    d = gpu(t, n, pos, sl, cs, *w)
    out = torch.empty(len(slots), H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(x, out, k1, v1, s1, d[2], d[3], d[4], d[5], d[6], H, G, 1e-6, q_rows=0)
    st = torch.tensor(start, dtype=torch.int32, device=DEV)
    ops.scaled_attention_prefill(out, None, k1, v1, s1, d[0], d[1], st, *tiles(lens, new, H // G, rows), H // G, 0.1,
                                 tile_rows=rows, qprep=(x, d[2], d[4], d[5], 1e-6), max_len=max_len)
    torch.cuda.synchronize()
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, H, G, k1, v1, s1, None)
    eq = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
    entries = orc.codes(k1, v1) * s1.cpu().double()[..., None, None]
    want, bound = orc.attention(eq, entries, t, lens, start, 0.1)
    close(out, want, bound + q_bound(eq, entries, t, lens, start, 0.1))


def test_step_captured_and_replayed():
    """Steps of rising lengths in one graph: each replay against the same calls made eagerly, the page's scale
    growing on the way."""
    H, G, page = 8, 2, 32
    lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(71, H, G, page, [28, 60, 200], True, room=4)
    x, t, n, pos, sl, w0, w1 = gpu(qkv, t, n, pos, sl, *w)
    cs = ref.rope_cos_sin(512, D, 1e4).to(DEV)
    caches = [gpu(k.clone(), v.clone(), s.clone()) for _ in range(2)]
    outs = [torch.zeros(3, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    ws = [ops.decode_workspace(3, G, H // G, 2, DEV) for _ in range(2)]

    def step(i):
        ops.scaled_attention_decode_fused(outs[i], x, *caches[i], t, n, pos, sl, cs, w0, w1, H // G, 0.1, 1e-6,
                                          workspace=ws[i], num_parts=2, part_size=256)

    step(0)
    step(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    base = x.clone()
    for i in range(4):
        x.copy_(base * (1.0 + i))
        n += 1
        pos += 1
        at = pos.long() // page
        sl.copy_(torch.gather(t.long(), 1, at[:, None])[:, 0] * page + pos % page)
        graph.replay()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        for a, b in zip(*caches):
            assert torch.equal(a, b)


def test_append_captured_with_its_checks(monkeypatch):
    """AKAP_DEBUG_CHECKS=1 and a captured append: each replay as the eager call."""
    monkeypatch.setattr(ops, "DEBUG_CHECKS", True)
    H, G = 4, 2
    qkv, k, v, s, pos, sl, cs, w = make(72, H, G, 70, list(range(40, 110)), 32, 5, True)
    x, pos, sl, cs, w0, w1 = gpu(qkv, pos, sl, cs, *w)
    caches = [gpu(k.clone(), v.clone(), s.clone()) for _ in range(2)]
    qs = [torch.zeros(70, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def append(i):
        ops.scaled_cache_append(x, qs[i], *caches[i], pos, sl, cs, w0, w1, H, G, 1e-6)

    append(0)
    append(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append(0)
    for i in range(3):
        x.mul_(2)
        graph.replay()
        append(1)
        torch.cuda.synchronize()
        assert torch.equal(*qs) and all(torch.equal(a, b) for a, b in zip(*caches))


def test_on_another_stream():
    lens = [400, 33]
    c = attention_case(81, 4, 2, 32, lens, [1, 1])
    want = want_rows(c, lens)
    side = torch.cuda.Stream()
    args = gpu(*c)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, k, v, s, t, n, start = args
        out = torch.empty_like(q)
        ws = ops.decode_workspace(2, 2, 2, 4, DEV)
        ops.scaled_attention_decode(out, q, k, v, s, t, n, 2, 0.1, workspace=ws, num_parts=4, part_size=128)
    side.synchronize()
    close(out, *want)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: its last pages are written and read."""
    H, G, page = 2, 2, 32
    pages = (1 << 32) // (G * page * D) + 40
    k = torch.zeros(pages, G, page, D, dtype=torch.uint8, device=DEV)
    v = torch.zeros(pages, G, page // 8, D, 8, dtype=torch.uint8, device=DEV)
    s = torch.full((2, pages, G), 2.0 ** -100, device=DEV)
    slots = list(range((pages - 3) * page, (pages - 3) * page + 70))
    qkv, _, _, _, _, sl, cs, w = make(91, H, G, 70, slots, page, 2, True)
    pos = torch.arange(70)
    q = torch.empty(70, H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(*gpu(qkv), q, k, v, s, *gpu(pos, sl, cs, *w), H, G, 1e-6)
    table = torch.tensor([[pages - 3, pages - 2, pages - 1]], dtype=torch.int32)
    small = [x[..., pages - 3:, :, :, :].cpu() if x.dim() == 4 else x[pages - 3:].cpu() for x in (k, v)]
    entries = orc.codes(*small) * s[:, pages - 3:].cpu().double()[..., None, None]
    here = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    out = torch.empty_like(q)
    n, st = gpu(torch.tensor([70], dtype=torch.int32), torch.tensor([0, 70], dtype=torch.int32))
    ops.scaled_attention_prefill(out, q, k, v, s, table.to(DEV), n, st, *tiles([70], [70], 1, 128), 1, 0.1)
    close(out, *orc.attention(q, entries, here, [70], [0, 70], 0.1))
    one = torch.empty_like(q[69:])
    ops.scaled_attention_decode(one, q[69:].contiguous(), k, v, s, table.to(DEV), n, 1, 0.1)
    close(one, *orc.attention(q[69:], entries, here, [70], [0, 1], 0.1))
    assert not k[:pages - 3].any() and not v[:pages - 3].any()


# ------------------------------------------------------------------------------------------------ engine
@pytest.mark.parametrize("model", ["tiny-qwen3", "tiny-llama"])
@pytest.mark.parametrize("block", [32, 96])
def test_engine_on_a_scaled_cache(model, block):
    """--kv-cache-dtype fp8_scaled end to end: prompts, captured decode steps, mixed steps."""
    from test_engine_gpu import _check_teacher_forced, _engine
    from aws_k8s_ansible_provisioner_amd.engine.config import SamplingParams

    eng = _engine(model, kv_cache_dtype="fp8_scaled", block_size=block)
    assert eng.runner.kv.dtype == torch.uint8 and eng.runner.graphs
    prompts = [list(range(3, 80)), [17] * 33 + [5, 6, 7]]
    outs = eng.generate(None, SamplingParams(max_tokens=10, temperature=0, ignore_eos=True), prompt_ids=prompts)
    for p, o in zip(prompts, outs):
        assert len(o.output_ids) == 10
        _check_teacher_forced(eng, p, o.output_ids, tol=0.6)
    sp = SamplingParams(max_tokens=12, temperature=0, ignore_eos=True)
    eng.add_request("a", None, sp, prompt_ids=list(range(5, 90)))
    got, mixed = {}, False
    for step in range(100):
        if step == 3:
            eng.add_request("b", None, sp, prompt_ids=[9, 8, 7] * 30)
        for o in eng.step():
            if o.finished:
                got[o.req_id] = o.output_ids
        mixed |= eng.last_step_mixed
        if len(got) == 2:
            break
    assert mixed
    _check_teacher_forced(eng, list(range(5, 90)), got["a"], tol=0.6)
    _check_teacher_forced(eng, [9, 8, 7] * 30, got["b"], tol=0.6)
