"""The scaled cache's norm and rotation to the last bit: every product and sum rounded by itself, in the order that the
kernels state, and the three kernels that prepare rows (append, prompts, the fused step) alike."""
import pytest
import torch

import scaled_cache_oracle as orc
from aws_k8s_ansible_provisioner_amd import ops
from aws_k8s_ansible_provisioner_amd.ops import reference as ref
from test_scaled_cache_gpu import DEV, FORMS, tiles

pytestmark = pytest.mark.gpu
D = 128
EPS = 1e-6


def prepared(x, w, angle):
    """x [T, heads, D] fp32, angle [T, D] = cos | sin.  Torch's fp32 operations, one rounding each: squares by fours and
    those in pairs, neighbours of 8 dims, of 16, 32 and 64 added; 1 / sqrt to the nearest; x inv w from the left; the
    rotation's products before their sum.  Also which rows are `sure`: the reciprocal root in 64 bits lies 2^-40 or
    more from the border of two fp32 numbers (the kernel's, a Newton step from one with an error e of 2^-22 at most,
    is off by 3/8 e^2 and a few 2^-46 before its rounding)."""
    s = (x * x).view(*x.shape[:-1], 16, 8)
    a = ((s[..., 0] + s[..., 1]) + s[..., 2]) + s[..., 3]
    b = ((s[..., 4] + s[..., 5]) + s[..., 6]) + s[..., 7]
    s = a + b
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    m = s * (1 / D) + torch.tensor(EPS, dtype=torch.float32, device=x.device)
    root = 1 / m.double().sqrt()
    sure = (root * (1 - 2.0 ** -40)).float() == (root * (1 + 2.0 ** -40)).float()
    y = x * root.float() * w.float()
    lo, hi = y[..., :D // 2], y[..., D // 2:]
    c, s = angle[:, None, :D // 2], angle[:, None, D // 2:]
    lc, hs, hc, ls = lo * c, hi * s, hi * c, lo * s
    return torch.cat([lc - hs, hc + ls], -1), sure[..., 0]


def inputs(seed, T, H, G):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device=DEV).bfloat16()
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).bfloat16() for _ in range(2)]
    return qkv, w, ref.rope_cos_sin(2048, D, 1e4).to(DEV)


def empty_cache(pages, G, page=32):
    k = torch.zeros(pages, G, page, D, dtype=torch.uint8, device=DEV)
    v = torch.zeros(pages, G, page // 8, D, 8, dtype=torch.uint8, device=DEV)
    return k, v, ops.scaled_cache_scales(1, pages, G, DEV)[0]


@pytest.mark.parametrize("decode", [False, True])        # runs of a workgroup, of a wave
def test_append_to_the_last_bit(decode):
    """20 million query entries: the rotation's product and sum rounded once would move one in 60000 of them to a
    neighbour, some hundreds, a reciprocal root that is off by a unit one in 25000."""
    T, H, G = 20480, 8, 2
    qkv, w, cs = inputs(1, T, H, G)
    pos = torch.arange(T, device=DEV) % 2048
    k, v, s = empty_cache(T // 32, G)
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(qkv, q, k, v, s, pos, torch.arange(T, device=DEV), cs, *w, H, G, EPS, decode=decode)
    x = qkv.float().view(T, H + 2 * G, D)
    want, sure = prepared(x[:, :H], w[0], cs[pos])
    assert int((~sure).sum()) < 100
    assert torch.equal(q[sure], want.bfloat16()[sure])
    keys, sure = prepared(x[:, H:H + G], w[1], cs[pos])
    sure = sure.view(-1, 32, G).all(1)                    # pages and heads without a row that is not
    assert int((~sure).sum()) < 50
    got = orc.codes(k, v)
    for j, y in enumerate((keys, x[:, H + G:])):
        y = y.view(-1, 32, G, D).transpose(1, 2)          # [pages, G, 32, D]
        m, e = torch.frexp(y.abs().amax((2, 3)).double() / 448)       # = m 2^e, 0.5 <= m < 1
        scale = torch.exp2((e - (m == 0.5).int()).double()).float()
        ok = sure if j == 0 else torch.ones_like(sure)
        assert torch.equal(s[j][ok], scale[ok])
        codes = (y / scale[..., None, None]).cpu().to(torch.float8_e4m3fn).double()
        assert torch.equal(got[j][ok.cpu()], codes[ok.cpu()])


@pytest.mark.parametrize("rows,max_len", FORMS)
@pytest.mark.parametrize("norm", [True, False])
def test_prompts_prepare_the_rows_that_an_append_writes(rows, max_len, norm):
    """Attention over the projection's rows and over the append's query rows: the same outputs, bit for bit."""
    H, G, n, B = 16, 2, 500, 8
    T = n * B
    qkv, w, cs = inputs(2, T, H, G)
    w = w if norm else [None, None]
    per = -(-n // 32)
    pos = torch.arange(T, device=DEV) % n
    slots = torch.arange(T, device=DEV) // n * per * 32 + pos
    k, v, s = empty_cache(B * per, G)
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_cache_append(qkv, q, k, v, s, pos, slots, cs, *w, H, G, EPS)
    t = torch.arange(B * per, dtype=torch.int32, device=DEV).view(B, per)
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    start = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
    out = [torch.empty_like(q) for _ in range(2)]
    for o, prep in zip(out, (None, (qkv, pos, cs, w[0], EPS))):
        ops.scaled_attention_prefill(o, q if prep is None else None, k, v, s, t, lens, start,
                                     *tiles([n] * B, [n] * B, H // G, rows), H // G, 0.2, tile_rows=rows, qprep=prep,
                                     max_len=max_len)
    assert torch.equal(*out)


@pytest.mark.parametrize("B,size", [(300, 1280), (20, 1280), (12, 256)])     # four waves, eight, split rows
@pytest.mark.parametrize("norm", [True, False])
def test_a_fused_step_is_an_append_and_its_attention(B, size, norm):
    """The same cache and the same outputs, bit for bit."""
    H, G, room = 16, 2, 40
    qkv, w, cs = inputs(3, B, H, G)
    w = w if norm else [None, None]
    g = torch.Generator().manual_seed(4)
    full = orc.cache(g, B * room, G, 32)
    past = torch.randint(0, room * 32 - 1, (B,), generator=g)
    past[:4] = torch.tensor([0, 31, 32, room * 32 - 1])
    t = torch.arange(B * room, dtype=torch.int32, device=DEV).view(B, room)
    pos = past.to(DEV)
    slots = torch.arange(B, device=DEV) * room * 32 + pos
    lens = (pos + 1).int()
    one, two = [[x.to(DEV) for x in full] for _ in range(2)]
    parts = room * 32 // size
    q, out, fused = [torch.empty(B, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    kw = dict(num_parts=parts, part_size=size, workspace=ops.decode_workspace(B, G, H // G, parts, DEV))
    ops.scaled_cache_append(qkv, q, *one, pos, slots, cs, *w, H, G, EPS, decode=True)
    ops.scaled_attention_decode(out, q, *one, t, lens, H // G, 0.2, **kw)
    ops.scaled_attention_decode_fused(fused, qkv, *two, t, lens, pos, slots, cs, *w, H // G, 0.2, EPS, **kw)
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    assert torch.equal(out, fused)
