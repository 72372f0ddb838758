"""The scaled 8-bit cache in 64 bits, entry by entry from its definition; shares nothing with the package.

A cache is held in token order here: values [2, pages, G, page, D] (keys, values; what the codes stand for),
scales [2, pages, G]."""
import math

import torch

D = 128
F8 = torch.float8_e4m3fn


def k_index(page):
    """Flat position in a (page, head)'s K bytes of token o, dim d: [page, D]."""
    o, d = torch.arange(page)[:, None], torch.arange(D)[None]
    c, t = o // 32, o % 32
    half, row = (t // 4) % 2, 4 * (t // 8) + t % 4
    return c * 4096 + half * 2048 + (d // 32) * 512 + row * 32 + d % 32


def v_index(page):
    o, d = torch.arange(page)[:, None], torch.arange(D)[None]
    return (o // 8) * 1024 + d * 8 + o % 8


def codes(k, v):
    """[2, pages, G, page, D] codes as float64, in token order."""
    NB, G, page, _ = k.shape
    out = []
    for t, i in ((k, k_index(page)), (v, v_index(page))):
        flat = t.cpu().contiguous().view(F8).double().view(NB, G, page * D)
        out.append(flat[..., i.reshape(-1)].view(NB, G, page, D))
    return torch.stack(out)


def store(x, page):
    """Token-ordered codes [2, pages, G, page, D] (uint8) -> K and V tensors."""
    _, NB, G = x.shape[:3]
    k, v = torch.empty(2, NB, G, page * D, dtype=torch.uint8)
    k[..., k_index(page).reshape(-1)] = x[0].reshape(NB, G, -1)
    v[..., v_index(page).reshape(-1)] = x[1].reshape(NB, G, -1)
    return k.view(NB, G, page, D), v.view(NB, G, page // 8, D, 8)


def need(most):
    """least 2^e >= most / 448, e in -100 .. 100"""
    e = -100
    if most > 0:
        e = math.frexp(most / 448.0)[1]                   # most / 448 = m 2^e, 0.5 <= m < 1
        e -= math.frexp(most / 448.0)[0] == 0.5
    return 2.0 ** max(-100, min(100, e))


def cache(gen, pages, G, page, std=1.0):
    """K, V, scales of a cache that is full of entries of different loudness."""
    x = torch.randn(2, pages, G, page, D, generator=gen, dtype=torch.float64) * std
    x = x * 2.0 ** torch.randint(-3, 4, (2, pages, G, 1, 1), generator=gen)
    s = torch.tensor([need(float(m)) for m in x.abs().amax((3, 4)).flatten()], dtype=torch.float64)
    s = s.view(2, pages, G)
    k, v = store((x / s[..., None, None]).float().to(F8).view(torch.uint8), page)
    return k, v, s.float()


def prepared(qkv, positions, cos_sin, q_w, k_w, H, G, eps, rope=True):
    """q [T, H, D], k, v [T, G, D]."""
    x = qkv[:, :(H + 2 * G) * D].cpu().double().view(-1, H + 2 * G, D)
    cs = cos_sin.cpu().double()[positions.cpu().clamp(0, len(cos_sin) - 1)][:, None]
    c, s = cs[..., :D // 2], cs[..., D // 2:]

    def turned(y, w):
        if w is not None:
            y = y / ((y * y).mean(-1, keepdim=True) + eps).sqrt() * w.cpu().double()
        if not rope:
            return y
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    return turned(x[:, :H], q_w), turned(x[:, H:H + G], k_w), x[:, H + G:]


def append(before, scales, k, v, slots):
    """Scales after an append, and (entries [2, pages, G, page, D], which are new): new entries unrounded, old
    ones as they were.  Entries that are not finite: infinities the largest number, NaN 0."""
    _, NB, G, page, _ = before.shape
    after, now = before.clone(), scales.double().clone()
    new = torch.zeros(2, NB, G, page, D, dtype=torch.bool)
    at = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < NB * page:
            at.setdefault(s // page, []).append((t, s % page))
    for b, rows in at.items():
        for j, x in enumerate((k, v)):
            for h in range(G):
                mine = torch.stack([x[t, h] for t, _ in rows])
                fin = mine[torch.isfinite(mine)].abs()
                n = need(float(fin.max()) if fin.numel() else 0.0)
                now[j, b, h] = n if any(o == 0 for _, o in rows) else max(n, float(now[j, b, h]))
                for t, o in rows:
                    y = torch.nan_to_num(x[t, h], nan=0.0, posinf=math.inf, neginf=-math.inf)
                    after[j, b, h, o] = y.clamp(-448 * now[j, b, h], 448 * now[j, b, h])
                    new[j, b, h, o] = True
    return now, after, new


def attention(q, entries, tables, lens, start, scale):
    """(rows, bound): causal attention of each sequence's rows start[b] .. start[b + 1] - 1 in 64 bits, and how
    far a kernel may be off that takes q and the entries exactly, forms scores and sums in fp32 and rounds the
    weights and the result to bf16 (half a step: 2^-8)."""
    T, H, _ = q.shape
    _, NB, G, page, _ = entries.shape
    out, off = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    q = q.cpu().double()
    for b, n in enumerate(lens):
        r0, rows = start[b], start[b + 1] - start[b]
        n = min(int(n), tables.shape[1] * page)
        for h in range(H):
            ks, vs, pos = [], [], []
            for i in range(-(-max(n, 0) // page)):
                blk = int(tables[b, i])
                if 0 <= blk < NB:
                    m = min(page, n - i * page)
                    ks.append(entries[0, blk, h * G // H, :m])
                    vs.append(entries[1, blk, h * G // H, :m])
                    pos += range(i * page, i * page + m)
            if not pos:
                continue
            k, v, pos = torch.cat(ks), torch.cat(vs), torch.tensor(pos)
            x = q[r0:r0 + rows, h]
            seen = pos[None] <= torch.arange(int(lens[b]) - rows, int(lens[b]))[:, None]
            z = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(z, -1).masked_fill(~seen.any(-1, keepdim=True), 0.0)
            o, w = p @ v, p @ v.abs()
            size = (x.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            out[r0:r0 + rows, h] = o
            # weights and result rounded; a score of 128 products summed in fp32, taken to base 2: twice its error
            # in a weight and the weights' sum
            off[r0:r0 + rows, h] = 2 ** -8 * 1.02 * (w + o.abs()) + w * (4 * 132 * 2.0 ** -24 * size + 2 ** -16)
    return out, off
