"""Performance cases of the scaled cache: keys and values kept as e4m3 bytes with one power-of-two
scale for each page and kv head, the operators that append to it and those that attend over it.

A cache has pages of `page` tokens, a multiple of 32.  K [pages, G, page, D] and V [pages, G, page / 8,
D, 8] hold e4m3 codes in the orders of the framework's other caches, `scales` [2, pages, G] (keys,
values) the power of two that a page's codes are multiplied with.  An append takes a row's keys (normed
and rotated) and values into their page:

    need  = the least 2^e, -100 <= e <= 100, with every finite |x| of the page's new entries <= 448 2^e
    scale = need if the append writes the page's first token, else max(scale, need)
    code  = e4m3(clamp(x / scale, -448, 448)), to nearest even; of a NaN 0

and where a page that was begun before gets a larger scale, its other codes are rounded anew for it.

A case is a dict:
  kind      append   rows of the projection into the cache: q and k norms, rotation, codes, scales
            decode   one query row per sequence over its keys
            step     a decode step whole: the new token's q, k and v prepared, appended, attended over
            prompt   rows of prompts over the cache, causal
            chunk    a step of prompts whole: keys and values appended, queries prepared, attention
  seqs, tokens, past, spread   sequences; new tokens of the longest (decode rows: 1); cached tokens
            before them (of the longest); how many fewer the others may have (of `tokens` where
            there are several, else of `past`)
  heads, kv_heads, page, norm  the layer's heads of 128 dims, tokens per page, q and k norms
"""
import math

import torch

own = False

DEV = "cuda"
D = 128
EPS = 1e-6
TOP = 448.0         # the largest e4m3 number
LOW, HIGH = -100, 100


def _case(name, kind, seqs, tokens, past, spread, heads, kv_heads, norm, page=32):
    return dict(name=name, kind=kind, seqs=seqs, tokens=tokens, past=past, spread=spread,
                heads=heads, kv_heads=kv_heads, page=page, norm=norm)


def listed():
    return [
        # one sequence of a chat decoding: its row into the cache, its attention, the step whole
        _case("append 1 row", "append", 1, 1, 300, 0, 16, 8, True),
        _case("decode 1 x 333", "decode", 1, 1, 333, 0, 16, 8, False),
        # a step of prompt chunks as the scheduler fills it, ragged, all pages new
        _case("append 12 prompts", "append", 12, 1300, 0, 700, 32, 8, False),
        # serving at some hundred to some thousand keys
        _case("decode 64 x 2048", "decode", 64, 1, 2048, 1100, 32, 8, False),
        _case("decode 200 x 4000", "decode", 200, 1, 4000, 1500, 16, 8, False),
        # a few long documents, a head group as one of eight ranks has it
        _case("decode 3 x 30000", "decode", 3, 1, 30000, 9000, 8, 1, False),
        _case("step 16 x 500", "step", 16, 1, 500, 320, 16, 8, True),
        _case("step 128 x 1500", "step", 128, 1, 1500, 900, 32, 8, False),
        # a short question; long prompts; the rest of a long one behind what was cached; few pages of 64
        _case("prompt 1 x 77", "prompt", 1, 77, 0, 0, 16, 8, False),
        _case("prompt 8 x 2048", "prompt", 8, 2048, 0, 0, 32, 8, False),
        _case("chunk 1000 behind 9000", "chunk", 1, 1000, 9000, 0, 16, 8, True),
        _case("chunk 24 x 350", "chunk", 24, 350, 40, 260, 32, 4, False, page=64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "step", "prompt", "chunk"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    c = _case("", kind, 1, 1, 0, 0, heads, kv_heads, rng.random() < 0.5, rng.choice([32, 32, 64, 96]))
    del c["name"]
    if kind in ("decode", "step"):
        c["past"] = _spread(rng, 1, 30000)
        c["seqs"] = _spread(rng, 1, max(1, min(250, 1600000 // (c["past"] * kv_heads))))
        c["spread"] = rng.randint(0, c["past"] - 1)
    elif kind == "append":
        rows = _spread(rng, 1, 12000)
        c["seqs"] = min(rows, _spread(rng, 1, 64))
        c["tokens"] = -(-rows // c["seqs"])
        c["past"] = rng.choice([0, rng.randint(1, 2000)])
        c["spread"] = rng.randint(0, c["tokens"] - 1)
    else:
        c["tokens"] = _spread(rng, 2, 2000)
        c["past"] = rng.choice([0, 0, _spread(rng, 1, 8000)])
        most = 800000000 // (c["tokens"] * (c["tokens"] + c["past"]) * heads)
        c["seqs"] = _spread(rng, 1, max(1, min(32, most, 8000 // c["tokens"])))
        c["spread"] = rng.randint(0, c["tokens"] - 1)
    return c


def _shape(c):
    """[(cached tokens, new tokens)] of the sequences; of a decode row the cached ones are all but itself."""
    def less(i):
        return (i * 7919 + i * i) % (c["spread"] + 1) if i else 0

    if c["kind"] == "decode":
        return [(max(0, c["past"] - less(i) - 1), 1) for i in range(c["seqs"])]
    if c["tokens"] == 1:
        return [(max(0, c["past"] - less(i)), 1) for i in range(c["seqs"])]
    return [(c["past"], max(1, c["tokens"] - less(i))) for i in range(c["seqs"])]


# ---------------------------------------------------------------------------- inputs
def _need(most):
    """The least power of two with most <= 448 times it."""
    m, e = torch.frexp(most)                    # most = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(most > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, LOW))
    return torch.ldexp(torch.ones_like(most), e.clamp(LOW, HIGH))


def _codes(x, scale):
    y = torch.nan_to_num(x / scale, nan=0.0, posinf=TOP, neginf=-TOP).clamp(-TOP, TOP)
    return y.to(torch.float8_e4m3fn)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(*shape, device=DEV).normal_(mean, std, generator=g)

    H, G, page, shape = c["heads"], c["kv_heads"], c["page"], _shape(c)
    B, group = len(shape), c["heads"] // c["kv_heads"]
    count = [-(-(p + n) // page) for p, n in shape]
    width = max(count) + 1
    pages = sum(count) + 2
    order = torch.randperm(pages, generator=g, device=DEV).cpu()
    tables = torch.zeros(B, width, dtype=torch.int32)
    positions, slots, start, at, tiles = [], [], [0], 0, []
    long = max(n for _, n in shape) * group > 1024
    tile_rows = 256 if long else 128
    for b, (p, n) in enumerate(shape):
        mine = order[at:at + count[b]]
        at += count[b]
        tables[b, :count[b]] = mine.to(torch.int32)
        where = torch.arange(p, p + n)
        positions.append(where)
        slots.append(mine[where // page] * page + where % page)
        start.append(start[-1] + n)
        for r in range(0, n * group, tile_rows):
            tiles.append((p + min(n, (r + tile_rows + group - 1) // group), b, r))
    tiles.sort(key=lambda t: t[0])
    slots = torch.cat(slots)
    touched, row = torch.unique(slots // page, return_inverse=True)
    fresh = torch.zeros(len(touched), dtype=torch.bool)
    fresh[row[slots % page == 0]] = True
    T = start[-1]
    s = {
        "case": c, "rows": T, "tile_rows": tile_rows,
        "tables": tables.to(DEV), "positions": torch.cat(positions).to(DEV), "slots": slots.to(DEV),
        "lens": torch.tensor([p + n for p, n in shape], dtype=torch.int32, device=DEV),
        "start": torch.tensor(start, dtype=torch.int32, device=DEV),
        "tile_seq": torch.tensor([t[1] for t in tiles], dtype=torch.int32, device=DEV),
        "tile_row": torch.tensor([t[2] for t in tiles], dtype=torch.int32, device=DEV),
        # the pages that the new rows are in, each row's among them, and which of them they begin
        "touched": touched.to(DEV), "touched_row": row.to(DEV), "fresh": fresh.to(DEV),
        "longest": max(p + n for p, n in shape), "most": max(n for _, n in shape),
    }
    # keys with a few strong channels, smaller values, some heads louder than others
    loud = 1.0 + 7.0 * (torch.rand(D, generator=g, device=DEV) < 0.06)
    head = torch.exp2(normal(2, G))
    k = torch.empty(pages, G, page, D, dtype=torch.uint8, device=DEV)
    v = torch.empty(pages, G, page // 8, D, 8, dtype=torch.uint8, device=DEV)
    scales = torch.empty(2, pages, G, device=DEV)
    for a in range(0, pages, 4096):
        b = min(pages, a + 4096)
        x = normal(b - a, G, page, D) * loud * head[0][:, None, None] * 0.3
        scales[0, a:b] = _need(x.abs().amax((2, 3)))
        k[a:b] = _k_order(_codes(x, scales[0, a:b, :, None, None]), page).view(torch.uint8)
        x = normal(b - a, G, page // 8, D, 8) * head[1][:, None, None, None] * 0.2
        scales[1, a:b] = _need(x.abs().amax((2, 3, 4)))
        v[a:b] = _codes(x, scales[1, a:b, :, None, None, None]).view(torch.uint8)
        del x
    s["k"], s["v"], s["scales"] = k, v, scales
    angle = torch.arange(max(s["longest"], 16), dtype=torch.float64, device=DEV)[:, None] * (
        5e5 ** (-torch.arange(D // 2, dtype=torch.float64, device=DEV) / (D // 2)))[None]
    s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    s["q"] = normal(T, H, D).to(torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    if c["kind"] in ("append", "step", "chunk"):
        s["qkv"] = normal(T, (H + 2 * G) * D, std=0.7).to(torch.bfloat16)
        s["qw"], s["kw"] = [(normal(D, std=0.1, mean=1.0) * (loud ** 0.5)).to(torch.bfloat16)
                            if c["norm"] else None for _ in range(2)]
    if c["kind"] in ("decode", "step"):
        # partitions as an engine cuts a decode step: enough work items to fill the card
        parts = max(1, min(-(-2048 // (B * G)), -(-s["longest"] // 256)))
        size = -(-(-(-s["longest"] // parts)) // (4 * page)) * 4 * page
        s["parts"], s["part_size"] = -(-s["longest"] // size), size
        from aws_k8s_ansible_provisioner_amd import ops

        s["workspace"] = ops.decode_workspace(B, G, group, s["parts"], DEV)
    return s


# ---------------------------------------------------------------------------- plain forms
def _k_order(x, page):
    """[..., page, D] of tokens -> the cache's order: in each 32 tokens [2, D / 32, 16, 32], row r of
    half h token 8 (r // 4) + 4 h + r % 4."""
    y = x.reshape(*x.shape[:-2], page // 32, 4, 2, 4, D // 32, 32)
    n = y.dim()
    lead = list(range(n - 6))
    return y.permute(*lead, n - 6, n - 4, n - 2, n - 5, n - 3, n - 1).reshape(x.shape)


def _k_tokens(x, page):
    """The cache's order -> [..., page, D]."""
    y = x.reshape(*x.shape[:-2], page // 32, 2, D // 32, 4, 4, 32)
    n = y.dim()
    lead = list(range(n - 6))
    return y.permute(*lead, n - 6, n - 3, n - 5, n - 2, n - 4, n - 1).reshape(x.shape)


def _prepared(s):
    """q, k, v of the projection's rows, normed and rotated, in 32 bits."""
    c = s["case"]
    H, G, T = c["heads"], c["kv_heads"], s["rows"]
    x = s["qkv"].float().view(T, H + 2 * G, D)
    cs = s["cos_sin"][s["positions"]][:, None]
    cos, sin = cs[..., :D // 2], cs[..., D // 2:]

    def turned(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    return turned(x[:, :H], s["qw"]), turned(x[:, H:H + G], s["kw"]), x[:, H + G:]


def _append(s, k, v):
    """The rows' keys and values into their pages."""
    c, page = s["case"], s["case"]["page"]
    x = torch.stack([k, v])                                               # [2, T, G, D]
    at, row, off = s["touched"], s["touched_row"], s["slots"] % page
    most = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    need = torch.zeros(2, len(at), c["kv_heads"], device=DEV).index_reduce_(1, row, most, "amax")
    old = s["scales"][:, at]
    need = _need(need)
    new = torch.where(s["fresh"][None, :, None], need, torch.maximum(old, need))
    again = torch.where(s["fresh"][None, :, None], 1.0, old / new)[..., None, None]
    f8 = torch.float8_e4m3fn
    codes = torch.stack([_k_tokens(s["k"][at].view(f8).float(), page),
                         s["v"][at].view(f8).float().transpose(-1, -2).reshape(len(at), -1, page, D)])
    codes = _codes(codes * again, torch.ones_like(again)).view(torch.uint8)
    mine = _codes(x, new[:, row][..., None]).view(torch.uint8)
    codes[:, row, :, off] = mine.permute(1, 0, 2, 3)
    s["k"][at] = _k_order(codes[0], page)
    s["v"][at] = codes[1].reshape(len(at), -1, page // 8, 8, D).transpose(-1, -2)
    s["scales"][:, at] = new


def _padded(s):
    """Keys and values of all sequences, [B, G, keys, D] in 32 bits, up to the longest's last page."""
    c, page, f8 = s["case"], s["case"]["page"], torch.float8_e4m3fn
    t = s["tables"][:, :-(-s["longest"] // page)].long()
    k = _k_tokens(s["k"][t].view(f8).float() * s["scales"][0][t][..., None, None], page)
    v = s["v"][t].view(f8).float() * s["scales"][1][t][..., None, None, None]
    v = v.transpose(-1, -2)
    both = [x.transpose(1, 2).reshape(t.shape[0], c["kv_heads"], -1, D) for x in (k, v)]
    return both[0], both[1], torch.arange(both[0].shape[2], device=DEV)


def _softmaxed(scores, seen):
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _decode(s, q):
    c = s["case"]
    k, v, key = _padded(s)
    q = q.float().view(len(q), c["kv_heads"], -1, D)
    p = _softmaxed(q @ k.transpose(-1, -2) * D ** -0.5, (key[None] < s["lens"][:, None])[:, None, None])
    return (p @ v).reshape(len(q), -1, D).to(torch.bfloat16)


def _prompt(s, q):
    c = s["case"]
    k, v, key = _padded(s)
    B, G, n = len(s["lens"]), c["kv_heads"], s["most"]
    fresh = s["start"][1:] - s["start"][:-1]
    i = torch.arange(n, device=DEV)
    at = (s["start"][:-1, None] + torch.minimum(i[None], fresh[:, None] - 1)).long()     # [B, n]
    rows = q.float()[at].view(B, n, G, -1, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    seen = key[None, None] <= ((s["lens"] - fresh)[:, None] + i[None])[..., None]        # [B, n, keys]
    group = c["heads"] // G
    p = _softmaxed((rows @ k.transpose(-1, -2) * D ** -0.5).view(B, G, group, n, -1), seen[:, None, None])
    o = (p.view(B, G, group * n, -1) @ v).view(B, G * group, n, D).transpose(1, 2)
    return o[i[None] < fresh[:, None]].to(torch.bfloat16)


def _cache(s):
    f8 = torch.float8_e4m3fn
    return {"k": s["k"].view(f8), "v": s["v"].view(f8), "scales": s["scales"]}


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "decode":
        return {"out": _decode(s, s["q"])}
    if kind == "prompt":
        return {"out": _prompt(s, s["q"])}
    q, k, v = _prepared(s)
    _append(s, k, v)
    q = q.to(torch.bfloat16)            # query rows are bf16, as an append hands them on
    if kind == "append":
        return {"q": q, **_cache(s)}
    return {"out": _decode(s, q) if kind == "step" else _prompt(s, q), **_cache(s)}


def run(state):
    if not own:
        return _plain(state)
    from aws_k8s_ansible_provisioner_amd import ops

    s = state
    c, scale = s["case"], D ** -0.5
    H, G, kind = c["heads"], c["kv_heads"], c["kind"]
    if kind == "decode":
        ops.scaled_attention_decode(s["out"], s["q"], s["k"], s["v"], s["scales"], s["tables"],
                                    s["lens"], H // G, scale, workspace=s["workspace"],
                                    num_parts=s["parts"], part_size=s["part_size"])
        return {"out": s["out"]}
    if kind == "prompt":
        ops.scaled_attention_prefill(s["out"], s["q"], s["k"], s["v"], s["scales"], s["tables"],
                                     s["lens"], s["start"], s["tile_seq"], s["tile_row"], H // G,
                                     scale, tile_rows=s["tile_rows"])
        return {"out": s["out"]}
    if kind == "step":
        ops.scaled_attention_decode_fused(s["out"], s["qkv"], s["k"], s["v"], s["scales"],
                                          s["tables"], s["lens"], s["positions"], s["slots"],
                                          s["cos_sin"], s["qw"], s["kw"], H // G, scale, EPS,
                                          workspace=s["workspace"], num_parts=s["parts"],
                                          part_size=s["part_size"])
        return {"out": s["out"], **_cache(s)}
    if kind == "append":
        ops.scaled_cache_append(s["qkv"], s["q"], s["k"], s["v"], s["scales"], s["positions"],
                                s["slots"], s["cos_sin"], s["qw"], s["kw"], H, G, EPS,
                                decode=c["tokens"] == 1)
        return {"q": s["q"], **_cache(s)}
    # prompts: the attention prepares its own query rows from the projection
    ops.scaled_cache_append(s["qkv"], s["q"], s["k"], s["v"], s["scales"], s["positions"],
                            s["slots"], s["cos_sin"], s["qw"], s["kw"], H, G, EPS, q_rows=0)
    ops.scaled_attention_prefill(s["out"], s["q"], s["k"], s["v"], s["scales"], s["tables"],
                                 s["lens"], s["start"], s["tile_seq"], s["tile_row"], H // G,
                                 scale, tile_rows=s["tile_rows"],
                                 qprep=(s["qkv"], s["positions"], s["cos_sin"], s["qw"], EPS))
    return {"out": s["out"], **_cache(s)}


def work(case):
    c = case
    H, G, kind, shape = c["heads"], c["kv_heads"], c["kind"], _shape(c)
    T = sum(n for _, n in shape)
    b = f = 0.0
    if kind in ("append", "step", "chunk"):
        b += T * (H + 2 * G) * D * 2 + T * (D * 4 + 16)     # the projection's rows, angles, places
        b += 2 * T * G * D                                  # codes
        b += T * H * D * 2 if kind == "append" else 0       # q
    if kind in ("decode", "prompt"):
        b += T * H * D * 2                                  # q
    if kind != "append":
        b += T * H * D * 2                                  # out
        # every key and value once (those of a step's own rows are written, above), the scales
        b += sum((p if kind in ("step", "chunk") else p + n) for p, n in shape) * G * D * 2
        b += sum(-(-(p + n) // c["page"]) for p, n in shape) * (G * 8 + 4)
        f += sum(n * p + n * (n + 1) / 2 for p, n in shape) * H * D * 4
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, sequence by sequence; codes before their rounding (times 2^0: as run() gives
    them, without the scale), other results unrounded."""
    s = prepare(case, seed)
    c, page = case, case["page"]
    H, G, kind, shape = c["heads"], c["kv_heads"], c["kind"], _shape(case)
    per = H // G
    f8, f64 = torch.float8_e4m3fn, torch.float64
    tok = torch.arange(page, device=DEV)
    part, half, r = tok // 32, (tok // 4) % 2, 4 * ((tok % 32) // 8) + tok % 4

    def key_rows(x, pages):                 # [n, G, page, D]: a token's dims lie in four runs of 32
        runs = x[pages].reshape(len(pages), G, page // 32, 2, 4, 16, 32)
        return runs[:, :, part, half, :, r].permute(1, 2, 0, 3, 4).reshape(len(pages), G, page, D)

    def value_rows(x, pages):
        return x[pages][:, :, tok // 8, :, tok % 8].permute(1, 2, 0, 3)

    result = {}
    kc, vc, sc = s["k"].view(f8).to(f64), s["v"].view(f8).to(f64), s["scales"].to(f64)
    q = s["q"].to(f64)
    if kind in ("append", "step", "chunk"):
        x = s["qkv"].to(f64).view(-1, H + 2 * G, D)
        angle = s["cos_sin"][s["positions"]].to(f64)[:, None]
        rows = {}
        for name, a, b, w in (("q", 0, H, s["qw"]), ("k", H, H + G, s["kw"])):
            y = x[:, a:b]
            if w is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS) * w.to(f64)
            lo, hi = y[..., :D // 2], y[..., D // 2:]
            co, si = angle[..., :D // 2], angle[..., D // 2:]
            rows[name] = torch.cat([lo * co - hi * si, lo * si + hi * co], -1)
        rows["v"] = x[:, H + G:]
        q = rows["q"] if kind == "append" else rows["q"].to(torch.bfloat16).to(f64)
        where, off = s["slots"] // page, s["slots"] % page
        began = torch.zeros(len(kc), dtype=torch.bool, device=DEV)
        began[where[off == 0]] = True
        hit = torch.zeros(len(kc), dtype=torch.bool, device=DEV)
        hit[where] = True
        held = []
        for j, name in enumerate("kv"):
            top = torch.zeros(len(kc), G, dtype=f64, device=DEV)
            top.scatter_reduce_(0, where[:, None].expand(-1, G), rows[name].abs().amax(-1), "amax")
            e = torch.ceil(torch.log2(top.clamp_min(1e-300) / TOP)).clamp(LOW, HIGH)
            need = torch.exp2(e)
            now = torch.where(began[:, None], need, torch.maximum(sc[j], need))
            now = torch.where(hit[:, None], now, sc[j])
            ratio = torch.where(began[:, None], torch.ones_like(now), sc[j] / now)
            every = torch.arange(len(kc), device=DEV)
            t = (key_rows if j == 0 else value_rows)((kc, vc)[j], every) * ratio[..., None, None]
            t[where, :, off] = rows[name] / now[where][..., None]
            sc[j] = now
            held.append(t)
        kt, vt = held
        order = torch.empty(len(kc), G, page // 32, 2, 4, 16, 32, dtype=f64, device=DEV)
        order[:, :, part, half, :, r] = kt.reshape(len(kc), G, page, 4, 32).permute(2, 0, 1, 3, 4)
        result = {"k": order.reshape(kc.shape),
                  "v": vt.reshape(len(kc), G, page // 8, 8, D).transpose(-1, -2).contiguous(),
                  "scales": sc}
        if kind == "append":
            return {"q": q, **result}
        # the attention sees codes
        keys, values = (t.to(f8).to(f64) * sc[j][..., None, None] for j, t in enumerate(held))
    out = torch.empty(s["rows"], H, D, dtype=f64, device=DEV)
    at = 0
    for b, (p, n) in enumerate(shape):
        mine = s["tables"][b, :-(-(p + n) // page)].long()
        if kind in ("step", "chunk"):
            k, v = keys[mine], values[mine]
        else:
            k = key_rows(kc, mine) * sc[0][mine][..., None, None]
            v = value_rows(vc, mine) * sc[1][mine][..., None, None]
        k, v = (x.transpose(0, 1).reshape(G, -1, D)[:, :p + n] for x in (k, v))
        later = torch.arange(p + n, device=DEV)[None] > torch.arange(p, p + n, device=DEV)[:, None]
        for h in range(H):
            z = q[at:at + n, h] @ k[h // per].T / math.sqrt(D)
            out[at:at + n, h] = torch.softmax(z.masked_fill(later, -math.inf), -1) @ v[h // per]
        at += n
    return {"out": out, **result}
