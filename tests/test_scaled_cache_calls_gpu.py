"""The scaled cache's operators called as they may be beside the usual way: rows that are named, tables and projections
that are views, positions past the angles, a workspace that two graphs share."""
import pytest
import torch

import scaled_cache_oracle as orc
from aws_k8s_ansible_provisioner_amd import ops
from test_scaled_cache import D, attention_case, check_append, close, make
from test_scaled_cache_gpu import DEV, FORMS, gpu, q_bound, step_case, tiles, want_rows

pytestmark = pytest.mark.gpu


def wide_tables(t):
    """The same tables as rows of a wider tensor, which names pages outside the cache elsewhere."""
    w = torch.full((t.shape[0] + 1, t.shape[1] + 13), 1 << 30, dtype=torch.int32, device=DEV)
    w[:-1, :t.shape[1]] = t
    return w[:, :t.shape[1]]


@pytest.mark.parametrize("parts,size,tickets", [(1, 1280, False), (5, 256, False), (5, 256, True)])
def test_decode_rows_that_q_start_names(parts, size, tickets):
    """Rows in another order and apart; those that are not named keep what they hold."""
    H, G, lens = 6, 2, [1100, 0, 33, 700, 257]
    q, k, v, s, t, n, start = attention_case(101, H, G, 32, lens, [1] * 5)
    rows = torch.tensor([8, 2, 0, 5, 3], dtype=torch.int32)
    many = torch.full((10, H, D), 3.0, dtype=torch.bfloat16)
    many[rows.long()] = q
    x, k1, v1, s1, t1, n1, r1 = gpu(many, k, v, s, t, n, rows)
    out = torch.full_like(x, 9.0)
    ws = ops.decode_workspace(5, G, H // G, parts, DEV) if tickets else None
    ops.scaled_attention_decode(out, x, k1, v1, s1, wide_tables(t1), n1, H // G, 0.1, workspace=ws, num_parts=parts,
                                part_size=size, q_start=r1)
    close(out[r1.long()], *want_rows((q, k, v, s, t, n, start), lens))
    others = torch.ones(10, dtype=torch.bool)
    others[rows.long()] = False
    assert bool((out.cpu()[others] == 9).all())


@pytest.mark.parametrize("parts,size", [(1, 512), (3, 128)])
def test_fused_step_of_wide_rows_and_far_positions(parts, size):
    """Projection rows with others between them, and positions before and behind the angles, which take the first and
    the last."""
    H, G, page = 6, 2, 32
    lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(102, H, G, page, [5, 340, 63, 64], True)
    pos = torch.tensor([-7, 100000, 63, 1 << 40])
    wide = torch.full((4, qkv.shape[1] + 72), float("nan"), dtype=torch.bfloat16)
    wide[:, :qkv.shape[1]] = qkv
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    x, k1, v1, s1, t1, n1, p1, l1, c1, *w1 = gpu(wide, k, v, s, t, n, pos, sl, cs, *w)
    out = torch.empty(4, H, D, dtype=torch.bfloat16, device=DEV)
    ops.scaled_attention_decode_fused(out, x[:, :qkv.shape[1]], k1, v1, s1, wide_tables(t1), n1, p1, l1, c1, *w1, H // G,
                                      0.1, 1e-6, workspace=ops.decode_workspace(4, G, H // G, parts, DEV),
                                      num_parts=parts, part_size=size)
    check_append(qkv, k0, v0, s0, pos, sl, cs, w, H, G, k1, v1, s1, None)
    q = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
    entries = orc.codes(k1, v1) * s1.cpu().double()[..., None, None]
    start = list(range(5))
    want, bound = orc.attention(q, entries, t, lens, start, 0.1)
    close(out, want, bound + q_bound(q, entries, t, lens, start, 0.1))


@pytest.mark.parametrize("rows,max_len", FORMS)
def test_prompts_of_wide_rows_and_far_positions(rows, max_len):
    H, G, page = 6, 2, 32
    lens, new = [90, 640, 3], [90, 120, 3]
    _, k, v, s, t, n, start = attention_case(103, H, G, page, lens, new)
    T = start[-1]
    qkv, *_, cs, w = make(104, H, G, T, list(range(T)), page, 8, True)
    pos = torch.arange(T) * 7 - 100                        # (of 512 angles)
    wide = torch.full((T, qkv.shape[1] + 8), float("nan"), dtype=torch.bfloat16)
    wide[:, :qkv.shape[1]] = qkv
    x, k1, v1, s1, t1, n1, p1, c1, w0 = gpu(wide, k, v, s, t, n, pos, cs, w[0])
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    st = torch.tensor(start, dtype=torch.int32, device=DEV)
    ops.scaled_attention_prefill(out, None, k1, v1, s1, wide_tables(t1), n1, st, *tiles(lens, new, H // G, rows), H // G,
                                 0.1, tile_rows=rows, qprep=(x[:, :qkv.shape[1]], p1, c1, w0, 1e-6), max_len=max_len)
    q = orc.prepared(qkv, pos, cs, *w, H, G, 1e-6)[0]
    entries = orc.codes(k, v) * s.double()[..., None, None]
    want, bound = orc.attention(q, entries, t, lens, start, 0.1)
    close(out, want, bound + q_bound(q, entries, t, lens, start, 0.1))


def test_two_graphs_of_one_workspace():
    """Steps of different batches captured with the same workspace and replayed in turn, its tickets among what they
    share: each replay as the eager call."""
    G, H, page, parts, size = 2, 8, 32, 5, 256
    ws = ops.decode_workspace(6, G, H // G, parts, DEV)
    graphs, checks = [], []
    for i, past in enumerate(([1000, 33, 700, 0], [5, 1200, 300, 640, 1279, 64])):
        lens, qkv, k, v, s, t, n, pos, sl, cs, w = step_case(105 + 2 * i, H, G, page, past, True)
        x, t, n, pos, sl, cs, w0, w1 = gpu(qkv, t, n, pos, sl, cs, *w)
        caches = [gpu(k.clone(), v.clone(), s.clone()) for _ in range(2)]
        outs = [torch.zeros(len(past), H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        own = ops.decode_workspace(6, G, H // G, parts, DEV)

        def step(j, caches=caches, outs=outs, args=(t, n, pos, sl, cs, w0, w1), x=x, ws=(ws, own)):
            ops.scaled_attention_decode_fused(outs[j], x, *caches[j], *args, H // G, 0.1, 1e-6, workspace=ws[j],
                                              num_parts=parts, part_size=size)

        step(0)
        step(1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(0)
        graphs.append((graph, step, x, caches, outs))
    for turn in range(4):
        for graph, step, x, caches, outs in graphs:
            x.mul_(1.5)
            graph.replay()
            step(1)
        torch.cuda.synchronize()
        for _, _, _, caches, outs in graphs:
            assert torch.equal(*outs) and all(torch.equal(a, b) for a, b in zip(*caches))
