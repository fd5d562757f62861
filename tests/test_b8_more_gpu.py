"""The 8-bit cache where its calls meet others: a workspace that both caches' decodes use, in captured graphs too; page offsets beyond 32
bits; calls on two streams; writes without any slot."""
import pytest
import torch

import b8_ref as R
from cases import build_decode_case, bf16_tensor
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt
from test_b8_gpu import fresh, paged, put, rows, same, write
from test_rotary_gpu import check_queries, gen, parts, qkv, table

pytestmark = pytest.mark.gpu


def call8(lens, KVH, G, D, PS, fmt, ws, ql=1, seed=0):
    cache, bt = paged(lens, KVH, PS, D, fmt, 40 + seed)
    flat, st = Lt.b8_views(cache.cuda(), KVH, D)
    B = len(lens)
    q = torch.randn(B * ql, KVH * G, D, generator=gen(seed)).to(torch.bfloat16).cuda()
    qsl = (torch.arange(B + 1) * ql).to(torch.int32).cuda()
    lens_d, bt_d, one = torch.tensor(lens, dtype=torch.int32).cuda(), bt.cuda(), torch.ones(KVH, device="cuda")
    out = torch.zeros_like(q)
    return lambda: K.decode_b8(q, flat, st, PS, bt_d, lens_d, qsl, D ** -0.5, 1.0, one, one, ql, out, ws, fmt=fmt), out


@pytest.mark.parametrize("D,KVH,G", [(128, 8, 4), (256, 2, 8)])
def test_one_workspace_for_both_caches(D, KVH, G):
    """split sequences of either cache leave the counters at zero for the other, launch after launch and replay after replay"""
    lens = [3000, 40, 9000]
    c = build_decode_case(91 + D, lens, KVH, G, D, 16)
    cache = c["cache"]
    ws = K.alloc_workspace(3, KVH, G, D, 2)
    q = bf16_tensor(c["q"])
    bt, sl, qsl = (torch.from_numpy(c[k]).cuda() for k in ("bt", "seq_lens", "qsl"))
    gk, gv = torch.from_numpy(c["gk"]).cuda(), torch.from_numpy(c["gv"]).cuda()
    o4 = torch.zeros_like(q)

    def four():
        K.decode_ragged(q, cache.flat, cache.strides, cache.PS, bt, sl, qsl, c["sm"], 1.0, gk, gv, 1, o4, ws)
    eight, o8 = call8(lens, KVH, G, D, 16, "e4m3", ws)
    draft, od = call8([700, 5000], KVH, G, D, 32, "int8", ws, ql=2, seed=1)
    calls, outs = (four, eight, draft), (o4, o8, od)
    want = []
    for f, o in zip(calls, outs):
        f()
        want.append(o.clone())
        o.zero_()
    torch.cuda.synchronize()
    graphs = []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f()
        graphs.append(g)
    for i in range(12):
        k = (i * 5 + i // 3) % 3
        outs[k].zero_()
        (graphs[k].replay if i % 2 else calls[k])()
        assert torch.equal(outs[k], want[k]), i
    assert K.workspace_status(ws) == 0 and int(ws[256:256 + 4 * 4096].view(torch.int32).abs().sum()) == 0


def test_two_streams():
    """calls that run at the same time, each on its own workspace"""
    wss = [K.alloc_workspace(2, 8, 4, 128, 1) for _ in range(2)]
    made = [call8([6000, 900], 8, 4, 128, 16, f, ws, seed=i) for i, (f, ws) in enumerate(zip(("e4m3", "int8"), wss))]
    want = []
    for f, o in made:
        f()
        want.append(o.clone())
        o.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        for s, (f, o) in zip(streams, made):
            with torch.cuda.stream(s):
                o.zero_()
                f()
    torch.cuda.synchronize()
    for (f, o), w in zip(made, want):
        assert torch.equal(o, w)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_offsets_beyond_32_bits(fmt):
    """a pool of more than 4 GiB: the same tokens in its last pages and in a small cache give the same bytes and rows"""
    D, KVH, G, PS, L = 128, 8, 4, 16, 100
    page = 2 * KVH * PS * (D + 1)
    P = (5 << 30) // page
    big = torch.empty((P, 2 * KVH, PS, D + 1), dtype=torch.uint8, device="cuda")
    small = torch.zeros((8, 2 * KVH, PS, D + 1), dtype=torch.uint8, device="cuda")
    k, v = rows(L, KVH, D, 1)
    one = torch.ones(KVH, device="cuda")
    q = torch.randn(1, KVH * G, D, generator=gen(1)).to(torch.bfloat16).cuda()
    outs = []
    for cache, first in ((big, P - 7), (small, 1)):
        big[P - 7:].zero_()
        flat, st = Lt.b8_views(cache, KVH, D)
        slots = first * PS + torch.arange(L, device="cuda")
        K.write_b8(k.cuda(), v.cuda(), flat, st, PS, slots, one, one, fmt=fmt)
        K.write_b8(k.cuda()[40:41] * 9, v.cuda()[40:41], flat, st, PS, slots[40:41], one, one, fmt=fmt)
        bt = (first + torch.arange(7, device="cuda")).to(torch.int32)[None]
        lens, qsl = torch.tensor([L], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        o, p = torch.zeros_like(q), torch.zeros(20, KVH * G, D, dtype=torch.bfloat16, device="cuda")
        K.decode_b8(q, flat, st, PS, bt, lens, qsl, D ** -0.5, 1.0, one, one, 1, o, K.alloc_workspace(1, KVH, G, D, 1), fmt=fmt)
        K.prefill_b8(q.expand(20, -1, -1).contiguous(), flat, st, PS, bt, [(0, 0, 20, L)], D ** -0.5, 1.0, KVH, p, fmt=fmt)
        outs.append((cache[first:first + 7].clone(), o, p))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.any())


@pytest.mark.parametrize("b8", [False, True])
def test_no_slots(b8):
    """a batch of queries only: empty keys, values and slots"""
    D, KVH, HQ, NT, PS = 128, 2, 8, 5, 16
    x, t, pos = qkv(NT, HQ, KVH, D, 3), table(90, D, torch.float32), torch.arange(NT)
    q, k, v = parts(x.cuda(), HQ, KVH, D)
    cache = torch.full((2, 2 * KVH, PS, D + 1 if b8 else Lt.slot_bytes(D)), 9, dtype=torch.uint8, device="cuda")
    one = torch.ones(KVH, device="cuda")
    for kk, vv in ((k[:0], v[:0]), (k[:0].clone(), v[:0].clone())):
        out = torch.zeros_like(q)
        args = torch.zeros(0, dtype=torch.int64, device="cuda"), pos.cuda(), t.cuda(), one, one, out
        if b8:
            flat, st = Lt.b8_views(cache, KVH, D)
            K.write_rotary_b8(q, kk, vv, flat, st, PS, *args)
            K.write_b8(kk, vv, flat, st, PS, args[0], one, one)
        else:
            flat, st = Lt.flat_views(*Lt.slot_views(cache, KVH, D))
            K.write_rotary(q, kk, vv, flat, st, PS, *args)
        check_queries(out, q.cpu(), pos, t, False)
        none = torch.zeros(0, HQ, D, dtype=torch.bfloat16, device="cuda")
        rest = args[0], args[0], args[2], one, one, none
        (K.write_rotary_b8 if b8 else K.write_rotary)(none, kk, vv, flat, st, PS, *rest)
    assert bool((cache == 9).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH", [(128, 2), (256, 3)])
@pytest.mark.parametrize("n", [511, 600, 2100])
def test_single_tokens_and_drafts_of_a_large_batch(fmt, D, KVH, n):
    """one token each at any place of a tile (several tiles a warp), among them drafts of two and three and tokens without a slot; then
    the same tiles again with larger values, whose codes there are rounded"""
    PS, g = 32, gen(n + D)
    one = torch.tensor([1.0, 0.5, 0.37])[:KVH]
    P = n // 2 + 2
    tiles = torch.randperm(2 * P, generator=g)[:n]
    cache = fresh(P, KVH, PS, D, fmt, 6)
    for step, drafts in enumerate((False, True, False)):
        at = torch.randint(0, 13, (n,), generator=g)
        slots = []
        for i in range(n):
            m = int(torch.randint(1, 4, (1,), generator=g)) if drafts and i % 5 == 0 else 1
            slots += [int(tiles[i]) * 16 + int(at[i]) + j for j in range(m)]
            if i % 17 == 3:
                slots.append(-1)
        slots = torch.tensor(slots)
        k, v = rows(len(slots), KVH, D, 50 + step)
        k, v = k * 2 ** (3 * step), v * 2 ** (3 * step)
        want = R.append(cache, k, v, slots.tolist(), one, one, fmt)
        same(write(cache, k, v, slots, one, one, fmt, KVH), want, fmt)
        cache = want


def test_put_keeps_what_lies_between_pages():
    view, big = put(fresh(2, 1, 16, 128, "int8", 1))
    assert bool((big[:, :, -32:] == 0xc3).all()) and view.shape == (2, 2, 16, 129)


@pytest.mark.parametrize("side", ["key", "value"])
@pytest.mark.parametrize("D,G,kind", [(128, 4, "draft"), (256, 8, "draft"), (128, 4, "window"), (128, 4, "prompt"), (256, 8, "prompt")])
def test_nan_of_the_last_token(D, G, kind, side):
    """a NaN that only the last of a request's rows sees: a key's makes that row NaN in its kv head, a value's its channel there. Other
    channels, heads and requests are as without it, and so are the earlier rows, but for the channel of a value"""
    KVH, PS, lens, ql = 2, 16, [100, 230, 61], 3 if kind != "prompt" else 40
    cache, bt = paged(lens, KVH, PS, D, "e4m3", 17 + D)
    bad, at, head = cache.clone(), lens[1] - 1, 1
    t = bad.view(len(bad), 2 * KVH, PS // 16, 16 * D + 16)[int(bt[1, at // PS]), head + (KVH if side == "value" else 0), at % PS // 16]
    t[at % 16 * D + ((2 ^ (at % 8)) << 4) + 5] = 0x7f                       # channel 16 * 2 + 5
    q = torch.randn(3 * ql, KVH * G, D, generator=gen(D)).to(torch.bfloat16).cuda()
    ws, one = K.alloc_workspace(3, KVH, G, D, ql if kind != "prompt" else 1), torch.ones(KVH, device="cuda")
    bt_d, lens_d = bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    qsl = (torch.arange(4) * ql).to(torch.int32).cuda()
    got = []
    for c in (cache, bad):
        flat, st = Lt.b8_views(c.cuda(), KVH, D)
        out = torch.zeros_like(q)
        if kind == "prompt":
            K.prefill_b8(q, flat, st, PS, bt_d, [(b, b * ql, b * ql + ql, n) for b, n in enumerate(lens)], D ** -0.5, 1.0, KVH, out, workspace=ws)
        else:
            K.decode_b8(q, flat, st, PS, bt_d, lens_d, qsl, D ** -0.5, 1.0, one, one, ql, out, ws, window=50 if kind == "window" else 0)
        got.append(out.view(3, ql, KVH, G, D).cpu())
    assert K.workspace_status(ws) == 0 and bool(got[0].isfinite().all())
    touched = torch.zeros(got[0].shape, dtype=torch.bool)
    touched[1, -1, head, :, slice(None) if side == "key" else 37] = True
    assert bool(got[1][touched].isnan().all())
    if side == "value":
        touched[1, :, head, :, 37] = True
    assert torch.equal(got[0][~touched].view(torch.int16), got[1][~touched].view(torch.int16))


@pytest.mark.parametrize("D,G", [(128, 4), (256, 8)])
@pytest.mark.parametrize("prompt", [False, True])
def test_nan_outside_the_windows(D, G, prompt):
    """NaN keys and values of tokens that no row sees, in tiles whose other tokens rows do see: behind the sinks, before the first row's
    window, behind the context"""
    KVH, PS, lens, ql, window, sinks = 2, 32, [100, 230, 61, 700], 35 if prompt else 2, 50, 5
    cache, bt = paged(lens, KVH, PS, D, "e4m3", 71 + D)
    bad = cache.clone()
    for b, L in enumerate(lens):
        seen = torch.stack([R.sees(L - ql + t, L, window, sinks) for t in range(ql)]).any(0)
        for j in torch.nonzero(~seen).flatten().tolist():
            t = bad.view(len(bad), 2 * KVH, PS // 16, 16 * D + 16)[int(bt[b, j // PS]), :, j % PS // 16]
            t[:, j % 16 * D:(j % 16 + 1) * D] = 0xff
    q = torch.randn(4 * ql, KVH * G, D, generator=gen(D + ql)).to(torch.bfloat16).cuda()
    ws, one = K.alloc_workspace(4, KVH, G, D, 1 if prompt else ql), torch.ones(KVH, device="cuda")
    bt_d, lens_d = bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    qsl = (torch.arange(5) * ql).to(torch.int32).cuda()
    got = []
    for c in (cache, bad):
        flat, st = Lt.b8_views(c.cuda(), KVH, D)
        out, lse = torch.full_like(q, float("nan")), torch.zeros(4 * ql, KVH * G, device="cuda")
        if prompt:
            K.prefill_b8(q, flat, st, PS, bt_d, [(b, b * ql, b * ql + ql, n) for b, n in enumerate(lens)], D ** -0.5, 1.0, KVH, out,
                         window=window, sinks=sinks, workspace=ws, lse=lse)
        else:
            K.decode_b8(q, flat, st, PS, bt_d, lens_d, qsl, D ** -0.5, 1.0, one, one, ql, out, ws, window=window, sinks=sinks, lse=lse)
        got.append((out, lse))
    assert K.workspace_status(ws) == 0 and bool(got[0][0].isfinite().all() & got[0][1].isfinite().all())
    assert torch.equal(got[0][0].view(torch.int16), got[1][0].view(torch.int16)) and torch.equal(got[0][1], got[1][1])
