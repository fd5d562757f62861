"""The 8-bit cache on the GPU: appending byte for byte as the definition says, attention of single tokens, drafts and prompts against 64
bits within the error of the kernels' roundings, and the calls together as a server makes them."""
import math

import pytest
import torch

import b8_ref as R
from horizon_kernels_b200 import _lib
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt
from test_rotary_gpu import check_queries, gen, parts, qkv, table

pytestmark = pytest.mark.gpu


def same(got, want, fmt):
    """equal codes (any NaN is one), equal scales, unused bytes as they were"""
    (a, s, x), (b, t, y) = R.unpack(got.cpu()), R.unpack(want)
    va, vb = R.values(a, fmt), R.values(b, fmt)
    assert torch.equal(s.view(torch.int32), t.view(torch.int32)) and torch.equal(x, y)
    assert bool(((va == vb) | (va.isnan() & vb.isnan())).all())


def fresh(P, KVH, PS, D, fmt, seed):
    """a cache of finite codes and ordinary scales"""
    codes = torch.randint(0, 256, (P, 2 * KVH, PS, D), generator=gen(seed), dtype=torch.uint8)
    if fmt == "e4m3":
        codes[(codes & 0x7f) == 0x7f] = 0x55
    else:
        codes[codes == 0x80] = 1
    return R.pack(codes, torch.randint(-9, -4, (P, 2 * KVH, PS // 16), generator=gen(seed + 1)))


def put(cache):
    """on the GPU, every page and head 32 bytes further apart"""
    P, H, PS, D1 = cache.shape
    big = torch.full((P, H, PS * D1 + 32), 0xc3, dtype=torch.uint8, device="cuda")
    view = big.as_strided(cache.shape, (big.stride(0), big.stride(1), D1, 1))
    view.copy_(cache)
    return view, big


def write(cache, key, value, slots, gk, gv, fmt, KVH, host=None):
    view, big = put(cache)
    flat, st = Lt.b8_views(view, KVH, view.shape[3] - 1)
    was, _lib._host = _lib._host, host or _lib._host
    try:
        K.write_b8(key.cuda(), value.cuda(), flat, st, view.shape[2], slots.cuda(), gk.cuda(), gv.cuda(), fmt=fmt)
    finally:
        _lib._host = was
    assert bool((big[:, :, -32:] == 0xc3).all())
    return view.cpu()


def rows(NT, KVH, D, seed, wild=False):
    k, v = (torch.randn(NT, KVH, D, generator=gen(seed + i)).to(torch.bfloat16) for i in range(2))
    k[..., 5] *= 20
    k *= (torch.rand(NT, KVH, 1, generator=gen(seed + 2)) * 8 - 4).exp2().to(torch.bfloat16)           # scales that grow and shrink
    if wild:
        big = torch.tensor([float("inf"), float("-inf"), float("nan"), 1e30, -7e4, 1e-30, 0.0, -0.0, 448.0, 127.0]).to(torch.bfloat16)
        at = torch.randint(0, NT * KVH * D, (max(2, NT // 4),), generator=gen(seed + 3))
        for x in (k, v):
            x.view(-1)[at] = big[torch.randint(0, 10, at.shape, generator=gen(seed + 4))]
        k[NT // 2] = 0
        v[:2] = float("nan")
    return k, v


def runs(kind, PS, P, seed):
    """slots of a call, the tokens of a tile side by side"""
    g = gen(seed)
    pages = torch.randperm(P, generator=g).tolist()
    if kind == "prompt":                                              # two prompts, one from the middle of a tile on
        a = torch.tensor(pages[0]) * PS + torch.arange(PS)
        b = torch.cat([torch.tensor(p * PS + torch.arange(PS).numpy()) for p in pages[1:4]])[5:-3]
        return torch.cat((a[:-1], b))
    if kind == "tokens":                                              # one token each, and a few drafts of three
        return torch.cat([torch.arange(p * PS + (7 * p) % (PS - 3), p * PS + (7 * p) % (PS - 3) + (3 if p % 3 == 0 else 1)) for p in pages])
    if kind == "skips":                                               # tokens without a slot between the tiles, rows in any order
        out = []
        for p in pages:
            r = torch.randperm(16, generator=g)[:int(torch.randint(1, 17, (1,), generator=g))]
            out += [p * PS + r, torch.full((int(torch.randint(0, 3, (1,), generator=g)),), -1)]
        return torch.cat(out)
    if kind == "twice":                                               # slots named twice, and a whole batch on one slot
        return torch.cat((torch.tensor([3, 3, 4, 3, 5, 4]), torch.full((70,), pages[0] * PS + 16 * (PS > 16) + 2), torch.arange(32, 48),
                          torch.arange(32, 48)) if PS > 32 else (torch.tensor([3, 3, 4, 3, 5, 4]), torch.full((70,), (P - 1) * PS + 2)))
    raise AssertionError(kind)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,PS", [(128, 2, 16), (256, 1, 32), (128, 3, 64), (128, 5, 16), (256, 9, 16)])
@pytest.mark.parametrize("kind", ["prompt", "tokens", "skips", "twice"])
def test_append(fmt, D, KVH, PS, kind):
    P = 9
    cache = fresh(P, KVH, PS, D, fmt, 11 * D + PS)
    gk, gv = torch.tensor([1.0, 0.37, 2.0 ** -20] * 3)[:KVH], torch.tensor([0.011, 1.0, 3.0] * 3)[:KVH]
    for step in range(3):
        slots = runs(kind, PS, P, step)
        k, v = rows(len(slots) + 2, KVH, D, 100 * step + D, wild=step == 1)
        want = R.append(cache, k, v, slots.tolist(), gk, gv, fmt)
        got = write(cache, k, v, slots, gk, gv, fmt, KVH, host=_lib._NoHost() if step == 2 else None)
        same(got, want, fmt)
        cache = want


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,n", [(128, 8, 700), (256, 2, 4000)])
def test_append_many_tokens(fmt, D, KVH, n):
    """more tokens than warps start one by one: requests of 1 to 90 tokens at any place of a tile, single tokens among them"""
    PS, g = 16, gen(n)
    lens = torch.cat((torch.randint(1, 90, (n // 60,), generator=g), torch.ones(40, dtype=torch.int64)))
    lens = lens[torch.randperm(len(lens), generator=g)]
    first = torch.randint(0, 16, lens.shape, generator=g)
    per = (first + lens + PS - 1) // PS
    P = int(per.sum()) + 1
    pages = (torch.randperm(P - 1, generator=g) + 1).split(per.tolist())
    slots = torch.cat([p[(torch.arange(int(f), int(f + L))) // PS] * PS + torch.arange(int(f), int(f + L)) % PS for p, f, L in zip(pages, first, lens)])
    assert len(slots) * 2 * KVH > 8192
    cache, one = fresh(P, KVH, PS, D, fmt, 5), torch.ones(KVH)
    k, v = rows(len(slots), KVH, D, 3)
    same(write(cache, k, v, slots, one, one, fmt, KVH), R.append(cache, k, v, slots.tolist(), one, one, fmt), fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,HQ,rot,interleaved,dtype,n", [(128, 8, 32, 128, False, torch.float32, 40), (256, 2, 6, 64, True, torch.bfloat16, 23),
                                                            (128, 1, 3, 48, False, torch.bfloat16, 7), (256, 4, 24, 256, False, torch.float32, 1100),
                                                            (128, 5, 10, 128, False, torch.float32, 2100), (256, 9, 9, 192, True, torch.bfloat16, 9000)])
def test_append_turned(fmt, D, KVH, HQ, rot, interleaved, dtype, n):
    PS, NT = 32, n + 5
    x = qkv(NT, HQ, KVH, D, n)
    t, pos = table(3000, rot, dtype), torch.arange(NT) * 2 - 3
    slots = torch.cat((torch.arange(n) + 37, torch.tensor([-1, -1])))
    one = torch.ones(KVH)
    cache = fresh((n + 37) // PS + 1, KVH, PS, D, fmt, 8)
    q, k, v = parts(x.cuda(), HQ, KVH, D)
    want = R.append(cache, R.turn(k.cpu(), pos, t, interleaved), v.cpu(), slots.tolist(), one, one, fmt)
    for host in (None, _lib._NoHost()):
        view, _ = put(cache)
        flat, st = Lt.b8_views(view, KVH, D)
        out = torch.full((NT, HQ, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        was, _lib._host = _lib._host, host or _lib._host
        try:
            K.write_rotary_b8(q, k, v, flat, st, PS, slots.cuda(), pos.cuda(), t.cuda(), one.cuda(), one.cuda(), out, interleaved=interleaved,
                              fmt=fmt)
        finally:
            _lib._host = was
        check_queries(out, q.cpu(), pos, t, interleaved)
        same(view.cpu(), want, fmt)


# ----------------------------------------------------------------------------------------------------------- attention
def paged(lens, KVH, PS, D, fmt, seed, sound=None):
    """a cache whose pages lie at random, and what nothing may read: NaN codes, NaN scales and bad table entries past every context's
    last tile (and in tiles that `sound`, a list of visible tiles per request, does not name), NaN codes behind the last token"""
    need = [(L + PS - 1) // PS for L in lens]
    P = sum(need) + 2
    cache = fresh(P, KVH, PS, D, fmt, seed)
    perm = (torch.randperm(P - 1, generator=gen(seed)) + 1).tolist()
    MP = max(need + [1]) + 1
    bt = torch.full((len(lens), MP), 0, dtype=torch.int32)
    tiles = cache.view(P, 2 * KVH, PS // 16, 16 * D + 16)
    tiles[0], tiles[perm[sum(need):]] = 0xff, 0xff
    for b, L in enumerate(lens):
        mine, perm = perm[:need[b]], perm[need[b]:]
        bt[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
        for i, p in enumerate(mine):
            for s in range(PS // 16):
                first = i * PS + 16 * s
                if first >= L or (sound is not None and first // 16 not in sound[b]):
                    tiles[p, :, s] = 0xff
                elif first + 16 > L:
                    tiles[p, :, s, (L - first) * D:16 * D] = 0x7f if fmt == "e4m3" else 0x80
    return cache, bt


def context(cache, bt, b, L, KVH, PS, fmt):
    codes, scales, _ = R.unpack(cache)
    pos = torch.arange(L)
    page = bt[b, pos // PS].long()
    c = R.values(codes, fmt)[page, :, pos % PS]                        # (L, 2 KVH, D)
    s = scales.double()[page, :, pos % PS // 16]
    return c, s


def check_rows(got, lse, cache, bt, b, L, q, KVH, PS, fmt, sm, gk, gv, window, sinks, D, out_step, prefill):
    """the rows of request b against 64 bits. Weights are rounded to f16 (half a step: 2^-11, at least 2^-25 of the largest weight times
    value scale), scores summed in fp32 over D products, sums of N weights in fp32; exponentials are within 2^-21."""
    c, s = context(cache, bt, b, L, KVH, PS, fmt)
    x = c * s[..., None]
    k, v = x[:, :KVH] * gk.double()[:, None], x[:, KVH:]
    ql, HQ, _ = q.shape
    G = HQ // KVH
    qd = q.double().view(ql, KVH, G, D)
    out, want, w, reach = R.attention(qd, k, v, sm, window, sinks)
    out = out * gv.double()[None, :, None, None]
    see = w > 0
    vis = see.any((0, 1, 2)) if L else torch.zeros(0, dtype=torch.bool)
    va = torch.where(vis[:, None, None], v.abs(), 0.0).nan_to_num(0.0)
    mean = torch.einsum("hgtj,jhd->thgd", w, va) * gv.double().abs()[None, :, None, None]
    serr = (reach * (D + 8) * 2.0 ** -23 + D * 2.0 ** -25 * abs(sm) * (k.abs().nan_to_num(0.0).max() if L else 0)).permute(2, 0, 1)     # (t, h, g)
    N = max(L, 1)
    c_rel = 2.0 ** -11 + 2 * serr + 2.0 ** -20 + N * 2.0 ** -24
    if prefill:
        low = 2.0 ** -25 * torch.einsum("jhd,thg->thgd", va, w.amax(-1).permute(2, 0, 1)) if L else 0.0
    else:
        sv = torch.where(vis[:, None], s[:, KVH:], 1.0)
        top = (w * sv.T[:, None, None]).amax(-1).permute(2, 0, 1) if L else 0.0
        low = 2.0 ** -25 * torch.einsum("jhd,thg->thgd", (va / sv[..., None]).nan_to_num(0.0), top) if L else 0.0
    tol = out_step * out.abs() + (1 + out_step) * (c_rel[..., None] * mean + (low * gv.double().abs()[None, :, None, None] if L else 0.0)) + 1e-30
    diff = (got.double().view(ql, KVH, G, D) - out).abs()
    assert bool((diff <= tol).all()), (float((diff - tol).max()), float((diff / tol).max()))
    if lse is not None:
        l = lse.double().view(ql, KVH, G)
        e = want.permute(2, 0, 1)
        assert torch.equal(l == -math.inf, e == -math.inf)
        ok = e != -math.inf
        assert bool(((l - e).abs()[ok] <= (serr + N * 2.0 ** -24 + 2.0 ** -19 + e.abs() * 2.0 ** -22)[ok]).all())


DECODE = [  # KVH, G, D, PS, lens, ql, window, sinks
    (8, 4, 128, 16, [1, 15, 16, 17, 0, 300, 33], [1] * 7, 0, 0), (2, 8, 128, 32, [700, 5, 64], [1, 2, 2], 0, 0),
    (1, 1, 128, 64, [129], [1], 0, 0), (2, 8, 256, 16, [250, 16, 0, 1, 900], [1] * 5, 0, 0), (2, 6, 256, 32, [97, 400], [2, 4], 0, 0),
    (1, 16, 256, 16, [333, 40], [1, 1], 0, 0), (4, 5, 128, 16, [60, 61, 62], [3, 0, 5], 0, 0), (1, 8, 256, 64, [500], [8], 0, 0),
    (2, 4, 128, 16, [500, 40, 3, 0, 77], [1, 2, 2, 1, 1], 33, 4), (2, 8, 256, 16, [700, 90], [2, 1], 100, 0), (1, 4, 128, 32, [300], [4], 1, 20),
    (2, 2, 256, 16, [17, 18, 400], [1, 1, 3], 16, 17)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("KVH,G,D,PS,lens,ql,window,sinks", DECODE)
def test_decode(fmt, KVH, G, D, PS, lens, ql, window, sinks):
    HQ, B = KVH * G, len(lens)
    sound = None
    if window:                                                         # tiles that some row sees
        sound = [{j // 16 for t in range(q) for j in torch.nonzero(R.sees(L - q + t, L, window, sinks)).flatten().tolist()} for L, q in zip(lens, ql)]
    cache, bt = paged(lens, KVH, PS, D, fmt, 7 * KVH + D + sum(lens), sound)
    qsl = torch.tensor([0] + ql).cumsum(0).to(torch.int32)
    T = int(qsl[-1])
    q = torch.randn(T, HQ, D, generator=gen(T)).to(torch.bfloat16)
    gk, gv = torch.rand(KVH, generator=gen(1)) + 0.5, torch.rand(KVH, generator=gen(2)) + 0.5
    gk[0] = -gk[0]
    view, _ = put(cache)
    flat, st = Lt.b8_views(view, KVH, D)
    qlmax, sm = max(ql), 0.7 * D ** -0.5
    ws = K.alloc_workspace(B, KVH, G, D, qlmax)
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    args = q.cuda(), flat, st, PS, bt.cuda(), lens_d, qsl.cuda(), sm, 1.5, gk.cuda(), gv.cuda(), qlmax
    got = {}
    for want_lse, host, splits in ((True, None, None), (False, None, None), (True, _lib._NoHost(), 1)):
        out = torch.full((T + 2, HQ, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        lse = torch.full((T + 1, HQ), 123.0, device="cuda") if want_lse else None
        was, _lib._host = _lib._host, host or _lib._host
        try:
            K.decode_b8(*args, out, ws, fmt=fmt, window=window, sinks=sinks, splits=splits, lse=lse)
        finally:
            _lib._host = was
        assert K.workspace_status(ws) == 0
        assert bool(out[T:].isnan().all()) and (lse is None or bool((lse[T:] == 123.0).all()))
        for b in range(B):
            a, e = int(qsl[b]), int(qsl[b + 1])
            if a < e:
                check_rows(out[a:e].cpu(), None if lse is None else lse[a:e].cpu(), cache, bt, b, lens[b], q[a:e], KVH, PS, fmt, sm, gk, gv * 1.5,
                           window, sinks, D, 2.0 ** -8, False)
        got[want_lse, splits] = out
    again = torch.full_like(out, float("nan"))
    K.decode_b8(*args, again, ws, fmt=fmt, window=window, sinks=sinks)
    assert torch.equal(again.view(torch.int16), got[False, None].view(torch.int16))


def test_decode_leaves_rows_that_are_not_its_own():
    """requests with more query tokens than qlmax, and none"""
    KVH, G, D, PS, lens, ql = 2, 4, 128, 16, [50, 60, 70], [1, 6, 2]
    cache, bt = paged(lens, KVH, PS, D, "e4m3", 3)
    qsl = torch.tensor([0] + ql).cumsum(0).to(torch.int32)
    q = torch.randn(9, 8, D, generator=gen(3)).to(torch.bfloat16)
    view, _ = put(cache)
    flat, st = Lt.b8_views(view, KVH, D)
    one = torch.ones(KVH, device="cuda")
    out = torch.full((9, 8, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    K.decode_b8(q.cuda(), flat, st, PS, bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), qsl.cuda(), 0.1, 1.0, one, one, 2, out,
                K.alloc_workspace(3, KVH, G, D, 2))
    nan = out.isnan().all(-1).all(-1).cpu()
    assert nan.tolist() == [False] + [True] * 6 + [False] * 2


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,G,ql", [(128, 8, 4, 1), (256, 2, 8, 2)])
def test_decode_long_and_split(fmt, D, KVH, G, ql):
    """sequences in many pieces, one of them merged in two steps, against 64 bits on the GPU; scales of values far apart"""
    lens, PS = [70001, 3, 5000], 64
    need = [(L + PS - 1) // PS for L in lens]
    P = sum(need)
    cache = fresh(P, KVH, PS, D, fmt, 9).cuda()
    tiles = cache.view(P, 2 * KVH, PS // 16, 16 * D + 16)
    e = torch.randint(-14, 3, (P, KVH, PS // 16), generator=gen(4))
    tiles[:, KVH:, :, 16 * D:16 * D + 4] = torch.ldexp(torch.ones(e.shape), e.float())[..., None].contiguous().view(torch.uint8).cuda()
    bt = torch.zeros((3, max(need)), dtype=torch.int32)
    perm = torch.randperm(P, generator=gen(5)).to(torch.int32).split(need)
    for b, p in enumerate(perm):
        bt[b, :need[b]] = p
    flat, st = Lt.b8_views(cache, KVH, D)
    ql_d = torch.tensor([0, ql, 2 * ql, 3 * ql], dtype=torch.int32)
    q = torch.randn(3 * ql, KVH * G, D, generator=gen(6)).to(torch.bfloat16)
    one, sm = torch.ones(KVH, device="cuda"), 0.3 * D ** -0.5
    out, lse = torch.zeros_like(q, device="cuda"), torch.zeros(3 * ql, KVH * G, device="cuda")
    ws = K.alloc_workspace(3, KVH, G, D, ql)
    K.decode_b8(q.cuda(), flat, st, PS, bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ql_d.cuda(), sm, 1.0, one, one, ql, out, ws,
                fmt=fmt, lse=lse)
    host = cache.cpu()
    for b in range(3):
        check_rows(out[b * ql:(b + 1) * ql].cpu(), lse[b * ql:(b + 1) * ql].cpu(), host, bt, b, lens[b], q[b * ql:(b + 1) * ql], KVH, PS, fmt, sm,
                   one.cpu(), one.cpu(), 0, 0, D, 2.0 ** -8, False)


PREFILL = [  # KVH, G, D, PS, [(q tokens, context)], window, sinks, chunk
    (2, 4, 128, 16, [(130, 130)], 0, 0, 65536), (8, 4, 128, 16, [(1, 1), (17, 40), (3, 129)], 0, 0, 65536), (2, 8, 256, 32, [(65, 300)], 0, 0, 65536),
    (1, 6, 256, 64, [(200, 200), (40, 77)], 0, 0, 65536), (2, 3, 128, 16, [(300, 700)], 0, 0, 256), (2, 4, 128, 16, [(150, 600)], 64, 5, 65536),
    (1, 8, 256, 16, [(50, 500), (9, 9)], 100, 0, 128), (1, 1, 128, 16, [(20, 16)], 0, 0, 65536)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("KVH,G,D,PS,reqs,window,sinks,chunk", PREFILL)
def test_prefill(fmt, KVH, G, D, PS, reqs, window, sinks, chunk):
    HQ, lens = KVH * G, [L for _, L in reqs]
    sound = None
    if window:
        sound = [{j // 16 for t in range(q) for j in torch.nonzero(R.sees(L - q + t, L, window, sinks)).flatten().tolist()} for q, L in reqs]
    cache, bt = paged(lens, KVH, PS, D, fmt, 5 * KVH + D + sum(lens), sound)
    T = sum(q for q, _ in reqs) + 3
    q = torch.randn(T, HQ, D, generator=gen(T)).to(torch.bfloat16)
    rows_, at = [], 1
    for b, (n, L) in enumerate(reqs):
        rows_.append((b, at, at + n, L))
        at += n
    view, _ = put(cache)
    flat, st = Lt.b8_views(view, KVH, D)
    one, sm = torch.ones(KVH), 0.7 * D ** -0.5
    ws = K.alloc_workspace(len(reqs), KVH, G, D, 1)
    for dtype, qt, sign, want_lse, host in ((torch.float32, torch.bfloat16, 1, True, None), (torch.bfloat16, torch.bfloat16, -1, False, None),
                                            (torch.float32, torch.float16, 1, True, _lib._NoHost())):
        out = torch.full((T, HQ, D), float("nan"), dtype=dtype, device="cuda")
        lse = torch.full((T, HQ), 5.0, device="cuda") if want_lse else None
        was, _lib._host = _lib._host, host or _lib._host
        try:
            K.prefill_b8(q.to(qt).cuda(), flat, st, PS, bt.cuda(), rows_, sign * sm, 2.0, KVH, out, fmt=fmt, window=window, sinks=sinks,
                         chunk=chunk, workspace=ws, lse=lse)
        finally:
            _lib._host = was
        assert K.workspace_status(ws) == 0
        assert bool(out[0].isnan().all()) and bool(out[-2:].isnan().all())
        for b, a, e, L in rows_:
            check_rows(out[a:e].cpu(), None if lse is None else lse[a:e].cpu(), cache, bt, b, L, q[a:e].to(qt), KVH, PS, fmt, sign * sm, one, 2 * one,
                       window, sinks, D, 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23, True)


# ------------------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,G", [(128, 2, 4), (256, 2, 8)])
def test_a_server_s_steps(fmt, D, KVH, G):
    """two prompts, then tokens one by one from a captured graph, every step's cache and rows against the definitions"""
    HQ, PS, prompts, steps = KVH * G, 16, [37, 16], 20
    t, one, sm = table(500, D, torch.float32), torch.ones(KVH), D ** -0.5
    lens = list(prompts)
    bt = (torch.randperm(16, generator=gen(1)) + 1).to(torch.int32).view(2, 8)
    cache = torch.full((17, 2 * KVH, PS, D + 1), 0x7f, dtype=torch.uint8)         # (stale bytes everywhere, scales among them)
    dev = cache.cuda()
    flat, st = Lt.b8_views(dev, KVH, D)
    ws = K.alloc_workspace(2, KVH, G, D, 1)
    slot = lambda b, p: int(bt[b, p // PS]) * PS + p % PS  # noqa: E731
    NT = sum(prompts)
    x = qkv(NT, HQ, KVH, D, 77)
    pos = torch.cat([torch.arange(n) for n in prompts])
    slots = torch.tensor([slot(b, p) for b, n in enumerate(prompts) for p in range(n)])
    q, k, v = parts(x.cuda(), HQ, KVH, D)
    qo, out = torch.zeros(NT, HQ, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(NT, HQ, D, dtype=torch.bfloat16, device="cuda")
    K.write_rotary_b8(q, k, v, flat, st, PS, slots.cuda(), pos.cuda(), t.cuda(), one.cuda(), one.cuda(), qo, fmt=fmt)
    K.prefill_b8(qo, flat, st, PS, bt.cuda(), [(0, 0, 37, 37), (1, 37, 53, 16)], sm, 1.0, KVH, out, fmt=fmt, workspace=ws)
    cache = R.append(cache, R.turn(k.cpu(), pos, t, False), v.cpu(), slots.tolist(), one, one, fmt)
    assert torch.equal(R.unpack(dev.cpu())[1].view(torch.int32), R.unpack(cache)[1].view(torch.int32))
    for b, a, e, L in ((0, 0, 37, 37), (1, 37, 53, 16)):
        check_rows(out[a:e].cpu(), None, cache, bt, b, L, qo[a:e].cpu(), KVH, PS, fmt, sm, one, one, 0, 0, D, 2.0 ** -8, True)
    # a step: fixed buffers, captured once
    x1 = torch.zeros(3, (HQ + 2 * KVH) * D, dtype=torch.bfloat16, device="cuda")
    q1, k1, v1 = parts(x1, HQ, KVH, D)
    p1, s1 = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.full((3,), -1, dtype=torch.int64, device="cuda")
    lens_d = torch.tensor(lens + [0], dtype=torch.int32).cuda()
    bt_d = torch.cat((bt, torch.zeros(1, 8, dtype=torch.int32))).cuda()
    qsl = torch.tensor([0, 1, 2, 2], dtype=torch.int32).cuda()                     # (a third row of the graph has no request)
    qo1, o1, l1 = torch.zeros_like(q1.contiguous()), torch.zeros(3, HQ, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, HQ, device="cuda")
    g, td = one.cuda(), t.cuda()

    def step():
        K.write_rotary_b8(q1, k1, v1, flat, st, PS, s1, p1, td, g, g, qo1, fmt=fmt)
        K.decode_b8(qo1, flat, st, PS, bt_d, lens_d, qsl, sm, 1.0, g, g, 1, o1, ws, fmt=fmt, lse=l1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        x1.copy_(qkv(3, HQ, KVH, D, 1000 + i) * (1.0 if i % 3 else 2.5))
        p = torch.tensor([lens[0], lens[1], 0])
        s = torch.tensor([slot(0, lens[0]), slot(1, lens[1]), -1])
        lens = [n + 1 for n in lens]
        p1.copy_(p), s1.copy_(s), lens_d.copy_(torch.tensor(lens + [0], dtype=torch.int32))
        graph.replay()
        cache = R.append(cache, R.turn(k1.cpu(), p, t, False), v1.cpu(), s.tolist(), one, one, fmt)
        for b, L in enumerate(lens):
            a, w = R.unpack(dev.cpu()), R.unpack(cache)
            page = bt[b, torch.arange(L) // PS].long()
            r = torch.arange(L) % PS
            assert torch.equal(a[0][page, :, r], w[0][page, :, r]) and torch.equal(a[1][page, :, r // 16], w[1][page, :, r // 16])
            check_rows(o1[b:b + 1].cpu(), l1[b:b + 1].cpu(), cache, bt, b, L, qo1[b:b + 1].cpu(), KVH, PS, fmt, sm, one, one, 0, 0, D, 2.0 ** -8, False)
    assert K.workspace_status(ws) == 0
