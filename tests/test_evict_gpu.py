"""kernels.evict against a plain sort: which tokens stay, their slots byte for byte, their weights, the new lengths, and that
nothing else of the cache changes."""
import numpy as np
import pytest
import torch

import window_ref as R
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt

pytestmark = pytest.mark.gpu


def cache_of(kind, pages, PS, KVH, D, g):
    if kind == "k8":
        shape = (pages, KVH, PS, Lt.K8_SLOT)
    elif kind == "nhd":
        shape = (pages, PS, 2 * KVH, Lt.slot_bytes(D))
    else:
        shape = (pages, 2 * KVH, PS, Lt.slot_bytes(D))
    phys = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
    v = R.views(phys, kind, KVH, D)
    flat, st = Lt.k8_flat_views(*v) if kind == "k8" else Lt.flat_views(*v)
    return phys, flat, st


def weights_of(how, B, H, W, g):
    w = torch.exp(2 * torch.randn(B, H, W, device="cuda", generator=g))
    if how == "ties":                     # a few values, zeros of both signs among them
        w = torch.randint(-1, 3, (B, H, W), device="cuda", generator=g).float() * 0.5
        w[..., ::7] = -0.0
    elif how == "equal":
        w.fill_(0.25)
    elif how == "special":
        w[..., ::5] = float("inf")
        w[..., 1::11] = float("nan")
        w[..., 2::13] = -float("inf")
        w[..., 3::17] = 1e-42              # subnormal
    elif how == "near":                    # neighbours in the last bits, below one common prefix
        w = (torch.randint(0, 1024, (B, H, W), device="cuda", generator=g, dtype=torch.int32) + 0x3f800000).view(torch.float32)
    return w


def call(kind, lens, keep, sinks, recent, KVH, D, PS, how="plain", where="new", seed=0, extra=0, garbage_beyond=True):
    """one call; everything that may and may not change is checked"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(lens)
    per = [max(1, -(-L // PS)) for L in lens]
    MP = max(per)
    OMP = -(-keep // PS)
    total = sum(max(p, OMP) for p in per) + (B * OMP if where == "new" else 0) + 3
    phys, flat, st = cache_of(kind, total, PS, KVH, D, g)
    perm = torch.randperm(total - 1, device="cuda", generator=g).to(torch.int32) + 1
    bt = torch.zeros((B, max(MP, OMP)), dtype=torch.int32, device="cuda")
    o = 0
    for b, p in enumerate(per):
        n = max(p, OMP)
        bt[b, :n] = perm[o:o + n]
        o += n
    W = max(max(lens), keep, 1) + extra
    w = weights_of(how, B, KVH, W, g)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept = torch.full((B, KVH, keep), -7, dtype=torch.int32, device="cuda")
    out_lens = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    ot = perm[o:o + B * OMP].view(B, OMP).contiguous() if where == "new" else None
    ow = torch.full((B, KVH, keep + 5), -3.0, device="cuda") if where == "new" else None
    before, w0 = phys.clone(), w.clone()
    K.evict(flat, st, PS, D, bt, sl, w, keep, sinks, recent, kept, out_lens, out_tables=ot, out_weights=ow, k8=kind == "k8")
    torch.cuda.synchronize()
    # the plain form
    want = before.cpu().clone()
    vb, vw = R.views(before.cpu(), kind, KVH, D), R.views(want, kind, KVH, D)
    new_w = (ow if ow is not None else w).cpu()
    tab = (ot if ot is not None else bt).cpu().long()
    bt_c = bt.cpu().long()
    for b, L in enumerate(lens):
        n = min(L, keep)
        assert int(out_lens[b]) == n
        for h in range(KVH):
            stay = R.kept_positions(w0[b, h, :L].cpu().numpy(), keep, sinks, recent)
            got = kept[b, h].cpu().numpy()
            assert np.array_equal(got[:n], stay), (b, h, L)
            assert (got[n:] == -1).all()
            j, r = torch.from_numpy(stay).long(), torch.arange(n)
            for x, y in zip(vb, vw):
                y[tab[b][r // PS], r % PS, h] = x[bt_c[b][j // PS], j % PS, h]
            assert torch.equal(new_w[b, h, :n].view(torch.int32), w0[b, h].cpu()[j].view(torch.int32))
            end = min(L, new_w.shape[2])
            assert (new_w[b, h, n:end] == 0).all()
            rest = new_w[b, h, max(n, end):]
            assert torch.equal(rest.view(torch.int32), (w0[b, h, max(n, end):].cpu() if ow is None else torch.full_like(rest, -3.0)).view(torch.int32))
    if ow is not None:
        assert torch.equal(w.view(torch.int32), w0.view(torch.int32))
    assert torch.equal(phys.cpu(), want)


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("kind,KVH,D,PS", [("hnd", 8, 128, 16), ("nhd", 2, 128, 32), ("region", 2, 128, 16), ("hnd", 2, 256, 64), ("nhd", 4, 256, 16),
                                           ("region", 2, 256, 32), ("k8", 2, 256, 16)])
def test_layouts(kind, KVH, D, PS, where):
    call(kind, [777, 40, 100, 1500], 100, 4, 30, KVH, D, PS, where=where, seed=D + KVH)


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("how", ["ties", "equal", "special", "near"])
def test_order_of_weights(how, where):
    call("hnd", [3000, 513, 700], 500, 3, 100, 2, 128, 16, how=how, where=where, seed=5)


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("lens,keep,sinks,recent", [
    ([0, 1, 2, 3], 1, 0, 0), ([0, 1, 2, 3], 1, 1, 0), ([0, 1, 2, 3], 1, 0, 1), ([5, 17, 1], 4, 2, 2), ([17, 33, 16], 16, 0, 16),
    ([17, 33, 16], 16, 16, 0), ([100, 101, 99], 100, 0, 0), ([64], 63, 0, 0), ([4097], 4096, 1, 4000), ([1], 1000, 4, 500),
    ([9000], 2, 1, 1), ([9000], 1, 0, 0)])
def test_small_and_borders(lens, keep, sinks, recent, where):
    call("hnd", lens, keep, sinks, recent, 2, 128, 16, where=where, seed=len(lens) + keep, extra=3)


@pytest.mark.parametrize("lens,keep,KVH,D,how,where", [
    ([70000], 3001, 1, 128, "plain", "own"), ([200001, 5], 20000, 1, 128, "plain", "new"), ([180000], 170000, 2, 128, "ties", "own"),
    ([40000, 16000], 12345, 2, 256, "near", "own")])
def test_long(lens, keep, KVH, D, how, where):
    """more tokens than the CTAs of a cluster hold weights of, and more than one round of moves"""
    call("hnd", lens, keep, 4, 1000, KVH, D, 32, how=how, where=where, seed=3)


def test_many_requests():
    rng = np.random.default_rng(0)
    call("hnd", [int(x) for x in rng.integers(0, 400, 300)], 64, 2, 10, 4, 128, 16, where="own", seed=9)


def test_repeats_on_another_stream_and_in_a_graph():
    """a captured call, replayed on changed weights and lengths, and a call on a side stream: the bits of the plain calls"""
    g = torch.Generator(device="cuda").manual_seed(1)
    PS, KVH, D, keep = 16, 2, 128, 128
    phys, flat, st = cache_of("hnd", 200, PS, KVH, D, g)
    src = phys.clone()
    bt = (torch.randperm(180, device="cuda", generator=g).to(torch.int32) + 1).view(3, 60)
    ot = torch.arange(181, 205, dtype=torch.int32, device="cuda").view(3, 8)
    ot[2] = bt[2, :8]                                   # one request in place, two to new pages
    w = torch.rand(3, KVH, 960, device="cuda", generator=g)
    sl = torch.tensor([960, 300, 700], dtype=torch.int32, device="cuda")
    kept, ol = torch.zeros((3, KVH, keep), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    ow = torch.zeros(3, KVH, keep, device="cuda")

    def go():
        K.evict(flat, st, PS, D, bt, sl, w, keep, 4, 16, kept, ol, out_tables=ot, out_weights=ow)

    def result():
        torch.cuda.synchronize()
        return [t.clone() for t in (phys, kept, ol, ow)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        go()
    first = result()
    phys.copy_(src)
    go()
    assert all(torch.equal(a, b) for a, b in zip(first, result()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        with torch.cuda.graph(graph, stream=side):
            go()
    w.copy_(torch.rand(3, KVH, 960, device="cuda", generator=g))
    sl.copy_(torch.tensor([100, 960, 129], dtype=torch.int32))
    phys.copy_(src)
    go()
    plain = result()
    phys.copy_(src)
    for t in (kept, ol, ow):
        t.fill_(9)
    ow.copy_(plain[3].new_zeros(ow.shape))
    graph.replay()
    replayed = result()
    for a, b in zip(plain[:3], replayed[:3]):
        assert torch.equal(a, b)
    assert torch.equal(plain[3][1:], replayed[3][1:])   # (request 0 keeps all of its 100 tokens: entries beyond are not written)
    assert torch.equal(plain[3][0, :, :100], replayed[3][0, :, :100])


def test_lengths_beyond_the_table_and_the_weights_are_cut():
    g = torch.Generator(device="cuda").manual_seed(2)
    phys, flat, st = cache_of("hnd", 40, 16, 2, 128, g)
    bt = torch.arange(1, 33, dtype=torch.int32, device="cuda").view(2, 16)
    w = torch.rand(2, 2, 200, device="cuda", generator=g)
    sl = torch.tensor([100000, -5], dtype=torch.int32, device="cuda")
    kept, ol = torch.zeros((2, 2, 32), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    w0 = w.clone()
    K.evict(flat, st, 16, 128, bt, sl, w, 32, 0, 0, kept, ol)
    assert ol.tolist() == [32, 0] and (kept[1] == -1).all()
    for h in range(2):
        assert np.array_equal(kept[0, h].cpu().numpy(), R.kept_positions(w0[0, h].cpu().numpy(), 32, 0, 0))


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("D,offset,pad", [(128, 8, 0), (128, 0, 8), (128, 24, 40), (256, 16, 48), (256, 48, 16)])
def test_caches_off_the_16_byte_grid(D, offset, pad, where):
    """a cache that begins at, or whose pages are apart by, an odd multiple of 8 bytes (head_dim 128), where no bulk copy may go"""
    g = torch.Generator(device="cuda").manual_seed(4)
    KVH, PS, pages, keep, L = 2, 16, 60, 70, 400
    slot = Lt.slot_bytes(D)
    page = 2 * KVH * PS * slot + pad
    mem = torch.randint(0, 256, (offset + pages * page,), dtype=torch.uint8, device="cuda", generator=g)
    cache = torch.as_strided(mem, (pages, 2 * KVH, PS, slot), (page, PS * slot, slot, 1), offset)
    flat, st = Lt.flat_views(*Lt.slot_views(cache, KVH, D))
    bt = torch.arange(1, 26, dtype=torch.int32, device="cuda").view(1, 25)
    ot = torch.arange(30, 35, dtype=torch.int32, device="cuda").view(1, 5) if where == "new" else None
    w = torch.rand(1, KVH, L, device="cuda", generator=g)
    w0, before = w.cpu(), mem.cpu().clone()
    kept, ol = torch.zeros((1, KVH, keep), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    K.evict(flat, st, PS, D, bt, torch.tensor([L], dtype=torch.int32, device="cuda"), w, keep, 2, 9, kept, ol, out_tables=ot,
            out_weights=None if ot is None else torch.zeros(1, KVH, keep, device="cuda"))
    want = before.clone()
    old, new = (torch.as_strided(m, cache.shape, cache.stride(), offset) for m in (before, want))
    tab = (bt if ot is None else ot).cpu().long()[0]
    r = torch.arange(keep)
    for h in range(KVH):
        j = torch.from_numpy(R.kept_positions(w0[0, h].numpy(), keep, 2, 9))
        for side in (h, KVH + h):
            new[tab[r // PS], side, r % PS] = old[bt.cpu().long()[0][j // PS], side, j % PS]
    assert torch.equal(mem.cpu(), want)


def test_pages_shared_by_requests_move_to_new_ones():
    """a prefix that two requests share is read by both and stays as it is"""
    g = torch.Generator(device="cuda").manual_seed(6)
    phys, flat, st = cache_of("hnd", 60, 16, 2, 128, g)
    bt = torch.tensor([list(range(1, 21)), list(range(1, 11)) + list(range(21, 31))], dtype=torch.int32, device="cuda")
    ot = torch.arange(40, 50, dtype=torch.int32, device="cuda").view(2, 5)
    w = torch.rand(2, 2, 320, device="cuda", generator=g)
    kept, ol = torch.zeros((2, 2, 80), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    ow, before = torch.zeros(2, 2, 80, device="cuda"), phys.cpu().clone()
    K.evict(flat, st, 16, 128, bt, torch.tensor([320, 311], dtype=torch.int32, device="cuda"), w, 80, 4, 16, kept, ol, out_tables=ot, out_weights=ow)
    after = phys.cpu()
    assert torch.equal(after[:40], before[:40])
    r = torch.arange(80)
    for b in range(2):
        for h in range(2):
            j = kept[b, h].long().cpu()
            for side in (h, 2 + h):
                assert torch.equal(after[ot[b].long().cpu()[r // 16], side, r % 16], before[bt[b].long().cpu()[j // 16], side, j % 16])


def test_weights_that_are_rows_of_a_wider_tensor():
    g = torch.Generator(device="cuda").manual_seed(8)
    phys, flat, st = cache_of("hnd", 40, 16, 2, 128, g)
    bt = torch.arange(1, 33, dtype=torch.int32, device="cuda").view(2, 16)
    big = torch.rand(2, 3, 2, 300, device="cuda", generator=g)
    w, rest = big[:, 1, :, 20:276], big.clone()
    kept, ol = torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    sl = torch.tensor([256, 100], dtype=torch.int32, device="cuda")
    K.evict(flat, st, 16, 128, bt, sl, w, 64, 1, 5, kept, ol)
    for b, L in enumerate(sl.tolist()):
        for h in range(2):
            old = rest[b, 1, h, 20:276].clone()
            assert torch.equal(w[b, h, :64], old[kept[b, h].long()]) and bool((w[b, h, 64:L] == 0).all()) and torch.equal(w[b, h, L:], old[L:])
    big[:, 1, :, 20:276] = rest[:, 1, :, 20:276]
    assert torch.equal(big, rest)
