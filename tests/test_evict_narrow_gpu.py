"""kernels.evict with weights that are narrower than a context: the first and the last tokens stay by their position, whatever the
weights reach, and of those between the ones without a weight count as lighter than all that have one."""
import numpy as np
import pytest
import torch

import window_ref as R
from horizon_kernels_b200 import kernels as K
from test_evict_gpu import cache_of, weights_of

pytestmark = pytest.mark.gpu


def stays(w, L, keep, sinks, recent):
    """positions that stay of a context of L, by a plain sort; w has the weights of the first tokens"""
    if L <= keep:
        return np.arange(L)
    x = np.asarray(w, np.float64)

    def rank(j):
        return (2, 0.0, j) if j >= len(x) else (0, 0.0, j) if np.isnan(x[j]) else (1, -x[j], j)
    mid = sorted(range(sinks, L - recent), key=rank)[:keep - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), np.asarray(mid, np.int64), np.arange(L - recent, L)])).astype(np.int64)


def check(lens, W, keep, sinks, recent, KVH=2, D=128, kind="hnd", how="plain", where="new", seed=0):
    PS, B = 16, len(lens)
    g = torch.Generator(device="cuda").manual_seed(seed)
    MP, OMP = max(-(-max(lens) // PS), -(-keep // PS)), -(-keep // PS)
    phys, flat, st = cache_of(kind, B * (MP + OMP) + 1, PS, KVH, D, g)
    perm = torch.randperm(B * (MP + OMP), device="cuda", generator=g).to(torch.int32) + 1
    bt, ot = perm[:B * MP].view(B, MP), perm[B * MP:].view(B, OMP)
    w = weights_of(how, B, KVH, W, g)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept, ol = torch.full((B, KVH, keep), -7, dtype=torch.int32, device="cuda"), torch.full((B,), -7, dtype=torch.int32, device="cuda")
    ow = torch.full((B, KVH, keep + 5), -3.0, device="cuda") if where == "new" else w
    before, w0, ow0 = phys.cpu(), w.cpu(), ow.cpu()
    K.evict(flat, st, PS, D, bt, sl, w, keep, sinks, recent, kept, ol, out_tables=ot if where == "new" else None,
            out_weights=ow if where == "new" else None, k8=kind == "k8")
    want = before.clone()
    vb, vw = R.views(before, kind, KVH, D), R.views(want, kind, KVH, D)
    bt, tab, ow, kept = bt.cpu().long(), (ot if where == "new" else bt).cpu().long(), ow.cpu(), kept.cpu()
    for b, L in enumerate(lens):
        n = min(L, keep)
        assert int(ol[b]) == n
        for h in range(KVH):
            j = torch.from_numpy(stays(w0[b, h].numpy(), L, keep, sinks, recent))
            assert torch.equal(kept[b, h, :n].long(), j) and bool((kept[b, h, n:] == -1).all()), (b, h, L)
            r = torch.arange(n)
            for x, y in zip(vb, vw):
                y[tab[b][r // PS], r % PS, h] = x[bt[b][j // PS], j % PS, h]
            moved = torch.where(j < W, w0[b, h][j.clamp(max=W - 1)], torch.tensor(0.0))
            assert torch.equal(ow[b, h, :n].view(torch.int32), moved.view(torch.int32))
            end = min(L, ow.shape[2])
            assert bool((ow[b, h, n:end] == 0).all())
            assert torch.equal(ow[b, h, max(n, end):].view(torch.int32), ow0[b, h, max(n, end):].view(torch.int32))
    assert torch.equal(phys.cpu(), want)


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("lens,W,keep,sinks,recent", [
    ([400, 300, 260, 90], 300, 100, 4, 20),           # the last tokens lie behind the weights
    ([400, 310, 1000, 80], 300, 100, 4, 0),           # others between do
    ([400, 300, 100], 60, 60, 50, 10), ([400, 61], 60, 60, 0, 60), ([400, 61], 60, 60, 60, 0),
    ([400, 101, 100], 100, 90, 80, 5), ([5000, 9000], 4097, 600, 3, 100), ([400, 500], 64, 64, 0, 10)])
def test_narrow_weights(lens, W, keep, sinks, recent, where):
    check(lens, W, keep, sinks, recent, where=where, seed=W)


@pytest.mark.parametrize("W", [1, 3, 10, 30, 63])
def test_fewer_weights_than_tokens_stay(W):
    """to new places the weights may be narrower than what stays: then every weighted token stays, and the first of the others"""
    check([400, 70, 64, 30], W, 64, 4, 12, where="new", seed=W)


@pytest.mark.parametrize("how", ["special", "ties"])
@pytest.mark.parametrize("kind,D", [("nhd", 256), ("k8", 256), ("region", 128)])
def test_layouts_and_orders(kind, D, how):
    check([700, 333], 400, 128, 4, 30, D=D, kind=kind, how=how, seed=D)


@pytest.mark.parametrize("W", [64, 200, 399])
def test_many_short_contexts(W):
    """more pairs than the clusters' selection is taken for"""
    rng = np.random.default_rng(2)
    check([int(x) for x in rng.integers(0, 400, 150)], W, 64, 2, 10, KVH=4, where="own", how="ties", seed=W)
