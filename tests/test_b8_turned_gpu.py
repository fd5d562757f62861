"""Appending to the 8-bit cache with the rotation of the keys on the way and without it, where a tile's tokens come in any order, leave
gaps, name a slot more than once or fill more entries than a warp has lanes: byte for byte what the definition says, for batches on both
sides of every line that the write draws by their size."""
import pytest
import torch

import b8_ref as R
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt
from test_b8_gpu import fresh, put, same
from test_rotary_gpu import check_queries, gen, parts, qkv, table

pytestmark = pytest.mark.gpu


def slots_of(kind, n, tiles, seed):
    """n slots, a tile's side by side: `kind` is the order of a tile's rows, or "mixed": all of them in one batch"""
    g = gen(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    kinds = ("ascending", "descending", "gaps", "shuffled", "twice", "long", "single", "whole", "skip")
    out, order = [], torch.randperm(tiles, generator=g).tolist()
    while sum(map(len, out)) < n:
        k = kinds[pick(0, len(kinds))] if kind == "mixed" else kind
        first, m = pick(0, 16), pick(2, 13)
        if k == "ascending":
            r = torch.arange(first, 16)
        elif k == "descending":
            r = torch.arange(first, -1, -1)
        elif k == "gaps":
            r = torch.arange(first % 3, 16, 2 + first % 3)
        elif k == "shuffled":
            r = torch.randperm(16, generator=g)[:m]
        elif k == "twice":
            r = torch.randint(0, 16, (m,), generator=g)
        elif k == "long":
            r = torch.cat((torch.arange(first, 16), torch.randint(0, 16, (pick(20, 50),), generator=g)))
        elif k == "single":
            r = torch.tensor([first])
        elif k == "whole":
            r = torch.arange(16)
        else:
            r = torch.full((pick(1, 4),), -1)
        out.append(r if k == "skip" else r + 16 * order.pop())
    return torch.cat(out)[:n]


def tiles_for(kind, n):
    return n if kind == "single" else n // 2 + 40


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,HQ,rot,interleaved,dtype", [(128, 2, 4, 128, False, torch.float32), (256, 1, 3, 64, True, torch.bfloat16)])
@pytest.mark.parametrize("kind,n", [("descending", 4), ("gaps", 6), ("twice", 9), ("shuffled", 100), ("long", 300), ("descending", 513), ("mixed", 512),
                                    ("mixed", 1000), ("long", 2047), ("mixed", 2048), ("shuffled", 3000), ("mixed", 8191), ("mixed", 8192),
                                    ("long", 8300), ("descending", 9001)])
def test_order_of_a_tile_s_tokens(fmt, D, KVH, HQ, rot, interleaved, dtype, kind, n):
    """two calls over the same tiles; every token has a position of its own"""
    PS, tiles = 32, tiles_for(kind, n)
    tiles += tiles % 2
    t = table(n + 50, rot, dtype)
    one = torch.tensor([1.0, 0.5])[:KVH]
    cache = fresh(tiles // 2, KVH, PS, D, fmt, n + D)
    view, _ = put(cache)
    flat, st = Lt.b8_views(view, KVH, D)
    for step in range(2):
        slots = slots_of(kind, n, tiles, 7 * n + step)
        pos = torch.randperm(n + 50, generator=gen(n + step))[:n]
        x = qkv(n, HQ, KVH, D, n + 3 * step)
        x *= 2.0 ** torch.randint(-3, 4, (n, 1), generator=gen(n + 5 * step)).to(torch.bfloat16)
        q, k, v = parts(x.cuda(), HQ, KVH, D)
        out = torch.full((n, HQ, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        K.write_rotary_b8(q, k, v, flat, st, PS, slots.cuda(), pos.cuda(), t.cuda(), one.cuda(), one.cuda(), out, interleaved=interleaved, fmt=fmt)
        check_queries(out, q.cpu(), pos, t, interleaved)
        cache = R.append(cache, R.turn(k.cpu(), pos, t, interleaved), v.cpu(), slots.tolist(), one, one, fmt)
        same(view.cpu(), cache, fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("D,KVH", [(128, 1), (128, 4), (128, 5), (256, 2), (256, 7)])
@pytest.mark.parametrize("n", [700, 2100, 8200])
def test_large_batches_of_every_kind(fmt, turned, D, KVH, n):
    """prompts from and to the middle of a tile, drafts, single tokens, repeated and shuffled rows and skipped tokens in one call, for heads of
    one CTA and of several; the second call grows the scales of the first one's tiles. What is without a slot at the end stays unread"""
    PS, HQ = 64, KVH
    cache = fresh(n // 6 + 20, KVH, PS, D, fmt, n + D)
    one = torch.tensor([1.0, 0.5, 2.0, 0.37, 4.0, 1.0, 1.0])[:KVH]
    view, _ = put(cache)
    flat, st = Lt.b8_views(view, KVH, D)
    t = table(300, D, torch.float32)
    for step in range(2):
        slots, tiles = slots_of("mixed", n // 2, n // 2, n + step), torch.arange(n // 2, n) * 16
        prompts, at = [], 0                                             # of 17 to 400 tokens, each in tiles of its own
        while sum(map(len, prompts)) < n - n // 2:
            m, first = int(torch.randint(17, 400, (1,), generator=gen(n + at))), int(torch.randint(0, 16, (1,), generator=gen(n + at + 1)))
            prompts.append(int(tiles[at]) + first + torch.arange(m))
            at += (first + m + 15) // 16
        slots = torch.cat((slots, *prompts))[:n]
        assert int(slots.max()) < len(cache) * PS
        pos = torch.randint(0, 300, (n + 3,), generator=gen(n + step))
        x = qkv(n + 3, HQ, KVH, D, n + 3 * step)
        x *= 2.0 ** (torch.randint(-3, 4, (n + 3, 1), generator=gen(n + 5 * step)) + step).to(torch.bfloat16)
        q, k, v = parts(x.cuda(), HQ, KVH, D)
        if turned:
            out = torch.zeros(n + 3, HQ, D, dtype=torch.bfloat16, device="cuda")
            K.write_rotary_b8(q, k, v, flat, st, PS, slots.cuda(), pos.cuda(), t.cuda(), one.cuda(), one.cuda(), out, fmt=fmt)
            check_queries(out, q.cpu(), pos, t, False)
        else:
            K.write_b8(k, v, flat, st, PS, slots.cuda(), one.cuda(), one.cuda(), fmt=fmt)
        cache = R.append(cache, R.turn(k.cpu(), pos, t, False) if turned else k.cpu(), v.cpu(), slots.tolist(), one, one, fmt)
        same(view.cpu(), cache, fmt)
