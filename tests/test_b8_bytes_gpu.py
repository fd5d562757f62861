"""The bytes that the 8-bit cache's writes leave, compared as bytes: the sign of a zero, and scale words over pages of any
contents."""
import pytest
import torch

import b8_ref as R
from test_b8_gpu import fresh, rows, same, write
from test_rotary_gpu import gen

pytestmark = pytest.mark.gpu


def same_bytes(got, want, fmt):
    """code for code (any NaN is one), the scales and what nobody reads"""
    same(got, want, fmt)
    a, b = R.unpack(got)[0], R.unpack(want)[0]
    nan = R.values(a, fmt).isnan()
    assert torch.equal(a[~nan], b[~nan])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D,KVH,n", [(128, 4, 3), (256, 2, 40), (128, 4, 700), (256, 3, 2200), (128, 2, 8200)])
def test_zeros_keep_their_sign(fmt, D, KVH, n):
    """zeros of both signs, the smallest numbers and those that round to a code of zero, under global scales that are powers of two and
    that are not, of both signs; single tokens over them afterwards, which round codes to a larger scale"""
    PS, g = 16, gen(n)
    gk, gv = torch.tensor([0.37, -0.37, 1.0, -0.25])[:KVH], torch.tensor([3.0, -2.0, -0.011, 1.0])[:KVH]
    small = torch.tensor([0.0, -0.0, 1e-38, -1e-38, 1e-40, -1e-40, 1e-9, -1e-9, -1e-5, 2e-6]).to(torch.bfloat16)
    P = n // PS + 2
    cache = fresh(P, KVH, PS, D, fmt, n + 1)
    k, v = rows(n, KVH, D, n)
    for x in (k, v):
        at = torch.randperm(x.numel(), generator=g)[:x.numel() // 2]
        x.view(-1)[at] = small[torch.randint(0, 10, at.shape, generator=g)]
        x[n // 2] = -0.0
    slots = torch.arange(n) + 5
    want = R.append(cache, k, v, slots.tolist(), gk, gv, fmt)
    same_bytes(write(cache, k, v, slots, gk, gv, fmt, KVH), want, fmt)
    one = torch.arange(1, P, 2) * PS + 3                                # a token of every other page, far larger
    k, v = rows(len(one), KVH, D, n + 7)
    k[..., ::3], v[..., ::5] = -0.0, 0.0
    k, v = k * 64, v * 64
    same_bytes(write(want, k, v, one, gk, gv, fmt, KVH), R.append(want, k, v, one.tolist(), gk, gv, fmt), fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [7, 600, 2200, 8300])
@pytest.mark.parametrize("start", ["one", "few", "many"])
def test_scale_words_of_stale_pages(fmt, n, start):
    """a tile whose first slot the call does not name, over bytes that no write of this cache has left: its scale is a power of two
    afterwards, at least the smallest one that the call's rows need, and these rows are right under it"""
    D, KVH, PS, g = 128, 2, 16, gen(n)
    one = torch.ones(KVH)
    length = {"one": 1, "few": 3, "many": 11}[start]
    P = n // length + 1
    cache = torch.randint(0, 256, (P, 2 * KVH, PS, D + 1), generator=g, dtype=torch.uint8)
    tiles = cache.view(P, 2 * KVH, 16 * D + 16)
    word = torch.randint(110, 140, (P, 2 * KVH), generator=g) << 23 | torch.randint(0, 1 << 23, (P, 2 * KVH), generator=g)
    word |= torch.randint(0, 2, (P, 2 * KVH), generator=g) << 31
    odd = torch.tensor([0, 1, 0x7f800000, 0x7fc00001, 0x80000000, 0xff800000, 0x42f00000, 0xc0800000])
    word[::2] = odd[torch.randint(0, 8, word[::2].shape, generator=g)]
    tiles[..., 16 * D:16 * D + 4] = word.to(torch.int32)[..., None].view(torch.uint8)
    slots = torch.cat([p * PS + 2 + torch.arange(length) for p in torch.randperm(P, generator=g).tolist()])[:n]
    k, v = rows(n, KVH, D, n + 1)
    got = write(cache, k, v, slots, one, one, fmt, KVH)
    codes, scales, rest = R.unpack(got)
    assert torch.equal(rest, R.unpack(cache)[2])
    lo, hi = R.RANGE[fmt]
    x = torch.cat((k, v), 1).double()
    page, row = slots // PS, slots % PS
    touched = torch.zeros(P, dtype=torch.bool)
    touched[page] = True
    top = torch.zeros(P, 2 * KVH, dtype=torch.float64).scatter_reduce(0, page[:, None].expand(-1, 2 * KVH), x.abs().amax(-1), "amax")
    for p in torch.nonzero(touched).flatten().tolist():
        for h in range(2 * KVH):
            old = min(max((int(word[p, h]) >> 23 & 255) - 127, lo), hi)
            want = 2.0 ** max(old, R.exponent(float(top[p, h]), fmt))
            assert float(scales[p, h, 0]) == want, (p, h)
    s = scales[page, :, 0].double()
    assert torch.equal(codes[page, :, row], R.encode(x / s[..., None], fmt))
    assert torch.equal(got[~touched], cache[~touched])
