"""The bytes that the 8-bit cache's writes leave, compared as bytes: the sign of a zero among them."""
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
