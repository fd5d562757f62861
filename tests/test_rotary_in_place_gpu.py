"""Queries turned where they lie: under other views of the same rows, among the heads of keys and values, through the custom
ops. Every entry point, natively and through ctypes."""
import pytest
import torch

import b8_ref as R
from horizon_kernels_b200 import _lib
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt
from horizon_kernels_b200 import ops
from test_b8_gpu import fresh, same
from test_rotary_gpu import cache_of, check_queries, gen, parts, table

pytestmark = pytest.mark.gpu


def in_place(x, query, key, value, out, b8, interleaved=False):
    """one call whose query_out lies on the query; `x` holds all three. Queries, cache and the rest of x as the definition says"""
    (NT, HQ, D), KVH, PS = query.shape, key.shape[1], 16
    t, pos, slots = table(400, D, torch.float32), torch.arange(NT) * 3 + 1, torch.arange(NT) + 5
    g = torch.full((KVH,), 0.01)
    before, q0, k0, v0 = x.cpu(), query.cpu(), key.cpu(), value.cpu()
    for host in (None, _lib._NoHost()):
        x.copy_(before)
        args = slots.cuda(), pos.cuda(), t.cuda(), g.cuda(), g.cuda(), out
        was, _lib._host = _lib._host, host or _lib._host
        try:
            if b8:
                start = fresh(NT // PS + 2, KVH, PS, D, b8, 4)
                cache = start.cuda()
                flat, st = Lt.b8_views(cache, KVH, D)
                K.write_rotary_b8(query, key, value, flat, st, PS, *args, interleaved=interleaved, fmt=b8)
                same(cache, R.append(start, R.turn(k0, pos, t, interleaved), v0, slots.tolist(), g, g, b8), b8)
            else:
                phys, flat, st = cache_of("slot", NT // PS + 2, PS, KVH, D, False)
                ref, flat_r, _ = cache_of("slot", NT // PS + 2, PS, KVH, D, False)
                K.write_rotary(query, key, value, flat, st, PS, *args, interleaved=interleaved)
                K.write(R.turn(k0, pos, t, interleaved).cuda(), v0.cuda(), flat_r, st, PS, args[0], args[3], args[4])
                assert torch.equal(phys, ref)
        finally:
            _lib._host = was
        check_queries(query, q0, pos, t, interleaved)
        assert torch.equal(key.cpu(), k0) and torch.equal(value.cpu(), v0)
        query.copy_(q0)
        assert torch.equal(x.cpu(), before)                             # nothing beside the queries was written


@pytest.mark.parametrize("b8", [None, "e4m3", "int8"])
@pytest.mark.parametrize("NT,HQ", [(1, 8), (1, 1), (9, 1)])
def test_strides_of_single_rows(b8, NT, HQ):
    """one token, or one head: strides that differ where there is nothing to stride over"""
    D, KVH = 128, 1
    W = (HQ + 2 * KVH) * D
    x = torch.randn(NT, W, generator=gen(HQ)).to(torch.bfloat16).cuda()
    q = x.as_strided((NT, HQ, D), (W, D, 1))
    out = x.as_strided((NT, HQ, D), (W if NT > 1 else HQ * D, D if HQ > 1 else 5 * D, 1))
    assert q.stride() != out.stride()
    k, v = (x[:, (HQ + i) * D:(HQ + i + 1) * D].view(NT, 1, D) for i in range(2))
    in_place(x, q, k, v, out, b8)


@pytest.mark.parametrize("b8", [None, "e4m3", "int8"])
@pytest.mark.parametrize("NT,H,interleaved", [(1, 2, False), (21, 4, False), (40, 3, True)])
def test_heads_of_queries_keys_and_values_in_turn(b8, NT, H, interleaved):
    """(tokens, heads, 3, head_dim), as a fused product may leave them"""
    D = 128
    x = torch.randn(NT, H, 3, D, generator=gen(H)).to(torch.bfloat16).cuda()
    in_place(x, x[:, :, 0], x[:, :, 1], x[:, :, 2], x[:, :, 0], b8, interleaved)


@pytest.mark.parametrize("b8", [None, "int8"])
def test_custom_ops_in_place(b8):
    """query_out may be the query, as an out= argument may be an input"""
    hkv = ops.register()
    D, KVH, HQ, PS, NT = 128, 2, 6, 16, 30
    x = torch.randn(NT, (HQ + 2 * KVH) * D, generator=gen(1)).to(torch.bfloat16).cuda()
    q, k, v = parts(x, HQ, KVH, D)
    t, pos, slots = table(200, D, torch.float32).cuda(), torch.arange(NT).cuda() * 5, torch.arange(NT).cuda()
    g, q0 = torch.full((KVH,), 0.02, device="cuda"), q.cpu()
    got = []
    for out in (torch.zeros(NT, HQ, D, dtype=torch.bfloat16, device="cuda"), q):
        if b8:
            cache = torch.zeros((2, 2 * KVH, PS, D + 1), dtype=torch.uint8, device="cuda")
            flat, st = Lt.b8_views(cache, KVH, D)
            hkv.write_rotary_b8(q, k, v, *flat, list(st), PS, slots, pos, t, g, g, False, b8, out)
        else:
            cache, flat, st = cache_of("slot", 2, PS, KVH, D, False)
            hkv.write_rotary(q, k, v, *flat, list(st), PS, slots, pos, t, g, g, False, True, None, False, out)
        check_queries(out, q0, pos.cpu(), t.cpu(), False)
        got.append(cache)
    assert torch.equal(*got) and torch.equal(q.cpu(), out.cpu())
