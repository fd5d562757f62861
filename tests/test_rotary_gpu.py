"""Keys and queries turned by their positions on the way into the NVFP4 cache: the queries bit for bit those of the formula in fp32
steps and within their rounding of the one in 64 bits, the cache's bytes those of a write over the turned keys."""
import pytest
import torch

import b8_ref as R
from horizon_kernels_b200 import _lib
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def table(rows, rot, dtype, base=10000.0):
    half = rot // 2
    a = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat((a.cos(), a.sin()), 1).to(dtype)


def qkv(NT, HQ, KVH, D, seed):
    x = torch.randn(NT, (HQ + 2 * KVH) * D, generator=gen(seed)).to(torch.bfloat16)
    x[:, HQ * D:(HQ + KVH) * D] *= torch.where(torch.arange(KVH * D) % 37 == 3, 20.0, 1.0).to(torch.bfloat16)
    return x


def parts(x, HQ, KVH, D):
    return [t.view(x.shape[0], -1, D) for t in x.split((HQ * D, KVH * D, KVH * D), 1)]


def cache_of(order, pages, PS, KVH, D, k8):
    heads, slot = (KVH, Lt.K8_SLOT) if k8 else (2 * KVH, Lt.slot_bytes(D))
    if order == "nhd":
        phys = torch.full((pages, PS, heads, slot), 0xa5, dtype=torch.uint8, device="cuda")
        c = phys.permute(0, 2, 1, 3)
    else:
        phys = c = torch.full((pages, heads, PS, slot), 0xa5, dtype=torch.uint8, device="cuda")
    if k8:
        flat, st = Lt.k8_flat_views(*Lt.k8_views(c, D))
    elif order == "region":
        flat, st = Lt.flat_views(*Lt.split_views(c, KVH))
    else:
        flat, st = Lt.flat_views(*Lt.slot_views(c, KVH, D))
    return phys, flat, st


def check_queries(got, q, positions, t, interleaved):
    got = got.cpu()
    assert torch.equal(got.view(torch.int16), R.turn(q, positions, t, interleaved).view(torch.int16))
    want, mag = R.turn(q, positions, t, interleaved, exact=True)
    # two products and a sum, half a step of fp32 each, then half a step of bf16
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 3 * 2.0 ** -24 * (1 + 2.0 ** -8) * mag + 2.0 ** -134).all())


CASES = [(128, 8, 32, 128, False, torch.float32, "slot", {}, 5, 0), (128, 8, 32, 128, False, torch.float32, "slot", {}, 301, 7),
         (128, 2, 6, 64, True, torch.bfloat16, "nhd", {}, 33, 1), (128, 1, 1, 16, False, torch.bfloat16, "region", {}, 19, 0),
         (128, 4, 12, 112, False, torch.float32, "slot", {"had": True}, 70, 3), (256, 2, 16, 256, True, torch.float32, "slot", {}, 17, 2),
         (256, 4, 24, 64, False, torch.bfloat16, "nhd", {}, 400, 0), (256, 2, 10, 48, False, torch.float32, "slot", {"k8": True}, 25, 4),
         (256, 2, 16, 240, True, torch.float32, "slot", {"had": True}, 9, 0), (256, 1, 5, 256, False, torch.bfloat16, "region", {}, 1, 0),
         (128, 8, 32, 128, True, torch.float32, "slot", {"plain": True}, 190, 0), (128, 3, 9, 128, False, torch.float32, "slot", {}, 0, 6)]


@pytest.mark.parametrize("D,KVH,HQ,rot,interleaved,dtype,order,opt,n,pad", CASES)
def test_rotary_write(D, KVH, HQ, rot, interleaved, dtype, order, opt, n, pad):
    PS, NT = 16, n + pad
    x = qkv(NT, HQ, KVH, D, 7 * D + n)
    t = table(900, rot, dtype)
    pos = torch.randint(-3, 905, (NT,), generator=gen(n))              # (some outside the table: the nearest row)
    pages = (n + PS - 1) // PS + 2
    slots = torch.randperm(pages * PS, generator=gen(n + 1))[:n]
    slots[2::5] = -1
    slots = torch.cat((slots, torch.full((pad // 2,), -1)))             # (the rest of the tokens have no entry at all)
    gk, gv = torch.rand(KVH, generator=gen(3)) * 0.02 + 0.002, torch.rand(KVH, generator=gen(4)) * 0.02 + 0.002
    signs = K.hadamard_signs(D, device="cuda") if opt.get("had") else None
    more = dict(search=not opt.get("plain"), signs=signs, k8=bool(opt.get("k8")))
    dev = x.cuda()
    q, k, v = parts(dev, HQ, KVH, D)
    ref, flat_r, st = cache_of(order, pages, PS, KVH, D, more["k8"])
    turned = R.turn(k.cpu(), pos, t, interleaved).cuda() if NT else k
    K.write(turned, v, flat_r, st, PS, slots.cuda(), gk.cuda(), gv.cuda(), **more)
    for host in (None, _lib._NoHost()):                                 # natively and through ctypes
        was, _lib._host = _lib._host, host or _lib._host
        try:
            phys, flat, st = cache_of(order, pages, PS, KVH, D, more["k8"])
            out = torch.full((NT, HQ, D), float("nan"), dtype=torch.bfloat16, device="cuda")
            got = K.write_rotary(q, k, v, flat, st, PS, slots.cuda(), pos.cuda(), t.cuda(), gk.cuda(), gv.cuda(), out, interleaved=interleaved,
                                 **more)
        finally:
            _lib._host = was
        assert got is out
        check_queries(out, q.cpu(), pos, t, interleaved)
        assert torch.equal(phys, ref)
        assert torch.equal(dev.cpu().view(torch.int16), x.view(torch.int16))          # nothing but the outputs is written
    # the queries where they lie
    phys, flat, st = cache_of(order, pages, PS, KVH, D, more["k8"])
    K.write_rotary(q, k, v, flat, st, PS, slots.cuda(), pos.cuda(), t.cuda(), gk.cuda(), gv.cuda(), q, interleaved=interleaved, **more)
    assert torch.equal(q.reshape(out.shape), out) and torch.equal(phys, ref)
    assert torch.equal(dev[:, HQ * D:].cpu().view(torch.int16), x[:, HQ * D:].contiguous().view(torch.int16))


def test_rows_of_any_stride():
    """queries whose heads lie apart and keys whose tokens do, on a stream of their own"""
    D, KVH, HQ, NT, PS = 128, 2, 4, 21, 32
    q = torch.randn(NT, HQ, 2 * D, generator=gen(1)).to(torch.bfloat16).cuda()[..., :D]
    out = torch.zeros(HQ, NT, D, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    kv = torch.randn(KVH, 2 * NT, D, generator=gen(2)).to(torch.bfloat16).cuda()
    k, v = kv[:, ::2].transpose(0, 1), kv[:, 1::2].transpose(0, 1)
    t, pos = table(100, D, torch.float32), torch.arange(NT) * 3 + 5
    slots = torch.arange(NT).flip(0).contiguous()
    g = torch.full((KVH,), 0.01, device="cuda")
    phys, flat, st = cache_of("slot", 2, PS, KVH, D, False)
    ref, flat_r, _ = cache_of("slot", 2, PS, KVH, D, False)
    s = torch.cuda.Stream()
    args = slots.cuda(), pos.cuda(), t.cuda()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.write_rotary(q, k, v, flat, st, PS, *args, g, g, out)
    s.synchronize()
    check_queries(out, q.cpu(), pos, t, False)
    K.write(R.turn(k.cpu(), pos, t, False).cuda(), v, flat_r, st, PS, args[0], g, g)
    assert torch.equal(phys, ref)


def test_overlapping_outputs_are_refused_through_every_path():
    D, KVH, HQ, NT, PS = 128, 2, 4, 6, 16
    buf = torch.zeros(NT + 1, HQ, D, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(NT, KVH, D, dtype=torch.bfloat16, device="cuda")
    phys, flat, st = cache_of("slot", 2, PS, KVH, D, False)
    slots, pos, t = torch.arange(NT).cuda(), torch.arange(NT).cuda(), table(50, D, torch.float32).cuda()
    g = torch.ones(KVH, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        K.write_rotary(buf[:-1], k, k, flat, st, PS, slots, pos, t, g, g, buf[1:])
    with pytest.raises((ValueError, _lib.HkvError)):
        K.write_rotary(buf[:-1], k, k, flat, st, PS, slots, pos, t, g, g, torch.zeros(1, HQ, D, dtype=torch.bfloat16, device="cuda").expand(NT, -1, -1))
    assert bool((phys == 0xa5).all())


def test_graph_replays_with_new_positions_and_slots():
    D, KVH, HQ, NT, PS = 128, 8, 32, 12, 16
    t = table(5000, D, torch.float32)
    x = qkv(NT, HQ, KVH, D, 5).cuda()
    q, k, v = parts(x, HQ, KVH, D)
    out = torch.zeros(NT, HQ, D, dtype=torch.bfloat16, device="cuda")
    slots, pos = torch.zeros(NT, dtype=torch.int64, device="cuda"), torch.zeros(NT, dtype=torch.int64, device="cuda")
    slots.copy_(torch.arange(NT))
    phys, flat, st = cache_of("slot", 8, PS, KVH, D, False)
    g, td = torch.full((KVH,), 0.01, device="cuda"), t.cuda()
    K.write_rotary(q, k, v, flat, st, PS, slots, pos, td, g, g, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.write_rotary(q, k, v, flat, st, PS, slots, pos, td, g, g, out)
    ref, flat_r, _ = cache_of("slot", 8, PS, KVH, D, False)
    phys.copy_(ref)
    for i in range(3):
        p = torch.randint(0, 5000, (NT,), generator=gen(i))
        s = torch.randperm(8 * PS, generator=gen(i + 9))[:NT]
        x.copy_(qkv(NT, HQ, KVH, D, 20 + i))
        pos.copy_(p)
        slots.copy_(s)
        graph.replay()
        check_queries(out, q.cpu(), p, t, False)
        K.write(R.turn(k.cpu(), p, t, False).cuda(), v, flat_r, st, PS, s.cuda(), g, g)
        assert torch.equal(phys, ref)
