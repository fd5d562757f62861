"""The plugin surface with the 8-bit cache, the rotation on the way through it, and the torch custom ops of both, on the GPU."""
import os
from types import SimpleNamespace

import pytest
import torch

os.environ["HORIZON_KVFP4_STANDALONE"] = "1"
import b8_ref as R  # noqa: E402
from horizon_kernels_b200 import backend as BE  # noqa: E402
from horizon_kernels_b200 import kernels as K  # noqa: E402
from horizon_kernels_b200 import layout as Lt  # noqa: E402
from horizon_kernels_b200 import ops  # noqa: E402
from test_b8_gpu import check_rows, fresh, paged, same  # noqa: E402
from test_rotary_gpu import cache_of, check_queries, gen, parts, qkv, table  # noqa: E402

pytestmark = pytest.mark.gpu


def metadata(lens, qls, bt):
    qsl = torch.tensor([0] + qls).cumsum(0).to(torch.int32)
    cam = SimpleNamespace(num_reqs=len(lens), num_actual_tokens=int(qsl[-1]), query_start_loc=qsl.cuda(), query_start_loc_cpu=qsl,
                          seq_lens=torch.tensor(lens, dtype=torch.int32).cuda(), block_table_tensor=bt.cuda(),
                          slot_mapping=torch.zeros(int(qsl[-1]), dtype=torch.int64, device="cuda"),
                          seq_lens_cpu_upper_bound=torch.tensor(lens, dtype=torch.int32))
    return BE.HorizonFp4Builder().build(0, cam), qsl


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("KVH,G,D,PS,window", [(2, 4, 128, 16, 0), (1, 8, 256, 32, 0), (2, 4, 128, 16, 50)])
def test_update_then_forward(fmt, KVH, G, D, PS, window, monkeypatch):
    monkeypatch.setenv("HORIZON_KVFP4_B8", fmt)
    monkeypatch.setenv("HORIZON_KVFP4_WINDOW", str(window))
    HQ, lens, qls = KVH * G, [100, 33, 260, 1], [1, 33, 40, 1]
    sinks = 4 if window else 0
    _, bt = paged(lens, KVH, PS, D, fmt, 4)
    P = int(bt.max()) + 1
    cache = torch.full((P, 2 * KVH, PS, D + 1), 0x7f, dtype=torch.uint8)
    dev = cache.cuda()
    layer = SimpleNamespace(_k_scale_float=0.5, _v_scale_float=0.3, layer_name="l")
    impl = BE.HorizonFp4Impl(HQ, D, D ** -0.5, num_kv_heads=KVH, kv_cache_dtype="nvfp4", max_num_seqs=8)
    gk, gv = torch.full((KVH,), 0.5), torch.full((KVH,), 0.3)
    slots = torch.cat([bt[b, torch.arange(L) // PS].long() * PS + torch.arange(L) % PS for b, L in enumerate(lens)])
    x = qkv(len(slots), HQ, KVH, D, 9)
    _, k, v = parts(x.cuda(), HQ, KVH, D)
    impl.do_kv_cache_update(layer, k.reshape(len(slots), KVH * D), v.reshape(len(slots), KVH * D), dev, slots.cuda())
    cache = R.append(cache, k.cpu(), v.cpu(), slots.tolist(), gk, gv, fmt)
    same(dev, cache, fmt)
    meta, qsl = metadata(lens, qls, bt)
    NT = int(qsl[-1])
    q = torch.randn(NT, HQ * D, generator=gen(1)).to(torch.bfloat16)
    out = torch.full((NT + 1, HQ * D), 7.0, dtype=torch.bfloat16, device="cuda")
    assert impl.forward(layer, q.cuda(), None, None, dev, meta, out) is out
    assert bool((out[NT:] == 7.0).all())
    o = out[:NT].view(NT, HQ, D).cpu()
    for b, L in enumerate(lens):
        a, e = int(qsl[b]), int(qsl[b + 1])
        check_rows(o[a:e], None, cache, bt, b, L, q[a:e].view(-1, HQ, D), KVH, PS, fmt, D ** -0.5, gk, gv, window, sinks, D, 2.0 ** -8, qls[b] > 1)


@pytest.mark.parametrize("cache", ["fp4", "had", "k8", "e4m3", "int8"])
def test_rotary_update(cache, monkeypatch):
    D, KVH, G, PS, NT = (256 if cache == "k8" else 128), 2, 3, 16, 29
    HQ = KVH * G
    for name, on in (("HAD", cache == "had"), ("K8", cache == "k8")):
        monkeypatch.setenv("HORIZON_KVFP4_" + name, "1" if on else "0")
    b8 = cache if cache in Lt.B8_FORMATS else None
    monkeypatch.setenv("HORIZON_KVFP4_B8", b8 or "0")
    layer = SimpleNamespace(_k_scale_float=0.02, _v_scale_float=0.01, layer_name="l")
    x, t = qkv(NT, HQ, KVH, D, 2), table(500, D, torch.float32)
    pos = torch.arange(NT) * 7
    slots = torch.arange(NT) + 3
    q, k, v = parts(x.cuda(), HQ, KVH, D)
    caches = []
    for turned in (True, False):
        impl = BE.HorizonFp4Impl(HQ, D, 0.1, num_kv_heads=KVH, kv_cache_dtype="nvfp4", max_num_seqs=4)
        kv = fresh(3, KVH, PS, D, b8, 1).cuda() if b8 else cache_of("slot", 3, PS, KVH, D, cache == "k8")[0]
        if turned:
            flat = [z.reshape(NT, -1) for z in (q, k, v)]                       # (tokens, heads * head_dim), as an engine has them
            out = torch.zeros_like(flat[0])
            got = impl.rotary_kv_cache_update(layer, *flat, kv, slots.cuda(), pos.cuda(), t.cuda(), query_out=out)
            assert got is out
            check_queries(out.view(NT, HQ, D), q.cpu(), pos, t, False)
        else:
            impl.do_kv_cache_update(layer, R.turn(k.cpu(), pos, t, False).cuda(), v.contiguous(), kv, slots.cuda())
        caches.append(kv.cpu())
    assert torch.equal(*caches)
    before = q.clone()
    kv = caches[0].cuda()
    assert impl.rotary_kv_cache_update(layer, q, k, v, kv, slots.cuda(), pos.cuda(), t.cuda()) is q        # in place
    check_queries(q, before.cpu(), pos, t, False)


def test_custom_ops():
    hkv = ops.register()
    D, KVH, HQ, PS, NT, fmt = 128, 2, 8, 16, 40, "int8"
    x, t, pos = qkv(NT, HQ, KVH, D, 3).cuda(), table(300, 64, torch.bfloat16).cuda(), (torch.arange(NT) * 2).cuda()
    q, k, v = parts(x, HQ, KVH, D)
    slots, one = torch.arange(NT).cuda() + 16, torch.full((KVH,), 0.02, device="cuda")
    # NVFP4 cache
    a, fa, st = cache_of("slot", 4, PS, KVH, D, False)
    b, fb, _ = cache_of("slot", 4, PS, KVH, D, False)
    oa, ob = (torch.zeros(NT, HQ, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    hkv.write_rotary(q, k, v, *fa, list(st), PS, slots, pos, t, one, one, True, True, None, False, oa)
    K.write_rotary(q, k, v, fb, st, PS, slots, pos, t, one, one, ob, interleaved=True)
    assert torch.equal(a, b) and torch.equal(oa, ob)
    # 8-bit cache
    ca, cb = (fresh(4, KVH, PS, D, fmt, 2).cuda() for _ in range(2))
    (fa, st), (fb, _) = Lt.b8_views(ca, KVH, D), Lt.b8_views(cb, KVH, D)
    hkv.write_b8(k, v, *fa, list(st), PS, slots, one, one, fmt)
    K.write_b8(k, v, fb, st, PS, slots, one, one, fmt=fmt)
    assert torch.equal(ca, cb)
    hkv.write_rotary_b8(q, k, v, *fa, list(st), PS, slots, pos, t, one, one, False, fmt, oa)
    K.write_rotary_b8(q, k, v, fb, st, PS, slots, pos, t, one, one, ob, fmt=fmt)
    assert torch.equal(ca, cb) and torch.equal(oa, ob)
    bt = torch.tensor([[1, 2, 3]], dtype=torch.int32, device="cuda")
    lens, qsl = torch.tensor([NT], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    ws = K.alloc_workspace(1, KVH, HQ // KVH, D, 1)
    l1, l2 = torch.zeros(NT, HQ, device="cuda"), torch.zeros(NT, HQ, device="cuda")
    hkv.decode_b8(oa[:1], *fa, list(st), PS, bt, lens, qsl, 0.1, 1.0, one, one, 1, ws, 0, fmt, 9, 2, q1 := torch.zeros_like(oa[:1]), l1)
    K.decode_b8(oa[:1], fa, st, PS, bt, lens, qsl, 0.1, 1.0, one, one, 1, q2 := torch.zeros_like(q1), ws, fmt=fmt, window=9, sinks=2, lse=l2)
    assert torch.equal(q1, q2) and torch.equal(l1, l2) and bool(q1.any())
    hkv.prefill_b8(oa, *fa, list(st), PS, bt, [0, 0, NT, NT], 0.1, 1.0, KVH, 65536, fmt, 0, 0, p1 := torch.zeros_like(oa), None)
    K.prefill_b8(oa, fa, st, PS, bt, [(0, 0, NT, NT)], 0.1, 1.0, KVH, p2 := torch.zeros_like(oa), fmt=fmt)
    assert torch.equal(p1, p2) and bool(p1.any())
    with pytest.raises(ValueError):
        hkv.prefill_b8(oa, *fa, list(st), PS, bt, [0, 0, NT], 0.1, 1.0, KVH, 65536, fmt, 0, 0, p1, None)
    with pytest.raises((RuntimeError, NotImplementedError)):
        hkv.write_b8(k.cpu(), v.cpu(), *(z.cpu() for z in fa), list(st), PS, slots.cpu(), one.cpu(), one.cpu(), fmt)
