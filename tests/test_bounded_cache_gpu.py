"""The operators for bounded caches together, as a server uses them: attention over a window whose log-sum-exps feed the gathered
weights, an eviction that goes by them, and attention over what is left; through the wrappers, the torch ops and the plugin."""
import os
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import synth
import window_ref as R
from cases import Cache, bf16_tensor
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt
from horizon_kernels_b200 import ops
from test_weights_gpu import EACH, NORM
from test_window_gpu import close

os.environ["HORIZON_KVFP4_STANDALONE"] = "1"
from horizon_kernels_b200 import backend as BE  # noqa: E402

pytestmark = pytest.mark.gpu


def wide_table(seed, lens, spare, KVH, G, D, PS):
    """a case whose block table has `spare` more pages per request, and its cache, filled by the write kernel"""
    c = synth.paged_case(seed, lens, KVH, G, D, PS, extra_pages=3 + spare * len(lens))
    B, MP = c["bt"].shape
    used = {int(p) for b, L in enumerate(lens) for p in c["bt"][b, :-(-L // PS)]}
    free = [p for p in range(1, c["NP"]) if p not in used]
    bt = np.zeros((B, MP + spare), np.int32)
    for b, L in enumerate(lens):
        n = -(-L // PS)
        bt[b, :n] = c["bt"][b, :n]
        bt[b, n:n + spare] = [free.pop() for _ in range(spare)]
    cache = Cache(c["NP"], PS, KVH, D, "hnd", 0x7f)
    gk = torch.full((KVH,), synth.tensor_scale(c["key"]) * 2, device="cuda")
    gv = torch.full((KVH,), synth.tensor_scale(c["val"]), device="cuda")
    K.write(bf16_tensor(c["key"]), bf16_tensor(c["val"]), cache.flat, cache.strides, PS, torch.from_numpy(c["slots"]).cuda(), gk, gv)
    return c, cache, torch.from_numpy(bt).cuda(), gk, gv


@pytest.mark.parametrize("D,G,window,sinks", [(128, 4, 0, 0), (256, 8, 150, 4)])
def test_a_conversation_that_is_cut_and_goes_on(D, G, window, sinks):
    """five decode steps, an eviction in place, and five more: every step against 64 bits over what the cache then holds"""
    KVH, PS, keep, recent, lens = 2, 16, 160, 40, [300, 90, 410]
    c, cache, bt, gk, gv = wide_table(41, lens, 2, KVH, G, D, PS)
    B, sm = len(lens), D ** -0.5
    g = torch.Generator(device="cuda").manual_seed(1)
    qsl = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = K.alloc_workspace(B, KVH, G, D)
    weights = torch.zeros(B, KVH, bt.shape[1] * PS, device="cuda")
    total = torch.zeros(B, KVH, weights.shape[2], dtype=torch.float64)
    scale, vscale = [float(x) * sm for x in gk], [float(x) for x in gv]
    kept, new_lens = torch.zeros((B, KVH, keep), dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    for step in range(10):
        if step == 5:
            K.evict(cache.flat, cache.strides, PS, D, bt, sl, weights, keep, 4, recent, kept, new_lens)
            assert new_lens.tolist() == [min(n, keep) for n in sl.tolist()]
            for b in range(B):
                n = int(new_lens[b])
                for h in range(KVH):
                    j = kept[b, h, :n].long().cpu()
                    assert j.tolist() == sorted(set(j.tolist())) and int(j[-1]) == int(sl[b]) - 1
                    # what stays is heavier than what went, but for what the kernel's weights are off by
                    mid = total[b, h, 4:int(sl[b]) - recent].clone()
                    if n == keep:
                        stay = torch.zeros(int(sl[b]), dtype=torch.bool)
                        stay[j] = True
                        s = stay[4:int(sl[b]) - recent]
                        assert mid[s].min() >= mid[~s].max() - 2 * EACH * float(mid[~s].max())
                    total[b, h, :n] = total[b, h, j]
                    total[b, h, n:] = 0
            sl.copy_(new_lens)
        # a token per request is appended, then attends
        sl += 1
        kv = torch.randn(2, B, KVH, D, generator=g, device="cuda").to(torch.bfloat16)
        pos = sl.long() - 1
        slots = bt[torch.arange(B, device="cuda"), pos // PS].long() * PS + pos % PS
        K.write(kv[0], kv[1], cache.flat, cache.strides, PS, slots, gk, gv)
        q = torch.randn(B, KVH * G, D, generator=g, device="cuda").to(torch.bfloat16)
        out, lse = torch.zeros_like(q), torch.zeros(B, KVH * G, device="cuda")
        K.decode_window(q, cache.flat, cache.strides, PS, bt, sl, qsl, sm, 1.0, gk, gv, 1, out, ws, window, sinks, lse=lse)
        K.accumulate_weights(q, cache.flat, cache.strides, PS, bt, sl, qsl, sm, gk, 1, lse, weights, window=window, sinks=sinks)
        assert K.workspace_status(ws) == 0 and K.workspace_status(None) == 0
        want, want_lse = [], []
        for b, L in enumerate(sl.tolist()):
            k, v = R.dense(cache.phys, "hnd", KVH, D, bt[b], PS, L)
            qb = q[b:b + 1].cpu().view(1, KVH, G, D)
            o, l = R.attention(qb, k, v, scale, vscale, window, sinks)
            want.append(o.view(1, KVH * G, D))
            want_lse.append(l.view(1, KVH * G))
            total[b, :, :L] += R.gathered(qb, k, scale, l, window, sinks)
        close(out, torch.cat(want), lse, torch.cat(want_lse))
        err = (weights.cpu().double() - total).abs()
        assert bool((err <= 2 * EACH * total + 2.0 ** -21 * total + 1e-37).all()) and float(err.norm()) <= 2 * NORM * float(total.norm())


def test_the_last_tokens_of_prompts_vote():
    """prefill with log-sum-exps, the weights of each prompt's last eight tokens, and the eviction to new pages"""
    KVH, G, D, PS, lens, keep = 2, 4, 128, 16, [500, 333], 128
    c = synth.paged_case(43, lens, KVH, G, D, PS, ql_list=lens, extra_pages=30)
    cache = Cache(c["NP"], PS, KVH, D, "hnd", 0x7f)
    gk = torch.full((KVH,), synth.tensor_scale(c["key"]) * 2, device="cuda")
    gv = torch.full((KVH,), synth.tensor_scale(c["val"]), device="cuda")
    K.write(bf16_tensor(c["key"]), bf16_tensor(c["val"]), cache.flat, cache.strides, PS, torch.from_numpy(c["slots"]).cuda(), gk, gv)
    q, bt = bf16_tensor(c["q"]), torch.from_numpy(c["bt"]).cuda()
    rows = [(0, 0, lens[0], lens[0]), (1, lens[0], sum(lens), lens[1])]
    sm = D ** -0.5
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
    K.prefill_window(q, cache.flat, cache.strides, PS, bt, rows, sm * float(gk[0]), float(gv[0]), KVH, out, 0, 0, lse=lse)
    last = torch.cat([torch.arange(e - 8, e) for _, _, e, _ in rows]).cuda()
    qsl = torch.tensor([0, 8, 16], dtype=torch.int32, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    w = torch.zeros(2, KVH, max(lens), device="cuda")
    K.accumulate_weights(q[last].contiguous(), cache.flat, cache.strides, PS, bt, sl, qsl, sm, gk, 8, lse[last].contiguous(), w)
    assert abs(float(w.sum()) - 16 * KVH * G) < 1e-2            # every row gives away a weight of one
    used = {int(p) for b, L in enumerate(lens) for p in c["bt"][b, :-(-L // PS)]}
    new = torch.tensor([p for p in range(1, c["NP"]) if p not in used][:16], dtype=torch.int32, device="cuda").view(2, 8)
    kept, nl = torch.zeros((2, KVH, keep), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    nw = torch.zeros(2, KVH, keep, device="cuda")
    K.evict(cache.flat, cache.strides, PS, D, bt, sl, w, keep, 4, 32, kept, nl, out_tables=new, out_weights=nw)
    for b in range(2):
        old_k, old_v = R.dense(cache.phys, "hnd", KVH, D, bt[b], PS, lens[b])
        new_k, new_v = R.dense(cache.phys, "hnd", KVH, D, new[b], PS, keep)
        for h in range(KVH):
            j = torch.from_numpy(R.kept_positions(w[b, h, :lens[b]].cpu().numpy(), keep, 4, 32))
            assert torch.equal(kept[b, h].cpu().long(), j)
            assert torch.equal(new_k[:, h], old_k[j, h]) and torch.equal(new_v[:, h], old_v[j, h])
            assert torch.equal(nw[b, h].cpu(), w[b, h].cpu()[j])


def test_custom_ops_give_the_wrappers_bits():
    hkv = ops.register()
    KVH, G, D, PS, lens = 2, 4, 128, 16, [200, 70]
    c, cache, bt, gk, gv = wide_table(47, lens, 0, KVH, G, D, PS)
    q, qsl = bf16_tensor(c["q"]), torch.from_numpy(c["qsl"]).cuda()
    sl = torch.from_numpy(c["seq_lens"]).cuda()
    sm, flat, st = D ** -0.5, cache.flat, cache.strides
    ws = K.alloc_workspace(2, KVH, G, D)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    la, lb = torch.zeros(2, KVH * G, device="cuda"), torch.zeros(2, KVH * G, device="cuda")
    K.decode_window(q, flat, st, PS, bt, sl, qsl, sm, 1.0, gk, gv, 1, a, ws, 64, 4, lse=la)
    hkv.decode_window(q, *flat, list(st), PS, bt, sl, qsl, sm, 1.0, gk, gv, 1, ws, 0, 64, 4, None, False, b, lb)
    assert torch.equal(a, b) and torch.equal(la, lb)
    rows = [(0, 0, 1, 200), (1, 1, 2, 70)]
    K.prefill_window(q, flat, st, PS, bt, rows, sm * float(gk[0]), float(gv[0]), KVH, a, 64, 4)
    hkv.prefill_window(q, *flat, list(st), PS, bt, [x for r in rows for x in r], sm * float(gk[0]), float(gv[0]), KVH, 65536, 64, 4, None, False,
                       b, None)
    assert torch.equal(a, b)
    wa, wb = torch.zeros(2, KVH, 200, device="cuda"), torch.zeros(2, KVH, 200, device="cuda")
    K.accumulate_weights(q, flat, st, PS, bt, sl, qsl, sm, gk, 1, la, wa, window=64, sinks=4)
    hkv.accumulate_weights(q, *flat, list(st), PS, bt, sl, qsl, sm, gk, 1, la, 64, 4, None, False, wb)
    assert torch.equal(wa, wb) and float(wa.sum()) > 0
    src = cache.phys.clone()
    ka, kb = (torch.zeros((2, KVH, 48), dtype=torch.int32, device="cuda") for _ in range(2))
    na, nb = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    K.evict(flat, st, PS, D, bt, sl, wa, 48, 4, 8, ka, na)
    first = cache.phys.clone()
    cache.phys.copy_(src)
    hkv.evict(*flat, list(st), PS, D, bt, sl, wb, 48, 4, 8, kb, nb, None, None, False)
    assert torch.equal(cache.phys, first) and torch.equal(ka, kb) and torch.equal(na, nb) and torch.equal(wa, wb)
    with pytest.raises((RuntimeError, NotImplementedError)):
        hkv.evict(*[f.cpu() for f in flat], list(st), PS, D, bt.cpu(), sl.cpu(), wb.cpu(), 48, 4, 8, kb.cpu(), nb.cpu(), None, None, False)


@pytest.mark.parametrize("D,had", [(128, "0"), (256, "1")])
def test_the_plugin_over_a_window(monkeypatch, D, had):
    """HORIZON_KVFP4_WINDOW: a step of decode and prefill rows through the plugin gives the bits of the wrappers"""
    monkeypatch.setenv("HORIZON_KVFP4_WINDOW", "100")
    monkeypatch.setenv("HORIZON_KVFP4_SINKS", "7")
    monkeypatch.setenv("HORIZON_KVFP4_HAD", had)
    KVH, G, PS, lens, ql = 2, 4, 16, [400, 77, 260], [1, 1, 130]
    c = synth.paged_case(51, lens, KVH, G, D, PS, ql_list=ql)
    impl = BE.HorizonFp4Impl(KVH * G, D, D ** -0.5, num_kv_heads=KVH, kv_cache_dtype="nvfp4", max_num_seqs=4)
    layer = SimpleNamespace(_k_scale_float=0.01, _v_scale_float=0.005)
    kv = torch.full((c["NP"], 2 * KVH, PS, Lt.slot_bytes(D)), 0x7f, dtype=torch.uint8, device="cuda")
    T = int(c["qsl"][-1])
    impl.do_kv_cache_update(layer, bf16_tensor(c["key"]), bf16_tensor(c["val"]), kv, torch.from_numpy(c["slots"]).cuda())
    sl = torch.from_numpy(c["seq_lens"]).cuda()
    cam = SimpleNamespace(num_reqs=3, num_actual_tokens=T, query_start_loc=torch.from_numpy(c["qsl"]).cuda(),
                          query_start_loc_cpu=torch.from_numpy(c["qsl"]), seq_lens=sl, seq_lens_cpu_upper_bound=sl.cpu(),
                          block_table_tensor=torch.from_numpy(c["bt"]).cuda(), slot_mapping=None)
    m = BE.HorizonFp4Builder().build(0, cam)
    q = bf16_tensor(c["q"]).view(T, -1)
    out = torch.full_like(q, float("nan"))
    impl.forward(layer, q, None, None, kv, m, out)
    flat, st = Lt.flat_views(*Lt.slot_views(kv, KVH, D))
    signs = K.hadamard_signs(D, device="cuda") if had == "1" else None
    gk, gv = torch.full((KVH,), 0.01, device="cuda"), torch.full((KVH,), 0.005, device="cuda")
    want = torch.full((T, KVH * G, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    q3 = q.view(T, KVH * G, D)
    K.decode_window(q3, flat, st, PS, m.block_table, sl, m.query_start_loc, D ** -0.5, 0.005, gk, gv, 1, want, K.alloc_workspace(4, KVH, G, D),
                    100, 7, signs=signs)
    K.prefill_window(q3, flat, st, PS, m.block_table, [(2, 2, 132, 260)], D ** -0.5 * 0.01, 0.005, KVH, want, 100, 7, signs=signs)
    assert torch.equal(out.view(T, KVH * G, D), want)
    monkeypatch.delenv("HORIZON_KVFP4_WINDOW")
    full = BE.HorizonFp4Impl(KVH * G, D, D ** -0.5, num_kv_heads=KVH, kv_cache_dtype="nvfp4", max_num_seqs=4)
    other = torch.zeros_like(q)
    full.forward(layer, q, None, None, kv, m, other)
    assert not torch.equal(other, out)


def test_a_captured_step_with_other_lengths():
    """decode, weights and eviction captured once and replayed with other lengths: the bits of the plain calls; the decode on a
    workspace of its own, as graphs that may overlap need it"""
    KVH, G, D, PS, lens = 2, 4, 128, 16, [700, 300]
    c, cache, bt, gk, gv = wide_table(53, lens, 0, KVH, G, D, PS)
    q, qsl = bf16_tensor(c["q"]), torch.from_numpy(c["qsl"]).cuda()
    sl = torch.from_numpy(c["seq_lens"]).cuda()
    flat, st, sm, keep = cache.flat, cache.strides, D ** -0.5, 96
    ws = K.alloc_workspace(2, KVH, G, D)
    out, lse = torch.zeros_like(q), torch.zeros(2, KVH * G, device="cuda")
    w, kept = torch.zeros(2, KVH, 700, device="cuda"), torch.zeros((2, KVH, keep), dtype=torch.int32, device="cuda")
    nl = torch.zeros(2, dtype=torch.int32, device="cuda")
    src = cache.phys.clone()

    def go():
        K.decode_window(q, flat, st, PS, bt, sl, qsl, sm, 1.0, gk, gv, 1, out, ws, 200, 4, lse=lse)
        K.accumulate_weights(q, flat, st, PS, bt, sl, qsl, sm, gk, 1, lse, w, window=200, sinks=4, workspace=ws)
        K.evict(flat, st, PS, D, bt, sl, w, keep, 4, 32, kept, nl)

    def reset(lengths):
        cache.phys.copy_(src)
        w.zero_()
        sl.copy_(torch.tensor(lengths, dtype=torch.int32))
        for t in (out, lse, kept, nl):
            t.fill_(3)

    def result():
        torch.cuda.synchronize()
        return [t.clone() for t in (out, lse, w, kept, nl, cache.phys)]
    reset(lens)
    go()
    result()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            go()
    torch.cuda.current_stream().wait_stream(side)
    for lengths in (lens, [1, 699], [64, 0], [97, 96]):
        reset(lengths)
        go()
        plain = result()
        reset(lengths)
        graph.replay()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(plain, result())), lengths
        assert K.workspace_status(ws) == 0
