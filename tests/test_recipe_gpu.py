"""The integration guide's recipe for bounded caches over two layers on the GPU: each layer keeps its own heaviest tokens, and the
steps after the cut attend what stayed, against 64 bits."""
from types import SimpleNamespace

import pytest
import torch

import window_ref as R
from cases import Cache, bf16_tensor
from horizon_kernels_b200 import kernels as K
from test_bounded_cache_gpu import wide_table
from test_recipe_cpu import recipe
from test_window_gpu import close

pytestmark = pytest.mark.gpu


def test_two_layers_are_cut_and_go_on():
    KVH, G, D, PS, keep, sinks, recent, lengths = 2, 4, 128, 16, 96, 4, 20, [300, 80, 190]
    c, first, bt, gk, gv = wide_table(61, lengths, 2, KVH, G, D, PS)
    second = Cache(c["NP"], PS, KVH, D, "hnd", 0x7f)
    g = torch.Generator(device="cuda").manual_seed(7)
    kv = torch.randn(2, c["slots"].size, KVH, D, generator=g, device="cuda").to(torch.bfloat16)
    K.write(kv[0], kv[1], second.flat, second.strides, PS, torch.from_numpy(c["slots"]).cuda(), gk, gv)
    B, sm, vs, qlmax, st = len(lengths), D ** -0.5, 1.0, 1, first.strides
    lens, new_lens = torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    qsl = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    lse, ws = torch.zeros(B, KVH * G, device="cuda"), K.alloc_workspace(B, KVH, G, D)
    kept = torch.zeros((B, KVH, keep), dtype=torch.int32, device="cuda")
    layers = [SimpleNamespace(cache=x, flat=x.flat, gk=gk, gv=gv, weights=torch.zeros(B, KVH, bt.shape[1] * PS, device="cuda"),
                              q=torch.zeros(B, KVH * G, D, dtype=torch.bfloat16, device="cuda")) for x in (first, second)]
    def evict(flat, st, PS, D, bt, lens, weights, *more):
        x = next(x for x in layers if x.weights is weights)
        x.seen = weights.cpu().clone()
        K.evict(flat, st, PS, D, bt, lens, weights, *more)
    calls = SimpleNamespace(decode_window=K.decode_window, accumulate_weights=K.accumulate_weights, evict=evict)
    env = dict(K=calls, layers=layers, st=st, PS=PS, D=D, bt=bt, lens=lens, qsl=qsl, sm=sm, vs=vs, qlmax=qlmax, ws=ws, lse=lse, keep=keep, sinks=sinks,
               recent=recent, kept=kept, new_lens=new_lens)
    scale, vscale = [float(x) * sm for x in gk], [float(x) for x in gv]
    cut_at = 3
    for step in range(6):
        lens += 1                                         # a token a request
        pos = lens.long() - 1
        slots = bt[torch.arange(B, device="cuda"), pos // PS].long() * PS + pos % PS
        for x in layers:
            k, v, x.q = (torch.randn(B, n, D, generator=g, device="cuda").to(torch.bfloat16) for n in (KVH, KVH, KVH * G))
            K.write(k, v, x.flat, st, PS, slots, gk, gv)
            x.out = torch.zeros_like(x.q)
        before, old = lens.tolist(), [x.cache.phys.cpu().clone() for x in layers]
        exec(recipe(), dict(env, cut=step == cut_at))
        torch.cuda.synchronize()
        for x, phys in zip(layers, old):
            want = []
            for b, L in enumerate(before):
                k, v = R.dense(phys, "hnd", KVH, D, bt[b], PS, L)
                o, _ = R.attention(x.q[b:b + 1].cpu().view(1, KVH, G, D), k, v, scale, vscale, 0, 0)
                want.append(o.view(1, KVH * G, D))
                if step == cut_at:                        # this layer's own heaviest tokens, from a context of L
                    n = min(L, keep)
                    now_k, now_v = R.dense(x.cache.phys, "hnd", KVH, D, bt[b], PS, n)
                    for h in range(KVH):
                        j = torch.from_numpy(R.kept_positions(x.seen[b, h, :L].numpy(), keep, sinks, recent))
                        assert torch.equal(now_k[:, h], k[j, h]) and torch.equal(now_v[:, h], v[j, h])
            close(x.out, torch.cat(want))
        assert lens.tolist() == ([min(n, keep) for n in before] if step == cut_at else before)
