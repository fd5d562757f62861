"""kernels.accumulate_weights against the definition in 64 bits: layouts, ragged batches, several query tokens, windows, lengths
from none to long, and what must stay untouched.

Tolerance. A score is a sum of D products of f16 numbers, exact one by one, added in fp32: at most D roundings (the tensor
core truncates, a step of 2^-23) of the sum of the magnitudes, |q| . |k| * scale, here below A = 60 nats for every case (checked). The
scaled score, its product with log2(e) and the log-sum-exp's each add 2^-24 of at most A, the exponential 2^-22. Their sum, as
a relative error of a weight: A * (D * 2^-23 + 3 * 2^-24) + 2^-22, under the assumption that all roundings go the same way;
D = 256: 1.9e-3. Roundings that go either way give about sqrt(D) of them instead of D: the tests ask for 1.9e-3 per entry and
for 16 * A / 60 * 2^-23 * 60 = 1.2e-4 in the 2-norm. To it comes the addition, 2^-24 of the entry's value."""
import numpy as np
import pytest
import torch

import synth
import window_ref as R
from cases import Cache, bf16_tensor, build_decode_case
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt

pytestmark = pytest.mark.gpu
EACH, NORM = 1.9e-3, 1.2e-4


def k8_case(seed, lens, KVH, G, D, PS, ql_list):
    """a case over the FP8-key slot: keys e4m3(k / gk), values any codes"""
    c = synth.paged_case(seed, lens, KVH, G, D, PS, outliers=True, ql_list=ql_list)
    gk = np.full(KVH, synth.tensor_scale(c["key"]) * 6, np.float32)
    phys = torch.full((c["NP"], KVH, PS, Lt.K8_SLOT), 0x7f, dtype=torch.uint8, device="cuda")
    flat, st = Lt.k8_flat_views(*Lt.k8_views(phys, D))
    gkt = torch.from_numpy(gk).cuda()
    gv = torch.full((KVH,), synth.tensor_scale(c["val"]), device="cuda")
    if c["slots"].size:
        K.write(bf16_tensor(c["key"]), bf16_tensor(c["val"]), flat, st, PS, torch.from_numpy(c["slots"]).cuda(), gkt, gv, False, k8=True)
    c.update(phys=phys, flat=flat, strides=st, gk=gk, gv=gv.cpu().numpy(), sm=D ** -0.5, kind="k8")
    return c


def case(seed, lens, KVH, G, D, PS, kind="hnd", ql_list=None, gscale=None):
    if kind == "k8":
        return k8_case(seed, lens, KVH, G, D, PS, ql_list)
    c = build_decode_case(seed, lens, KVH, G, D, PS, kind=kind, ql_list=ql_list, gscale=gscale)
    c.update(phys=c["cache"].phys, flat=c["cache"].flat, strides=c["cache"].strides, kind=kind)
    return c


def tensors(c):
    return dict(q=bf16_tensor(c["q"]), bt=torch.from_numpy(c["bt"]).cuda(), sl=torch.from_numpy(c["seq_lens"]).cuda(),
                qsl=torch.from_numpy(c["qsl"]).cuda(), gk=torch.from_numpy(np.asarray(c["gk"], np.float32)).cuda(),
                gv=torch.from_numpy(np.asarray(c["gv"], np.float32)).cuda())


def reference(c, window, sinks, qlmax, signs=None):
    """(log-sum-exps (tokens, heads), weights to add (B, KVH, longest)), in 64 bits"""
    KVH, G, D = c["KVH"], c["G"], c["D"]
    q = bf16_tensor(c["q"], "cpu")
    if signs is not None:
        q = K.rotate(q, signs.cpu()).to(torch.bfloat16)
    lse = torch.full((q.shape[0], KVH * G), 3.25, dtype=torch.float64)
    W = max(1, max(int(x) for x in c["seq_lens"]))
    add = torch.zeros(len(c["seq_lens"]), KVH, W, dtype=torch.float64)
    scale = [c["sm"] * float(g) for g in c["gk"]]
    worst = 0.0
    for b, L in enumerate(int(x) for x in c["seq_lens"]):
        a, e = int(c["qsl"][b]), int(c["qsl"][b + 1])
        if not 0 < e - a <= qlmax:
            continue
        qb = q[a:e].view(e - a, KVH, G, D)
        if L == 0:
            lse[a:e] = -torch.inf
            continue
        k, v = R.dense(c["phys"], c["kind"], KVH, D, torch.from_numpy(c["bt"])[b], c["PS"], L)
        worst = max(worst, float(R.scores(qb.abs(), k.abs(), [abs(s) for s in scale]).max()))
        see = R.seen(L, e - a, window, sinks)[:, None, None, :]
        x = R.scores(qb, k, scale).masked_fill(~see, -torch.inf)
        l = torch.logsumexp(x, -1).float()
        lse[a:e] = l.view(e - a, KVH * G).double()
        add[b, :, :L] = R.gathered(qb, k, scale, torch.where(l == -torch.inf, torch.tensor(0.0), l), window, sinks)
    assert worst < 60, worst
    return lse, add


def check(c, window=0, sinks=0, qlmax=None, signs=None, extra=0, ws=None):
    t = tensors(c)
    qlmax = int(max(1, (c["qsl"][1:] - c["qsl"][:-1]).max())) if qlmax is None else qlmax
    lse, add = reference(c, window, sinks, qlmax, signs)
    B, KVH, W = add.shape
    g = torch.Generator(device="cuda").manual_seed(3)
    w = 1e-3 * torch.rand(B, KVH, W + extra, device="cuda", generator=g)
    w0 = w.clone()
    args = (t["q"], c["flat"], c["strides"], c["PS"], t["bt"], t["sl"], t["qsl"], c["sm"], t["gk"], qlmax, lse.float().cuda())
    K.accumulate_weights(*args, w, window=window, sinks=sinks, signs=signs, k8=c["kind"] == "k8", workspace=ws)
    assert K.workspace_status(ws) == 0
    got, want = w.cpu().double()[..., :W], w0.cpu().double()[..., :W] + add
    assert torch.equal(w[..., W:], w0[..., W:])
    zero = add == 0
    assert torch.equal(got[zero & (got == w0.cpu().double()[..., :W])], want[zero & (got == w0.cpu().double()[..., :W])])
    err = (got - want).abs()
    assert bool((err <= EACH * add + 2.0 ** -23 * want + 1e-37).all()), float((err / (EACH * add + 2.0 ** -23 * want + 1e-37)).max())
    assert float((got - want).norm()) <= NORM * float(add.norm()) + 2.0 ** -23 * float(want.norm())
    # the same bits again
    w2 = w0.clone()
    K.accumulate_weights(*args, w2, window=window, sinks=sinks, signs=signs, k8=c["kind"] == "k8", workspace=ws)
    assert torch.equal(w, w2)
    return w


@pytest.mark.parametrize("kind,KVH,G,D,PS", [("hnd", 8, 4, 128, 16), ("nhd", 2, 8, 128, 32), ("region", 2, 3, 128, 16), ("hnd", 2, 8, 256, 64),
                                             ("nhd", 4, 6, 256, 16), ("region", 2, 1, 256, 32), ("k8", 2, 8, 256, 16), ("k8", 1, 5, 256, 64)])
def test_layouts(kind, KVH, G, D, PS):
    check(case(7000 + D + KVH, [700, 33, 1, 0, 64, 2049], KVH, G, D, PS, kind), extra=5)


@pytest.mark.parametrize("kind,G,D,qls", [("hnd", 4, 128, [4, 1, 0, 2, 3]), ("hnd", 8, 256, [2, 2, 2, 2, 2]), ("k8", 8, 256, [3, 1, 4, 2, 0]),
                                          ("nhd", 8, 128, [8, 1, 8, 0, 5]), ("hnd", 16, 128, [4, 4, 4, 1, 1]), ("hnd", 1, 128, [64, 3, 40, 9, 1])])
def test_several_query_tokens(kind, G, D, qls):
    check(case(7100 + G, [300, 5, 77, 2, 40], 2, G, D, 16, kind, ql_list=qls), qlmax=max(qls))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 3), (33, 40), (0, 7), (5000, 2), (64, 0)])
@pytest.mark.parametrize("kind,D", [("hnd", 128), ("hnd", 256), ("k8", 256), ("nhd", 128)])
def test_windows(kind, D, window, sinks):
    check(case(7200, [500, 64, 97, 1, 0, 1023], 2, 4, D, 16, kind, ql_list=[1, 2, 3, 1, 1, 4]), window=window, sinks=sinks, qlmax=4)


def test_rotated_keys():
    """keys written rotated: the rotated queries (to bf16, as decode does) give the scores"""
    signs = K.hadamard_signs(128, device="cuda")
    c = synth.paged_case(7300, [400, 65], 2, 4, 128, 16)
    cache = Cache(c["NP"], 16, 2, 128, "hnd", 0x7f)
    gk = np.full(2, synth.tensor_scale(c["key"]) * 2, np.float32)
    gkt = torch.from_numpy(gk).cuda()
    K.write(bf16_tensor(c["key"]), bf16_tensor(c["val"]), cache.flat, cache.strides, 16, torch.from_numpy(c["slots"]).cuda(), gkt, gkt,
            signs=signs)
    c.update(phys=cache.phys, flat=cache.flat, strides=cache.strides, kind="hnd", gk=gk, gv=gk, sm=128 ** -0.5)
    check(c, signs=signs)


def test_requests_that_are_not_for_this_call():
    """more than qlmax query tokens, or none: nothing changes, whatever the log-sum-exps of those rows hold"""
    c = case(7400, [300, 200, 100], 2, 4, 128, 16, ql_list=[1, 9, 0])
    w = check(c, qlmax=2)
    g = torch.Generator(device="cuda").manual_seed(3)
    assert torch.equal(w[1:], (1e-3 * torch.rand(3, 2, 300, device="cuda", generator=g))[1:])


def test_scales():
    """per-head scales, a zero and a negative softmax scale"""
    c = case(7500, [300, 90], 4, 4, 128, 16, gscale=(0.002, 0.001))
    for sm in (0.05, 0.0, -0.05):
        check(dict(c, sm=sm))


def test_strided_rows_and_a_workspace():
    c = case(7600, [300, 20], 2, 4, 128, 16)
    t = tensors(c)
    lse, add = reference(c, 0, 0, 1)
    big = torch.full((2, 3, 2, 640), 7.0, device="cuda")
    w = big[:, 1, :, 100:400]
    w.zero_()
    ws = K.alloc_workspace(2, 2, 4, 128, 1)
    K.accumulate_weights(t["q"], c["flat"], c["strides"], 16, t["bt"], t["sl"], t["qsl"], c["sm"], t["gk"], 1, lse.float().cuda(), w, workspace=ws)
    assert K.workspace_status(ws) == 0
    assert float((w.cpu().double() - add).norm()) <= NORM * float(add.norm())
    big[:, 1, :, 100:400] = 7.0
    assert bool((big == 7.0).all())


def test_a_length_beyond_the_weights_is_cut():
    c = case(7700, [300], 2, 4, 128, 16)
    t = tensors(c)
    w = torch.zeros(1, 2, 100, device="cuda")
    lse, _ = reference(dict(c, seq_lens=np.array([100], np.int32)), 0, 0, 1)
    _, add = reference(dict(c, seq_lens=np.array([100], np.int32)), 0, 0, 1)
    K.accumulate_weights(t["q"], c["flat"], c["strides"], 16, t["bt"], t["sl"], t["qsl"], c["sm"], t["gk"], 1, lse.float().cuda(), w)
    assert float((w.cpu().double() - add).norm()) <= NORM * float(add.norm())


def test_a_long_batch():
    rng = np.random.default_rng(1)
    check(case(7800, [20000] + [int(x) for x in rng.integers(1, 500, 60)], 2, 4, 128, 16))
