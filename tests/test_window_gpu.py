"""kernels.decode_window and kernels.prefill_window against the definition in 64 bits: layouts, windows and sinks of every kind,
several query tokens, split and whole sequences, chunked prefills, the log-sum-exps, and pages that are gone.

Tolerances. Outputs are bf16: half a step of 2^-8, relative; probabilities are f16 under a running maximum (2^-11 of each, so at
most 2^-11 of sum p |v|, and sum p |v| is below max |v| where the output itself may be small). The gate that this repository's
other attention tests use: relative 2-norm 2.5e-3, max-abs 2e-2 and mean-abs 2e-3 at values of order one (tests/cases.py).
Log-sum-exps are fp32: as for the weights (tests/test_weights_gpu.py) every score is off by at most A (D 2^-23 + 3 2^-24) for
magnitudes that sum to A < 60, absolute: 1.9e-3, and the log-sum-exp by no more than the scores are, plus 2^-22 for the
exponentials; over a row of scores the roundings go either way, for which 1.2e-4 is asked in the root mean square."""
import numpy as np
import pytest
import torch

import window_ref as R
from cases import bf16_tensor
from horizon_kernels_b200 import kernels as K
from test_weights_gpu import case, tensors

pytestmark = pytest.mark.gpu
LSE_EACH, LSE_RMS = 1.9e-3, 1.2e-4


def close(got, want, lse=None, want_lse=None):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    d = (got - want).abs()
    assert float(d.max()) <= 2e-2 and float(d.mean()) <= 2e-3 and float(d.norm()) <= 2.5e-3 * max(float(want.norm()), 1e-300)
    if lse is not None:
        lse = lse.double().cpu()
        gone = want_lse == -torch.inf
        assert torch.equal(lse == -torch.inf, gone)
        e = (lse - want_lse)[~gone].abs()
        if e.numel():
            assert float(e.max()) <= LSE_EACH and float(e.square().mean().sqrt()) <= LSE_RMS


def reference(c, rows, window, sinks, vscale, signs=None):
    """rows: [(request, first query token, one past the last, context)]; (out, lse) with NaN where no row writes"""
    KVH, G, D = c["KVH"], c["G"], c["D"]
    q = bf16_tensor(c["q"], "cpu")
    if signs is not None:
        q = K.rotate(q, signs.cpu()).to(torch.bfloat16)
    out = torch.full(q.shape, torch.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], torch.nan, dtype=torch.float64)
    scale = [c["sm"] * float(g) for g in c["gk"]]
    for b, a, e, L in rows:
        if L == 0:
            out[a:e], lse[a:e] = 0.0, -torch.inf
            continue
        k, v = R.dense(c["phys"], c["kind"], KVH, D, torch.from_numpy(c["bt"])[b], c["PS"], L)
        o, l = R.attention(q[a:e].view(e - a, KVH, G, D), k, v, scale, vscale, window, sinks)
        out[a:e], lse[a:e] = o.reshape(e - a, KVH * G, D), l.reshape(e - a, KVH * G)
    return out, lse


def lose_pages(c, rows, window, sinks):
    """every page of a request none of whose tokens is visible: its table entry becomes an unused page of NaN scales"""
    bt = c["bt"].copy()
    for b, a, e, L in rows:
        see = R.seen(L, e - a, window, sinks).any(0) if L else torch.zeros(0, dtype=torch.bool)
        for p in range(bt.shape[1]):
            if not bool(see[p * c["PS"]:(p + 1) * c["PS"]].any()):
                bt[b, p] = 0
    return dict(c, bt=bt)


def decode(c, window, sinks, qlmax=None, signs=None, vs=0.75, splits=None, lse=True):
    qlens = c["qsl"][1:] - c["qsl"][:-1]
    qlmax = int(max(1, qlens.max())) if qlmax is None else qlmax
    rows = [(b, int(c["qsl"][b]), int(c["qsl"][b + 1]), int(L)) for b, L in enumerate(c["seq_lens"]) if 0 < qlens[b] <= qlmax]
    if window:
        c = lose_pages(c, rows, window, sinks)
        c["phys"][0] = 0xff
    t = tensors(c)
    want, want_lse = reference(c, rows, window, sinks, [float(g) * vs for g in c["gv"]], signs)
    out = torch.full(t["q"].shape, float("nan"), dtype=torch.bfloat16, device="cuda")
    got_lse = torch.full(t["q"].shape[:2], float("nan"), device="cuda") if lse else None
    ws = K.alloc_workspace(len(c["seq_lens"]), c["KVH"], c["G"], c["D"], qlmax)

    def go():
        K.decode_window(t["q"], c["flat"], c["strides"], c["PS"], t["bt"], t["sl"], t["qsl"], c["sm"], vs, t["gk"], t["gv"], qlmax, out, ws,
                        window, sinks, splits=splits, signs=signs, k8=c["kind"] == "k8", lse=got_lse)
    go()
    assert K.workspace_status(ws) == 0
    on = torch.zeros(t["q"].shape[0], dtype=torch.bool)
    for _, a, e, _ in rows:
        on[a:e] = True
    close(out.cpu()[on], want[on], got_lse.cpu()[on] if lse else None, want_lse[on])
    assert out.cpu()[~on].isnan().all()
    first, first_lse = out.clone(), got_lse.clone() if lse else None
    go()
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), first.view(torch.int16))
    assert not lse or torch.equal(got_lse.view(torch.int32), first_lse.view(torch.int32))
    return out, got_lse


SHAPES = [("hnd", 8, 4, 128, 16), ("nhd", 2, 8, 128, 32), ("region", 2, 3, 128, 16), ("hnd", 2, 8, 256, 64), ("nhd", 4, 6, 256, 16),
          ("region", 2, 1, 256, 32), ("k8", 2, 8, 256, 16)]


@pytest.mark.parametrize("kind,KVH,G,D,PS", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (1, 0), (333, 50)])
def test_decode_layouts(kind, KVH, G, D, PS, window, sinks):
    decode(case(8000 + D + KVH, [700, 33, 1, 0, 64, 2049], KVH, G, D, PS, kind), window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 0), (17, 16), (31, 33), (32, 32), (33, 31), (64, 1), (5, 200), (100000, 3), (47, 95), (0, 9)])
@pytest.mark.parametrize("D", [128, 256])
def test_decode_windows(D, window, sinks):
    decode(case(8100, [500, 64, 97, 1, 0, 1023, 130], 2, 4, D, 16, ql_list=[1, 2, 3, 1, 1, 4, 2]), window, sinks, qlmax=4)


@pytest.mark.parametrize("kind,G,D,qls", [("hnd", 4, 128, [4, 1, 0, 2, 3]), ("hnd", 8, 256, [2, 2, 2, 2, 2]), ("k8", 8, 256, [3, 1, 4, 2, 0]),
                                          ("nhd", 8, 128, [8, 1, 8, 0, 5]), ("hnd", 16, 128, [4, 4, 4, 1, 1]), ("hnd", 1, 128, [64, 3, 40, 9, 1])])
@pytest.mark.parametrize("window,sinks", [(40, 3), (2, 0)])
def test_decode_several_query_tokens(kind, G, D, qls, window, sinks):
    """rows of one request with different windows, more rows than a pass serves, and rows that see no key (more query tokens than
    context)"""
    decode(case(8200 + G, [300, 5, 77, 2, 40], 2, G, D, 16, kind, ql_list=qls), window, sinks, qlmax=max(qls))


@pytest.mark.parametrize("KVH,G,D,lens,window,sinks", [
    (1, 4, 128, [70000], 60000, 4), (2, 8, 256, [30000], 25001, 100), (1, 8, 128, [9000, 20, 4000], 3000, 4), (1, 16, 256, [9000, 300], 6000, 33),
    (2, 4, 128, [40000], 0, 0)])
def test_decode_split_sequences(KVH, G, D, lens, window, sinks):
    """windows that are cut among many CTAs: merged directly, by weights, and by groups"""
    decode(case(8300 + D, lens, KVH, G, D, 16), window, sinks)


@pytest.mark.parametrize("splits", [1, 2])
def test_decode_split_caps(splits):
    decode(case(8310, [2000, 700], 2, 4, 128, 16), 600, 4, splits=splits)


def test_decode_without_a_window_gives_the_bits_of_decode():
    for D, G, kind in ((128, 4, "hnd"), (256, 8, "nhd"), (128, 16, "hnd")):
        c = case(8400, [700, 33, 1500], 2, G, D, 16, kind)
        t = tensors(c)
        out, _ = decode(c, 0, 0, lse=False)
        want = torch.full_like(out, float("nan"))
        K.decode_ragged(t["q"], c["flat"], c["strides"], 16, t["bt"], t["sl"], t["qsl"], c["sm"], 0.75, t["gk"], t["gv"], 1, want,
                        K.alloc_workspace(3, 2, G, D, 1))
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_decode_rotated():
    signs = K.hadamard_signs(256, device="cuda")
    c = case(8500, [400, 65], 2, 8, 256, 16)
    decode(c, 64, 4, signs=signs)


def test_decode_scales():
    c = case(8600, [300, 90], 4, 4, 128, 16, gscale=(0.002, 0.001))
    for sm in (0.05, 0.0, -0.05):
        decode(dict(c, sm=sm), 100, 4)


# ------------------------------------------------------------------------------------------------------------- prefill
def prefill(c, rows, window, sinks, chunk=65536, signs=None, out_dtype=torch.bfloat16, q_dtype=torch.bfloat16, ws=None, lse=True):
    if window:
        c = lose_pages(c, rows, window, sinks)
        c["phys"][0] = 0xff
    t = tensors(c)
    gk, gv = float(c["gk"][0]), float(c["gv"][0])
    want, want_lse = reference(c, rows, window, sinks, [gv] * c["KVH"], signs)
    q = t["q"].to(q_dtype)
    out = torch.full(q.shape, float("nan"), dtype=out_dtype, device="cuda")
    got_lse = torch.full(q.shape[:2], float("nan"), device="cuda") if lse else None

    def go():
        K.prefill_window(q, c["flat"], c["strides"], c["PS"], t["bt"], rows, c["sm"] * gk, gv, c["KVH"], out, window, sinks, chunk=chunk,
                         signs=signs, k8=c["kind"] == "k8", workspace=ws, lse=got_lse)
    go()
    assert K.workspace_status(ws) == 0
    on = torch.zeros(q.shape[0], dtype=torch.bool)
    for _, a, e, _ in rows:
        on[a:e] = True
    close(out.cpu()[on], want[on], got_lse.cpu()[on] if lse else None, want_lse[on])
    assert out.cpu()[~on].isnan().all() and (not lse or got_lse.cpu()[~on].isnan().all())
    first = out.clone()
    go()
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.uint8), first.view(torch.uint8))
    return out


def rows_of(c):
    return [(b, int(c["qsl"][b]), int(c["qsl"][b + 1]), int(L)) for b, L in enumerate(c["seq_lens"]) if c["qsl"][b + 1] > c["qsl"][b]]


@pytest.mark.parametrize("kind,KVH,G,D,PS", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (1, 0), (300, 150)])
def test_prefill_layouts(kind, KVH, G, D, PS, window, sinks):
    c = case(8700 + D + KVH, [700, 33, 300], KVH, G, D, PS, kind, ql_list=[200, 33, 2])
    prefill(c, rows_of(c), window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 1), (127, 0), (128, 128), (129, 127), (17, 300), (255, 1), (500, 129), (100000, 5), (0, 9), (1000, 4)])
@pytest.mark.parametrize("D", [128, 256])
def test_prefill_windows(D, window, sinks):
    c = case(8800, [1300, 1000, 513, 40], 2, 4, D, 16, ql_list=[300, 1000, 1, 60])       # (60 tokens, 40 of context)
    prefill(c, rows_of(c), window, sinks)


@pytest.mark.parametrize("chunk", [128, 384, 1024])
@pytest.mark.parametrize("window,sinks", [(700, 4), (130, 260), (2000, 0), (0, 0)])
def test_prefill_chunks(chunk, window, sinks):
    """contexts beyond the chunk, piece by piece: row tiles whose keys lie in some of the pieces only"""
    for D, G in ((128, 4), (256, 8)):
        c = case(8900 + D, [2500, 1500], 2, G, D, 16, ql_list=[400, 1500])
        prefill(c, rows_of(c), window, sinks, chunk=chunk)


def test_prefill_divided_row_tiles():
    """few tokens over a wide window: row tiles divided among CTAs, cut between the sinks and the window as well"""
    for D, G, ql in ((128, 8, 16), (256, 8, 5)):
        c = case(9000 + D, [20000], 1, G, D, 16, ql_list=[ql])
        for window, sinks in ((15000, 700), (300, 128), (129, 1000)):
            prefill(c, rows_of(c), window, sinks)


def test_prefill_types_and_options():
    c = case(9100, [600, 90], 2, 4, 128, 16, ql_list=[150, 90])
    prefill(c, rows_of(c), 200, 4, out_dtype=torch.float32, q_dtype=torch.float16)
    prefill(c, rows_of(c), 200, 4, ws=K.alloc_workspace(2, 2, 4, 128, 1), lse=False)
    prefill(c, rows_of(c), 200, 4, signs=K.hadamard_signs(128, device="cuda"))
    prefill(c, [rows_of(c)[1]], 50, 0)                   # the other request's rows stay as they are
    prefill(dict(c, sm=-0.05), rows_of(c), 200, 4)


def test_prefill_without_a_window_gives_the_bits_of_prefill():
    c = case(9200, [900, 300], 2, 4, 128, 16, ql_list=[500, 300])
    t = tensors(c)
    out = prefill(c, rows_of(c), 0, 0, lse=False)
    want = torch.full_like(out, float("nan"))
    K.prefill(t["q"], c["flat"], c["strides"], 16, t["bt"], rows_of(c), c["sm"] * float(c["gk"][0]), float(c["gv"][0]), 2, want)
    assert torch.equal(out, want)


def test_prefill_of_the_last_tokens_agrees_with_decode():
    """the same rows through both operators: their log-sum-exps agree"""
    c = case(9300, [1200, 800], 2, 4, 128, 16, ql_list=[4, 4])
    t = tensors(c)
    _, a = decode(c, 300, 4, vs=1.0)
    b = torch.zeros_like(a)
    out = torch.zeros_like(t["q"])
    K.prefill_window(t["q"], c["flat"], c["strides"], 16, t["bt"], rows_of(c), c["sm"] * float(c["gk"][0]), float(c["gv"][0]), 2, out, 300, 4, lse=b)
    assert float((a - b).abs().max()) <= 2 * LSE_EACH
