"""kernels.accumulate_weights with weights that are narrower than a context: the query tokens stay at the end of the whole context,
and the tokens that the weights have no entry for gather nothing. Against the definition in 64 bits, entry by entry, with the
tolerances of tests/test_weights_gpu.py; entries that no row sees keep their bits."""
import pytest
import torch

import window_ref as R
from horizon_kernels_b200 import kernels as K
from test_weights_gpu import EACH, NORM, case, reference, tensors

pytestmark = pytest.mark.gpu


def check(c, W, window=0, sinks=0, qlmax=None, signs=None):
    """one call over weights W wide"""
    t = tensors(c)
    qlens = [int(x) for x in c["qsl"][1:] - c["qsl"][:-1]]
    qlmax = max(1, max(qlens)) if qlmax is None else qlmax
    lse, add = reference(c, window, sinks, qlmax, signs)
    B, KVH, n = add.shape
    add = torch.nn.functional.pad(add, (0, max(0, W - n)))[..., :W]
    seen = torch.zeros(B, W, dtype=torch.bool)
    for b, L in enumerate(int(x) for x in c["seq_lens"]):
        if 0 < qlens[b] <= qlmax and L:
            see = R.seen(L, qlens[b], window, sinks).any(0)[:W]
            seen[b, :see.numel()] = see
    g = torch.Generator(device="cuda").manual_seed(5)
    w = 1e-3 * torch.rand(B, KVH, W, device="cuda", generator=g)
    w0 = w.cpu()
    K.accumulate_weights(t["q"], c["flat"], c["strides"], c["PS"], t["bt"], t["sl"], t["qsl"], c["sm"], t["gk"], qlmax, lse.float().cuda(), w,
                         window=window, sinks=sinks, signs=signs, k8=c["kind"] == "k8")
    assert K.workspace_status(None) == 0
    w = w.cpu()
    untouched = ~seen[:, None].expand(B, KVH, W)
    assert torch.equal(w[untouched].view(torch.int32), w0[untouched].view(torch.int32))
    want = w0.double() + add
    err = (w.double() - want).abs()
    assert bool((err <= EACH * add + 2.0 ** -23 * want + 1e-37).all()), float((err / (EACH * add + 2.0 ** -23 * want + 1e-37)).max())
    assert float(err.norm()) <= NORM * float(add.norm()) + 2.0 ** -23 * float(want.norm())


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4), (1, 0), (230, 3), (450, 0), (60, 400), (5000, 1)])
@pytest.mark.parametrize("W", [1, 33, 100, 256])
@pytest.mark.parametrize("G,qls", [(4, [1, 1, 1, 1, 1]), (4, [4, 2, 3, 1, 0]), (8, [4, 1, 3, 4, 2])])
def test_narrow_weights(G, qls, W, window, sinks):
    """8, 16 and 32 query rows a pass; windows that lie behind the weights, across their end and before it"""
    check(case(9600 + G, [300, 90, 500, 33, 257], 2, G, 128, 16, ql_list=qls), W, window, sinks, qlmax=4)


@pytest.mark.parametrize("kind,D,PS", [("nhd", 128, 32), ("region", 128, 16), ("hnd", 256, 64), ("k8", 256, 16)])
@pytest.mark.parametrize("G", [4, 8])
def test_layouts(kind, D, PS, G):
    check(case(9700, [300, 90, 0, 700], 2, G, D, PS, kind, ql_list=[4, 1, 2, 3]), 150, 170, 5, qlmax=4)
