"""kernels.accumulate_weights with more than 16 query rows per kv head, which go through a kernel of their own: every layout of the cache
at both head_dims, second passes, windows and sinks, rotated keys, batches of more than 32 requests. Against the definition in 64
bits, with the tolerances of tests/test_weights_gpu.py; entries that no row sees keep their bits."""
import numpy as np
import pytest
import torch

import synth
from cases import Cache, bf16_tensor
from horizon_kernels_b200 import kernels as K
from test_weights_gpu import case
from test_weights_narrow_gpu import check

pytestmark = pytest.mark.gpu

LAYOUTS = [("hnd", 128, 16), ("nhd", 128, 32), ("region", 128, 16), ("hnd", 256, 64), ("nhd", 256, 16), ("region", 256, 32), ("k8", 256, 16)]


def width(c):
    return int(c["seq_lens"].max()) + 5


@pytest.mark.parametrize("kind,D,PS", LAYOUTS)
@pytest.mark.parametrize("G,qls", [(8, [3, 1, 4, 2, 0, 4]), (6, [4, 4, 1, 2, 3, 4]), (16, [4, 1, 3, 4, 2, 0]), (1, [64, 40, 17, 3, 33, 1])])
def test_layouts(kind, D, PS, G, qls):
    """24 to 64 rows: one pass and two, tiles of eight rows that are cut, rows that see no key (more query tokens than context)"""
    c = case(9400 + G, [700, 33, 64, 1, 300, 2049], 2, G, D, PS, kind, ql_list=qls)
    check(c, width(c), qlmax=max(qls))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 3), (33, 40), (0, 7), (5000, 2), (64, 0), (300, 129)])
@pytest.mark.parametrize("kind,D", [("hnd", 128), ("hnd", 256), ("nhd", 256), ("region", 128), ("k8", 256)])
@pytest.mark.parametrize("G", [8, 16])
def test_windows(kind, D, window, sinks, G):
    c = case(9500, [500, 64, 97, 1, 0, 1023], 2, G, D, 16, kind, ql_list=[1, 2, 3, 1, 1, 4])
    check(c, width(c), window, sinks, qlmax=4)


@pytest.mark.parametrize("D,kind", [(128, "hnd"), (256, "hnd"), (256, "nhd")])
@pytest.mark.parametrize("window", [0, 90])
def test_rotated_keys(D, kind, window):
    signs = K.hadamard_signs(D, device="cuda")
    c = synth.paged_case(9550 + D, [400, 65, 130], 2, 8, D, 16, ql_list=[4, 3, 4])
    cache = Cache(c["NP"], 16, 2, D, kind, 0x7f)
    gk = np.full(2, synth.tensor_scale(c["key"]) * 2, np.float32)
    gkt = torch.from_numpy(gk).cuda()
    K.write(bf16_tensor(c["key"]), bf16_tensor(c["val"]), cache.flat, cache.strides, 16, torch.from_numpy(c["slots"]).cuda(), gkt, gkt, signs=signs)
    c.update(phys=cache.phys, flat=cache.flat, strides=cache.strides, kind=kind, gk=gk, gv=gk, sm=D ** -0.5)
    check(c, width(c), window, 4, signs=signs)


@pytest.mark.parametrize("G,D,window", [(8, 128, 0), (8, 256, 0), (16, 128, 200), (4, 128, 60), (2, 256, 0)])
def test_many_requests(G, D, window):
    """more than 32 requests, some of which have no rows in the call (and fewer rows a pass, for the same search)"""
    rng = np.random.default_rng(3)
    lens = [9000, 3000] + [int(x) for x in rng.integers(1, 400, 70)]
    qls = [4, 1] + [int(x) for x in rng.integers(0, 5, 70)]
    c = case(9560, lens, 2, G, D, 16, ql_list=qls)
    check(c, width(c), window, 3, qlmax=4)


def test_scales():
    c = case(9570, [300, 90], 4, 8, 128, 16, ql_list=[4, 3], gscale=(0.002, 0.001))
    for sm in (0.05, 0.0, -0.05):
        check(dict(c, sm=sm), 300)
