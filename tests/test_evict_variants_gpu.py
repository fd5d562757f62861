"""kernels.evict in the forms that its rules choose for many short contexts (a warp selects) and for few long ones that are moved in place
(more warps a cluster), with every order of weights and every layout; against a plain sort, byte for byte."""
import numpy as np
import pytest

from test_evict_gpu import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("how", ["plain", "ties", "equal", "special", "near"])
@pytest.mark.parametrize("longest,keep,sinks,recent", [(1024, 64, 2, 10), (1024, 600, 0, 0), (1000, 100, 40, 60), (300, 7, 0, 3), (33, 1, 0, 0)])
def test_many_short_contexts(longest, keep, sinks, recent, how, where):
    rng = np.random.default_rng(longest + keep)
    lens = [longest, 0, 1, keep, keep + 1] + [int(x) for x in rng.integers(0, longest + 1, 75)]
    call("hnd", lens, keep, sinks, recent, 4, 128, 16, how=how, where=where, seed=longest)


@pytest.mark.parametrize("where", ["new", "own"])
@pytest.mark.parametrize("kind,KVH,D,PS", [("nhd", 4, 256, 16), ("region", 4, 128, 16), ("k8", 4, 256, 32)])
def test_layouts_of_many_short_contexts(kind, KVH, D, PS, where):
    rng = np.random.default_rng(1)
    call(kind, [int(x) for x in rng.integers(0, 200, 80)], 48, 2, 10, KVH, D, PS, how="ties", where=where, seed=D)


@pytest.mark.parametrize("kind,KVH,D,PS", [("k8", 2, 256, 16), ("nhd", 2, 256, 32), ("region", 2, 128, 16), ("hnd", 1, 128, 64)])
@pytest.mark.parametrize("how", ["plain", "special"])
def test_long_in_place(kind, KVH, D, PS, how):
    call(kind, [9000, 5000, 4500], 4400, 4, 500, KVH, D, PS, how=how, where="own", seed=KVH)


@pytest.mark.parametrize("longest", [12288, 12289, 16384, 16385, 16400])
@pytest.mark.parametrize("how", ["plain", "near"])
def test_lines_between_one_cta_and_several(longest, how):
    call("hnd", [longest, longest - 1, 9000], 3000, 4, 100, 1, 128, 16, how=how, where="new", seed=longest)
