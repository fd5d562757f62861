"""kernels.decode_window with nine to sixteen query rows per kv head, which are one pass over all slot layouts: positions-outermost pages
at head_dim 256 above all. Tolerances as in tests/test_window_gpu.py."""
import pytest

from horizon_kernels_b200 import kernels as K
from test_weights_gpu import case
from test_window_gpu import decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,D,PS", [("nhd", 256, 16), ("nhd", 128, 32), ("hnd", 256, 16), ("k8", 256, 16), ("region", 256, 16)])
@pytest.mark.parametrize("G,qls", [(8, [2, 1, 2, 0, 2]), (12, [1, 1, 1, 1, 1]), (4, [4, 3, 1, 4, 2]), (16, [1, 2, 1, 1, 2])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (1, 0), (333, 50)])
def test_rows(kind, D, PS, G, qls, window, sinks):
    decode(case(9900 + G, [700, 33, 1, 0, 2049], 2, G, D, PS, kind, ql_list=qls), window, sinks, qlmax=max(qls))


@pytest.mark.parametrize("window,sinks", [(0, 0), (6000, 33)])
def test_split_sequences(window, sinks):
    decode(case(9950, [9000, 300], 1, 16, 256, 16, "nhd"), window, sinks)


def test_rotated():
    decode(case(9960, [400, 65], 2, 8, 256, 16, "nhd", ql_list=[2, 2]), 64, 4, signs=K.hadamard_signs(256, device="cuda"))
