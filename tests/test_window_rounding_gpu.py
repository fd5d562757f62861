"""Attention of prompts over a window is as exact as without one: a 16-bit output is the rounded fp32 output of the same call, and a
window that no context exceeds gives the bits of `prefill`."""
import pytest
import torch

from horizon_kernels_b200 import kernels as K
from test_weights_gpu import case, tensors
from test_window_gpu import rows_of

pytestmark = pytest.mark.gpu

SHAPES = [("hnd", 8, 4, 128, [1500, 900, 64]), ("hnd", 2, 8, 256, [1300, 700]), ("nhd", 2, 8, 128, [2000]), ("k8", 2, 8, 256, [600, 900])]


def call(c, t, rows, window, sinks, dtype, chunk=65536):
    out = torch.full(t["q"].shape, float("nan"), dtype=dtype, device="cuda")
    args = (t["q"], c["flat"], c["strides"], c["PS"], t["bt"], rows, c["sm"] * float(c["gk"][0]), float(c["gv"][0]), c["KVH"], out)
    if window is None:
        K.prefill(*args, chunk=chunk, k8=c["kind"] == "k8")
    else:
        K.prefill_window(*args, window, sinks, chunk=chunk, k8=c["kind"] == "k8")
    return out


@pytest.mark.parametrize("kind,KVH,G,D,lens", SHAPES)
@pytest.mark.parametrize("window,sinks", [(100, 4), (800, 0), (1100, 130)])
def test_a_16_bit_output_is_the_rounded_fp32_output(kind, KVH, G, D, lens, window, sinks):
    c = case(9800 + D, lens, KVH, G, D, 16, kind, ql_list=[(n + 1) // 2 for n in lens])
    t = tensors(c)
    for chunk in (65536, 512):
        a, b = (call(c, t, rows_of(c), window, sinks, dt, chunk) for dt in (torch.bfloat16, torch.float32))
        assert torch.isfinite(b).all() and torch.equal(a, b.to(torch.bfloat16))


@pytest.mark.parametrize("kind,KVH,G,D,lens", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_window_that_no_context_exceeds_gives_the_bits_of_prefill(kind, KVH, G, D, lens, dtype):
    c = case(9900 + D, lens, KVH, G, D, 16, kind, ql_list=lens)
    t = tensors(c)
    want = call(c, t, rows_of(c), None, 0, dtype)
    for window, sinks in ((max(lens), 0), (100000, 4), ((1 << 31) - 1, 0)):
        assert torch.equal(call(c, t, rows_of(c), window, sinks, dtype), want)
