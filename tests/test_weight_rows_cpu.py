"""Rows of weights that overlap one another are refused where they are written: two CTAs would add to one number."""
import ctypes as C

import pytest
import torch

from horizon_kernels_b200 import _lib, build
from horizon_kernels_b200 import kernels as K

APART = [((2, 3, 8), (24, 8, 1)), ((2, 3, 8), (8, 16, 1)), ((2, 3, 8), (100, 30, 1)), ((1, 3, 8), (1, 8, 1)), ((2, 1, 8), (8, 1, 1)), ((1, 1, 8), (1, 1, 1)),
         ((2, 3, 1), (1, 2, 1)), ((2, 3, 0), (1, 1, 1))]
ACROSS = [((2, 3, 8), (24, 7, 1)), ((2, 3, 8), (8, 8, 1)), ((2, 3, 8), (23, 8, 1)), ((2, 3, 8), (8, 15, 1)), ((1, 3, 8), (24, 1, 1)), ((2, 1, 8), (7, 8, 1)),
          ((2, 3, 1), (1, 1, 1))]


def view(shape, strides):
    return torch.as_strided(torch.zeros(400), shape, strides)


def test_the_wrappers(monkeypatch):
    monkeypatch.setattr(K, "_need_cuda", lambda *t: None)
    for shape, strides in APART:
        K._check_weights(view(shape, strides), shape[0])
    for shape, strides in ACROSS:
        with pytest.raises(ValueError, match="overlap"):
            K._check_weights(view(shape, strides), shape[0])


def test_the_abi():
    build.build()
    lib, p = _lib.load(), C.c_void_p
    st, one = (C.c_int64 * 6)(18432, 72, 1152, 18432, 72, 1152), p(0x1000)
    for (B, KVH, W), (w_b, w_h, _) in ACROSS:
        assert lib.hkv_accumulate_weights(one, one, p(0x1040), st, 16, one, 8, one, one, B, KVH, 4, 128, 1, 0.088, one, one, one, w_b, w_h, W, 0, 0,
                                          None, 0, one, None) == -3
        assert lib.hkv_evict(one, p(0x1040), p(0x3400), p(0x3440), st, 16, one, 8, p(0x1000), B, KVH, 128, 0, p(0x100000), 64 * KVH, 64, 64, 1, 0, 0,
                             one, 2, one, p(0x2000), p(0x200000), w_b, w_h, W, None) == -3
