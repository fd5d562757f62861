"""hkv_evict refuses outputs that lie across its inputs, in the C ABI too: tokens' weights and lengths are read while others are
written. (Every call here is refused, or has no requests: nothing is launched.)"""
import ctypes as C

import pytest

from horizon_kernels_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_outputs_across_inputs_are_refused(lib):
    one, st = 0x1000, (C.c_int64 * 6)(18432, 72, 1152, 18432, 72, 1152)
    base = dict(B=4, KVH=8, w=0x100000, w_b=1024, w_h=128, W=128, sl=0x1000, ol=0x2000, ow=0x100000, ow_b=1024, ow_h=128, OW=128)

    def call(**kw):
        a = dict(base, **kw)
        p = C.c_void_p
        return lib.hkv_evict(p(one), p(0x1040), p(0x3400), p(0x3440), st, 16, p(one), 8, p(a["sl"]), a["B"], a["KVH"], 128, 0, p(a["w"]), a["w_b"],
                             a["w_h"], a["W"], 32, 4, 8, p(one), 2, p(one), p(a["ol"]), p(a["ow"]), a["ow_b"], a["ow_h"], a["OW"], None)
    # the same address with other strides: one head's new weights lie where another's are read
    assert call(ow_b=256, ow_h=32, OW=32) == call(ow_h=64, OW=64) == call(w_b=2048) == -3
    # a part of them
    assert call(ow=0x100000 + 16) == call(ow=0x100000 - 16) == call(ow=0x100000 + 4 * (4 * 1024 - 1), ow_b=256, ow_h=32, OW=32) == -3
    # lengths that begin inside the others
    assert call(ol=0x1004) == call(ol=0x100c) == call(sl=0x2008) == -3
