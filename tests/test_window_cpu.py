"""What the operators for bounded caches refuse, before anything is launched: in the C ABI, in the Python wrappers and in the
backend's switches; and that none of their kernels spills more than it is known to."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import window_ref as R
from horizon_kernels_b200 import _lib, build
from horizon_kernels_b200 import kernels as K

os.environ["HORIZON_KVFP4_STANDALONE"] = "1"
from horizon_kernels_b200 import backend as BE  # noqa: E402

ONE = C.c_void_p(0x1000)


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def strides(*v):
    return (C.c_int64 * 6)(*v)


SLOT = strides(18432, 72, 1152, 18432, 72, 1152)


def test_decode_window_rejects_misuse(lib):
    base = dict(q=ONE, kd=ONE, ksf=C.c_void_p(0x1040), vd=C.c_void_p(0x3400), vsf=C.c_void_p(0x3440), st=SLOT, PS=16, bt=ONE, MP=8, sl=ONE,
                qsl=ONE, B=4, KVH=8, G=4, D=128, qlmax=1, gk=ONE, gv=ONE, ws=ONE, wsb=1 << 20, splits=0, signs=None, k8=0, window=64,
                sinks=4, lse=None, out=ONE)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_decode_window(a["q"], a["kd"], a["ksf"], a["vd"], a["vsf"], a["st"], a["PS"], a["bt"], a["MP"], a["sl"], a["qsl"],
                                     a["B"], a["KVH"], a["G"], a["D"], a["qlmax"], 0.088, 1.0, a["gk"], a["gv"], a["ws"], a["wsb"],
                                     a["splits"], a["signs"], a["k8"], a["window"], a["sinks"], a["lse"], a["out"], None)
    for name in ("q", "kd", "ksf", "vd", "vsf", "bt", "sl", "qsl", "gk", "gv", "ws", "out"):
        assert call(**{name: None}) == -1, name
    assert call(window=-1) == call(sinks=-1) == call(B=-1) == call(MP=-1) == -6
    assert call(B=0) == 0
    assert call(lse=C.c_void_p(0x1002)) == call(q=C.c_void_p(0x1008)) == call(ws=C.c_void_p(0x1010)) == -2
    assert call(D=64) == call(G=65) == call(qlmax=17) == call(PS=24) == call(k8=1) == -3
    assert call(splits=65) == -4
    assert call(window=(1 << 30) + 1, MP=1 << 28) == -6                   # (a table that reaches further)


def test_prefill_window_rejects_misuse(lib):
    rows = (C.c_int32 * 4)(1, 0, 40, 100)
    base = dict(q=ONE, f16=0, kd=ONE, ksf=ONE, vd=ONE, vsf=ONE, st=SLOT, PS=16, bt=ONE, B=2, MP=8, rows=rows, n=1, NT=40, KVH=8, G=4,
                D=128, signs=None, k8=0, chunk=65536, window=64, sinks=4, lse=None, scratch=ONE, nb=1 << 40, out=ONE, ws=ONE)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_prefill_window(a["q"], a["f16"], a["kd"], a["ksf"], a["vd"], a["vsf"], a["st"], a["PS"], a["bt"], a["B"], a["MP"],
                                      a["rows"], a["n"], a["NT"], a["KVH"], a["G"], a["D"], 0.088, 1.0, a["signs"], a["k8"], a["chunk"],
                                      a["window"], a["sinks"], a["lse"], a["scratch"], a["nb"], a["out"], 0, a["ws"], None)
    assert call(n=0) == 0
    for name in ("q", "kd", "ksf", "vd", "vsf", "bt", "scratch", "out", "rows"):
        assert call(**{name: None}) == -1, name
    assert call(window=-1) == call(sinks=-1) == call(n=-1) == -6
    assert call(lse=C.c_void_p(0x1002)) == call(q=C.c_void_p(0x1008)) == call(scratch=C.c_void_p(0x1080)) == -2
    assert call(D=64) == call(G=129) == call(KVH=0) == call(k8=1) == call(signs=ONE, f16=1) == -3
    for r in ((-1, 0, 40, 100), (2, 0, 40, 100), (1, -1, 40, 100), (1, 7, 7, 100), (1, 0, 41, 100), (1, 0, 40, 0), (1, 0, 40, 129)):
        assert call(rows=(C.c_int32 * 4)(*r)) == -6, r
    need = lib.hkv_prefill_window_scratch_bytes(rows, 1, 40, 8, 4, 128, 65536, 0, 64, 4)
    assert need > 0 and call(nb=need - 1) == -5
    full = (C.c_int32 * 4)(0, 0, 40, 20000)                             # tokens that no row sees take no scratch
    win = lib.hkv_prefill_window_scratch_bytes(full, 1, 40, 8, 4, 128, 65536, 0, 64, 4)
    assert win < lib.hkv_prefill_scratch_bytes(full, 1, 40, 8, 4, 128, 65536, 0)
    assert lib.hkv_prefill_window_scratch_bytes(full, 1, 40, 8, 4, 128, 65536, 0, 0, 4) == lib.hkv_prefill_scratch_bytes(
        full, 1, 40, 8, 4, 128, 65536, 0)
    assert lib.hkv_prefill_window_scratch_bytes(full, 1, 40, 8, 4, 128, 65536, 0, -1, 4) == 0
    assert lib.hkv_prefill_window_scratch_bytes(full, 1, 40, 8, 4, 96, 65536, 0, 64, 4) == 0


def test_accumulate_weights_rejects_misuse(lib):
    base = dict(q=ONE, kd=ONE, ksf=C.c_void_p(0x1040), st=SLOT, PS=16, bt=ONE, MP=8, sl=ONE, qsl=ONE, B=4, KVH=8, G=4, D=128, qlmax=1, gk=ONE,
                lse=ONE, w=ONE, W=128, window=0, sinks=0, signs=None, k8=0, ws=ONE)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_accumulate_weights(a["q"], a["kd"], a["ksf"], a["st"], a["PS"], a["bt"], a["MP"], a["sl"], a["qsl"], a["B"], a["KVH"],
                                          a["G"], a["D"], a["qlmax"], 0.088, a["gk"], a["lse"], a["w"], 8 * 128, 128, a["W"], a["window"],
                                          a["sinks"], a["signs"], a["k8"], a["ws"], None)
    for name in ("q", "kd", "ksf", "bt", "sl", "qsl", "gk", "lse", "w"):
        assert call(**{name: None}) == -1, name
    assert call(B=0) == 0
    assert call(B=-1) == call(MP=-1) == call(W=-1) == call(window=-1) == call(sinks=-1) == call(B=100000) == -6
    assert call(D=64) == call(G=65) == call(qlmax=17) == call(G=0) == call(PS=8) == call(PS=24) == call(k8=1) == -3
    assert call(k8=1, D=256, signs=ONE, st=strides(102400, 400, 6400, 102400, 400, 6400)) == -3
    assert call(st=strides(18432, 2304, 144, 18432, 1152, 144)) == -3      # scales not behind their token's codes
    for name, at in (("q", 0x1008), ("lse", 0x1002), ("w", 0x1002), ("ws", 0x1010), ("signs", 0x1008)):
        assert call(**{name: C.c_void_p(at)}) == -2, name
    assert call(kd=C.c_void_p(0x1008), ksf=C.c_void_p(0x1048)) == -2
    assert call(st=strides(1 << 31, 72, 1152, 1 << 31, 72, 1152)) == -6


def test_evict_rejects_misuse(lib):
    base = dict(kd=ONE, ksf=C.c_void_p(0x1040), vd=C.c_void_p(0x3400), vsf=C.c_void_p(0x3440), st=SLOT, PS=16, bt=ONE, MP=8, sl=ONE, B=4, KVH=8,
                D=128, k8=0, w=ONE, W=128, keep=32, sinks=4, recent=8, ot=ONE, OMP=2, kept=ONE, ol=C.c_void_p(0x2000), ow=ONE, OW=32)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_evict(a["kd"], a["ksf"], a["vd"], a["vsf"], a["st"], a["PS"], a["bt"], a["MP"], a["sl"], a["B"], a["KVH"], a["D"],
                             a["k8"], a["w"], 1024, 128, a["W"], a["keep"], a["sinks"], a["recent"], a["ot"], a["OMP"], a["kept"], a["ol"],
                             a["ow"], 256, 32, a["OW"], None)
    for name in ("kd", "ksf", "vd", "vsf", "bt", "sl", "w", "ot", "kept", "ol", "ow"):
        assert call(**{name: None}) == -1, name
    assert call(B=0) == 0
    assert call(B=-1) == call(MP=-1) == call(OMP=-1) == call(W=-1) == call(OW=-1) == call(B=100000) == -6
    assert call(keep=0) == call(sinks=-1) == call(recent=-1) == call(sinks=30) == call(keep=33) == call(OW=31) == call(OMP=1) == -6
    assert call(sinks=(1 << 31) - 1, recent=(1 << 31) - 1) == -6
    assert call(D=64) == call(k8=1) == call(KVH=0) == call(KVH=1025) == call(PS=8) == call(PS=24) == -3
    assert call(ol=ONE) == -3                                              # the lengths' own array
    assert call(kd=C.c_void_p(0x1004)) == call(st=strides(18432, 70, 1152, 18432, 72, 1152)) == call(w=C.c_void_p(0x1002)) == -2
    assert call(D=256, st=strides(18432, 152, 1152, 18432, 152, 1152)) == -2


def tensors():
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    flat, st, g = tuple(torch.zeros(64, dtype=torch.uint8) for _ in range(4)), (1, 1, 1, 1, 1, 1), torch.ones(2)
    bt, lens, qsl = (torch.zeros(s, dtype=torch.int32) for s in ((2, 4), (2,), (3,)))
    return q, flat, st, g, bt, lens, qsl


def test_wrappers_check_before_any_launch():
    q, flat, st, g, bt, lens, qsl = tensors()
    out, ws, lse, w = q.clone(), flat[0], torch.zeros(2, 8), torch.zeros(2, 2, 64)

    def decode(**kw):
        a = dict(dict(q=q, bt=bt, window=4, sinks=1, lse=None, signs=None, k8=False, out=out), **kw)
        K.decode_window(a["q"], flat, st, 16, a["bt"], lens, qsl, 1.0, 1.0, g, g, 1, a["out"], ws, a["window"], a["sinks"], signs=a["signs"],
                        k8=a["k8"], lse=a["lse"])

    def prefill(**kw):
        a = dict(dict(q=q, rows=[(0, 0, 2, 5)], window=4, sinks=1, lse=None, signs=None, k8=False), **kw)
        K.prefill_window(a["q"], flat, st, 16, bt, a["rows"], 1.0, 1.0, 2, out, a["window"], a["sinks"], signs=a["signs"], k8=a["k8"],
                         lse=a["lse"])

    def gather(**kw):
        a = dict(dict(q=q, lse=lse, w=w, window=0, sinks=0, signs=None, k8=False), **kw)
        K.accumulate_weights(a["q"], flat, st, 16, bt, lens, qsl, 1.0, g, 1, a["lse"], a["w"], window=a["window"], sinks=a["sinks"],
                             signs=a["signs"], k8=a["k8"])
    for call in (decode, prefill, gather):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
        for bad in (dict(window=-1), dict(sinks=-1), dict(window=1 << 31), dict(k8=True, signs=g)):
            with pytest.raises(ValueError):
                call(**bad)
        with pytest.raises(TypeError):
            call(q=q.float())
    with pytest.raises(TypeError):
        decode(bt=bt.long())
    with pytest.raises(ValueError):
        prefill(rows=[(0, 0, 2, 65)])                                      # positions beyond the table
    with pytest.raises(TypeError):
        gather(lse=None)


def test_lse_and_weights_are_checked(monkeypatch):
    """the checks behind the one for CUDA tensors, which these stand-ins pass"""
    monkeypatch.setattr(K, "_need_cuda", lambda *t: None)
    for bad in (torch.zeros(2, 8, dtype=torch.float64), torch.zeros(1, 8), torch.zeros(2, 9), torch.zeros(8, 2).T, torch.zeros(16)):
        with pytest.raises(TypeError):
            K._check_lse(bad, 2, 8)
    K._check_lse(torch.zeros(3, 8), 2, 8)
    K._check_lse(None, 2, 8)
    for bad in (torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, 64), torch.zeros(3, 2, 64)):
        with pytest.raises(TypeError):
            K._check_weights(bad, 2)
    for bad in (torch.zeros(2, 64, 2).transpose(1, 2), torch.zeros(2, 1, 64).expand(2, 2, 64), torch.zeros(1, 2, 64).expand(2, 2, 64)):
        with pytest.raises(ValueError):
            K._check_weights(bad, 2)
    K._check_weights(torch.zeros(2, 4, 64)[:, 1:3], 2)

    q, flat, st, _, bt, lens, _ = tensors()
    w, kept, ol = torch.zeros(2, 2, 64), torch.zeros(2, 2, 16, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def evict(**kw):
        a = dict(dict(w=w, keep=16, sinks=2, recent=3, kept=kept, ol=ol, ot=None, ow=None, bt=bt, lens=lens), **kw)
        K.evict(flat, st, 16, 128, a["bt"], a["lens"], a["w"], a["keep"], a["sinks"], a["recent"], a["kept"], a["ol"], out_tables=a["ot"],
                out_weights=a["ow"])
    both = torch.zeros(4, dtype=torch.int32)
    wide = torch.zeros(2, 2, 80)
    for bad in (dict(keep=0), dict(sinks=-1), dict(recent=-1), dict(sinks=14), dict(keep=17), dict(kept=kept[:1]), dict(ol=ol[:1]),
                dict(ot=bt[:1]), dict(ot=bt[:, :0].contiguous()), dict(ow=torch.zeros(2, 2, 15)), dict(ow=torch.zeros(2, 3, 16)), dict(ol=lens),
                dict(lens=both[:2], ol=both[1:3]), dict(w=wide[..., :64], ow=wide[..., 8:72]), dict(keep=65, kept=torch.zeros(2, 2, 65, dtype=torch.int32))):
        with pytest.raises(ValueError):
            evict(**bad)
    for bad in (dict(bt=bt.long()), dict(lens=lens.long()), dict(kept=kept.long()), dict(w=w.double()), dict(w=w[0]), dict(ow=w.half())):
        with pytest.raises(TypeError):
            evict(**bad)


def test_backend_switches(monkeypatch):
    def impl():
        return BE.HorizonFp4Impl(32, 128, 0.088, num_kv_heads=8, kv_cache_dtype="nvfp4")
    assert impl().window == 0 and impl().sinks == 0
    monkeypatch.setenv("HORIZON_KVFP4_WINDOW", "4096")
    assert (impl().window, impl().sinks) == (4096, 4)
    monkeypatch.setenv("HORIZON_KVFP4_SINKS", "0")
    assert (impl().window, impl().sinks) == (4096, 0)
    monkeypatch.setenv("HORIZON_KVFP4_SINKS", "-1")
    with pytest.raises(ValueError):
        impl()
    monkeypatch.setenv("HORIZON_KVFP4_SINKS", "4")
    monkeypatch.setenv("HORIZON_KVFP4_WINDOW", "-5")
    with pytest.raises(ValueError):
        impl()


def test_the_plain_forms():
    """the references of the GPU tests, on cases worked out by hand"""
    assert R.seen(6, 2, 3, 1).int().tolist() == [[1, 0, 1, 1, 1, 0], [1, 0, 0, 1, 1, 1]]
    assert R.seen(2, 3, 1, 0).int().tolist() == [[0, 0], [1, 0], [0, 1]]
    w = [5.0, 1.0, float("nan"), 1.0, -2.0, 1.0, 0.5, 9.0]
    assert R.kept_positions(w, 8, 0, 0).tolist() == list(range(8))
    assert R.kept_positions(w, 4, 1, 1).tolist() == [0, 1, 2, 7]
    assert R.kept_positions(w, 3, 0, 0).tolist() == [0, 2, 7]
    assert R.kept_positions([0.0, -0.0, 0.0, -1.0], 2, 0, 0).tolist() == [0, 1]
    code = torch.tensor([[0x21, 0xf9, 0, 0, 0, 0, 0, 0]], dtype=torch.uint8)
    sf = torch.tensor([[0x40]], dtype=torch.uint8)                          # 2.0
    assert R.fp4(code, sf)[0, :4].tolist() == [1.0, 2.0, -1.0, -12.0]
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(2, 1, 2, 8, generator=g), torch.randn(5, 1, 8, generator=g).double(), torch.randn(5, 1, 8, generator=g).double()
    out, lse = R.attention(q, k, v, [0.5], [2.0], 0, 0)
    x = (q[1, 0, 1].double() @ k[:, 0].T) * 0.5
    assert torch.allclose(out[1, 0, 1], torch.softmax(x, 0) @ v[:, 0] * 2) and torch.allclose(lse[1, 0, 1], torch.logsumexp(x, 0))
    assert abs(float(R.gathered(q, k, [0.5], lse, 0, 0).sum()) - 4) < 1e-12      # four rows give away a weight of one each


def test_no_kernel_of_a_bounded_cache_spills_more_than_known(tmp_path):
    """the sixteen-row decode kernels at head_dim 256 over a window keep 32 bytes in local memory (FP8 keys: 4), the prefill's at 256 8, the
    selection 4; the others none"""
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    flags = [f for f in build.NVCC_FLAGS if f not in ("-shared", "-cudart", "static")]
    jobs = {s: subprocess.Popen([nvcc, *flags, "-Xptxas", "-v", "-c", "-o", str(tmp_path / (s + ".o")), os.path.join(build.CSRC, s)],
                                stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
            for s in ("hkv_decode.cu", "hkv_prefill.cu", "hkv_weights.cu", "hkv_evict.cu")}
    spills, name = {}, None
    for s, j in jobs.items():
        _, err = j.communicate()
        assert j.returncode == 0, err
        for line in err.splitlines():
            if "Function properties for" in line:
                name = line.split()[-1]
            elif "bytes spill stores" in line:
                spills[name] = int(line.split("frame, ")[1].split()[0])
    ours = {k: v for k, v in spills.items() if any(x in k for x in ("window_kernel", "weights_kernel", "select_kernel", "move_kernel"))
            or ("attend_kernel" in k and "ELb0ELb1E" in k)}
    assert len(ours) == 12 + 21 + 1 + 9 + 2, sorted(ours)
    known = {"window_kernelILi256ELi0ELi2E": 32, "window_kernelILi256ELi3ELi2E": 32, "window_kernelILi256ELi2ELi2E": 4, "attend_kernelILi256": 8, "select_kernel": 4}
    over = {k: v for k, v in ours.items() if v > max([0] + [n for x, n in known.items() if x in k])}
    assert not over, over
