"""The 8-bit cache and the rotating writes without a GPU: the layout, what the C ABI and the wrappers refuse before anything is
launched, and the plain forms that the GPU tests go by, on values worked out by hand."""
import ctypes as C

import pytest
import torch

import b8_ref as R
from horizon_kernels_b200 import _lib, build
from horizon_kernels_b200 import kernels as K
from horizon_kernels_b200 import layout as Lt


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


ONE = C.c_void_p(0x100000)


def at(x):
    return C.c_void_p(x)


def two(*v):
    return (C.c_int64 * 2)(*v)


def rotary(**kw):
    """queries (8 heads) at 2 MB, turned ones at 4 MB, keys and values of the calls below at 1 MB"""
    a = dict(query=0x200000, qs0=1024, qs1=128, query_out=0x400000, os0=1024, os1=128, n_tokens=4, positions=0x500000, table=0x600000,
             rows=100, HQ=8, rot=128, table_bf16=0, interleaved=0)
    a.update(kw)
    return _lib.Rotary(*[a[n] for n, _ in _lib.Rotary._fields_])


BAD_ROTARY = [(dict(query=None), -1), (dict(query_out=None), -1), (dict(positions=None), -1), (dict(table=None), -1),
              (dict(n_tokens=3), -6), (dict(rows=0), -6), (dict(qs0=-8), -6), (dict(os1=-8), -6), (dict(n_tokens=1 << 31), -6),
              (dict(rot=0), -3), (dict(rot=8), -3), (dict(rot=24), -3), (dict(rot=144), -3), (dict(HQ=0), -3),
              (dict(query=0x200008), -2), (dict(query_out=0x400008), -2), (dict(table=0x600008), -2), (dict(positions=0x500004), -2),
              (dict(qs0=1028), -2), (dict(os1=132), -2),
              (dict(os1=64), -6), (dict(os0=512), -6),                                        # turned rows over one another
              (dict(query_out=0x200010), -6), (dict(query_out=0x200000, os0=2048), -6),       # .. over the queries
              (dict(query_out=0x200000 + 2 * 512), -6),
              (dict(query_out=0x100000, os0=1024), -6), (dict(query_out=0x100800 - 16), -6)]  # .. over the keys


def test_write_rotary_refuses(lib):
    st = (C.c_int64 * 6)(18432, 72, 1152, 18432, 72, 1152)

    def call(r=None, signs=None, k8=0, D=128, n=4, key=ONE, none=False):
        return lib.hkv_write_rotary(key, ONE, 1024, 128, 1024, 128, ONE, ONE, ONE, ONE, st, 16, ONE, n, ONE, ONE, 8, D, 1, signs, k8,
                                    None if none else C.byref(r or rotary()), None)
    assert call(none=True) == -1
    assert call(signs=ONE, k8=1) == -3
    assert call(k8=1) == -3                                   # FP8 keys at head_dim 256 only
    assert call(D=64) == -3 and call(key=None) == -1 and call(key=at(0x100008)) == -2 and call(n=-1) == -6
    assert call(rotary(n_tokens=0), n=0) == 0                 # nothing to do
    for kw, code in BAD_ROTARY:
        assert call(rotary(**kw)) == code, kw


def test_write_b8_refuses(lib):
    base = dict(key=ONE, val=ONE, ks=(1024, 128, 1024, 128), kt=ONE, vt=ONE, st=two(2 * 8 * 2064, 2064), PS=16, slots=ONE, n=4, gk=ONE, gv=ONE,
                KVH=8, D=128, fmt=0, r=None)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_write_b8(a["key"], a["val"], *a["ks"], a["kt"], a["vt"], a["st"], a["PS"], a["slots"], a["n"], a["gk"], a["gv"],
                                a["KVH"], a["D"], a["fmt"], None if a["r"] is None else C.byref(a["r"]), None)
    assert call(n=0) == 0 and call(n=0, r=rotary(n_tokens=0)) == 0
    for name in ("key", "val", "kt", "vt", "st", "slots", "gk", "gv"):
        assert call(**{name: None}) == -1, name
    assert call(n=-1) == call(n=1 << 31) == -6
    for kw in (dict(D=64), dict(fmt=2), dict(fmt=-1), dict(KVH=0), dict(KVH=1025), dict(PS=8), dict(PS=24), dict(PS=0)):
        assert call(**kw) == -3, kw
    for kw in (dict(key=at(0x100008)), dict(val=at(0x100008)), dict(kt=at(0x100008)), dict(vt=at(0x100008)), dict(st=two(33032, 2064)),
               dict(st=two(33024, 2056)), dict(ks=(1024, 132, 1024, 128))):
        assert call(**kw) == -2, kw
    for kw, code in BAD_ROTARY:
        assert call(r=rotary(**kw)) == code, kw


def test_decode_b8_refuses(lib):
    base = dict(q=ONE, kt=ONE, vt=ONE, st=two(2 * 8 * 2064, 2064), PS=16, bt=ONE, MP=8, sl=ONE, qsl=ONE, B=4, KVH=8, G=4, D=128, qlmax=1, gk=ONE,
                gv=ONE, ws=ONE, wsb=1 << 20, splits=0, fmt=0, window=0, sinks=0, lse=None, out=ONE)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_decode_b8(a["q"], a["kt"], a["vt"], a["st"], a["PS"], a["bt"], a["MP"], a["sl"], a["qsl"], a["B"], a["KVH"], a["G"],
                                 a["D"], a["qlmax"], 0.1, 1.0, a["gk"], a["gv"], a["ws"], a["wsb"], a["splits"], a["fmt"], a["window"],
                                 a["sinks"], a["lse"], a["out"], None)
    assert call(B=0) == 0
    for name in ("q", "kt", "vt", "st", "bt", "sl", "qsl", "gk", "gv", "ws", "out"):
        assert call(**{name: None}) == -1, name
    for kw in (dict(D=64), dict(fmt=2), dict(fmt=-1), dict(KVH=0), dict(G=0), dict(G=65), dict(qlmax=17), dict(qlmax=0), dict(PS=8),
               dict(PS=48), dict(G=1 << 20, qlmax=1 << 12)):
        assert call(**kw) == -3, kw
    for kw in (dict(B=-1), dict(B=100000), dict(MP=-1), dict(window=-1), dict(sinks=-1), dict(splits=-1), dict(st=two(-16, 2064)),
               dict(st=two(1 << 31, 2064))):
        assert call(**kw) == -6, kw
    assert call(splits=65) == -4
    for kw in (dict(q=at(0x100008)), dict(out=at(0x100008)), dict(kt=at(0x100008)), dict(vt=at(0x100008)), dict(st=two(33032, 2064)),
               dict(st=two(33024, 2056)), dict(ws=at(0x100010)), dict(lse=at(0x100002))):
        assert call(**kw) == -2, kw


def test_prefill_b8_refuses(lib):
    base = dict(q=ONE, kt=ONE, vt=ONE, st=two(2 * 8 * 2064, 2064), PS=16, bt=ONE, B=2, MP=8, rows=(C.c_int32 * 4)(1, 0, 40, 100), n=1, NT=40, KVH=8,
                G=4, D=128, fmt=0, window=0, sinks=0, lse=None, scratch=ONE, nb=1 << 40, out=ONE, ws=ONE)

    def call(**kw):
        a = dict(base, **kw)
        return lib.hkv_prefill_b8(a["q"], 0, a["kt"], a["vt"], a["st"], a["PS"], a["bt"], a["B"], a["MP"], a["rows"], a["n"], a["NT"],
                                  a["KVH"], a["G"], a["D"], 0.1, 1.0, 65536, a["fmt"], a["window"], a["sinks"], a["lse"], a["scratch"],
                                  a["nb"], a["out"], 0, a["ws"], None)
    assert call(n=0) == 0 and call(n=-1) == -6
    for window in (0, 16):
        for name in ("q", "kt", "vt", "st", "bt", "scratch", "out", "rows"):
            assert call(**{name: None}, window=window) == -1, name
        for kw in (dict(D=64), dict(fmt=2), dict(G=129), dict(KVH=0), dict(PS=0), dict(PS=8), dict(PS=40)):
            assert call(**kw, window=window) == -3, kw
        for kw in (dict(q=at(0x100008)), dict(out=at(0x100008)), dict(kt=at(0x100008)), dict(vt=at(0x100008)), dict(st=two(33032, 2064)),
                   dict(scratch=at(0x100080)), dict(ws=at(0x100010)), dict(lse=at(0x100002))):
            assert call(**kw, window=window) == -2, kw
        for r in ((-1, 0, 40, 100), (2, 0, 40, 100), (1, 7, 7, 100), (1, 0, 41, 100), (1, 0, 40, 0), (1, 0, 40, 129)):
            assert call(rows=(C.c_int32 * 4)(*r), window=window) == -6, r
        need = lib.hkv_prefill_window_scratch_bytes(base["rows"], 1, 40, 8, 4, 128, 65536, 0, window, 0)
        assert need > 0 and call(nb=need - 1, window=window) == -5
    assert call(window=-1) == call(sinks=-1) == -6


# ------------------------------------------------------------------------------------------------------------ wrappers
D, KVH, HQ, PS, B, NT = 128, 2, 8, 16, 2, 2
ST6, ST2 = (1, 1, 1, 1, 1, 1), (16, 16)


def base():
    i32, b16 = torch.int32, torch.bfloat16
    return dict(query=torch.zeros(NT, HQ, D, dtype=b16), out=torch.zeros(NT, HQ, D, dtype=b16), key=torch.zeros(NT, KVH, D, dtype=b16),
                value=torch.zeros(NT, KVH, D, dtype=b16), slots=torch.zeros(NT, dtype=torch.int64), pos=torch.zeros(NT, dtype=torch.int64),
                table=torch.zeros(16, D), kd=torch.zeros(64, dtype=torch.uint8), ksf=torch.zeros(64, dtype=torch.uint8),
                vd=torch.zeros(64, dtype=torch.uint8), vsf=torch.zeros(64, dtype=torch.uint8), bt=torch.zeros(B, 4, dtype=i32),
                lens=torch.zeros(B, dtype=i32), qsl=torch.zeros(B + 1, dtype=i32), gk=torch.ones(KVH), gv=torch.ones(KVH),
                signs=torch.ones(D), ws=torch.zeros(256, dtype=torch.uint8), lse=torch.zeros(NT, HQ), fmt="e4m3", rows=[(0, 0, 2, 5)],
                window=4, sinks=1)


def _rot(a):
    return K.write_rotary(a["query"], a["key"], a["value"], (a["kd"], a["ksf"], a["vd"], a["vsf"]), ST6, PS, a["slots"], a["pos"],
                          a["table"], a["gk"], a["gv"], a["out"], signs=a["signs"])


def _w8(a):
    return K.write_b8(a["key"], a["value"], (a["kd"], a["vd"]), ST2, PS, a["slots"], a["gk"], a["gv"], fmt=a["fmt"])


def _rot8(a):
    return K.write_rotary_b8(a["query"], a["key"], a["value"], (a["kd"], a["vd"]), ST2, PS, a["slots"], a["pos"], a["table"], a["gk"],
                             a["gv"], a["out"], fmt=a["fmt"])


def _dec8(a):
    return K.decode_b8(a["query"], (a["kd"], a["vd"]), ST2, PS, a["bt"], a["lens"], a["qsl"], 1.0, 1.0, a["gk"], a["gv"], 1, a["out"],
                       a["ws"], fmt=a["fmt"], window=a["window"], sinks=a["sinks"], lse=a["lse"])


def _pre8(a):
    return K.prefill_b8(a["query"], (a["kd"], a["vd"]), ST2, PS, a["bt"], a["rows"], 1.0, 1.0, KVH, a["out"], fmt=a["fmt"],
                        window=a["window"], sinks=a["sinks"], workspace=a["ws"], lse=a["lse"])


WRITE = ("key", "value", "slots", "gk", "gv")
TURN = ("query", "pos", "table", "out")
CALLS = {"write_rotary": (WRITE + TURN + ("kd", "ksf", "vd", "vsf", "signs"), _rot), "write_b8": (WRITE + ("kd", "vd"), _w8),
         "write_rotary_b8": (WRITE + TURN + ("kd", "vd"), _rot8),
         "decode_b8": (("query", "kd", "vd", "bt", "lens", "qsl", "gk", "gv", "out", "ws", "lse"), _dec8),
         "prefill_b8": (("query", "kd", "vd", "bt", "out", "ws", "lse"), _pre8)}


@pytest.mark.parametrize("name", CALLS)
def test_cpu_tensors_and_other_devices_are_refused(lib, monkeypatch, name):
    names, call = CALLS[name]
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(base())
    monkeypatch.setattr(K, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(K._lib, "_host", K._lib._NoHost())
    monkeypatch.setattr(K._lib, "load", lambda: pytest.fail("a launch was prepared"))
    for n in names:
        a = base()
        a[n] = a[n].to("meta")
        with pytest.raises(ValueError, match="more than one device|on the query's device"):
            call(a)
            pytest.fail(f"{n} on another device was taken")


def _bad(**kw):
    return dict(base(), **kw)


WRONG = {
    "write_rotary": [dict(query=torch.zeros(NT, HQ, D)), dict(query=torch.zeros(NT, HQ, 64, dtype=torch.bfloat16)),
                     dict(out=torch.zeros(NT, HQ + 1, D, dtype=torch.bfloat16)), dict(pos=torch.zeros(NT, dtype=torch.int32)),
                     dict(pos=torch.zeros(NT + 1, dtype=torch.int64)), dict(table=torch.zeros(16, D, dtype=torch.float16)),
                     dict(table=torch.zeros(16, 24)), dict(table=torch.zeros(16, 2 * D)), dict(table=torch.zeros(16, 2 * D)[:, :D]),
                     dict(query=torch.zeros(NT, HQ, 2 * D, dtype=torch.bfloat16)[..., ::2]), dict(slots=torch.zeros(NT, dtype=torch.int32)),
                     dict(slots=torch.zeros(NT + 1, dtype=torch.int64)), dict(gk=torch.ones(KVH + 1))],
    "write_b8": [dict(fmt="e5m2"), dict(key=torch.zeros(NT, KVH, D)), dict(slots=torch.zeros(NT + 1, dtype=torch.int64)),
                 dict(value=torch.zeros(NT, KVH, D + 16, dtype=torch.bfloat16))],
    "write_rotary_b8": [dict(fmt=0), dict(pos=torch.zeros(NT - 1, dtype=torch.int64)), dict(table=torch.zeros(16, 8))],
    "decode_b8": [dict(fmt="fp8"), dict(window=-1), dict(sinks=-2), dict(lse=torch.zeros(NT, HQ + 1)), dict(lse=torch.zeros(NT, HQ).double()),
                  dict(bt=torch.zeros(B, 4, dtype=torch.int64)), dict(query=torch.zeros(NT, HQ, D)), dict(gk=torch.ones(3), gv=torch.ones(3))],
    "prefill_b8": [dict(fmt=None), dict(window=-1), dict(rows=[(0, 0, 3, 5)]), dict(rows=[(0, 0, 2, 65)]), dict(rows=[(2, 0, 2, 5)]),
                   dict(lse=torch.zeros(NT - 1, HQ)), dict(out=torch.zeros(NT, HQ, D, dtype=torch.float16))],
}


@pytest.mark.parametrize("name", CALLS)
def test_wrong_arguments_are_refused(lib, monkeypatch, name):
    monkeypatch.setattr(K, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(K._lib, "_host", K._lib._NoHost())
    monkeypatch.setattr(K._lib, "load", lambda: pytest.fail("a launch was prepared"))
    for kw in WRONG[name]:
        with pytest.raises((TypeError, ValueError)):
            CALLS[name][1](_bad(**kw))
            pytest.fail(f"{kw} was taken")


@pytest.mark.parametrize("name", ["write_rotary", "write_rotary_b8"])
def test_turned_queries_lie_apart_from_what_is_read(lib, monkeypatch, name):
    monkeypatch.setattr(K, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(K._lib, "_host", K._lib._NoHost())
    qkv = torch.zeros(4, (HQ + 2 * KVH) * D, dtype=torch.bfloat16)
    parts = [x[:NT].view(NT, -1, D) for x in qkv.split((HQ * D, KVH * D, KVH * D), 1)]
    a = dict(base(), query=parts[0], key=parts[1], value=parts[2])

    class Reached(Exception):
        pass

    def load():
        raise Reached
    monkeypatch.setattr(K._lib, "load", load)
    whole = torch.zeros(NT, 2 * HQ * D, dtype=torch.bfloat16)
    for q, out in ((parts[0], parts[0]), (parts[0], torch.zeros_like(parts[0])),
                   (whole[:, :HQ * D].view(NT, HQ, D), whole[:, HQ * D:].view(NT, HQ, D))):
        with pytest.raises(Exception) as e:
            with torch.no_grad():
                monkeypatch.setattr(torch.cuda, "device", lambda d: __import__("contextlib").nullcontext())
                CALLS[name][1](dict(a, query=q, out=out))
        assert e.type is Reached
    shifted = qkv.view(-1)[D:D + NT * qkv.shape[1]].view(NT, -1)[:, :HQ * D].view(NT, HQ, D)
    keys_too = qkv.view(-1)[2 * KVH * D:2 * KVH * D + NT * qkv.shape[1]].view(NT, -1)[:, :HQ * D].view(NT, HQ, D)
    for q, out in ((parts[0], shifted), (torch.zeros(NT, HQ, D, dtype=torch.bfloat16), keys_too)):
        with pytest.raises(ValueError, match="apart"):
            CALLS[name][1](dict(a, query=q, out=out))


# -------------------------------------------------------------------------------------------------- layout, plain forms
def test_views():
    c = torch.arange(3 * 4 * 32 * 129 % 251, dtype=torch.int64)
    cache = torch.zeros((3, 4, 32, 129), dtype=torch.uint8)
    (kt, vt), st = Lt.b8_views(cache, 2, 128)
    assert st == (4 * 32 * 129, 32 * 129) and Lt.b8_slot_bytes(128) == 129 and all(s % 16 == 0 for s in st)
    kt[st[0] + st[1]] = 7
    vt[2 * st[0]] = 9
    assert cache[1, 1, 0, 0] == 7 and cache[2, 2, 0, 0] == 9 and len(c)
    for bad in (cache.transpose(1, 2), cache.permute(0, 1, 3, 2), cache[..., :128], cache.int(), cache[:, :3],
                torch.zeros((3, 32, 4, 129), dtype=torch.uint8).permute(0, 2, 1, 3)):
        with pytest.raises(ValueError):
            Lt.b8_views(bad, 2, 128)


def test_plain_forms_by_hand():
    assert R.exponent(448.0, "e4m3") == 0 and R.exponent(448.5, "e4m3") == 1 and R.exponent(224.0, "e4m3") == -1
    assert R.exponent(127.0, "int8") == 0 and R.exponent(127.5, "int8") == 1 and R.exponent(1.0, "int8") == -6
    assert R.exponent(0.0, "e4m3") == -15 and R.exponent(1e9, "int8") == 9 and R.exponent(float("inf"), "e4m3") == 7
    assert R.encode(torch.tensor([0.5, 1.5, -2.5, 300.0, float("nan")]).double(), "int8").view(torch.int8).tolist() == [0, 2, -2, 127, 0]
    assert R.values(R.encode(torch.tensor([17.0, 19.0, 500.0, -2.0 ** -10, 3 * 2.0 ** -10]).double(), "e4m3"), "e4m3").tolist() == \
        [16.0, 20.0, 448.0, 0.0, 2 * 2.0 ** -9]
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (2, 2, 32, 128), generator=g, dtype=torch.uint8)
    exps = torch.randint(-5, 3, (2, 2, 2), generator=g)
    c, s, rest = R.unpack(R.pack(codes, exps))
    assert torch.equal(c, codes) and torch.equal(s, 2.0 ** exps.float()) and bool((rest == 0xff).all())
    assert int(R.pack(codes, exps).view(2, 2, 2, -1)[0, 0, 0, 5 * 128 + 0]) == int(codes[0, 0, 5, 5 * 16])      # chunk 0 of token 5 is channel chunk 5
    # one token after another, then a larger one: the tile's scale grows by two powers of two, its codes are rounded
    one = torch.ones(1)
    cache = R.pack(torch.zeros((1, 2, 16, 128), dtype=torch.uint8), torch.zeros((1, 2, 1)))
    k = torch.full((1, 1, 128), 100.0, dtype=torch.bfloat16)
    cache = R.append(cache, k, k, [0], one, one, "int8")
    cache = R.append(cache, k * 4.5, k, [3], one, one, "int8")
    c, s, _ = R.unpack(cache)
    assert s.flatten().tolist() == [4.0, 1.0]
    v = R.values(c, "int8")
    assert v[0, 0, 0, 0] == 25 and v[0, 0, 3, 0] == round(450 / 4) and v[0, 1, 0, 0] == 100 and v[0, 0, 1, 0] == 0
    t = torch.tensor([[1.0, 0.0], [0.6, 0.8]]).repeat_interleave(8, 1)
    x = torch.arange(1, 17, dtype=torch.bfloat16).view(1, 1, 16)
    assert R.turn(x, torch.tensor([0]), t, False).flatten().tolist() == x.flatten().tolist()
    y, mag = R.turn(x, torch.tensor([1]), t, False, exact=True)
    assert abs(float(y[0, 0, 0]) - (0.6 - 9 * 0.8)) < 1e-6 and abs(float(y[0, 0, 8]) - (9 * 0.6 + 0.8)) < 1e-6 and abs(float(mag[0, 0, 0]) - 7.8) < 1e-6
    z = R.turn(x, torch.tensor([1]), t, True).double()
    assert abs(float(z[0, 0, 0]) - (0.6 - 2 * 0.8)) < 2 ** -8 and abs(float(z[0, 0, 1]) - (2 * 0.6 + 0.8)) < 2 ** -7
