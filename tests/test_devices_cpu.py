"""A call whose tensors lie on more than one device is refused by every wrapper, before anything is launched: a kernel that is
given another device's pointer reads or writes outside of its own memory. Shown without a GPU: CPU tensors stand in for those of
the call's device and a meta tensor for one of another device, behind the check for CUDA tensors."""
import pytest
import torch

from horizon_kernels_b200 import kernels as K

D, KVH, HQ, PS, B, NT = 128, 2, 8, 16, 2, 2


def base():
    i32, f32 = torch.int32, torch.float32
    return dict(query=torch.zeros(NT, HQ, D, dtype=torch.bfloat16), out=torch.zeros(NT, HQ, D, dtype=torch.bfloat16),
                key=torch.zeros(NT, KVH, D, dtype=torch.bfloat16), value=torch.zeros(NT, KVH, D, dtype=torch.bfloat16),
                slots=torch.zeros(NT, dtype=torch.int64), kd=torch.zeros(64, dtype=torch.uint8), ksf=torch.zeros(64, dtype=torch.uint8),
                vd=torch.zeros(64, dtype=torch.uint8), vsf=torch.zeros(64, dtype=torch.uint8), bt=torch.zeros(B, 4, dtype=i32),
                lens=torch.zeros(B, dtype=i32), qsl=torch.zeros(B + 1, dtype=i32), gk=torch.ones(KVH), gv=torch.ones(KVH), signs=torch.ones(D),
                ws=torch.zeros(256, dtype=torch.uint8), lse=torch.zeros(NT, HQ), weights=torch.zeros(B, KVH, 64), kept=torch.zeros(B, KVH, 16, dtype=i32),
                out_lens=torch.zeros(B, dtype=i32), out_bt=torch.zeros(B, 1, dtype=i32), out_w=torch.zeros(B, KVH, 16, dtype=f32),
                dk=torch.zeros(NT, KVH, D, dtype=torch.float16), dv=torch.zeros(NT, KVH, D, dtype=torch.float16), rows=torch.zeros(B, dtype=i32),
                cu=torch.zeros(B + 1, dtype=i32))


def flat(a):
    return a["kd"], a["ksf"], a["vd"], a["vsf"]


ST = (1, 1, 1, 1, 1, 1)
CACHE = ("kd", "ksf", "vd", "vsf")
DECODE = ("query", *CACHE, "bt", "lens", "qsl", "gk", "gv", "out", "ws", "signs")
CALLS = {
    "write": (("key", "value", *CACHE, "slots", "gk", "gv", "signs"),
              lambda a: K.write(a["key"], a["value"], flat(a), ST, PS, a["slots"], a["gk"], a["gv"], signs=a["signs"])),
    "decode_ragged": (DECODE, lambda a: K.decode_ragged(a["query"], flat(a), ST, PS, a["bt"], a["lens"], a["qsl"], 1.0, 1.0, a["gk"], a["gv"], 1,
                                                        a["out"], a["ws"], signs=a["signs"])),
    "decode_window": (DECODE + ("lse",), lambda a: K.decode_window(
        a["query"], flat(a), ST, PS, a["bt"], a["lens"], a["qsl"], 1.0, 1.0, a["gk"], a["gv"], 1, a["out"], a["ws"], 4, 1, signs=a["signs"],
        lse=a["lse"])),
    "prefill": (("query", *CACHE, "bt", "out", "signs", "ws"), lambda a: K.prefill(
        a["query"], flat(a), ST, PS, a["bt"], [(0, 0, 2, 5)], 1.0, 1.0, KVH, a["out"], signs=a["signs"], workspace=a["ws"])),
    "prefill_window": (("query", *CACHE, "bt", "out", "signs", "ws", "lse"), lambda a: K.prefill_window(
        a["query"], flat(a), ST, PS, a["bt"], [(0, 0, 2, 5)], 1.0, 1.0, KVH, a["out"], 4, 1, signs=a["signs"], workspace=a["ws"], lse=a["lse"])),
    "accumulate_weights": (("query", *CACHE, "bt", "lens", "qsl", "gk", "lse", "weights", "signs", "ws"), lambda a: K.accumulate_weights(
        a["query"], flat(a), ST, PS, a["bt"], a["lens"], a["qsl"], 1.0, a["gk"], 1, a["lse"], a["weights"], signs=a["signs"],
        workspace=a["ws"])),
    "evict": ((*CACHE, "bt", "lens", "weights", "kept", "out_lens", "out_bt", "out_w"), lambda a: K.evict(
        flat(a), ST, PS, D, a["bt"], a["lens"], a["weights"], 16, 1, 2, a["kept"], a["out_lens"], out_tables=a["out_bt"], out_weights=a["out_w"])),
    "dequant_tokens": ((*CACHE, "bt", "dk", "dv"), lambda a: K.dequant_tokens(flat(a), ST, PS, a["bt"][0], 0, 2, a["dk"], a["dv"])),
    "dequant_multi": ((*CACHE, "bt", "rows", "cu", "dk", "dv"), lambda a: K.dequant_multi(
        flat(a), ST, PS, a["bt"], a["rows"], a["cu"], B, 2, a["dk"], a["dv"])),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_tensor_on_another_device_is_refused(monkeypatch, name):
    monkeypatch.setattr(K, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(K._lib, "_host", K._lib._NoHost())                # (the native side takes CUDA tensors only)
    monkeypatch.setattr(K._lib, "load", lambda: pytest.fail("a launch was prepared"))
    names, call = CALLS[name]
    for n in names:
        a = base()
        a[n] = a[n].to("meta")
        with pytest.raises(ValueError, match="more than one device|on the query's device"):
            call(a)
            pytest.fail(f"{n} on another device was taken")
