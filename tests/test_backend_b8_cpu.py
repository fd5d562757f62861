"""The plugin surface with the 8-bit cache, without a GPU: the spec, the page orders, what does not go together."""
import os
from dataclasses import dataclass
from types import SimpleNamespace

import pytest

os.environ["HORIZON_KVFP4_STANDALONE"] = "1"
from horizon_kernels_b200 import backend as BE  # noqa: E402


@dataclass
class Spec:
    head_size: int
    head_size_v: int
    num_kv_heads: int
    kv_quant_mode: object
    state_content_bytes: object = None
    num_head_slots: object = None


def impl(D=128):
    return BE.HorizonFp4Impl(16, D, 0.1, num_kv_heads=4, kv_cache_dtype="nvfp4")


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_spec_and_layouts(monkeypatch, fmt):
    monkeypatch.delenv("HORIZON_KVFP4_K8", raising=False)
    assert impl().b8 is None and BE.HorizonFp4Backend.supported_kv_cache_layouts() == ("LBHNC", "LBNHC")
    monkeypatch.setenv("HORIZON_KVFP4_B8", fmt)
    for D in (128, 256):
        s = BE.HorizonFp4Backend.customize_spec(Spec(D, D, 4, SimpleNamespace(is_nvfp4=True)))
        assert s.num_head_slots == 8 and s.state_content_bytes == D + 1
        assert impl(D).b8 == fmt
    assert BE.HorizonFp4Backend.supported_kv_cache_layouts() == ("LBHNC",)
    monkeypatch.setenv("HORIZON_KVFP4_B8", "0")
    assert impl().b8 is None


def test_what_does_not_go_together(monkeypatch):
    monkeypatch.setenv("HORIZON_KVFP4_B8", "fp8")
    with pytest.raises(ValueError, match="HORIZON_KVFP4_B8"):
        impl()
    monkeypatch.setenv("HORIZON_KVFP4_B8", "int8")
    for other in ("HORIZON_KVFP4_K8", "HORIZON_KVFP4_HAD"):
        monkeypatch.setenv(other, "1")
        with pytest.raises(ValueError, match="neither"):
            impl(256)
        monkeypatch.setenv(other, "0")
