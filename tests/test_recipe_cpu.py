"""The recipe for bounded caches in the integration guide, run as it is written over several layers: the lengths are shared by the
layers, so every layer's eviction must see those of the step, and they change once."""
import os
import re
from types import SimpleNamespace

GUIDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


def recipe():
    """the first python block of the guide's section on bounded caches"""
    section = open(GUIDE).read().split("## 2a. Bounded caches")[1]
    return re.search(r"```python\n(.*?)```", section, re.S).group(1)


class Lengths(list):
    def copy_(self, other):
        self[:] = other


def test_every_layer_is_cut_from_the_lengths_of_the_step():
    layers = [SimpleNamespace(q=f"q{i}", flat=f"flat{i}", gk=f"gk{i}", gv=f"gv{i}", out=f"out{i}", weights=f"weights{i}") for i in range(3)]
    lens, new_lens, calls = Lengths([300, 90]), Lengths([0, 0]), []

    class K:
        @staticmethod
        def decode_window(q, flat, st, PS, bt, lens, qsl, sm, vs, gk, gv, qlmax, out, ws, window, sinks=0, lse=None):
            calls.append(("decode", flat, list(lens)))

        @staticmethod
        def accumulate_weights(q, flat, st, PS, bt, lens, qsl, sm, gk, qlmax, lse, weights, window=0, sinks=0):
            calls.append(("weights", flat, weights, list(lens)))

        @staticmethod
        def evict(flat, st, PS, D, bt, lens, weights, keep, sinks, recent, kept, out_lens, out_tables=None, out_weights=None):
            calls.append(("evict", flat, weights, list(lens)))
            out_lens[:] = [min(n, keep) for n in lens]
    env = dict(K=K, layers=layers, lens=lens, new_lens=new_lens, keep=128, cut=True)
    for name in ("st", "PS", "D", "bt", "qsl", "sm", "vs", "qlmax", "ws", "lse", "sinks", "recent", "kept"):
        env[name] = name
    # (names that a recipe for one layer alone would use)
    env.update(q="q0", flat="flat0", gk="gk0", gv="gv0", out="out0", weights="weights0")
    exec(recipe(), env)
    assert [c for c in calls if c[0] == "evict"] == [("evict", f"flat{i}", f"weights{i}", [300, 90]) for i in range(3)]
    assert [c[2] for c in calls if c[0] == "decode"] == [[300, 90]] * 3
    assert lens == [128, 90]
