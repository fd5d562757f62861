"""Which turned queries lie apart from what a rotating write reads: the rule of the C ABI (compiled from its source) and that of the wrapper,
against the addresses themselves. Neither may call rows apart that share a byte, and both take the layouts that models have."""
import os
import re
import subprocess

import pytest
import torch

from horizon_kernels_b200 import build
from horizon_kernels_b200 import kernels as K

D = 16
HARNESS = r"""
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <numeric>
@CODE@
int main() {
  long long o[2], s0[2], s1[2], n[2], h[2], D;
  while (scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld %lld %lld", &D, &o[0], &s0[0], &s1[0], &n[0], &h[0], &o[1], &s0[1], &s1[1], &n[1], &h[1]) == 11) {
    RowSet r[2];
    for (int i = 0; i < 2; ++i) r[i] = RowSet{(const void*)(uintptr_t)(0x100000 + 2 * o[i]), s0[i], s1[i], n[i], h[i]};
    printf("%d\n", (int)rows_disjoint(r[0], r[1], D));
  }
}
"""


@pytest.fixture(scope="module")
def c_rule(tmp_path_factory):
    src = open(os.path.join(build.CSRC, "hkv_rotary.cuh")).read()
    code = re.search(r"struct RowSet \{.*?\n\}\n", src, re.S)
    d = tmp_path_factory.mktemp("rows")
    (d / "t.cpp").write_text(HARNESS.replace("@CODE@", code.group(0)))
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-o", str(d / "t"), str(d / "t.cpp")], check=True)

    def rule(cases):
        text = "\n".join(" ".join(map(str, (D, *a, *b))) for a, b in cases)
        return [x == "1" for x in subprocess.run([str(d / "t")], input=text, capture_output=True, text=True, check=True).stdout.split()]
    return rule


def wrapper_rule(cases):
    buf = torch.zeros(1 << 14, dtype=torch.bfloat16)
    return [K._rows_apart(*(buf.as_strided((n, h, D), (s0, s1, 1), o) for o, s0, s1, n, h in c)) for c in cases]


def elements(o, s0, s1, n, h):
    return {o + i * s0 + j * s1 + d for i in range(n) for j in range(h) for d in range(D)}


def test_rows_that_share_a_byte_are_never_apart(c_rule):
    g = torch.Generator().manual_seed(1)
    pick = lambda *v: v[int(torch.randint(0, len(v), (1,), generator=g))]  # noqa: E731
    cases = []
    for _ in range(6000):
        # (offset, stride between tokens, between heads, tokens, heads): multiples of 8, many of D, often the same strides
        a = [8 * int(torch.randint(0, 60, (1,), generator=g)), 8 * pick(0, 1, 2, 3, 4, 6, 8, 12, 16, 24), 8 * pick(0, 1, 2, 4, 6, 8, 12, 48), pick(1, 2, 3, 5), pick(1, 2, 3)]
        b = [8 * int(torch.randint(0, 60, (1,), generator=g)), *pick(a[1:3], [a[1], 8 * pick(2, 4, 6)], [8 * pick(2, 4, 8, 12), a[2]]), pick(1, 2, 4), pick(1, 2, 3)]
        cases.append((a, b))
    want = [not (elements(*a) & elements(*b)) for a, b in cases]
    for rule in (c_rule, wrapper_rule):
        got = rule(cases)
        assert not any(x and not w for x, w in zip(got, want))
        assert sum(got) > 0.5 * sum(want) and not all(want)


def test_layouts_of_models(c_rule):
    H, n = 3, 5
    fused = ((0, 5 * D, D, n, H), (3 * D, 5 * D, D, n, 1))                                  # queries, then a key head, a value head
    turns = ((0, 9 * D, 3 * D, n, H), (D, 9 * D, 3 * D, n, H))                              # query, key, value of a head in turn
    pairs = ((0, 6 * D, 2 * D, n, H), (D, 6 * D, 2 * D, n, H))                              # queries and turned queries in turn
    outer = ((0, D, n * D, n, H), (H * n * D, D, n * D, n, H))                              # heads outermost
    for rule in (c_rule, wrapper_rule):
        assert rule([fused, turns, pairs, outer, fused[::-1], turns[::-1]]) == [True] * 6
        # half a row further, a row further where there is no room, the rows themselves
        assert rule([(turns[0], (8, *turns[0][1:])), (pairs[0], (D + 8, *pairs[0][1:])), (turns[0], (3 * D, *turns[0][1:])), (fused[0], fused[0])]) == [False] * 4
