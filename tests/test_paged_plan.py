"""The arithmetic by which the paged prompt kernel finds the keys of its tiles (csrc/zs_paged_plan.cuh), compiled for
the host with checks of signed overflow, against whole numbers of any size; and on the GPU the calls that reach its
ends."""
import random
import shutil
import subprocess

import pytest
import torch

from conftest import PKG

I_MAX, CAP_MAX = 2 ** 31 - 1, 2 ** 31 - 256

HARNESS = r"""
#include "zs_paged_plan.cuh"
#include <cstdio>
using namespace zs::paged;
int main() {
  long long len, cap, n, window, skip, rows;
  while (std::scanf("%lld %lld %lld %lld %lld %lld", &len, &cap, &n, &window, &skip, &rows) == 6) {
    const int l = length_within((int)len, (int)cap), w = window_within((int)window, cap);
    const int p0 = l - (int)n + (int)skip;
    const KeyTiles k = key_tiles<128>(p0, (int)rows, w);
    std::printf("%d %d %d %d %d\n", l, w, first_seen(l - (int)n, w), k.lo, k.cnt);
  }
}
"""


def _want(len_, cap, n, window, skip, rows):
    l = min(max(len_, 0), cap)
    w = window if window < cap else 0
    first = lambda p: max(0, p - w + 1) if w else 0
    p0 = l - n + skip
    p1 = p0 + rows - 1
    lo = first(p0) // 128
    return [l, w, first(l - n), lo, p1 // 128 - lo + 1 if rows > 0 and p1 >= 0 else 0]


def _cases():
    r = random.Random(0)
    sizes = [0, 1, 2, 3, 127, 128, 129, 1000, 4096, 2 ** 20 + 1, 2 ** 30, 2 ** 31 - 1000]
    for cap in (16, 128, 4096, 2 ** 30, CAP_MAX):
        for len_ in (-2 ** 31, -5, 0, 1, 5, 100, 4000, 2 ** 30 + 7, CAP_MAX, I_MAX):
            for n in sizes[1:]:
                for window in (0, 1, 2, 100, 129, cap - 1, cap, cap + 1, 2 ** 30, I_MAX - 1, I_MAX):
                    skip = r.choice([0, n // 2, n - 1])
                    yield len_, cap, n, window, skip, min(r.choice([0, 1, 10, 128]), n - skip)


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_plan_arithmetic_has_no_overflow(tmp_path):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow,float-cast-overflow",
                    "-fno-sanitize-recover=all", "-I", str(PKG / "csrc"), str(src), "-o", str(exe)],
                   check=True)
    cases = list(_cases())
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases), text=True,
                         capture_output=True)
    assert out.returncode == 0, out.stderr
    got = [[int(x) for x in line.split()] for line in out.stdout.splitlines()]
    assert len(got) == len(cases)
    for c, g in zip(cases, got):
        assert g == _want(*c), c
        assert g[4] >= 0 and g[3] <= 2 ** 24


@pytest.mark.gpu
@pytest.mark.parametrize("window", [I_MAX, I_MAX - 5, 2 ** 30, 1000])
@pytest.mark.parametrize("lens,new", [([5], [9]), ([0, 3], [30, 200]), ([130], [400]), ([300, 0, 40], [7, 5, 40])])
def test_longest_windows(lens, new, window):
    """Windows of no end, with sequences shorter than their new tokens (the first of those are padding)."""
    from zs_b200 import paged
    from test_paged_gpu import _check, _world

    kw = dict(H=6, Hkv=2, hd=64, page=16, dtype=torch.bfloat16, sink=torch.float32, gate=True)
    w = _world(lens, new, **kw)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], window=window,
                                          k_sink=w["ks"], gate=w["gate"], return_lse=True)
    _check(w, o, lse)
    w = _world(lens, [1] * len(lens), **kw)
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], window=window,
                                          k_sink=w["ks"], gate=w["gate"], return_lse=True)
    _check(w, o, lse)


@pytest.mark.gpu
def test_lengths_far_below_zero_are_empty():
    from zs_b200 import _lib as Z
    from zs_b200 import paged
    from test_paged_gpu import _world

    w = _world([128, 40], [4, 9], H=2, Hkv=1, hd=64, page=16, dtype=torch.bfloat16, poison=False)
    for window in (None, 3, I_MAX):
        lens = torch.tensor([-2 ** 31, -7], dtype=torch.int32, device="cuda")
        o = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], lens, w["cu"], window=window)
        assert (o == 0).all()
        assert (paged.paged_decode_attention(w["q"][:2], w["k"], w["v"], w["table"], lens, window=window) == 0).all()
    assert Z.device_error() == 0
