"""The rules that choose between the tiles of the products (csrc/product_cut.h, host code alone), asked on the CPU:
the sizes of the GPU tests take the tiles that those tests name, and every kind of tile has a size."""

import ctypes
import shutil
import subprocess

import pytest

import test_linear_mx_tiles_gpu as linear
import test_swiglu_tiles_gpu as swiglu
from tinytrain_amd import build as B

SOURCE = """
#include "product_cut.h"
extern "C" void mx_cut(int M, int K, int N, int x_quantised, int *out) {
  const ttfa::Cut c = ttfa::mx_cut(M, K, N, x_quantised != 0);
  out[0] = c.wide, out[1] = c.splits, out[2] = c.deep, out[3] = ttfa::linear_mx_few_rows(M, N);
}
extern "C" void cut_of(int M, int N, int K, int segs, int z, int dual, int *out) {
  const ttfa::Cut c = ttfa::cut_of(M, N, K, segs, z, dual != 0);
  out[0] = c.wide, out[1] = c.splits, out[2] = c.deep;
}
extern "C" int swiglu_few_rows(int M, int N) { return ttfa::swiglu_few_rows(M, N); }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{B.CSRC}", str(d / "rules.cpp"),
                    "-o", str(d / "rules.so")], check=True, timeout=120)
    return ctypes.CDLL(str(d / "rules.so"))


def _named(kind, tm, tn, M, N, splits, z=1):
    return kind + (f"/{splits}" if splits > 1 else ""), z * splits * -(-M // tm) * -(-N // tn)


def _linear(rules, M, K, N, x8):
    c = (ctypes.c_int * 4)()
    rules.mx_cut(M, K, N, int(x8), c)
    wide, splits, deep, few = c
    assert not few
    if not x8:
        assert not deep
        return _named("wide" if wide else "narrow", 128, 256 if wide else 128, M, N, splits)
    t = 256 if wide else 128
    return _named("wide" if wide else "deep" if deep else "two", t, t, M, N, splits)


def _kinds(found):
    """Kinds of tiles, whole or in parts."""
    return {name.split("/")[0] + ("/" if "/" in name else "") for name, _ in found}


def test_linear_mx_sizes_take_the_tiles_that_they_name(rules):
    for (M, K, N), want in linear.CASES.items():
        assert tuple(_linear(rules, M, K, N, x8) for x8 in (True, False)) == want, (M, K, N)
    x8, bf = zip(*linear.CASES.values())
    assert _kinds(x8) == {k + p for k in ("wide", "two", "deep") for p in ("", "/")}
    assert _kinds(bf) == {k + p for k in ("wide", "narrow") for p in ("", "/")}
    for found, slots in ((x8, {"wide": 256, "two": 512}), (bf, {"wide": 256, "narrow": 256})):
        for kind, n in slots.items():
            assert any(name.startswith(kind) and items > n for name, items in found), kind


def _product(rules, M, N, K, segs, z, dual):
    c = (ctypes.c_int * 3)()
    rules.cut_of(M, N, K, segs, z, int(dual), c)
    wide, splits, deep = c
    t = 256 if wide else 128
    return _named("wide" if wide else "deep" if deep else "two", t, t // 2 if dual else t, M, N, splits, z)


def _swiglu(rules, M, K, N):
    """Tiles of the forward, of dx and of the weights' gradients."""
    assert not rules.swiglu_few_rows(M, N)
    return (_product(rules, M, N, K, 1, 1, True), _product(rules, M, K, N, 2, 1, False),
            _product(rules, N, K, M, 1, 2, False))


def test_swiglu_sizes_take_the_tiles_that_they_name(rules):
    for size, want in swiglu.CASES.items():
        assert _swiglu(rules, *size) == want, size
    forward, dx, dw = zip(*swiglu.CASES.values())
    assert _kinds(forward) == {"wide", "two", "deep"}
    for found in (dx, dw):
        assert _kinds(found) == {k + p for k in ("wide", "two", "deep") for p in ("", "/")}
    for found in (forward, dx, dw):
        for kind, n in (("wide", 256), ("two", 512)):
            assert any(name.startswith(kind) and items > n for name, items in found), kind


def test_swiglu_sizes_on_two_streams_are_in_parts(rules):
    for size in swiglu.STREAMS:
        assert all("/" in name for name, _ in _swiglu(rules, *size)[1:]), size
