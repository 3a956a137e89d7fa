"""A contract of the tiled products (gemm.h, linear_mx.hip), checked on the compiled device assembly (CPU only:
hipcc cross-compiles gfx950 without a GPU).

Their waits count memory accesses: a tile's stores may still be on their way while the loads that are older must have
arrived.  So the stores of a tile are as many as the source counts, in every wave, and none of them, nor any load into
LDS of a tile, lies behind a branch on lanes.
"""

from __future__ import annotations

import re
import subprocess

import pytest

from tinytrain_amd import build as B

STORE, PARTIAL, GATED, GATED_SAVE = range(4)


@pytest.fixture(scope="module", params=["swiglu", "linear_mx"])
def asm(request, tmp_path_factory):
    try:
        hipcc = B._hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / f"{request.param}.s"
    subprocess.run([hipcc, *B.HIPCC_FLAGS, f"-I{B.INCLUDE}", f"-I{B.CSRC}", "--cuda-device-only", "-S",
                    str(B.CSRC / f"{request.param}.hip"), "-o", str(out)], check=True, capture_output=True, timeout=600)
    return out.read_text()


def _kernels(asm, name):
    """(template arguments, instructions and labels) of each instantiation."""
    for m in re.finditer(rf"^(_ZN4ttfa\S*{name}I\S+):", asm, re.M):
        args = re.match(r"((?:L(?:[ib]|N\S+?E)\d+E)+)", m.group(1).split(f"{name}I")[1]).group(1)
        body = asm[m.end():asm.index("s_endpgm", m.end())]
        yield [int(a) for a in re.findall(r"L(?:[ib]|N\S+?E)(\d+)E", args)], [l.strip() for l in body.split("\n")]


def _accesses(lines, kind):
    """The number of such instructions, and those that a branch on lanes may jump over."""
    hits = [i for i, l in enumerate(lines) if l.startswith("buffer_") and kind(l)]
    behind = []
    for i, l in enumerate(lines):
        m = re.match(r"s_cbranch_execn?z (\S+)", l)
        if m:
            to = next((j for j, t in enumerate(lines) if t.startswith(m.group(1) + ":")), len(lines))
            behind += [lines[j] for j in hits if i < j < to]
    return len(hits), behind


def _gemm_stores(tm, tn, wm, wn, bk, s, xtr, wtr, e):
    mb, nb = tm // wm // 32, tn // wn // 32
    return mb * {STORE: 2 * nb, PARTIAL: 4 * nb, GATED: 2, GATED_SAVE: 8}[e]


def _mx_stores(tm, tn, wm, wn, s, bits, xmx, partial):
    n = (tm // wm // 16) * (tn // wn // 16)
    return n if partial else n // 2


def test_stores_are_as_many_as_the_waits_count(asm):
    kernels = 0
    for name, stores in (("gemm_kernel", _gemm_stores), ("linear_mx_tile_kernel", _mx_stores)):
        for args, lines in _kernels(asm, name):
            kernels += 1
            n, behind = _accesses(lines, lambda l: l.startswith("buffer_store"))
            assert n == stores(*args) and not behind, (name, args, n, behind[:2])
            n, behind = _accesses(lines, lambda l: l.startswith("buffer_load_dwordx4") and l.endswith("lds"))
            assert n and not behind, (name, args, behind[:2])
    assert kernels >= 10
