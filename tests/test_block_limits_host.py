"""The largest calls that the block's operators take, as their documents state them: the sizes on both sides of each
limit, asked of the entries that compute sizes alone."""

import pytest

from tinytrain_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(),
                                reason="libttfa.so not built (python -m tinytrain_amd.build)")
MOST = 1 << 20


def _swiglu(M, K, N):
    return _lib.load().ttfa_swiglu_workspace_bytes(M, K, N)


def _linear(M, K, N):
    return _lib.load().ttfa_linear_mx_workspace_bytes(M, K, N, 4, 0)


def _norm(M, C):
    return _lib.load().ttfa_rms_norm_workspace_bytes(M, C)


@pytest.mark.parametrize("entry, taken, refused", [
    (_swiglu, ((1 << 30) - 128, 128, 128), ((1 << 30) - 127, 128, 128)),
    (_swiglu, ((1 << 29) - 128, 8, 256), ((1 << 29) - 127, 8, 256)),       # a, from 256 columns on fewer rows
    (_swiglu, ((1 << 17) - 128, 8, MOST), ((1 << 17) - 127, 8, MOST)),     # a
    (_swiglu, ((1 << 17) - 128, MOST, 8), ((1 << 17) - 127, MOST, 8)),     # dx
    (_swiglu, (8, MOST, (1 << 16) - 64), (8, MOST, (1 << 16) - 56)),       # both weights' gradients
    (_linear, ((1 << 30) - 128, 32, 128), ((1 << 30) - 127, 32, 128)),
    (_linear, ((1 << 29) - 128, 32, 256), ((1 << 29) - 127, 32, 256)),
    (_linear, ((1 << 17) - 128, 32, MOST), ((1 << 17) - 127, 32, MOST)),
    (_norm, (1 << 37, 8), ((1 << 37) + 1, 8)), (_norm, (1 << 26, 16384), ((1 << 26) + 1, 16384))])
def test_sizes(entry, taken, refused):
    assert entry(*taken) >= 0 and entry(*refused) == -1


@pytest.mark.parametrize("K", [32, 4096, MOST])
def test_rows_to_quantise(K):
    """The entry launches, so only sizes that it refuses are asked, and one it takes with a pointer it does not."""
    f, most = _lib.load().ttfa_mx_quantize, ((1 << 34) - (1 << 13)) // K
    assert f(0x100000, 0x200000, 0x300000, most + 1, K, 4, 0, None) == _lib.E_SEQ
    assert f(None, 0x200000, 0x300000, most, K, 4, 0, None) == _lib.E_NULL
