"""The compiled 112M model with its blocks as HIP operators: the gradients of every kind of parameter, within the bound
that test_block_model_gpu.py gives the eager one (which has the reasons)."""

import pytest
import torch

from helpers import announce
from test_block_model_gpu import GRAD_RATIO, _off, _pass, model  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_112m_compiled_gradients(model):  # noqa: F811
    announce("112M training pass, hip attention and blocks, torch.compile, gradients")
    m, x = model
    _, ref = _pass(m, x, "sdpa", "eager", bf16=False)
    _, eager = _pass(m, x, "hip", "eager")
    _, got = _pass(m, x, "hip", "hip", compiled=True)
    assert got.keys() == ref.keys()
    kinds = {}
    for n in ref:
        kinds.setdefault(".".join(p for p in n.split(".") if not p.isdigit()), []).append(n)
    assert len(kinds) >= 10
    for kind, names in kinds.items():
        cat = lambda g: torch.cat([g[n].flatten() for n in names])  # noqa: E731
        r = cat(ref)
        off, off_eager = _off(cat(got), r), _off(cat(eager), r)
        assert off <= GRAD_RATIO * off_eager, (kind, off, off_eager)
