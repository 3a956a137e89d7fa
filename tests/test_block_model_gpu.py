"""The model with its blocks' norms, residual additions and gated feed-forward as HIP operators: logits and
gradients at the reference's 112M shape against the same model in fp32.

The bound is the eager path's own bf16 noise, as in test_model_112m_gpu.py (which has the reasons): the
operators round no more often than the eager lines do (the norm's product with the weight, the gate, its
activation and the up projection stay in fp32 there), so their deviation from fp32 must not be larger, within
the spread of a mean over 33 million logits and of a gradient's norm; the largest deviation is set by a handful
of values.
"""

import pytest
import torch

from helpers import announce
from tinytrain_amd.kernels.rms_norm import BlockInputError
from tinytrain_amd.model import ModelConfig, ModelForCausalLM

pytestmark = pytest.mark.gpu
MAX_RATIO, MEAN_RATIO, GRAD_RATIO = 1.15, 1.05, 1.1


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(0)
    c = ModelConfig()
    m = ModelForCausalLM(c).to("cuda")
    g = torch.Generator(device="cpu").manual_seed(1)
    x = torch.randint(0, c.vocab_size, (2, c.max_seq_len), generator=g).to("cuda")
    yield m, x
    torch._dynamo.reset()


def _pass(m, x, attn, block, bf16=True, compiled=False):
    """(logits, gradients by parameter) of a training pass."""
    m.set_attn_impl(attn, fused_prologue=attn == "hip")
    m.set_block_impl(block)
    f = m
    if compiled:
        torch._dynamo.reset()
        f = torch.compile(m)
    m.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=bf16):
        logits, loss = f(x, x.roll(-1, dims=1))
    loss.backward()
    return logits.detach().float(), {n: p.grad.float() for n, p in m.named_parameters()}


def _off(got, ref):
    return (got - ref).norm().item() / ref.norm().item()


@pytest.mark.parametrize("attn", ["sdpa", "hip"])
def test_112m_logits_and_gradients(model, attn):
    announce(f"112M training pass, {attn} attention, hip blocks vs eager blocks vs fp32")
    m, x = model
    ref, gref = _pass(m, x, "sdpa", "eager", bf16=False)
    eager, geager = _pass(m, x, attn, "eager")
    got, ggot = _pass(m, x, attn, "hip")
    e, h = (eager - ref).abs(), (got - ref).abs()
    assert h.max() <= MAX_RATIO * e.max() and h.mean() <= MEAN_RATIO * e.mean(), (h.max(), e.max(), h.mean(), e.mean())
    assert ggot.keys() == gref.keys()
    # every kind of parameter, over the layers
    kinds = {}
    for n in gref:
        kinds.setdefault(".".join(p for p in n.split(".") if not p.isdigit()), []).append(n)
    for kind, names in kinds.items():
        cat = lambda g: torch.cat([g[n].flatten() for n in names])  # noqa: E731
        r, off_e, off_h = cat(gref), _off(cat(geager), cat(gref)), _off(cat(ggot), cat(gref))
        assert torch.isfinite(r).all() and off_h <= GRAD_RATIO * off_e, (kind, off_h, off_e)


def test_112m_compiled(model):
    """Traced, the same operators run: the compiled model stays as near to fp32 as the eager one."""
    announce("112M training pass, hip attention and blocks, torch.compile")
    m, x = model
    ref, _ = _pass(m, x, "sdpa", "eager", bf16=False)
    eager, _ = _pass(m, x, "hip", "eager")
    got, grads = _pass(m, x, "hip", "hip", compiled=True)
    assert (got - ref).abs().mean() <= MEAN_RATIO * (eager - ref).abs().mean()
    assert all(torch.isfinite(g).all() for g in grads.values())


def test_fp32_compute_is_refused(model):
    m, x = model
    m.set_attn_impl("hip")
    m.set_block_impl("hip")
    with pytest.raises(BlockInputError), torch.no_grad():
        m(x)
    with pytest.raises(ValueError):
        m.set_block_impl("triton")
