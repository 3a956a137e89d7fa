"""``set_block_impl("hip")`` on the CPU, with the operators replaced by their formulas: what a module does when it is
called (hooks, adapters, biases, wrappers) is not lost where its weights are read by an operator."""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from tinytrain_amd import model as M

CONFIG = dict(vocab_size=64, hidden_size=32, num_hidden_layers=3, num_attention_heads=2, num_key_value_heads=1,
              head_dim=16, intermediate_size=64, max_seq_len=8)
CALLS = []


def _rms_norm(x, w, eps, dtype=None):
    CALLS.append("rms_norm")
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + eps) * w).to(dtype or x.dtype)


def _add_rms_norm(x, r, w, eps, dtype=None):
    CALLS.append("add_rms_norm")
    h = (r.float() + x.float()).to(r.dtype)
    return _rms_norm(h, w, eps, dtype or x.dtype), h


def _swiglu(x, wg, wu):
    CALLS.append("swiglu")
    return F.silu(x @ wg.t()) * (x @ wu.t())


@pytest.fixture
def model(monkeypatch):
    for name, f in (("rms_norm", _rms_norm), ("add_rms_norm", _add_rms_norm), ("swiglu", _swiglu)):
        monkeypatch.setattr(M, name, f)
    torch.manual_seed(0)
    m = M.ModelForCausalLM(M.ModelConfig(**CONFIG))
    with torch.no_grad():
        for p in m.parameters():   # so that every branch counts
            p.add_(0.2 * torch.randn_like(p))
    return m, torch.randint(0, 64, (2, 8))


def _logits(m, ids, impl):
    m.set_block_impl(impl)
    CALLS.clear()
    return m(ids)[0].detach()


def _same(m, ids):
    want = _logits(m, ids, "eager")
    assert not CALLS
    got = _logits(m, ids, "hip")
    # fp32 on both sides, in another order: a few roundings a layer
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    return CALLS


def test_plain_modules_run_as_operators(model):
    # one norm without a residual (the first), six with one, each of which calls the formula of the other
    assert sorted(_same(*model)) == ["add_rms_norm"] * 6 + ["rms_norm"] * 7 + ["swiglu"] * 3


MODULES = ["layers.1", "layers.0.input_layernorm", "layers.1.input_layernorm", "layers.2.post_attention_layernorm",
           "layers.0.mlp.gate_proj", "layers.1.mlp.up_proj", "layers.1.mlp.down_proj", "layers.2.mlp", "layers.0.self_attn",
           "norm", "lm_head", "embed_tokens"]


@pytest.mark.parametrize("name", MODULES)
def test_hooks_are_called(model, name):
    """A forward hook that changes the output, a pre-hook that changes the input and a backward hook."""
    m, ids = model
    mod, plain = m.get_submodule(name), _logits(*model, "eager")
    seen = []
    mod.register_forward_hook(lambda mod, args, out: seen.append("forward") or 1.5 * out)
    if name != "embed_tokens":
        mod.register_forward_pre_hook(lambda mod, args: seen.append("pre") or (args[0] + 0.25, *args[1:]))
    assert (_logits(m, ids, "eager") - plain).abs().max() > 1e-2 * plain.abs().max()
    first = list(seen)
    seen.clear()
    _same(m, ids)
    assert first and seen == 2 * first
    if name == "embed_tokens":  # no input that a gradient flows to
        return
    mod.register_full_backward_hook(lambda mod, grad_in, grad_out: seen.append("backward"))
    for impl in ("eager", "hip"):
        seen.clear()
        m.set_block_impl(impl)
        m(ids)[0].square().mean().backward()
        assert seen == first + ["backward"], impl


def test_hooks_on_all_modules_are_called(model):
    m, ids = model
    counts = {}
    for impl in ("eager", "hip"):
        seen = []
        handle = nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(type(mod).__name__))
        try:
            _logits(m, ids, impl)
        finally:
            handle.remove()
        counts[impl] = seen
    assert counts["hip"] == counts["eager"] and len(counts["hip"]) > 20


class Adapter(nn.Module):
    """A low-rank term beside a layer whose weight it shows."""

    def __init__(self, base):
        super().__init__()
        self.base, self.a, self.b = base, nn.Parameter(torch.randn(4, base.in_features)), nn.Parameter(
            torch.randn(base.out_features, 4))

    weight = property(lambda self: self.base.weight)
    bias = None

    def forward(self, x):
        return self.base(x) + x @ self.a.t() @ self.b.t()


class Scaled(M.RMSNorm):
    def forward(self, x):
        return 0.5 * super().forward(x)


class Half(M.Block):
    def forward(self, x, cos, sin):
        return x + 0.5 * (super().forward(x, cos, sin) - x)


def _adapter(m):
    m.layers[1].mlp.gate_proj = Adapter(m.layers[1].mlp.gate_proj)


def _bias(m):
    m.layers[0].mlp.up_proj = nn.Linear(32, 64, bias=True)


def _norm_class(m):
    m.layers[1].post_attention_layernorm = Scaled(32)


def _block_class(m):
    m.layers[1].__class__ = Half


def _own_forward(m):
    gate = m.layers[2].mlp.gate_proj
    gate.forward = lambda x: 2 * F.linear(x, gate.weight)


def _parametrized(m):
    class Double(nn.Module):
        def forward(self, w):
            return 2 * w
    nn.utils.parametrize.register_parametrization(m.layers[0].mlp.up_proj, "weight", Double())


def _only_layers(m):
    m.layers = nn.ModuleList()


@pytest.mark.parametrize("change", [_adapter, _bias, _norm_class, _block_class, _own_forward, _parametrized, _only_layers])
def test_other_modules_are_called(model, change):
    m, ids = model
    plain = _logits(m, ids, "eager")
    change(m)
    assert (_logits(m, ids, "eager") - plain).abs().max() > 1e-3 * plain.abs().max()
    _same(m, ids)


@pytest.mark.parametrize("hooked", [False, True])
def test_traces_in_one_graph(hooked, monkeypatch):
    """Compiled, the same choice is made, without a graph break."""
    ops = []

    def backend(gm, _):
        ops.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function")
        return gm.forward

    torch._dynamo.reset()
    monkeypatch.setattr(nn.init, "normal_", lambda t, **kw: t)
    with FakeTensorMode(), torch.device("cuda"):
        torch.set_default_dtype(torch.bfloat16)
        try:
            m = M.ModelForCausalLM(M.ModelConfig(**(CONFIG | dict(head_dim=64))))
        finally:
            torch.set_default_dtype(torch.float32)
        m.set_attn_impl("hip")
        m.set_block_impl("hip")
        if hooked:
            m.layers[1].mlp.gate_proj.register_forward_hook(lambda mod, args, out: 2 * out)
            m.layers[2].input_layernorm.register_forward_hook(lambda mod, args, out: 2 * out)
        torch.compile(m, backend=backend, fullgraph=True)(torch.zeros(2, 8, dtype=torch.long, device="cuda"))
    torch._dynamo.reset()
    counts = [sum(f"tinytrain.{n}." in o for o in ops) for n in ("rms_norm_fwd", "swiglu_fwd")]
    assert counts == ([6, 2] if hooked else [7, 3]), counts
