"""The feed-forward block's operators without a GPU: their wrappers as tools that read a program take them, their shapes
when traced, the C ABI's answers to what it refuses, and the reference formulas against differences."""
import inspect

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.overrides import TorchFunctionMode

import driss_torch as d
import feed_forward_reference as ref
from driss_torch_amd import cabi, feed_forward

X = torch.randn(4, 16, dtype=torch.bfloat16)
W = torch.randn(8, 16, dtype=torch.bfloat16)
P = torch.randn(16, dtype=torch.bfloat16)
Q = torch.zeros(4, 16, dtype=torch.int8)
CALLS = {"int8_quantize": (X,), "int8_bf16": (Q, Q.t(), torch.ones(4, 1), torch.ones(4, 1)), "gated_linear": (X, W, W), "pre_norm": (X, P), "post_norm": (X, X, P),
         "post_pre_norm": (X, X, P, P)}


def test_every_wrapper_is_here_and_public():
    assert set(feed_forward.__all__) == set(CALLS)
    for name in CALLS:
        assert getattr(d, name) is getattr(feed_forward, name) and inspect.getdoc(getattr(d, name))


@pytest.mark.parametrize("name", CALLS)
def test_script_trace_and_function_mode(name):
    wrapper, op = getattr(d, name), getattr(torch.ops.DrissTorch, name)
    assert "DrissTorch::" + name in str(torch.jit.script(wrapper).inlined_graph)
    concrete = {p.name: p.default for p in inspect.signature(wrapper).parameters.values() if p.default is not p.empty}
    assert op in [n.target for n in torch.fx.symbolic_trace(wrapper, concrete_args=concrete).graph.nodes if n.op == "call_function"]
    seen = []

    class Watch(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return args[0]

    with Watch():
        wrapper(*CALLS[name])
    assert op in seen


@pytest.mark.parametrize("name", CALLS)
def test_no_kernel_on_the_cpu(name):
    with pytest.raises(NotImplementedError):
        getattr(d, name)(*CALLS[name])


def test_traced_shapes():
    with FakeTensorMode():
        x = torch.empty(2, 3, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        w = torch.empty(8, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        p = torch.empty(16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        gate = torch.empty(2, 1, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        h = d.gated_linear(x, w, w, "gelu")
        assert h.shape == (2, 3, 8) and h.dtype == torch.bfloat16
        assert h.grad_fn is not None
        _, g, u = d.ops.gated_linear_forward(x, w, w, "gelu")
        grads = d.ops.gated_linear_backward(h, x, w, w, g, u, "gelu", True, True)
        assert [t.shape for t in grads] == [x.shape, w.shape, w.shape]
        r, n = d.post_pre_norm(x, x, p, p, gate)
        assert r.grad_fn is not None and r.shape == n.shape == x.shape
        r, n, iy, ir = d.ops.norm_forward(x, x, p, p, gate, 1.0, 1e-6, True)
        assert iy.shape == ir.shape == (6,)
        grads = d.ops.norm_backward(r, None, r, x, p, p, gate, iy, ir, 1.0)
        assert [t.shape for t in grads] == [x.shape, x.shape, p.shape, p.shape, gate.shape]
        assert d.pre_norm(x, p).shape == x.shape and d.post_norm(x, x, p).shape == x.shape
        q, s = d.int8_quantize(torch.empty(5, 16, device="cuda"))
        assert q.dtype == torch.int8 and s.shape == (5, 1) and d.int8_bf16(q, q.t(), s, s).shape == (5, 5)


def test_host_validation():
    L, p = cabi.lib(), 0x1000  # never dereferenced
    assert L.dt_int8_quantize(p, cabi.F16, 4, 8, p, p, None) == 1
    assert L.dt_int8_quantize(p, cabi.BF16, -1, 8, p, p, None) == 2
    assert L.dt_int8_quantize(p, cabi.BF16, 4, 0, p, p, None) == 8
    assert L.dt_int8_quantize(p, cabi.BF16, 0, 8, None, None, None) == 0
    assert L.dt_int8_quantize(p, cabi.BF16, 4, 8, p, None, None) == 3
    assert L.dt_int8_quantize(p + 1, cabi.BF16, 4, 8, p, p, None) == 4
    big = 1 << 40
    assert L.dt_int8_bf16(p, p, p, p, 4, 8, 1 << 17, 1 << 17, 1 << 17, p, 8, p, big, None) == 2
    assert L.dt_int8_bf16(p, p, p, p, 4, 8, 16, 15, 16, p, 8, p, big, None) == 2
    assert L.dt_int8_bf16(p, p, p, p, 4, 8, 16, 16, 16, p, 7, p, big, None) == 2
    assert L.dt_int8_bf16(p, None, p, p, 4, 8, 16, 16, 16, p, 8, p, big, None) == 3
    assert L.dt_int8_bf16(p, p, p + 2, p, 4, 8, 16, 16, 16, p, 8, p, big, None) == 4
    assert L.dt_int8_bf16(None, None, None, None, 0, 8, 16, 16, 16, None, 8, None, 0, None) == 0
    assert L.dt_gated_linear(p, p, p, 4, 8, 16, 8, 8, 8, 3, p, None, None, p, big, None) == 6
    assert L.dt_gated_linear(p, p, p, 4, 8, 16, 7, 8, 8, 0, p, None, None, p, big, None) == 2
    assert L.dt_gated_linear(p, p, p, 4, 1 << 22, 16, 1 << 22, 1 << 22, 1 << 22, 0, p, None, None, p, big, None) == 2
    assert L.dt_gated_linear(p, p, p, 4, 8, 1 << 22, 8, 8, 8, 0, p, None, None, p, big, None) == 2
    assert L.dt_gated_linear(p, p, p, 4, 8, 16, 8, 8, 8, 0, p, p, None, p, big, None) == 3
    assert L.dt_gated_linear(p, p + 1, p, 4, 8, 16, 8, 8, 8, 0, p, None, None, p, big, None) == 4
    assert L.dt_gated_linear(None, None, None, 0, 8, 16, 8, 8, 8, 0, None, None, None, None, 0, None) == 0
    need = L.dt_gated_linear_backward_workspace_bytes(p, p, p, 4, 8, 16, 8, 8, 8)
    assert need >= 4 * 16 * 4
    args = (p, p, p, p, p, p, 4, 8, 16, 8, 8, 8)
    assert L.dt_gated_linear_backward(*args, 0, p, p, p, p, need - 1, None) == 5
    assert L.dt_gated_linear_backward(*args, 0, p, p, None, p, need, None) == 3
    assert L.dt_gated_linear_backward(*args, 5, p, p, p, p, need, None) == 6
    forward = lambda form, gate, gates, dtype, rows, cols, normed=p: L.dt_norm_forward(form, p, p, p, p, gate, gates, dtype, rows, cols, 1.0, 1e-6, p, normed, None, None, None)  # noqa: E731
    assert forward(0, None, 0, cabi.F32, 4, 8) == 6 and forward(3, None, 0, cabi.F16, 4, 8) == 1 and forward(3, None, 0, cabi.F32, 4, 32769) == 2
    assert forward(3, p, 3, cabi.F32, 4, 8) == 2 and forward(3, p, 0, cabi.F32, 4, 8) == 6 and forward(2, p, 1, cabi.F32, 4, 8) == 6
    assert forward(3, None, 0, cabi.F32, 4, 0) == 8 and forward(3, None, 0, cabi.F32, 0, 8) == 0 and forward(3, None, 0, cabi.F32, 4, 8, None) == 3
    assert forward(3, None, 0, cabi.F32, 4, 8, p + 2) == 4
    need = L.dt_norm_backward_workspace_bytes(3, 2, cabi.F32, 64, 100)
    assert need >= 2 * 100 * 4
    assert L.dt_norm_backward(3, p, p, p, p, p, p, p, 2, cabi.F32, 64, 100, 1.0, p, p, p, p, p, p, p, p, need - 1, None) == 5
    assert L.dt_norm_backward(3, p, p, p, p, p, p, p, 2, cabi.F32, 64, 100, 1.0, p, p, p, p, p, p, None, p, need, None) == 3


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_reference_gradients_of_the_gated_projections(act):
    """the formulas of the reference against autograd over its value, and its slope against differences"""
    g = torch.Generator().manual_seed(1)
    x, wg, wu, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (6, 7), (6, 7), (5, 6)))
    leaves = [v.clone().requires_grad_() for v in (x, wg, wu)]
    h = ref.act(leaves[0] @ leaves[1].t(), act)[0] * (leaves[0] @ leaves[2].t())
    for want, (value, _) in zip(torch.autograd.grad(h, leaves, dh), ref.gated_grads(dh, x, wg, wu, act).values()):
        assert torch.allclose(want, value, rtol=1e-12, atol=1e-12)
    z = torch.linspace(-6, 6, 101, dtype=torch.float64)
    step = 1e-5
    differences = (ref.act(z + step, act)[0] - ref.act(z - step, act)[0]) / (2 * step)
    assert torch.allclose(ref.act(z, act)[1], differences, rtol=1e-8, atol=1e-9)  # the third derivative, at most 2, times step^2 / 6, and 1e-16 / step
    assert ref.act(z, act)[1].abs().max() < ref.SLOPE
    curve = (ref.act(z + 1e-4, act)[1] - ref.act(z - 1e-4, act)[1]) / 2e-4
    assert curve.abs().max() < ref.CURVE


@pytest.mark.parametrize("gates", [0, 1, 2, 6])
def test_reference_gradients_of_the_norms(gates):
    g = torch.Generator().manual_seed(2)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    r, y, p, w, gate = n(6, 9), n(6, 9), n(9), n(9), n(gates, 9) if gates else None
    dr, dn = n(6, 9), n(6, 9)
    leaves = [v.clone().requires_grad_() for v in (r, y, p, w)] + ([gate.clone().requires_grad_()] if gates else [])
    norm = lambda v: v / (v.square().mean(1, keepdim=True) + 1e-3).sqrt()  # noqa: E731
    gr = leaves[4].repeat_interleave(6 // gates, 0) if gates else 1.0
    stream = leaves[0] + 0.3 * gr * leaves[2] * norm(leaves[1])
    normed = leaves[3] * norm(stream)
    got = ref.norms(r, y, p, w, gate, 0.3, 1e-3, dr, dn)
    assert torch.allclose(got["residual"][0], stream) and torch.allclose(got["normed"][0], normed)
    names = ["d_residual", "d_branch", "d_post_weight", "d_pre_weight"] + (["d_gate"] if gates else [])
    for name, want in zip(names, torch.autograd.grad([stream, normed], leaves, [dr, dn])):
        assert torch.allclose(got[name][0], want, rtol=1e-11, atol=1e-12), name


def test_new_residual_built_again_is_of_both_norms_in_bf16():
    L, p = cabi.lib(), 0x1000  # never dereferenced
    backward = lambda form, dtype, room: L.dt_norm_backward(form, p, p, p, p, p, p, p, 2, dtype, 64, 100, 1.0, p, p, p, p, p, p, p, p, room, None)  # noqa: E731
    need = L.dt_norm_backward_workspace_bytes(7, 2, cabi.BF16, 64, 100)
    assert need == L.dt_norm_backward_workspace_bytes(3, 2, cabi.BF16, 64, 100)
    assert backward(7, cabi.BF16, need - 1) == 5 and backward(7, cabi.F32, need) == 6 and backward(5, cabi.BF16, need) == 6 and backward(6, cabi.BF16, need) == 6
    assert backward(4, cabi.BF16, need) == 6 and L.dt_norm_forward(7, p, p, p, p, None, 0, cabi.BF16, 4, 8, 1.0, 1e-6, p, p, None, None, None) == 6


TRAINED = {"gated_linear": 3, "pre_norm": 2, "post_norm": 4, "post_pre_norm": 5}


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("name,of", [(name, of) for name, n in TRAINED.items() for of in range(n)])
def test_a_tangent_is_refused(name, of, no_grad):
    """forward-mode derivatives there are none: a dual tensor or torch.func.jvp raises, of whichever input, with gradients recorded or not"""
    with FakeTensorMode():
        x, w, p = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((4, 16), (8, 16), (16,)))
        args = list({"gated_linear": (x, w, w), "pre_norm": (x, p), "post_norm": (x, x, p, p), "post_pre_norm": (x, x, p, p, p)}[name])
        call = lambda v: getattr(d, name)(*args[:of], v, *args[of + 1:])  # noqa: E731
        if name == "post_pre_norm" and of == 4:
            call = lambda v: d.post_pre_norm(*args[:4], gate=v)  # noqa: E731
        with torch.set_grad_enabled(not no_grad):
            call(args[of])
            with torch.autograd.forward_ad.dual_level():
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(torch.autograd.forward_ad.make_dual(args[of], torch.empty_like(args[of])))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.func.jvp(call, (args[of],), (torch.empty_like(args[of]),))
