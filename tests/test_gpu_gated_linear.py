"""The gated projections and their gradients against 64 bits, with bounds that follow each rounding and sum
(feed_forward_reference.py)."""
import pytest
import torch

import driss_torch as d
import feed_forward_reference as ref
from driss_torch_amd import cabi

pytestmark = pytest.mark.gpu
ACTS = ["silu", "gelu", "gelu_tanh"]


def inputs(t, dim, f, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, dim, generator=g).to(torch.bfloat16)
    wg, wu = ((torch.randn(f, dim, generator=g) * max(1, dim) ** -0.5).to(torch.bfloat16) for _ in range(2))
    dh = torch.randn(t, f, generator=g).to(torch.bfloat16)
    return tuple(v.to(device) for v in (x, wg, wu, dh))


FORWARD = [(1, 1, 1), (1, 8, 8), (1, 128, 64), (1, 1001, 333), (2, 512, 1000), (3, 7, 5), (5, 4096, 200), (15, 1000, 130), (16, 520, 1024), (17, 264, 96), (32, 64, 513), (33, 2048, 128),
           (64, 100, 100), (65, 129, 127), (100, 640, 700), (128, 256, 256), (130, 1032, 1000), (200, 72, 1433), (256, 512, 264), (257, 255, 511), (512, 128, 1000), (1001, 333, 257),
           (1, 70, 40), (20, 1018, 33), (9, 4, 100), (70, 130, 50), (150, 1002, 64), (300, 134, 260), (128, 2, 128)]


@pytest.mark.parametrize("t,dim,f", FORWARD)
def test_forward(gpu_device, t, dim, f):
    act = ACTS[(t + dim + f) % 3]
    x, wg, wu, _ = inputs(t, dim, f, t * 31 + dim * 7 + f, gpu_device)
    h = d.gated_linear(x, wg, wu, act)
    assert h.dtype == torch.bfloat16
    ref.assert_within(h, *ref.gated(x, wg, wu, act), (t, dim, f, act))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [1, 40, 300])
def test_activations_far_out(gpu_device, t, act):
    """products from far below to far above zero, where exp overflows or vanishes"""
    x, wg, wu, dh = inputs(t, 64, 520, t, gpu_device)
    x *= 40
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    h = d.gated_linear(*leaves, act)
    ref.assert_within(h, *ref.gated(x, wg, wu, act), act)
    grads = torch.autograd.grad(h, leaves, dh)
    for g, (name, (want, bound)) in zip(grads, ref.gated_grads(dh, x, wg, wu, act).items()):
        ref.assert_within(g, want, bound, (name, act))


BACKWARD = [(1, 8, 8), (1, 1, 1), (1, 333, 130), (3, 5, 7), (16, 64, 128), (40, 1001, 37), (65, 129, 130), (100, 72, 1000), (128, 256, 256), (130, 520, 264), (256, 128, 512), (257, 255, 513),
            (511, 1000, 96), (1001, 201, 273), (2048, 264, 136),
            (2, 70, 40), (70, 130, 50), (150, 1002, 66), (300, 134, 262), (128, 2, 128), (66, 6, 10)]


@pytest.mark.parametrize("t,dim,f", BACKWARD)
def test_gradients(gpu_device, t, dim, f):
    act = ACTS[(t + dim + f) % 3]
    x, wg, wu, dh = inputs(t, dim, f, t * 31 + dim * 7 + f, gpu_device)
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    h = d.gated_linear(*leaves, act)
    ref.assert_within(h, *ref.gated(x, wg, wu, act), (t, dim, f, act))
    grads = torch.autograd.grad(h, leaves, dh)
    for g, (name, (want, bound)) in zip(grads, ref.gated_grads(dh, x, wg, wu, act).items()):
        assert g.dtype == torch.bfloat16
        ref.assert_within(g, want, bound, (name, t, dim, f, act))


@pytest.fixture
def tiles(request):
    """the tiles and shares of K, as given"""
    cabi.set_tuning("mm.tiles", request.param[0])
    cabi.set_tuning("mm.splits", request.param[1])
    yield request.param
    cabi.set_tuning("mm.tiles", 0)
    cabi.set_tuning("mm.splits", 0)


@pytest.mark.parametrize("tiles", [(1, 0), (2, 1), (2, 3), (3, 1), (3, 2), (3, 7), (4, 1), (4, 2)], indirect=True)
@pytest.mark.parametrize("t,dim,f", [(33, 8, 8), (65, 129, 130), (130, 520, 264), (257, 255, 513), (300, 1000, 200)])
def test_tiles(gpu_device, t, dim, f, tiles):
    x, wg, wu, dh = inputs(t, dim, f, t + dim + f, gpu_device)
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    h = d.gated_linear(*leaves)
    ref.assert_within(h, *ref.gated(x, wg, wu, "silu"), tiles)
    for g, (name, (want, bound)) in zip(torch.autograd.grad(h, leaves, dh), ref.gated_grads(dh, x, wg, wu, "silu").items()):
        ref.assert_within(g, want, bound, (name, tiles))


def test_forward_is_the_same_with_and_without_gradients(gpu_device):
    for t in (1, 30, 200, 600):
        x, wg, wu, _ = inputs(t, 264, 520, t, gpu_device)
        h = d.gated_linear(x, wg, wu)
        assert torch.equal(h, d.gated_linear(x.clone().requires_grad_(), wg, wu).detach())
        with torch.no_grad():
            assert torch.equal(h, d.gated_linear(x.clone().requires_grad_(), wg, wu))


def test_gradients_on_demand(gpu_device):
    """of the inputs that want one, equal to those of all, and the same on every call"""
    x, wg, wu, dh = inputs(130, 264, 328, 1, gpu_device)
    every = [v.clone().requires_grad_() for v in (x, wg, wu)]
    want = torch.autograd.grad(d.gated_linear(*every), every, dh)
    for wanted in ([0], [1], [2], [0, 2], [1, 2]):
        leaves = [v.clone().requires_grad_(i in wanted) for i, v in enumerate((x, wg, wu))]
        grads = torch.autograd.grad(d.gated_linear(*leaves), [leaves[i] for i in wanted], dh)
        assert all(torch.equal(g, want[i]) for g, i in zip(grads, wanted))


@pytest.mark.parametrize("t", [2, 70, 300])
def test_strides_and_leading_dimensions(gpu_device, t):
    x, wg, wu, dh = inputs(2 * t, 200, 136, t, gpu_device)
    want = d.gated_linear(x, wg, wu)
    assert torch.equal(d.gated_linear(x.view(2, t, 200), wg, wu), want.view(2, t, 136))
    wide = torch.full((2 * t, 333), float("nan"), dtype=torch.bfloat16, device=gpu_device)
    wide[:, 5:205] = x
    both = torch.full((136, 512), float("nan"), dtype=torch.bfloat16, device=gpu_device)
    both[:, 8:208], both[:, 256:456] = wg, wu
    views = [wide[:, 5:205].detach().requires_grad_(), both[:, 8:208].detach().requires_grad_(), both[:, 256:456].detach().requires_grad_()]
    h = d.gated_linear(*views)
    ref.assert_within(h, *ref.gated(x, wg, wu, "silu"), "strided")
    # gradients of views, and of a gradient that is itself a view or one value for all
    grads = torch.autograd.grad(h, views, dh.t().contiguous().t())
    for g, (name, (v, bound)) in zip(grads, ref.gated_grads(dh, x, wg, wu, "silu").items()):
        ref.assert_within(g, v, bound, name)
    one = torch.ones((), dtype=torch.bfloat16, device=gpu_device).expand_as(dh)
    grads = torch.autograd.grad(d.gated_linear(*views), views, one)
    for g, (name, (v, bound)) in zip(grads, ref.gated_grads(one, x, wg, wu, "silu").items()):
        ref.assert_within(g, v, bound, name)


@pytest.mark.parametrize("dim", [64, 200, 201])
def test_what_is_not_finite_stays_in_its_row(gpu_device, dim):
    for t in (5, 70, 300):
        x, wg, wu, dh = inputs(t, dim, 150, t, gpu_device)
        want = d.gated_linear(x, wg, wu)
        x[3, dim - 1] = float("nan")
        wg[7, 0] = float("inf")
        h = d.gated_linear(x, wg, wu)
        assert h[3].isnan().all()
        keep = torch.ones_like(h, dtype=torch.bool)
        keep[3], keep[:, 7] = False, False
        assert torch.equal(h[keep], want[keep])


def test_empty(gpu_device):
    x, wg, wu, dh = inputs(4, 16, 8, 0, gpu_device)
    assert d.gated_linear(x[:0], wg, wu).shape == (0, 8)
    assert d.gated_linear(x, wg[:0], wu[:0]).shape == (4, 0)
    assert torch.equal(d.gated_linear(x[:, :0], wg[:, :0], wu[:, :0]), torch.zeros_like(dh))
    leaves = [v.clone().requires_grad_() for v in (x[:0], wg, wu)]
    dx, dg, du = torch.autograd.grad(d.gated_linear(*leaves), leaves, dh[:0])
    assert dx.shape == (0, 16) and not dg.any() and not du.any()
    leaves = [v.clone().requires_grad_() for v in (x, wg[:0], wu[:0])]
    dx, dg, du = torch.autograd.grad(d.gated_linear(*leaves), leaves, dh[:, :0])
    assert not dx.any() and dx.shape == (4, 16) and dg.shape == (0, 16)


def test_on_another_stream_and_in_a_graph(gpu_device):
    for t in (1, 40, 300):
        x, wg, wu, dh = inputs(t, 264, 328, t, gpu_device)

        def step(v):
            leaves = [u.detach().requires_grad_() for u in (v, wg, wu)]
            h = d.gated_linear(*leaves)
            return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

        want = [v.clone() for v in step(x)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = step(x)
        stream.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        static = x.clone()
        with torch.cuda.graph(graph):
            out = step(static)
        for seed in range(3):
            static.copy_(torch.randn(static.shape, generator=torch.Generator().manual_seed(seed)).to(static.dtype))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(step(static), out))


def test_refusals(gpu_device):
    x, wg, wu, dh = inputs(4, 16, 8, 0, gpu_device)
    for bad, text in [(lambda: d.gated_linear(x, wg, wu, "relu"), "activation"), (lambda: d.gated_linear(x.float(), wg, wu), "bfloat16"), (lambda: d.gated_linear(x, wg, wu[:4]), "same shape"),
                      (lambda: d.gated_linear(x[:, :8], wg, wu), "Incompatible"), (lambda: d.gated_linear(x, wg[0], wu), "matrices"), (lambda: d.gated_linear(x, wg.cpu(), wu), "on the GPU")]:
        with pytest.raises(RuntimeError, match=text):
            bad()
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient of its gradient"):
        torch.autograd.grad(d.gated_linear(leaf, wg, wu), leaf, dh, create_graph=True)


@pytest.mark.parametrize("t", [3, 20, 70, 300])
def test_last_columns_of_wide_tensors(gpu_device, t):
    """views whose rows end where their storage does, with rows that end inside a 16-byte chunk: nothing past the storage counts"""
    dim, f = 202, 150
    x, wg, wu, dh = inputs(t, dim, f, t, gpu_device)
    views = []
    for v in (x, wg, wu):
        wide = torch.full((v.shape[0], 330), float("nan"), dtype=torch.bfloat16, device=gpu_device)
        wide[:, 330 - dim:] = v
        views.append(wide[:, 330 - dim:].detach().requires_grad_())
    h = d.gated_linear(*views)
    ref.assert_within(h, *ref.gated(x, wg, wu, "silu"), t)
    for g, (name, (want, bound)) in zip(torch.autograd.grad(h, views, dh), ref.gated_grads(dh, x, wg, wu, "silu").items()):
        ref.assert_within(g, want, bound, (name, t))


# the products of the forward pass, of dx, of both weights' gradients take two launches each
@pytest.mark.parametrize("t,dim,f", [(1515, 2102, 2811), (3559, 4898, 150), (2430, 4703, 1583)])
def test_two_launches(gpu_device, t, dim, f):
    x, wg, wu, dh = inputs(t, dim, f, t, gpu_device)
    h = d.gated_linear(x, wg, wu)
    ref.assert_within(h, *ref.gated(x, wg, wu, "silu"), t)
    if f > dim:
        return
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    grads = torch.autograd.grad(d.gated_linear(*leaves), leaves, dh)
    for g, (name, (want, bound)) in zip(grads, ref.gated_grads(dh, x, wg, wu, "silu").items()):
        ref.assert_within(g, want, bound, (name, t, dim, f))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [2, 40, 300])
def test_gradients_where_squares_overflow(gpu_device, t, act):
    """gates of +-2^66, whose squares are no fp32 numbers: activations and slopes are at their limits, g and 1 above zero, 0 and 0 below.  Every sum has one
    term, a product of powers of two, and half the rows have a gate of either sign."""
    dim, f = 16, 8
    x, wg, wu = (torch.zeros(n, dim, dtype=torch.bfloat16, device=gpu_device) for n in (t, f, f))
    x[::2, 0], x[1::2, 0], x[:, 1] = 2.0**66, -(2.0**66), 1.0
    wg[:, 0], wu[:, 1] = 1.0, 0.5
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    h = d.gated_linear(*leaves, act)
    assert (h[::2] == 2.0**65).all() and (h[1::2] == 0).all()
    dh = torch.zeros_like(h)
    dh[0, 0] = dh[1, 1] = 1.0
    dx, dg, du = torch.autograd.grad(h, leaves, dh)
    want = torch.zeros_like(x)
    want[0, 0], want[0, 1] = 0.5, 2.0**65  # u times the slope 1, times the weight 1; the activation times the weight 0.5
    assert torch.equal(dx, want)
    want_g, want_u = torch.zeros_like(wg), torch.zeros_like(wu)
    want_g[0, 0], want_g[0, 1], want_u[0, 0], want_u[0, 1] = 2.0**65, 0.5, float("inf"), 2.0**66  # (2^132 is past bf16)
    assert torch.equal(dg, want_g) and torch.equal(du, want_u)


# at most 32 rows and more groups of columns than CUs: a workgroup takes several in turn, with rows of whole words and off them, one and two tiles of rows,
# and few groups of rows off the words with sixteen waves a workgroup
@pytest.mark.parametrize("t,dim,f", [(1, 256, 14336), (3, 1032, 9001), (8, 130, 16001), (12, 520, 7000), (20, 256, 9000), (32, 64, 20011), (1, 2048, 2731), (3, 129, 9001), (16, 65, 8500),
                                     (24, 333, 200), (24, 333, 5000), (32, 1001, 4097), (17, 129, 9003), (32, 77, 13000)])
def test_few_rows_and_many_columns(gpu_device, t, dim, f):
    act = ACTS[(t + dim + f) % 3]
    x, wg, wu, _ = inputs(t, dim, f, t + dim + f, gpu_device)
    want = ref.gated(x, wg, wu, act)
    h = d.gated_linear(x, wg, wu, act)
    ref.assert_within(h, *want, (t, dim, f, act))
    # and with both products kept
    kept, g, u = d.ops.gated_linear_forward(x, wg, wu, act)
    assert torch.equal(kept, h)
    n = dim * 2.0**-24 + ref.E
    for got, w in ((g, wg), (u, wu)):
        ref.assert_within(got, ref.f64(x) @ ref.f64(w).t(), n * (ref.f64(x).abs() @ ref.f64(w).abs().t()))


def test_offsets_past_32_bits(gpu_device):
    """more than 2^31 gated elements: rows at the end as in a call of those rows alone, and weights' gradients of the last rows, the others' being zero"""
    t, dim, f = 70001, 64, 32760
    if torch.cuda.mem_get_info()[0] < 96 << 30:
        pytest.skip("needs 96 GiB of free device memory")
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device, dtype=torch.bfloat16)  # noqa: E731
    x, wg, wu = (v.requires_grad_() for v in (n(t, dim), n(f, dim), n(f, dim)))
    h = d.gated_linear(x, wg, wu)
    dh = torch.zeros_like(h)
    last = t - 50
    dh[last:] = n(50, f)
    dx, dg, du = torch.autograd.grad(h, (x, wg, wu), dh)
    for part in (slice(0, 50), slice(65536, 65586), slice(last, t)):
        ref.assert_within(h[part], *ref.gated(x[part], wg, wu, "silu"), part)
    assert not dx[:last].any()
    want = ref.gated_grads(dh[last:], x[last:], wg, wu, "silu")
    ref.assert_within(dx[last:], *want["dx"], "dx")
    # (the zero rows add nothing, of however many steps the sum is)
    ref.assert_within(dg, *want["dw_gate"], "dw_gate")
    ref.assert_within(du, *want["dw_up"], "dw_up")
