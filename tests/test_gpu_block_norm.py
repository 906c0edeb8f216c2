"""The norms before and after a block and their gradients against 64 bits, with bounds that follow each rounding and
sum (feed_forward_reference.py), and the fp32 gradients against differences of the kernels' own results."""
import pytest
import torch

import driss_torch as d
import feed_forward_reference as ref
from driss_torch_amd import cabi

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
EPS = 1e-6


def inputs(rows, cols, gates, dtype, seed, device, form="post_pre"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    v = {"residual": n(rows, cols) * 2, "branch": n(rows, cols) * torch.exp(n(rows, 1)), "post_weight": 1 + 0.2 * n(cols), "pre_weight": 1 + 0.2 * n(cols),
         "gate": n(gates, cols) if gates else None, "d_residual": n(rows, cols), "d_normed": n(rows, cols)}
    gone = {"pre": ("branch", "post_weight", "gate", "d_residual"), "post": ("pre_weight", "d_normed"), "post_pre": ()}[form]
    return {k: None if k in gone or t is None else t.to(dtype).to(device) for k, t in v.items()}


def call(v, form, scale=0.7):
    if form == "pre":
        return {"normed": d.pre_norm(v["residual"], v["pre_weight"], EPS)}
    if form == "post":
        return {"residual": d.post_norm(v["residual"], v["branch"], v["post_weight"], v["gate"], scale, EPS)}
    r, n = d.post_pre_norm(v["residual"], v["branch"], v["post_weight"], v["pre_weight"], v["gate"], scale, EPS)
    return {"residual": r, "normed": n}


def run(v, form, scale=0.7, skip=()):
    """values and gradients by name; `skip`: results whose gradient is not given"""
    names = [k for k in ("residual", "branch", "post_weight", "pre_weight", "gate") if v[k] is not None]
    leaves = {**v, **{k: v[k].detach().clone().requires_grad_() for k in names}}
    out = call(leaves, form, scale)
    ends = [k for k in out if k not in skip]
    grads = torch.autograd.grad([out[k] for k in ends], [leaves[k] for k in names], [v["d_" + k] for k in ends], allow_unused=True)
    return {**{k: t.detach() for k, t in out.items()}, **{"d_" + k: g for k, g in zip(names, grads) if g is not None}}


def reference(v, scale=0.7, skip=()):
    return ref.norms(v["residual"], v["branch"], v["post_weight"], v["pre_weight"], v["gate"], scale, EPS, None if "residual" in skip else v["d_residual"],
                     None if "normed" in skip else v["d_normed"])


def check(got, want, what):
    assert set(got) == set(want), (sorted(got), sorted(want))
    for k, (value, bound) in want.items():
        ref.assert_within(got[k], value, bound, (k, what))


# rows of one element to the longest, on and off the vectors; one row to more than the units the gradient is split into
SIZES = [(1, 1, 1), (3, 7, 3), (1, 64, 0), (5, 256, 1), (40, 512, 4), (1, 513, 1), (600, 520, 0), (7, 1001, 7), (64, 1024, 2), (9, 2048, 0), (30, 2056, 3), (2, 4096, 1), (20, 4100, 5),
         (520, 1000, 520), (3, 8192, 1), (12, 8191, 2), (4, 16384, 1), (6, 16390, 3), (2, 32768, 2), (3, 30001, 1), (4100, 72, 4100), (5000, 40, 1), (6000, 33, 1500), (1100, 264, 550),
         (2048, 128, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,gates", SIZES)
def test_post_pre(gpu_device, rows, cols, gates, dtype):
    v = inputs(rows, cols, gates, dtype, rows + cols, gpu_device)
    check(run(v, "post_pre"), reference(v), (rows, cols, gates))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["pre", "post"])
@pytest.mark.parametrize("rows,cols,gates", [(1, 1, 0), (5, 100, 1), (70, 1000, 0), (33, 2048, 33), (10, 4104, 2), (3, 9001, 0), (2, 32768, 1), (3000, 96, 3)])
def test_one_norm_alone(gpu_device, rows, cols, gates, form, dtype):
    v = inputs(rows, cols, 0 if form == "pre" else gates, dtype, rows + cols, gpu_device, form)
    check(run(v, form), reference(v), (rows, cols, gates, form))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("skip", ["residual", "normed"])
def test_a_result_without_gradient(gpu_device, skip, dtype):
    v = inputs(60, 328, 2, dtype, 4, gpu_device)
    check(run(v, "post_pre", skip=(skip,)), reference(v, skip=(skip,)), skip)


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dimensions_strides_and_alignment(gpu_device, dtype):
    v = inputs(24, 200, 4, dtype, 1, gpu_device)
    want = run(v, "post_pre")
    shaped = {k: t.view(4, 6, 200) if k in ("residual", "branch", "d_residual", "d_normed") else t.view(4, 1, 200) if k == "gate" else t for k, t in v.items()}
    got = run(shaped, "post_pre")
    assert all(torch.equal(got[k].reshape(want[k].shape), want[k]) for k in want)
    for skip in (1, 2, 3):
        moved = {}
        for k, t in v.items():
            wide = torch.full((skip + t.numel(),), float("nan"), dtype=dtype, device=gpu_device)
            moved[k] = wide[skip:].view(t.shape).copy_(t)
        check(run(moved, "post_pre"), reference(v), skip)
    wide = torch.full((24, 333), float("nan"), dtype=dtype, device=gpu_device)
    wide[:, 7:207] = v["branch"]
    got = run({**v, "branch": wide[:, 7:207], "d_normed": v["d_normed"].t().contiguous().t()}, "post_pre")
    assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_anything_and_rows_that_are_not_finite(gpu_device, dtype):
    v = inputs(40, 264, 0, dtype, 2, gpu_device)
    v["branch"][3] = 0
    v["residual"][3] = 0
    check(run(v, "post_pre"), reference(v), "zero rows")
    want = call(v, "post_pre")
    v["branch"][5, 263] = float("nan")
    v["residual"][9, 0] = float("inf")
    got = call(v, "post_pre")
    keep = [i for i in range(40) if i not in (5, 9)]
    assert all(torch.equal(got[k][keep], want[k][keep]) for k in want)
    assert got["normed"][5].isnan().all() and not got["normed"][9, 0].isfinite()


def test_same_bits_every_time(gpu_device):
    """the sums over rows are always taken in the same order"""
    v = inputs(3000, 520, 3, torch.bfloat16, 6, gpu_device)
    want = run(v, "post_pre")
    for _ in range(3):
        got = run(v, "post_pre")
        assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("rows,cols,gates", [(6, 40, 1), (8, 257, 2), (5, 1000, 5)])
def test_gradients_against_differences(gpu_device, rows, cols, gates):
    """fp32: the change of <results, their gradients> along a direction of all inputs.  With a step of 2^-7 the third-order term is
    measured by the same difference at twice the step (four times as large), and the results' rounding, E of
    each, is divided by the step."""
    v = inputs(rows, cols, gates, torch.float32, rows, gpu_device)
    names = ("residual", "branch", "post_weight", "pre_weight", "gate")
    g = torch.Generator().manual_seed(9)
    way = {k: torch.randn(v[k].shape, generator=g).to(gpu_device) for k in names}
    grads = run(v, "post_pre")
    along = sum((grads["d_" + k].double() * way[k].double()).sum() for k in names)

    def value(step):
        out = call({**v, **{k: v[k] + step * way[k] for k in names}}, "post_pre")
        return sum((out[k].double() * v["d_" + k].double()).sum() for k in out), sum((out[k].double() * v["d_" + k].double()).abs().sum() for k in out)

    h = 2.0**-7
    (up, size), (down, _) = value(h), value(-h)
    (up2, _), (down2, _) = value(2 * h), value(-2 * h)
    near, far = (up - down) / (2 * h), (up2 - down2) / (4 * h)
    assert (near - along).abs() <= (far - near).abs() + ref.E * size / h * 2


def test_on_another_stream_and_in_a_graph(gpu_device):
    v = inputs(300, 520, 3, torch.bfloat16, 8, gpu_device)
    want = run(v, "post_pre")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(v, "post_pre")
    stream.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(v, "post_pre")
    for seed in range(3):
        v["branch"].copy_(torch.randn(300, 520, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = run(v, "post_pre")
        assert all(torch.equal(got[k], out[k]) for k in got)


def test_empty_and_refusals(gpu_device):
    v = inputs(6, 40, 2, torch.float32, 0, gpu_device)
    empty = {**{k: t[:0] if k in ("residual", "branch", "d_residual", "d_normed") else t for k, t in v.items()}, "gate": None}
    got = run(empty, "post_pre")
    assert got["normed"].shape == (0, 40) and not got["d_post_weight"].any() and not got["d_pre_weight"].any()
    r, y, p, w, g = (v[k] for k in ("residual", "branch", "post_weight", "pre_weight", "gate"))
    for bad, text in [(lambda: d.pre_norm(r.half(), w.half()), "BFloat16 or Float"), (lambda: d.pre_norm(r, w.bfloat16()), "dtype"), (lambda: d.pre_norm(r, w[:39]), "40 elements"),
                      (lambda: d.pre_norm(r, w.cpu()), "on the GPU"), (lambda: d.pre_norm(r[:, :0], w[:0]), "empty"), (lambda: d.post_norm(r, y[:5], p), "shape"),
                      (lambda: d.post_norm(r, y, p, g[:, :8]), "gate"), (lambda: d.post_norm(r, y, p, torch.cat([g, g])), "divide"),
                      (lambda: d.post_pre_norm(r, y, p, w.unsqueeze(0)), "40 elements"), (lambda: d.pre_norm(torch.zeros(1, 32769, device=gpu_device), torch.ones(32769, device=gpu_device)), "32768")]:
        with pytest.raises(RuntimeError, match=text):
            bad()
    leaf = r.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient of its gradient"):
        torch.autograd.grad(d.pre_norm(leaf, w), leaf, r, create_graph=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,gates", [(1100, 9224, 1), (600, 12288, 0), (520, 12290, 520), (530, 16384, 2), (530, 13001, 530), (30, 9000, 30), (2, 12000, 2), (700, 5000, 350)])
def test_long_rows(gpu_device, rows, cols, gates, dtype):
    """several rows a unit, in front of a gate row's end and over it"""
    v = inputs(rows, cols, gates, dtype, rows + cols, gpu_device)
    check(run(v, "post_pre"), reference(v), (rows, cols, gates))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["pre", "post"])
@pytest.mark.parametrize("rows,cols,gates", [(600, 12288, 1), (530, 9001, 530), (520, 16384, 0)])
def test_long_rows_of_one_norm(gpu_device, rows, cols, gates, form, dtype):
    v = inputs(rows, cols, 0 if form == "pre" else gates, dtype, rows + cols, gpu_device, form)
    check(run(v, form), reference(v), (rows, cols, gates, form))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["pre", "post", "post_pre"])
@pytest.mark.parametrize("gate_shape", [None, (40,), (1, 40), (3, 1, 40)])
def test_no_rows_with_a_gate(gpu_device, gate_shape, form, dtype):
    """a rank that is given no tokens: gradients of weights and gate are zero, whatever the memory held that they are made in"""
    if form == "pre" and gate_shape:
        return
    v = inputs(6, 40, 0, dtype, 0, gpu_device, form)
    v = {k: t[:0] if t is not None and t.dim() == 2 else t for k, t in v.items()}
    v["gate"] = torch.ones(gate_shape, dtype=dtype, device=gpu_device) if gate_shape else None
    names = [k for k in ("post_weight", "pre_weight", "gate") if v[k] is not None]
    for _ in range(3):
        held = [torch.full((n,), float("nan"), dtype=dtype, device=gpu_device) for n in (40, 120) for _ in range(8)]
        del held
        got = run(v, form)
        for k in names:
            assert got["d_" + k].shape == v[k].shape and got["d_" + k].eq(0).all(), k


@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, cabi.BF16), (torch.float32, cabi.F32)])
def test_no_rows_through_the_c_interface(gpu_device, dtype, code):
    """zeros in what is not NULL, nothing behind it, no workspace"""
    p, cols, gates = torch.ones(40, dtype=dtype, device=gpu_device), 33, 2
    stream = torch.cuda.current_stream().cuda_stream
    for given in ((1, 1, 1), (1, 0, 1), (0, 1, 0)):
        out = [torch.full((n + 3,), 5.0, dtype=dtype, device=gpu_device) for n in (cols, cols, gates * cols)]
        d_post, d_pre, d_gate = (t.data_ptr() if there else None for t, there in zip(out, given))
        at = p.data_ptr()
        assert cabi.lib().dt_norm_backward(3, at, at, at, at, at, at, at, gates, code, 0, cols, 1.0, None, None, None, None, d_post, d_pre, d_gate, None, 0, stream) == 0
        for t, there in zip(out, given):
            assert (t[:-3] == (0 if there else 5)).all() and (t[-3:] == 5).all()


@pytest.mark.parametrize("rows,cols,gates", [(5, 40, 1), (64, 1001, 2), (300, 520, 0), (700, 256, 350), (9, 4096, 9), (520, 9224, 1), (30, 12290, 30), (40, 16384, 4), (3, 20000, 0)])
def test_bf16_gradients_take_the_new_residual_before_its_rounding(gpu_device, rows, cols, gates):
    """bounds as for fp32 tensors of the same values, which hold no rounding of the new residual, and one rounding of each result"""
    v = inputs(rows, cols, gates, torch.bfloat16, rows * 3 + cols, gpu_device)
    got = run(v, "post_pre")
    want = reference({k: None if t is None else t.float() for k, t in v.items()})
    for k, (value, bound) in want.items():
        ref.assert_within(got[k], value, bound + ref.R * (value.abs() + bound), (k, rows, cols, gates))


def test_gradients_from_the_new_residual(gpu_device):
    """the operator that takes the new residual itself: in fp32 the only form, in bf16 with its rounding"""
    for dtype in DTYPES:
        v = inputs(50, 264, 2, dtype, 3, gpu_device)
        r, n, iy, ir = d.ops.norm_forward(*(v[k] for k in ("residual", "branch", "post_weight", "pre_weight", "gate")), 0.7, EPS, True)
        rest = (v["branch"], v["post_weight"], v["pre_weight"], v["gate"], iy, ir, 0.7)
        names = ("d_residual", "d_branch", "d_post_weight", "d_pre_weight", "d_gate")
        got = dict(zip(names, d.ops.norm_backward(v["d_residual"], v["d_normed"], r, *rest)))
        check(got, {k: t for k, t in reference(v).items() if k in names}, dtype)
    with pytest.raises(RuntimeError, match="from_residual"):
        d.ops.norm_backward(v["d_residual"], v["d_normed"], v["residual"], *rest, True)


def test_saved_tensors_are_the_callers(gpu_device):
    """what the gradients read may not change before they are taken; a bf16 result may"""
    v = inputs(20, 64, 1, torch.bfloat16, 3, gpu_device)
    want = run(v, "post_pre")
    leaves = {**v, **{k: v[k].clone().requires_grad_() for k in ("branch", "post_weight")}}
    out = call(leaves, "post_pre")
    with torch.no_grad():
        out["residual"].zero_()
    got = torch.autograd.grad([out["residual"], out["normed"]], [leaves["branch"]], [v["d_residual"], v["d_normed"]])[0]
    assert torch.equal(got, want["d_branch"])
    out = call(leaves, "post_pre")
    leaves["residual"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([out["residual"], out["normed"]], [leaves["branch"]], [v["d_residual"], v["d_normed"]])


@pytest.mark.parametrize("shape,gate_shape", [((3, 4, 40), (4, 40)), ((3, 4, 40), (1, 4, 40)), ((2, 3, 4, 40), (2, 1, 4, 40)), ((2, 3, 4, 40), (3, 1, 40)), ((2, 3, 4, 40), (3, 4, 40)),
                                              ((2, 3, 4, 40), (4, 40)), ((2, 3, 4, 40), (1, 3, 4, 40))])
def test_a_gate_per_position_is_refused(gpu_device, shape, gate_shape):
    """shapes whose rows broadcasting would give to other rows than equal shares in turn do; expanded they are taken as they are meant"""
    v = inputs(1, 40, 0, torch.float32, 1, gpu_device)
    r, y = (torch.randn(shape, device=gpu_device) for _ in range(2))
    gate = torch.randn(gate_shape, device=gpu_device)
    for bad in (lambda: d.post_norm(r, y, v["post_weight"], gate), lambda: d.post_pre_norm(r, y, v["post_weight"], v["pre_weight"], gate)):
        with pytest.raises(RuntimeError, match="expanded to the residual's shape"):
            bad()
    got = d.post_norm(r, y, v["post_weight"], gate.expand(shape), 0.7, EPS)
    want, bound = ref.norms(r, y, v["post_weight"], None, gate.expand(shape), 0.7, EPS)["residual"]
    ref.assert_within(got, want, bound)


@pytest.mark.parametrize("shape,gate_shape", [((3, 4, 40), (40,)), ((3, 4, 40), (1, 1, 40)), ((3, 4, 40), (3, 40)), ((3, 4, 40), (3, 1, 40)), ((3, 4, 40), (3, 4, 40)), ((4, 4, 40), (4, 40)),
                                              ((3, 4, 40), (12, 40)), ((3, 4, 40), (6, 40)), ((1, 4, 40), (4, 40)), ((3, 1, 40), (3, 40)), ((2, 3, 4, 40), (2, 3, 1, 40)),
                                              ((2, 3, 4, 40), (2, 1, 1, 40)), ((2, 3, 4, 40), (2, 40)), ((1, 3, 4, 40), (3, 1, 40)), ((12, 40), (4, 1, 40)), ((1, 1, 40), (1, 40))])
def test_gates_of_equal_shares(gpu_device, shape, gate_shape):
    """every shape whose meaning is plain, of whatever number of dimensions"""
    v = inputs(1, 40, 0, torch.float32, 1, gpu_device)
    r, y = (torch.randn(shape, device=gpu_device) for _ in range(2))
    gate = torch.randn(gate_shape, device=gpu_device)
    want, bound = ref.norms(r, y, v["post_weight"], None, gate, 0.7, EPS)["residual"]
    ref.assert_within(d.post_norm(r, y, v["post_weight"], gate, 0.7, EPS), want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,gate_shape", [((0, 5, 40), (0, 1, 40)), ((0, 5, 40), (0, 40)), ((0, 5, 40), (0, 5, 40)), ((0, 40), (0, 40)), ((3, 0, 40), (3, 1, 40)), ((3, 0, 40), (3, 0, 40))])
def test_an_empty_batch_with_its_gate(gpu_device, shape, gate_shape, dtype):
    """a gate row per sequence where there are no sequences, or sequences without rows"""
    v = inputs(1, 40, 0, dtype, 1, gpu_device)
    p, w = v["post_weight"].requires_grad_(), v["pre_weight"].requires_grad_()
    r, y = (torch.zeros(shape, dtype=dtype, device=gpu_device, requires_grad=True) for _ in range(2))
    gate = torch.ones(gate_shape, dtype=dtype, device=gpu_device, requires_grad=True)
    new, normed = d.post_pre_norm(r, y, p, w, gate)
    assert new.shape == normed.shape == shape and d.post_norm(r, y, p, gate).shape == shape
    grads = torch.autograd.grad([new, normed], [r, y, p, w, gate], [torch.zeros_like(new), torch.zeros_like(normed)])
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (r, y, p, w, gate)))
    with pytest.raises(RuntimeError, match="gate must have rows"):
        d.post_norm(torch.zeros(2, 40, dtype=dtype, device=gpu_device), torch.zeros(2, 40, dtype=dtype, device=gpu_device), p, torch.zeros(0, 40, dtype=dtype, device=gpu_device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,gates", [(2064, 1000, 129), (1290, 4104, 129), (1530, 2056, 255), (774, 9224, 129), (1608, 520, 201), (2056, 521, 257), (1542, 4096, 257), (900, 12288, 300)])
def test_gate_rows_about_as_many_as_units(gpu_device, rows, cols, gates, dtype):
    """gate rows of several rows each, one unit to a gate row and several gate rows to a unit"""
    v = inputs(rows, cols, gates, dtype, rows + cols, gpu_device)
    check(run(v, "post_pre"), reference(v), (rows, cols, gates))


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_residual_stream_may_be_added_to_in_place(gpu_device, dtype):
    """neither the residual nor the result of a norm behind a block is needed for its gradients"""
    v = inputs(20, 72, 2, dtype, 5, gpu_device, "post")
    want = run(v, "post")
    leaves = {**v, **{k: v[k].clone().requires_grad_() for k in ("branch", "post_weight", "gate")}}
    out = call(leaves, "post")["residual"]
    out += 1
    leaves["residual"].zero_()
    got = torch.autograd.grad(out, [leaves[k] for k in ("branch", "post_weight", "gate")], v["d_residual"])
    assert all(torch.equal(g, want["d_" + k]) for g, k in zip(got, ("branch", "post_weight", "gate")))


def test_offsets_past_32_bits(gpu_device):
    """a row's values and gradients are the same at the end of tensors of more than 2^31 elements as in tensors of that row's neighbours alone"""
    rows, cols = 70000, 32760
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of free device memory")
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device, dtype=torch.bfloat16)  # noqa: E731
    v = {"residual": n(rows, cols), "branch": n(rows, cols), "post_weight": n(cols), "pre_weight": n(cols), "gate": n(2, cols), "d_residual": n(rows, cols), "d_normed": n(rows, cols)}
    got = run(v, "post_pre")
    for part in (slice(0, 40), slice(65560, 65600), slice(rows - 40, rows)):
        alone = {k: t[part] if t.shape[0] == rows else t for k, t in v.items()}
        alone["gate"] = v["gate"][0 if part.stop <= rows // 2 else 1]
        want = run(alone, "post_pre")
        assert all(torch.equal(got[k][part], want[k]) for k in ("residual", "normed", "d_residual", "d_branch"))
