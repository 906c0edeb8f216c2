"""8-bit integer quantization against its definition in 32 bits, bit for bit, and the scaled product of 8-bit integers
against 64 bits: |error| <= |y| (2^-8 for the rounding to bf16 + 4 * 2^-24 for the sum's conversion and both scales)."""
import pytest
import torch

import driss_torch as d
from driss_torch_amd import cabi
from feed_forward_reference import R, assert_within

pytestmark = pytest.mark.gpu


def quantized(x):
    """(q, scale) on the CPU, by the definition"""
    x = x.cpu().float()
    bits = x.view(torch.int32) & 0x7FFFFFFF  # NaN above infinity
    amax = bits.amax(dim=1, keepdim=True).view(torch.float32)
    c = torch.where(amax < 1e-12, torch.full_like(amax, 1e-12), amax)
    top = torch.full_like(c, 127.0)
    q = torch.round(x * (top / c))
    q = torch.where(torch.isfinite(amax), q, torch.zeros_like(q))
    return q.to(torch.int8), c / top


def check_quantize(x):
    q, scale = d.int8_quantize(x)
    want, ws = quantized(x)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == (x.shape[0], 1)
    assert torch.equal(q.cpu(), want)
    assert torch.equal(scale.cpu().view(torch.int32), ws.view(torch.int32)) or torch.equal(scale.cpu().nan_to_num(-1.0, -2.0, -3.0), ws.nan_to_num(-1.0, -2.0, -3.0))


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 63), (4, 64), (2, 511), (7, 512), (65, 513), (3, 1001), (2, 2048), (9, 2049), (2, 4104), (1, 8192), (5, 8190), (2, 16384), (3, 20001),
          (1, 33000), (1, 70001), (1, 140000), (1000, 130)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_shapes(gpu_device, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 7919 + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(4 * torch.randn(rows, 1, generator=g))
    check_quantize(x.to(dtype).to(gpu_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [40, 1003, 9000])
def test_quantize_special_rows(gpu_device, cols, dtype):
    """zero rows, tiny rows, rows of one value, ties, infinities and NaN: nothing leaves its row"""
    x = torch.randn(9, cols, generator=torch.Generator().manual_seed(cols))
    x[1] = 0
    x[2] *= 1e-30
    x[3] = 5.0
    x[4] = torch.arange(cols) % 128 - 0.5  # ties at a scale of one, where bf16 has them
    x[4, 0] = 127.0
    x[5, cols // 2] = float("inf")
    x[6, cols - 1] = float("nan")
    x[7, 0] = -float("inf")
    x[8] *= 1e30
    check_quantize(x.to(dtype).to(gpu_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_off_alignment(gpu_device, dtype):
    flat = torch.randn(3 * 520 + 8, generator=torch.Generator().manual_seed(3)).to(dtype).to(gpu_device)
    for skip in (0, 1, 3, 4, 8):
        check_quantize(flat[skip:skip + 3 * 520].view(3, 520))


def operands(m, n, k, seed, device):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    sa, sb = torch.rand(m, 1, generator=g) + 0.01, torch.rand(n, 1, generator=g) + 0.01
    return a.to(device), b.to(device), sa.to(device), sb.to(device)


def check_product(a, b, sa, sb, out=None):
    y = d.int8_bf16(a, b.t(), sa, sb) if out is None else out
    want = (a.cpu().double() @ b.cpu().double().t()) * sa.cpu().double().reshape(-1, 1) * sb.cpu().double().reshape(1, -1)
    assert y.dtype == torch.bfloat16
    assert_within(y, want, want.abs() * (R + 4 * 2.0**-24), (tuple(a.shape), tuple(b.shape)))


# one token to many, sizes on and off 16 bytes, a step of K, a tile; few and many tiles of each kind
PRODUCTS = [(1, 1, 1), (1, 8, 16), (1, 64, 128), (3, 5, 7), (1, 1000, 4096), (2, 257, 1000), (7, 640, 136), (15, 512, 2048), (16, 513, 2049), (17, 96, 4104), (31, 1024, 1024),
            (32, 100, 5000), (33, 200, 512), (48, 1111, 640), (64, 64, 64), (65, 130, 129), (100, 300, 1024), (128, 128, 1024), (129, 1000, 1040), (197, 1433, 1032), (255, 257, 255),
            (256, 256, 256), (257, 511, 4096), (300, 2000, 130), (512, 1024, 128), (700, 768, 1), (1000, 1000, 1000), (1024, 1280, 16), (2048, 520, 272), (2051, 1029, 1021), (1, 500, 4), (8, 77, 1036), (30, 300, 5132), (40, 64, 20), (90, 200, 1044), (260, 300, 4108)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_sizes(gpu_device, m, n, k):
    check_product(*operands(m, n, k, m * 31 + n * 7 + k, gpu_device))


@pytest.fixture
def tiles(request):
    """the tiles and shares of K of products of more than 32 rows, as given"""
    cabi.set_tuning("mm.tiles", request.param[0])
    cabi.set_tuning("mm.splits", request.param[1])
    yield request.param
    cabi.set_tuning("mm.tiles", 0)
    cabi.set_tuning("mm.splits", 0)


@pytest.mark.parametrize("tiles", [(1, 0), (2, 1), (2, 2), (2, 5), (3, 1), (3, 3), (3, 16), (4, 1), (4, 3)], indirect=True)
@pytest.mark.parametrize("m,n,k", [(33, 1, 16), (64, 300, 2000), (200, 129, 640), (129, 520, 4104), (513, 257, 127), (300, 1000, 1300)])
def test_product_tiles(gpu_device, m, n, k, tiles):
    check_product(*operands(m, n, k, m + n + k, gpu_device))


@pytest.mark.parametrize("m", [1, 9, 40, 130, 600])
def test_product_extreme_sums(gpu_device, m):
    """-128 in both operands at the largest K: the sum's largest magnitude fits 32 bits"""
    k = (1 << 17) - 1
    a = torch.full((m, k), -128, dtype=torch.int8, device=gpu_device)
    b = torch.full((24, k), -128, dtype=torch.int8, device=gpu_device)
    b[1::2] = 127
    check_product(a, b, torch.ones(m, 1, device=gpu_device), torch.ones(24, 1, device=gpu_device))


@pytest.mark.parametrize("m", [1, 20, 70, 300])
@pytest.mark.parametrize("k,lda,ldb,skip", [(256, 272, 288, 0), (256, 257, 256, 0), (100, 128, 4096, 0), (512, 512, 512, 3), (520, 700, 701, 16)])
def test_product_strides(gpu_device, m, k, lda, ldb, skip):
    """rows further apart than K and bases off 16 bytes; what lies between the rows does not count"""
    n = 150
    a, b, sa, sb = operands(m, n, k, m + k, gpu_device)
    wa = torch.full((skip + m * lda,), 101, dtype=torch.int8, device=gpu_device)
    wb = torch.full((skip + n * ldb,), -77, dtype=torch.int8, device=gpu_device)
    va, vb = wa[skip:].view(m, lda)[:, :k], wb[skip:].view(n, ldb)[:, :k]
    va.copy_(a)
    vb.copy_(b)
    check_product(va, vb, sa, sb)


def test_product_empty(gpu_device):
    a, b, sa, sb = operands(4, 8, 16, 0, gpu_device)
    assert d.int8_bf16(a[:0], b.t(), sa[:0], sb).shape == (0, 8)
    assert d.int8_bf16(a, b[:0].t(), sa, sb[:0]).shape == (4, 0)
    assert torch.equal(d.int8_bf16(a[:, :0], b[:, :0].t(), sa, sb).cpu(), torch.zeros(4, 8, dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [1, 40, 200])
def test_product_scales_that_are_not_finite(gpu_device, m):
    """a NaN or infinite scale stays in its row or column"""
    a, b, sa, sb = operands(m + 2, 72, 512, 5, gpu_device)
    sa[1] = float("nan")
    sb[3] = float("inf")
    y = d.int8_bf16(a, b.t(), sa, sb).cpu()
    assert y[1].isnan().all()
    ok = torch.ones_like(y, dtype=torch.bool)
    ok[1] = False
    ok[:, 3] = False
    assert y[ok].isfinite().all() and not y[0, 3].isfinite()


def test_product_rows_do_not_depend_on_their_neighbours(gpu_device):
    """the sums are exact, so the same row gives the same bits whatever kernel the number of rows selects"""
    a, b, sa, sb = operands(700, 520, 1024, 11, gpu_device)
    y = d.int8_bf16(a, b.t(), sa, sb)
    for m in (1, 5, 16, 33, 64, 65, 130, 257):
        assert torch.equal(d.int8_bf16(a[:m], b.t(), sa[:m], sb), y[:m])


def test_product_wide_operand(gpu_device):
    """offsets past 32 bits: rows of b that lie 40 MB apart"""
    n, k, ldb = 200, 256, 40_000_000
    wide = torch.empty(n * ldb, dtype=torch.int8, device=gpu_device)
    a, b, sa, sb = operands(70, n, k, 2, gpu_device)
    v = torch.as_strided(wide, (n, k), (ldb, 1))
    v.copy_(b)
    for m in (1, 70):
        check_product(a[:m], v, sa[:m], sb)


def test_on_another_stream_and_in_a_graph(gpu_device):
    x = torch.randn(40, 1024, device=gpu_device, dtype=torch.bfloat16)
    w = torch.randn(300, 1024, device=gpu_device, dtype=torch.bfloat16)
    wq, ws = d.int8_quantize(w)

    def step(v):
        q, s = d.int8_quantize(v)
        return q, s, d.int8_bf16(q, wq.t(), s, ws)

    want = [t.clone() for t in step(x)]
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
    for seed in range(4):
        static.copy_(torch.randn(40, 1024, generator=torch.Generator().manual_seed(seed)).to(static.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(step(static), out))


def test_refusals(gpu_device):
    a, b, sa, sb = operands(4, 8, 32, 0, gpu_device)
    x = torch.randn(4, 32, device=gpu_device)
    for bad, text in [(lambda: d.int8_quantize(x.half()), "BFloat16 or Float"), (lambda: d.int8_quantize(x[0]), "2D"), (lambda: d.int8_quantize(x.t()), "contiguous"),
                      (lambda: d.int8_quantize(x[:, :0]), "empty rows"), (lambda: d.int8_bf16(a, b, sa, sb), "Incompatible"), (lambda: d.int8_bf16(a.float(), b.t(), sa, sb), "int8"),
                      (lambda: d.int8_bf16(a, b.t().contiguous(), sa, sb), "contiguous in the K"), (lambda: d.int8_bf16(a.t().contiguous().t(), b.t(), sa, sb), "contiguous in the K"),
                      (lambda: d.int8_bf16(a, b.t(), sa[:3], sb), "a_scale"), (lambda: d.int8_bf16(a, b.t(), sa, sb.double()), "float32"), (lambda: d.int8_bf16(a[0], b.t(), sa, sb), "matrix"),
                      (lambda: d.int8_bf16(a, b.t(), sa.cpu(), sb), "on the GPU"), (lambda: d.int8_bf16(a[:1].expand(4, 32), b.t(), sa, sb), "overlap"),
                      (lambda: d.int8_bf16(torch.zeros(1, 1 << 17, dtype=torch.int8, device=gpu_device), torch.zeros(8, 1 << 17, dtype=torch.int8, device=gpu_device).t(), sa[:1], sb),
                       "131072")]:
        with pytest.raises(RuntimeError, match=text):
            bad()


@pytest.mark.parametrize("m,n,k", [(4011, 4442, 1659), (2677, 3136, 2984), (4449, 2640, 2164)])
def test_product_of_two_launches(gpu_device, m, n, k):
    """more tiles than CUs: whole rounds of large ones and the columns behind them in smaller ones, with and without shares of K and copies"""
    check_product(*operands(m, n, k, m, gpu_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", range(1, 18))
def test_quantize_narrow_rows(gpu_device, cols, dtype):
    """rows that begin and end inside one vector, and those just longer: each has a scale and codes of its own"""
    g = torch.Generator().manual_seed(cols)
    for rows in (2, 3, 64, 1031):
        check_quantize((torch.randn(rows, cols, generator=g) * torch.exp(4 * torch.randn(rows, 1, generator=g))).to(dtype).to(gpu_device))


@pytest.mark.parametrize("cols", [1, 3, 7])
def test_quantize_narrow_rows_write_nothing_else(gpu_device, cols):
    """codes and scales between words of a pattern, which stay; a row that is not finite leaves its neighbours alone"""
    rows = 37
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(cols))
    x[5, cols - 1], x[20, 0] = float("nan"), float("inf")
    want, scale = quantized(x)
    x = x.to(gpu_device)
    q = torch.full((64 + rows * cols + 64,), 85, dtype=torch.int8, device=gpu_device)
    s = torch.full((16 + rows + 16,), 7.0, device=gpu_device)
    stream = torch.cuda.current_stream().cuda_stream
    assert cabi.lib().dt_int8_quantize(x.data_ptr(), cabi.F32, rows, cols, q.data_ptr() + 64, s.data_ptr() + 64, stream) == 0
    q, s = q.cpu(), s.cpu()
    assert torch.equal(q[64:-64].view(rows, cols), want) and torch.equal(s[16:-16].nan_to_num(-1.0, -2.0).view(rows, 1), scale.nan_to_num(-1.0, -2.0))
    assert (q[:64] == 85).all() and (q[-64:] == 85).all() and (s[:16] == 7).all() and (s[-16:] == 7).all()


@pytest.mark.parametrize("rows,cols,dtype", [((1 << 26) + 5, 8, torch.bfloat16), ((1 << 24) + 3, 3, torch.float32), ((1 << 21) + 9, 1030, torch.bfloat16)])
def test_quantize_many_rows(gpu_device, rows, cols, dtype):
    """more rows than one launch has threads for, and tensors of more than 2^31 elements: 1021 rows over and over"""
    period = 1021
    g = torch.Generator().manual_seed(cols)
    block = (torch.randn(period, cols, generator=g) * torch.exp(4 * torch.randn(period, 1, generator=g))).to(dtype)
    x = torch.empty(rows, cols, dtype=dtype, device=gpu_device)
    whole = rows // period * period
    x[:whole].view(-1, period, cols).copy_(block.to(gpu_device))
    x[whole:] = block[:rows - whole].to(gpu_device)
    q, scale = d.int8_quantize(x)
    want, ws = (t.to(gpu_device) for t in quantized(block))
    for got, of in ((q, want), (scale, ws)):
        assert bool((got[:whole].view(-1, period, of.shape[1]) == of).all()) and torch.equal(got[whole:], of[:rows - whole])


# at most 32 rows and more groups of columns than CUs: a workgroup takes several in turn, with rows of whole words and off them, one and two tiles of rows
@pytest.mark.parametrize("m,n,k", [(1, 20000, 512), (1, 66000, 128), (8, 33001, 260), (12, 20000, 1040), (20, 20001, 640), (32, 40000, 132), (5, 9000, 257), (1, 20011, 1001), (16, 8500, 130),
                                   (24, 9000, 257), (32, 17003, 513), (24, 4000, 333)])
def test_product_of_few_rows_and_many_columns(gpu_device, m, n, k):
    check_product(*operands(m, n, k, m + n + k, gpu_device))


def test_product_offsets_past_32_bits(gpu_device):
    """results past element 2^31, and more than 2^32 bytes of either operand; a row's result is the same in a product of fewer"""
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GiB of free device memory")
    for m, n, k in ((70001, 32760, 64), (70001, 300, 65536), (300, 70001, 65536), (20, 70001, 65536)):
        a, b = (torch.randint(-127, 128, (r, k), dtype=torch.int8, device=gpu_device) for r in (m, n))
        sa, sb = (torch.rand(r, 1, device=gpu_device) + 0.01 for r in (m, n))
        y = d.int8_bf16(a, b.t(), sa, sb)
        for rows in (slice(0, 17), slice(m - 17, m)):
            for columns in (slice(0, 40), slice(n - 40, n)):
                check_product(a[rows], b[columns], sa[rows], sb[columns], y[rows, columns])
        del a, b, y
