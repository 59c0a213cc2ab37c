"""GPU tests of the 8-bit linear path: each kernel form at sizes that reach it.

Tolerances count roundings as in test_gpu_blocks.py (u = 2^-24).  For rows on the
16-byte grid: a square's own rounding and 7 additions in its vector, 2 over a thread's
vectors, 5 over a warp and 5 over a block's warps, 20, of which the square root passes
half; the division by the row's length and epsilon's addition, halved too, the square
root, the reciprocal and two products add 5: 15 u, without a residual.  x + residual is a
rounding of its own in every element and, twice, in every square: 2 u more."""
import pytest
import torch

import test_gpu_blocks as tb

pytestmark = pytest.mark.gpu
U, TYPES = tb.U, tb.TYPES


@pytest.fixture(scope="module")
def ctx(ob, handle):
    return ob.ExecutionContext(handle)


def check_norm(out, x, r, w, eps, quantize):
    h, y = tb.norm_ref(x, r, w, eps)
    t, cols = x.dtype, x.shape[-1]
    slack = (15 + 2 * (r is not None)) * U * (1 + 2 ** -10)
    if r is not None:
        assert ((out[-1].double() - h).abs() <= h.abs() * (tb.half(t) + U) * (1 + U) + tb.TINY[t]).all()
    if quantize:
        tb.check_quantized(out[0].reshape(-1, cols), out[1].reshape(-1, out[1].shape[-1]), y.reshape(-1, cols), 1, slack)
    else:
        off = (out[0].double() - y).abs()
        assert (off <= y.abs() * (tb.half(t) + slack) * (1 + tb.half(t)) + tb.TINY[t]).all(), (off / y.abs() / U).max()


@pytest.mark.parametrize("cols", [520, 768, 1024, 2056, 4096])
@pytest.mark.parametrize("eps", [0.0, 1e-5])
def test_norm_of_one_large_and_many_small_elements(ob, ctx, cols, eps):
    """Squares just below half a step of the row's largest: added to it one by one all are lost."""
    rows = 4096
    x = torch.full((rows, cols), 2.0 ** -12 * 0.999 ** 0.5, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(cols)
    x[:, 0] = 1 + 2.0 ** -5 * torch.rand(rows, generator=g, device="cuda")
    w = 1 + torch.rand(cols, generator=g, device="cuda")
    check_norm(ob.RMSNormalization(epsilon=eps).compute([x, w], ctx), x, None, w, eps, False)


def check_mm(y, a, sa, b, sb, bias, relu, t):
    """As in test_gpu_blocks.py, and past the type's range: from half a step above the largest value,
    top = (2 - eps / 2) 2^e with max = (2 - eps) 2^e (fp16: 65504 and 65520), the nearest is infinity.  1800 x
    5003 x 400 has one such output, 88643."""
    ref, mag = tb.mm_ref(a, sa, b, sb, bias, relu)
    sums = mag * (128 * 2 * U + (-(-a.shape[1] // 128) + 4) * U)
    assert y.dtype == t and y.shape == ref.shape
    f, v = torch.finfo(t), y.double()
    top = f.max + f.eps / 2 * f.max / (2 - f.eps)
    ok = (v - ref).abs() <= sums + (ref.abs() + sums) * tb.half(t) + tb.TINY[t]
    ok |= (ref.abs() + sums >= top) & (v == torch.copysign(torch.full_like(ref, float("inf")), ref))
    assert ok.all(), ((v - ref).abs() / (sums + ref.abs() * tb.half(t)))[~ok].max()


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(300, 512), (300, 520), (300, 1000), (300, 1032), (300, 2056), (300, 4096), (300, 8200),
                                       (297, 16384)])
def test_norm_with_rows_that_fill_the_gpu(ob, ctx, rows, cols, t, residual, quantize):
    """More rows than twice the SMs, on the grid: one to four vectors a thread, a row per warp up to 1024
    columns and per thread block above."""
    x = tb.normal((rows, cols), rows + cols, t)
    r = 3 * tb.normal((rows, cols), 7, t) if residual else None
    w = (1 + 0.3 * tb.normal((cols,), 9)).to(t)
    out = ob.RMSNormalization(epsilon=1e-5, quantize=quantize).compute([x, w], ctx, residual=r)
    check_norm(out, x, r, w, 1e-5, quantize)


# Which of these take tiles of 256 x 256 is checked in test_blocks_rules.py; the others take 256 x 128, all of
# them several for a pair of thread blocks, ragged in every direction.
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(1777, 5000, 300), (2300, 4700, 1100), (1800, 5003, 400), (1500, 6700, 128), (700, 6400, 1100),
                                   (600, 6404, 97)])
def test_product_with_many_tiles(ob, ctx, m, n, k, t):
    a, sa, b, sb = tb.operands(m, n, k, m + n)
    for bias, relu in ((tb.normal((n,), 3), True), (None, False)):
        y = ob.MatMulBlockScaled(t, relu=relu).compute([a, sa, b, sb, bias], ctx)[0]
        check_mm(y, a, sa, b, sb, bias, relu, t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n", [(1800, 5003), (700, 6401)])
def test_product_with_many_tiles_inside_a_larger_y(handle, m, n, t):
    """On and off the 16-byte grid, with bias: nothing but the m x n outputs is written."""
    k = 400
    a, sa, b, sb = tb.operands(m, n, k, 9)
    bias = tb.normal((n,), 4)
    for off, width in ((8, n + 24 - n % 8), (1, n + 24 - n % 8), (0, n + 2)):
        y = torch.full((m + 2, width), 3.0, dtype=t, device="cuda")
        inner = y[1:-1, off:off + n]
        tb.run_mm(handle, a, sa, b, sb, bias, inner, relu=True)
        check_mm(inner, a, sa, b, sb, bias, True, t)
        rest = y.clone()
        rest[1:-1, off:off + n] = 3.0
        assert (rest == 3.0).all()


@pytest.mark.parametrize("m,n,k", [(1777, 5000, 640), (700, 6400, 640)])
def test_product_with_many_tiles_whole_numbers(ob, ctx, m, n, k):
    """Whole numbers up to 15 and scales of powers of two: every sum is below 2^24 / 4, exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(m)
    a = torch.randint(-15, 16, (m, k), generator=g, device="cuda").float().to(tb.E4M3)
    b = torch.randint(-15, 16, (n, k), generator=g, device="cuda").float().to(tb.E4M3)
    sa = torch.exp2(torch.randint(-1, 2, (m, k // 128), generator=g, device="cuda").float())
    sb = torch.exp2(torch.randint(-1, 2, (-(-n // 128), k // 128), generator=g, device="cuda").float())
    ref, _ = tb.mm_ref(a, sa, b, sb, None, False)
    op = ob.MatMulBlockScaled()
    y = op.compute([a, sa, b, sb], ctx)[0]
    assert torch.equal(y.double(), ref)
    assert torch.equal(op.compute([a, sa, b, sb], ctx)[0], y)


@pytest.mark.parametrize("m,n", [(1777, 5000), (700, 6400)])
def test_product_with_many_tiles_nan_stays_in_its_row_and_column(ob, ctx, m, n):
    k = 384
    a, sa, b, sb = tb.operands(m, n, k, 5)
    ref = ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0]
    for row, col in ((m - 1, n - 1), (300, 250), (0, n // 2)):
        sa2, b2 = sa.clone(), b.clone()
        sa2[row, 1] = float("nan")
        b2.view(torch.uint8)[col, 130] = 0x7F
        for relu in (False, True):
            y = ob.MatMulBlockScaled(relu=relu).compute([a, sa2, b2, sb], ctx)[0]
            assert torch.isnan(y[row]).all() and torch.isnan(y[:, col]).all()
            y, want = y.clone(), ref.clamp(min=0) if relu else ref.clone()
            y[row], want[row] = 0, 0
            y[:, col], want[:, col] = 0, 0
            assert torch.equal(y, want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(256, 512, 2560), (100, 1000, 2048), (200, 1004, 3700), (129, 2565, 3700)])
def test_product_with_shared_tiles(handle, m, n, k, t):
    """Tiles shared by two or four pairs of thread blocks, in every type: 16 bytes of y at a time where its
    rows are on the grid, the last columns and other rows by elements, and nothing beside them."""
    a, sa, b, sb = tb.operands(m, n, k, m + n)
    bias = tb.normal((n,), 3)
    for off, width in ((8, n + 24 - n % 8), (1, n + 24 - n % 8), (0, n + 1)):
        y = torch.full((m + 2, width), 3.0, dtype=t, device="cuda")
        inner = y[1:-1, off:off + n]
        tb.run_mm(handle, a, sa, b, sb, bias, inner, relu=True)
        check_mm(inner, a, sa, b, sb, bias, True, t)
        rest = y.clone()
        rest[1:-1, off:off + n] = 3.0
        assert (rest == 3.0).all()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(3, 256), (400, 256), (400, 1000), (300, 2056), (2, 4096), (3, 1001), (3, 3001), (3, 6001),
                                       (2, 20000)])
def test_norm_of_a_node_has_the_type_of_its_scale(ob, ctx, rows, cols, t, wt, residual):
    """As ONNX defines it: y in the scale's type, rounded once; x + residual stays in x's.  The longest chain
    of roundings is a row's of 20000 columns in shared memory: a square's and 40 additions in a thread, 5 over
    its warp, 16 over the warps, of which the root passes half, and 7 as on the grid: 38 u."""
    node = {"op": "RMSNormalization", "inputs": ["x", "w"], "outputs": ["y"], "attrs": {"epsilon": 1e-5}}
    op = ob.OperatorRegistry.initialize_standard_operators().create_operator_for_node(node, opset=23)
    x = tb.normal((rows, cols), rows + cols, t)
    r = 3 * tb.normal((rows, cols), 7, t) if residual else None
    w = (1 + 0.3 * tb.normal((cols,), 9)).to(wt)
    out = op.compute([x, w], ctx, residual=r)
    h, y = tb.norm_ref(x, r, w, 1e-5)
    assert out[0].dtype == wt and out[0].shape == x.shape
    slack = 38 * U * (1 + 2 ** -10)
    assert ((out[0].double() - y).abs() <= y.abs() * (tb.half(wt) + slack) * (1 + tb.half(wt)) + tb.TINY[wt]).all()
    if residual:
        assert out[1].dtype == t and ((out[1].double() - h).abs() <= h.abs() * (tb.half(t) + U) * (1 + U) + tb.TINY[t]).all()


@pytest.mark.parametrize("cols", [256, 1001, 6001])
def test_norm_into_the_type_of_the_weight_writes_nothing_else(handle, cols):
    """fp32 rows of y inside a larger matrix, x in bf16."""
    x, w = tb.normal((5, cols), 1, torch.bfloat16), tb.normal((cols,), 2)
    for off in (4, 1):
        y = torch.full((7, cols + 16 - cols % 8), 3.0, device="cuda")
        inner = y[1:-1, off:off + cols]
        tb.run_norm(handle, x, None, w, None, inner, None)
        ref = tb.norm_ref(x, None, w, 1e-5)[1]
        assert ((inner.double() - ref).abs() <= ref.abs() * 39 * U * (1 + 2 ** -10)).all()
        rest = y.clone()
        rest[1:-1, off:off + cols] = 3.0
        assert (rest == 3.0).all()


@pytest.mark.parametrize("cols", [256, 1001, 6001])
def test_norm_past_the_range_of_its_sum(ob, ctx, cols):
    """A finite row whose sum of squares passes fp32's range gives zeros; with epsilon 0 one whose squares
    vanish gives values that are not finite.  Each row by itself."""
    x, w = tb.normal((4, cols), 1), tb.normal((cols,), 2)
    x[1] *= 1e25
    x[2] = 1e-30
    y = ob.RMSNormalization(epsilon=0.0).compute([x, w], ctx)[0]
    assert (y[1] == 0).all() and not torch.isfinite(y[2]).any()
    ref = tb.norm_ref(x[[0, 3]], None, w, 0.0)[1]
    assert ((y[[0, 3]].double() - ref).abs() <= ref.abs() * 39 * U * (1 + 2 ** -10)).all()
