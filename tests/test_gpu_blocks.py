"""GPU tests of the 8-bit linear path against plain forms in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, h(t) half a step
of the output's type relative to the value (torch.finfo(t).eps / 2: bf16 2^-8).

rmsnorm: h = x + r is one rounding; the sum of squares adds at most ceil(cols /
256) + 16 roundings in a row, of which the square root passes half; division,
square root, reciprocal and two products add 5 more; then the output's rounding.

matmul: the products of two e4m3 numbers are exact; a block's sum is at most 128
additions of at most one fp32 step (2 u) each, however the tensor cores order or
cut them; the scales' product, the scaled addition (one per block) and the bias
add u each; then the output's rounding.
"""
import ctypes
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

C = importlib.import_module("onnx-rs_b200")._capi
E4M3 = torch.float8_e4m3fn
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, E4M3: 3}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step at zero


def half(t):
    return torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def ctx(ob, handle):
    return ob.ExecutionContext(handle)


def normal(shape, seed, t=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(t)


def e4m3_step(v):
    """Distance of neighbouring e4m3 values at |v| (float64)."""
    e = torch.frexp(v.abs())[1].clamp(min=-5) - 1
    return torch.ldexp(torch.ones_like(v), e - 3)


def block_view(x, rows, value=0.0):
    """[row blocks, rows, column blocks, 128] of a matrix, filled up with `value`."""
    r, c = x.shape
    rb, cb = -(-r // rows), -(-c // 128)
    v = torch.full((rb * rows, cb * 128), value, dtype=x.dtype, device=x.device)
    v[:r, :c] = x
    return v.view(rb, rows, cb, 128)


def by_element(s, shape, rows):
    """Scales [row blocks, column blocks] at every element of `shape`."""
    return s.repeat_interleave(rows, 0)[:shape[0]].repeat_interleave(128, 1)[:, :shape[1]]


def check_quantized(q, s, x64, rows, slack):
    """q, s against float64 values: the scale is amax / 448, each q the nearest value (half a step) of x * 448 / amax.
    `slack`: relative error of the values that were quantised."""
    amax = block_view(x64.abs(), rows).amax((1, 3)).clamp(min=2.0 ** -96)
    assert s.shape == amax.shape and s.dtype == torch.float32
    assert ((s.double() - amax / 448).abs() <= amax / 448 * (slack + 2 * U)).all()
    want = x64 * 448 / by_element(amax, x64.shape, rows)
    got = q.double()
    assert got.shape == want.shape and torch.isfinite(got).all() and (got.abs() <= 448).all()
    # half a step, of the larger of the two neighbours' steps, and the values' own error (the amax's too)
    off = (got - want).abs() - e4m3_step(torch.maximum(got.abs(), want.abs())) / 2
    assert (off <= want.abs() * (2 * slack + 4 * U)).all(), off.max()


def exact_quantize(x, rows):
    """The defining formula in fp32, bit by bit, on the CPU."""
    x = x.float().cpu()
    amax = block_view(x.abs(), rows).amax((1, 3)).clamp(min=2.0 ** -96)
    inv = torch.tensor(448.0) / amax
    q = (x * by_element(inv, x.shape, rows)).clamp(-448, 448).to(E4M3)
    return q, amax / 448


# --------------------------------------------------------------------------- norm
def norm_ref(x, r, w, eps):
    h = x.double() if r is None else x.double() + r.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
    return h, y


def norm_slack(cols):
    return ((cols + 255) // 256 / 2 + 8 + 6) * U


def check_norm(out, x, r, w, eps, quantize):
    h, y = norm_ref(x, r, w, eps)
    t = x.dtype
    if r is not None:
        s = out[-1]
        assert s.dtype == t and s.shape == x.shape
        # x + r in fp32, then in t: two roundings
        assert ((s.double() - h).abs() <= h.abs() * (half(t) + U) * (1 + U) + TINY[t]).all()
    cols = x.shape[-1]
    slack = norm_slack(cols)
    if quantize:
        check_quantized(out[0].reshape(-1, cols), out[1].reshape(-1, out[1].shape[-1]), y.reshape(-1, cols), 1, slack)
    else:
        assert out[0].dtype == t and out[0].shape == x.shape
        off = (out[0].double() - y).abs()
        assert (off <= y.abs() * (half(t) + slack) * (1 + half(t)) + TINY[t]).all(), off.max()


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 128), (2, 130), (17, 768), (1, 4096), (4, 1000), (3, 5001),
                                       (2, 8192), (3, 12296), (2, 16384), (1, 20000), (2, 49152), (300, 64), (1025, 256)])
def test_rmsnorm(ob, ctx, rows, cols, t, residual, quantize):
    x = normal((rows, cols), rows + cols, t)
    r = 3 * normal((rows, cols), 7, t) if residual else None
    w = (1 + 0.3 * normal((cols,), 9)).to(t)
    out = ob.RMSNormalization(epsilon=1e-5, quantize=quantize).compute([x, w], ctx, residual=r)
    assert len(out) == 1 + quantize + residual
    check_norm(out, x, r, w, 1e-5, quantize)


@pytest.mark.parametrize("wt", TYPES)
def test_rmsnorm_weight_type_leading_dims_and_row_strides(ob, ctx, wt):
    big = normal((2, 5, 800), 3, torch.bfloat16)
    x = big[:, :, :512]
    assert not x.is_contiguous()
    r = normal((2, 5, 520), 4, torch.bfloat16)[:, :, :512]
    w = normal((512,), 5, wt)
    for quantize in (False, True):
        out = ob.RMSNormalization(quantize=quantize).compute([x, w], ctx, residual=r)
        check_norm(out, x, r, w, 1e-5, quantize)
        if quantize:
            assert out[0].shape == (2, 5, 512) and out[1].shape == (2, 5, 4)
    one = ob.RMSNormalization(quantize=True).compute([x[0, 0], w], ctx)
    assert one[0].shape == (512,) and one[1].shape == (4,)


@pytest.mark.parametrize("t", TYPES)
def test_rmsnorm_extreme_values(ob, ctx, t):
    """Zero rows, huge and tiny values, infinities and NaN: each row by itself."""
    cols = 384
    x = normal((7, cols), 1, t)
    big = 1e4 if t == torch.float16 else 1e15
    x[1] = 0
    x[2] *= big
    x[3] *= 1 / big
    x[4, 5] = float("inf")
    x[5, 300] = float("nan")
    w = torch.ones(cols, dtype=t, device="cuda")
    y = ob.RMSNormalization().compute([x, w], ctx)[0]
    assert (y[1] == 0).all()
    assert torch.isnan(y[4, 5]) and (y[4, :5] == 0).all() and torch.isnan(y[5]).all()
    keep = [0, 1, 2, 3, 6]
    check_norm([y[keep]], x[keep], None, w, 1e-5, False)
    q, s = ob.RMSNormalization(quantize=True).compute([x, w], ctx)
    check_quantized(q[keep], s[keep], norm_ref(x[keep], None, w, 1e-5)[1], 1, norm_slack(cols))
    assert (q[1].float() == 0).all() and torch.isfinite(s[1]).all()
    assert not torch.isfinite(s[4, 0]) and torch.isfinite(s[4, 1:]).all() and not torch.isfinite(s[5]).any()


def run_norm(handle, x, r, w, s, y, ys, **kw):
    d = C.RmsNormDesc(rows=x.shape[0], cols=x.shape[1], ldx=x.stride(0), ldr=r.stride(0) if r is not None else 0,
                      lds=s.stride(0) if s is not None else 0, ldy=y.stride(0), type=CODE[x.dtype],
                      weight_type=CODE[w.dtype], out_type=CODE[y.dtype], epsilon=1e-5)
    if ys is not None:
        d.y_scale_row, d.y_scale_block = ys.stride()
    p = [None if v is None else v.data_ptr() for v in (x, r, w, s, y, ys)]
    handle.check(C.lib().onnxb200_rmsnorm(handle.ptr, ctypes.byref(d), *p), "rmsnorm")
    handle.synchronize()


@pytest.mark.parametrize("cols", [256, 1001, 6000, 40000])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_rmsnorm_in_place_and_bounds(handle, cols, t):
    """sum over residual and y over x, and nothing written outside rows, columns and scales."""
    rows, pad = 5, 16
    x = normal((rows + 2, cols + pad), 1, t)
    r = normal((rows + 2, cols + pad), 2, t)
    w = normal((cols,), 3, t)
    x0, r0 = x.clone(), r.clone()
    xi, ri = x[1:-1, 8:-8], r[1:-1, 8:-8]
    run_norm(handle, xi, ri, w, ri, xi, None)
    check_norm([x[1:-1, 8:-8], r[1:-1, 8:-8]], x0[1:-1, 8:-8], r0[1:-1, 8:-8], w, 1e-5, False)
    q = torch.full((rows + 2, cols + pad), 0x55, dtype=torch.uint8, device="cuda")
    blocks = -(-cols // 128)
    ys = torch.full((blocks + 2, rows + 2), 77.0, device="cuda")
    run_norm(handle, x0[1:-1, 8:-8], r0[1:-1, 8:-8], w, None, q.view(E4M3)[1:-1, 8:-8], ys[1:-1, 1:-1].t())
    _, y = norm_ref(x0[1:-1, 8:-8], r0[1:-1, 8:-8], w, 1e-5)
    check_quantized(q.view(E4M3)[1:-1, 8:-8], ys[1:-1, 1:-1].t(), y, 1, norm_slack(cols))
    for v, v0 in ((x, x0), (r, r0), (q, torch.full_like(q, 0x55)), (ys, torch.full_like(ys, 77.0))):
        inner = v.clone()
        if v is ys:
            inner[1:-1, 1:-1] = v0[1:-1, 1:-1]
        else:
            inner[1:-1, 8:-8] = v0[1:-1, 8:-8]
        assert torch.equal(inner, v0)


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_rmsnorm_unaligned_rows(ob, ctx, shift):
    """Rows that start off the 16-byte grid, by pointer and by stride."""
    t = torch.bfloat16
    base = normal((9, 1031), 5, t)
    x = base[:, shift:shift + 1024]
    w = normal((1030,), 6, t)[shift:shift + 1024]
    for quantize in (False, True):
        check_norm(ob.RMSNormalization(quantize=quantize).compute([x, w], ctx, residual=base[:, :1024]), x, base[:, :1024], w, 1e-5, quantize)


# --------------------------------------------------------------------------- quantise
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (128, 128), (129, 127), (64, 4096), (300, 1000), (257, 16 * 9),
                                       (1000, 2056), (2, 14336)])
def test_quantize(ob, ctx, rows, cols, t, block_rows):
    x = (normal((rows, cols), rows * cols, t).float() * torch.exp(2 * normal((rows, 1), 5))).to(t)
    q, s = ob.QuantizeBlocks(block_rows).compute([x], ctx)
    check_quantized(q, s, x.double(), block_rows, 0.0)
    qe, se = exact_quantize(x, block_rows)
    assert torch.equal(q.view(torch.uint8).cpu(), qe.view(torch.uint8)) and torch.equal(s.cpu(), se)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("t", TYPES)
def test_quantize_extreme_values(ob, ctx, t, block_rows):
    """Zeros, the smallest and the largest values, ties, infinities and NaN, each in blocks of its own."""
    x = torch.zeros((128, 128 * 9), dtype=torch.float32)
    v = [x[:, 128 * i:128 * (i + 1)] for i in range(9)]
    top = torch.finfo(t).max
    v[1][:] = torch.finfo(t).tiny / 8 * torch.arange(128)  # subnormal
    v[2][:] = torch.linspace(-top, top, 128)
    v[3][:, 0] = 448.0                                     # scale 1: ties of the grid itself
    v[3][:, 1:17] = torch.arange(16) * 2.0 ** -10          # halfway between subnormals
    v[3][:, 17:49] = 16 + torch.arange(32) * 0.5
    v[4][:, 3] = float("inf")
    v[4][:, 4] = 1.0
    v[5][:, 7] = float("nan")
    v[5][:, 8] = 2.0
    v[6][:, 127] = -top
    v[7][:] = -0.0
    v[8][:, :4] = torch.tensor([1.0, -1.0, 2.0 ** -9, 1e-4])
    x = x.to(t).cuda()
    q, s = ob.QuantizeBlocks(block_rows).compute([x], ctx)
    qe, se = exact_quantize(x, block_rows)
    good = [c for c in range(9) if c not in (4, 5)]
    sel = torch.cat([torch.arange(128 * c, 128 * c + 128) for c in good])
    assert torch.equal(q.view(torch.uint8).cpu()[:, sel], qe.view(torch.uint8)[:, sel])
    # (fp32: linspace overflows between its ends, so its block holds NaN on both sides)
    assert torch.allclose(s.cpu()[:, good], se[:, good], rtol=0, atol=0, equal_nan=True)
    assert not torch.isfinite(s[:, 4]).any() and not torch.isfinite(s[:, 5]).any()
    stands_for = q.float() * by_element(s, q.shape, block_rows)
    assert torch.isnan(stands_for[:, 128 * 4:128 * 6]).all()


def run_quantize(handle, x, q, s, block_rows):
    d = C.QuantizeDesc(rows=x.shape[0], cols=x.shape[1], ldx=x.stride(0), ldq=q.stride(0), scale_row=s.stride(0),
                       scale_block=s.stride(1), type=CODE[x.dtype], block_rows=block_rows)
    handle.check(C.lib().onnxb200_quantize_blocks(handle.ptr, ctypes.byref(d), x.data_ptr(), q.data_ptr(), s.data_ptr()), "quantize")
    handle.synchronize()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("off", [0, 1, 16])
def test_quantize_strides_and_bounds(handle, t, off, block_rows):
    rows, cols = 200, 300
    x = normal((rows, cols + 40), 3, t)[:, off:off + cols]
    rb = rows if block_rows == 1 else 2
    q = torch.full((rows + 2, 352), 0x55, dtype=torch.uint8, device="cuda")
    for transposed in (False, True):
        s = torch.full((5, rb + 2) if transposed else (rb + 2, 5), 7.0, device="cuda")
        inner = s.t()[1:-1, 1:-1] if transposed else s[1:-1, 1:-1]
        run_quantize(handle, x, q.view(E4M3)[1:-1, off:off + cols], inner, block_rows)
        qe, se = exact_quantize(x, block_rows)
        assert torch.equal(q[1:-1, off:off + cols].cpu(), qe.view(torch.uint8)) and torch.equal(inner.cpu(), se)
        out, so = q.clone(), s.clone()
        out[1:-1, off:off + cols] = 0x55
        (so.t() if transposed else so)[1:-1, 1:-1] = 7.0
        assert (out == 0x55).all() and (so == 7.0).all()


def test_quantize_empty(ob, ctx):
    for shape in ((0, 256), (3, 0), (0, 0)):
        q, s = ob.QuantizeBlocks().compute([torch.empty(shape, device="cuda")], ctx)
        assert q.shape == shape and s.shape == (shape[0], -(-shape[1] // 128))
    y = ob.RMSNormalization().compute([torch.empty((0, 64), device="cuda"), torch.ones(64, device="cuda")], ctx)
    assert y[0].shape == (0, 64)


# --------------------------------------------------------------------------- product
def operands(m, n, k, seed, pad=True):
    """e4m3 operands and scales of normal values, quantised by torch; rows padded to 16 bytes if `pad`."""
    out = []
    for rows, block_rows, s in ((m, 1, seed), (n, 128, seed + 1)):
        g = torch.Generator().manual_seed(s)
        x = torch.randn((rows, k), generator=g) * torch.exp(torch.randn((rows, 1), generator=g))
        q, sc = exact_quantize(x, block_rows)
        hold = torch.zeros((rows, (k + 15) // 16 * 16 if pad else k), dtype=torch.uint8)
        hold[:, :k] = q.view(torch.uint8)
        out += [hold.cuda().view(E4M3)[:, :k], sc.cuda()]
    return out


def mm_ref(a, sa, b, sb, bias, relu):
    """(result, sum of magnitudes) in float64."""
    fa = a.double() * by_element(sa, a.shape, 1).double()
    fb = b.double() * by_element(sb, b.shape, 128).double()
    y, mag = fa @ fb.t(), fa.abs() @ fb.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return (y.clamp(min=0) if relu else y), mag


def check_mm(y, a, sa, b, sb, bias, relu, t):
    ref, mag = mm_ref(a, sa, b, sb, bias, relu)
    kb = -(-a.shape[1] // 128)
    sums = mag * (128 * 2 * U + (kb + 4) * U)
    assert y.dtype == t and y.shape == ref.shape
    off = (y.double() - ref).abs()
    assert (off <= sums + (ref.abs() + sums) * half(t) + TINY[t]).all(), (off / (sums + ref.abs() * half(t))).max()


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (1, 1000, 2048), (2, 300, 1000), (8, 8, 16), (15, 129, 127), (16, 256, 128),
          (17, 1000, 2048), (33, 100, 640), (64, 130, 4096), (65, 512, 256), (127, 257, 300), (128, 128, 1024), (129, 640, 48),
          (200, 2048, 512), (256, 256, 256), (257, 511, 129), (500, 1000, 1100), (1024, 512, 768), (777, 1300, 400), (2049, 300, 200),
          (1, 64, 60000), (2, 130, 30000), (3, 70, 20011), (40, 200, 12345), (65, 300, 2200), (100, 140, 9999), (300, 260, 7777)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(ob, ctx, m, n, k, t):
    a, sa, b, sb = operands(m, n, k, m + n + k)
    for bias, relu in ((None, False), (normal((n,), 3), True)):
        y = ob.MatMulBlockScaled(dtype=t, relu=relu).compute([a, sa, b, sb, bias], ctx)[0]
        check_mm(y, a, sa, b, sb, bias, relu, t)


@pytest.mark.parametrize("m,n,k", [(1, 384, 512), (60, 200, 256), (128, 512, 384), (300, 300, 512), (1500, 777, 1024)])
def test_matmul_exact_integers(ob, ctx, m, n, k):
    """Whole numbers up to 15 and scales of powers of two: every sum is exact in fp32, so is the result."""
    g = torch.Generator(device="cuda").manual_seed(m)
    a = torch.randint(-15, 16, (m, k), generator=g, device="cuda").float().to(E4M3)
    b = torch.randint(-15, 16, (n, k), generator=g, device="cuda").float().to(E4M3)
    sa = torch.exp2(torch.randint(-1, 2, (m, k // 128), generator=g, device="cuda").float())
    sb = torch.exp2(torch.randint(-1, 2, (-(-n // 128), k // 128), generator=g, device="cuda").float())
    ref, _ = mm_ref(a, sa, b, sb, None, False)
    y = ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0]
    assert torch.equal(y.double(), ref)
    r = ob.MatMulBlockScaled(relu=True).compute([a, sa, b, sb], ctx)[0]
    assert torch.equal(r.double(), ref.clamp(min=0))


@pytest.mark.parametrize("m", [3, 100, 700])
def test_matmul_every_scale_counts(ob, ctx, m):
    """Ones everywhere, each block with a scale of its own: the result names the scales that were used."""
    n, k = 300, 1100
    a = torch.ones((m, 1104), device="cuda").to(E4M3)[:, :k]
    b = torch.ones((n, 1104), device="cuda").to(E4M3)[:, :k]
    sa = normal((m, 9), 1)
    sb = normal((3, 9), 2)
    check_mm(ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0], a, sa, b, sb, None, False, torch.float32)
    # what lies behind the last column is not read as operands
    held = torch.full((m, 1104), 0x7F, dtype=torch.uint8, device="cuda")  # NaN
    held[:, :k] = a.view(torch.uint8)
    y = ob.MatMulBlockScaled().compute([held.view(E4M3)[:, :k], sa, b, sb], ctx)[0]
    check_mm(y, a, sa, b, sb, None, False, torch.float32)


@pytest.mark.parametrize("m", [5, 80, 400])
def test_matmul_nan_stays_in_its_row_and_column(ob, ctx, m):
    n, k = 260, 384
    a, sa, b, sb = operands(m, n, k, 5)
    ref = ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0]
    sa2, b2 = sa.clone(), b.clone()
    sa2[m // 2, 1] = float("nan")
    b2.view(torch.uint8)[200, 130] = 0x7F
    for relu in (False, True):
        y = ob.MatMulBlockScaled(relu=relu).compute([a, sa2, b2, sb], ctx)[0]
        assert torch.isnan(y[m // 2]).all() and torch.isnan(y[:, 200]).all()
        y, want = y.clone(), ref.clone().clamp(min=0) if relu else ref.clone()
        y[m // 2], want[m // 2] = 0, 0
        y[:, 200], want[:, 200] = 0, 0
        assert torch.equal(y, want)


def run_mm(handle, a, sa, b, sb, bias, y, relu=False):
    d = C.MatmulBlocksDesc(m=a.shape[0], n=b.shape[0], k=a.shape[1], lda=a.stride(0), ldb=b.stride(0), ldy=y.stride(0),
                           a_scale_row=sa.stride(0), a_scale_block=sa.stride(1), b_scale_row=sb.stride(0),
                           b_scale_block=sb.stride(1), out_type=CODE[y.dtype], flags=8 if relu else 0)
    p = [None if v is None else v.data_ptr() for v in (a, sa, b, sb, bias, y)]
    handle.check(C.lib().onnxb200_matmul_blocks(handle.ptr, ctypes.byref(d), *p), "matmul")
    handle.synchronize()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n", [(3, 200), (100, 301), (300, 520)])
def test_matmul_strides_and_bounds(handle, m, n, t):
    """Padded operands, both scale layouts, an output inside a larger one (aligned or not): nothing else is written."""
    k = 400
    a, sa, b, sb = operands(m, n, k, 9)
    bias = normal((n,), 4)
    for off in (0, 1, 8):
        for st in (False, True):
            y = torch.full((m + 2, n + 24), 3.0, dtype=t, device="cuda")
            inner = y[1:-1, off:off + n]
            s1 = sa.t().contiguous().t() if st else sa
            s2 = sb.t().contiguous().t() if st else sb
            run_mm(handle, a, s1, b, s2, bias, inner)
            check_mm(inner, a, sa, b, sb, bias, False, t)
            rest = y.clone()
            rest[1:-1, off:off + n] = 3.0
            assert (rest == 3.0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n", [(1, 517), (2, 129), (30, 517), (45, 130), (300, 517), (260, 1)])
def test_matmul_ragged_columns_on_the_grid(handle, m, n, t):
    """Output rows on the 16-byte grid whose last vector is cut: the columns behind it stay as they were."""
    a, sa, b, sb = operands(m, n, 272, 6)
    y = torch.full((m + 1, 544), 3.0, dtype=t, device="cuda")
    run_mm(handle, a, sa, b, sb, None, y[:m, :n])
    check_mm(y[:m, :n], a, sa, b, sb, None, False, t)
    assert (y[:m, n:] == 3.0).all() and (y[m] == 3.0).all()


@pytest.mark.parametrize("m,n,k", [(1, 77, 333), (9, 128, 200), (130, 70, 257)])
def test_matmul_unaligned_operands(ob, ctx, m, n, k):
    """Row strides and pointers that are no multiples of 16."""
    a, sa, b, sb = operands(m, n, k, 2, pad=False)
    check_mm(ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0], a, sa, b, sb, None, False, torch.float32)
    a, sa, b, sb = operands(m, n, k + 5, 3)
    a, b = a[:, 5:], b[:, 5:]
    check_mm(ob.MatMulBlockScaled().compute([a, sa[:, :-(-k // 128)], b, sb[:, :-(-k // 128)]], ctx)[0], a, sa[:, :-(-k // 128)],
             b, sb[:, :-(-k // 128)], None, False, torch.float32)


def test_matmul_empty_and_leading_dims(ob, ctx):
    a, sa, b, sb = operands(6, 40, 64, 1)
    y = ob.MatMulBlockScaled().compute([a.unflatten(0, (2, 3)), sa.unflatten(0, (2, 3)), b, sb], ctx)[0]
    assert y.shape == (2, 3, 40)
    check_mm(y.view(6, 40), a, sa, b, sb, None, False, torch.float32)
    one = ob.MatMulBlockScaled().compute([a[0], sa[0], b, sb], ctx)[0]
    assert one.shape == (40,)
    check_mm(one[None], a[:1], sa[:1], b, sb, None, False, torch.float32)
    z = ob.MatMulBlockScaled().compute([a[:0], sa[:0], b, sb], ctx)[0]
    assert z.shape == (0, 40)
    # k = 0: the sum of nothing, plus the bias
    e = torch.empty((3, 0), dtype=E4M3, device="cuda")
    w = torch.empty((5, 0), dtype=E4M3, device="cuda")
    bias = normal((5,), 1)
    y = ob.MatMulBlockScaled().compute([e, torch.empty((3, 0), device="cuda"), w, torch.empty((1, 0), device="cuda"), bias], ctx)[0]
    assert torch.equal(y, bias.expand(3, 5))


def test_refusals(ob, ctx):
    a, sa, b, sb = operands(4, 8, 256, 1)
    mm = ob.MatMulBlockScaled()
    x = normal((4, 256), 1)
    w = normal((256,), 2)
    bad = [lambda: mm.compute([a.float(), sa, b, sb], ctx), lambda: mm.compute([a[:, :128], sa[:, :1], b, sb], ctx),
           lambda: mm.compute([a, sa[:, :1], b, sb], ctx), lambda: mm.compute([a, sa, b, sb.double()], ctx),
           lambda: mm.compute([a, sa, b, sb, normal((7,), 1)], ctx), lambda: mm.compute([a, sa, b, sb, normal((8,), 1, torch.float16)], ctx),
           lambda: mm.compute([a.cpu(), sa, b, sb], ctx), lambda: mm.compute([a, sa, b[None], sb], ctx),
           lambda: ob.RMSNormalization().compute([x, w[:255]], ctx), lambda: ob.RMSNormalization().compute([x.double(), w], ctx),
           lambda: ob.RMSNormalization().compute([x, w], ctx, residual=x[:2]), lambda: ob.RMSNormalization().compute([x.t(), w[:4]], ctx),
           lambda: ob.RMSNormalization().compute([x, w], ctx, residual=x.half()), lambda: ob.RMSNormalization(epsilon=-1).compute([x, w], ctx),
           lambda: ob.QuantizeBlocks().compute([x.to(E4M3)], ctx), lambda: ob.QuantizeBlocks(128).compute([x[None]], ctx),
           lambda: ob.QuantizeBlocks().compute([x[:, ::2]], ctx)]
    for call in bad:
        with pytest.raises(ob.ValidationError):
            call()
    with pytest.raises(ob.UnsupportedFeature):
        ob.RMSNormalization().compute([normal((1, 49153), 1), normal((49153,), 1)], ctx)
    with pytest.raises(ob.UnsupportedFeature):
        ob.RMSNormalization(axis=0).compute([x, w], ctx)
    # a refusal leaves the handle usable
    assert torch.isfinite(mm.compute([a, sa, b, sb], ctx)[0]).all()
    ctx.handle.synchronize()


# --------------------------------------------------------------------------- together
def block(ob, ctx, x, res, layers):
    """Norm -> quantised product -> the product is the next layer's input, the sum its residual."""
    for w, b, sb, bias in layers:
        q, s, res = ob.RMSNormalization(quantize=True).compute([x, w], ctx, residual=res)
        x = ob.MatMulBlockScaled(dtype=x.dtype, relu=True).compute([q, s, b, sb, bias], ctx)[0]
    return x, res


def make_layers(ob, ctx, width, count):
    layers = []
    for i in range(count):
        b, sb = ob.QuantizeBlocks(128).compute([normal((width, width), 50 + i) * width ** -0.5], ctx)
        layers.append((1 + 0.1 * normal((width,), 60 + i).to(torch.bfloat16), b, sb, 0.1 * normal((width,), 70 + i)))
    return layers


@pytest.mark.parametrize("rows,width", [(1, 512), (33, 776), (300, 1000)])
def test_chain(ob, ctx, rows, width):
    """Four layers as a program runs them, each step against 64 bits from the step's own inputs."""
    layers = make_layers(ob, ctx, width, 4)
    x, res = normal((rows, width), 1, torch.bfloat16), normal((rows, width), 2, torch.bfloat16)
    for w, b, sb, bias in layers:
        out = ob.RMSNormalization(quantize=True).compute([x, w], ctx, residual=res)
        check_norm(out, x, res, w, 1e-5, True)
        q, s, res = out
        x = ob.MatMulBlockScaled(dtype=torch.bfloat16, relu=True).compute([q, s, b, sb, bias], ctx)[0]
        check_mm(x, q, s, b, sb, bias, True, torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 150, 600])
def test_captured_chains_side_by_side(ob, ctx, rows):
    """Two captured chains replayed on two streams at once, with new inputs in place, give what eager calls give."""
    width = 640
    layers = make_layers(ob, ctx, width, 3)
    xs = [[normal((rows, width), 10 * i + j, torch.bfloat16) for j in range(2)] for i in range(2)]
    graphs, outs = [], []
    for i in range(2):
        for _ in range(2):
            block(ob, ctx, *xs[i], layers)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(ob, ctx, *xs[i], layers))
        graphs.append(g)
    for turn in range(3):
        for i in range(2):
            for j in range(2):
                xs[i][j].copy_(normal((rows, width), 100 * turn + 10 * i + j, torch.bfloat16))
        want = [block(ob, ctx, *xs[i], layers) for i in range(2)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])
    ctx.handle.synchronize()


def test_calls_follow_the_current_stream(ob, ctx):
    """Inputs made on a side stream just before the call, outputs read there just after it."""
    layers = make_layers(ob, ctx, 512, 2)
    torch.cuda.synchronize()
    want = None
    for turn in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x = normal((64, 4096), 3, torch.bfloat16)
            for _ in range(20):  # a producer that is still running when the calls are made
                x = (x @ torch.eye(4096, dtype=x.dtype, device="cuda"))
            y, res = block(ob, ctx, x[:, :512].contiguous(), x[:, 512:1024].contiguous(), layers)
            got = y.float() + res.float()
        s.synchronize()
        want = got if want is None else want
        assert torch.equal(got, want) and torch.isfinite(got).all()


def test_results_do_not_depend_on_the_run(ob, ctx):
    """The same call gives the same bits, alone or behind others."""
    for m, n, k in ((1, 2048, 4096), (100, 1000, 8192), (600, 1024, 2048)):
        a, sa, b, sb = operands(m, n, k, 4)
        first = ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0]
        for _ in range(5):
            assert torch.equal(ob.MatMulBlockScaled().compute([a, sa, b, sb], ctx)[0], first)


def test_settings_changed_between_calls(ob, ctx):
    """Descriptors are kept by layout, but not past a change of the operator's own settings."""
    x, w = normal((4, 256), 1), normal((256,), 2)
    op = ob.RMSNormalization()
    op.compute([x, w], ctx)
    op.epsilon, op.quantize = 0.5, True
    out = op.compute([x, w], ctx)
    check_norm(out, x, None, w, 0.5, True)
    a, sa, b, sb = operands(4, 8, 256, 1)
    mm = ob.MatMulBlockScaled()
    mm.compute([a, sa, b, sb], ctx)
    mm.relu, mm.dtype = True, torch.float16
    check_mm(mm.compute([a, sa, b, sb], ctx)[0], a, sa, b, sb, None, True, torch.float16)
    q = ob.QuantizeBlocks()
    q.compute([x], ctx)
    q.block_rows = 128
    assert q.compute([x], ctx)[1].shape == (1, 2)


def test_first_call_of_a_process_inside_a_capture():
    """A capture may be the first thing a process does with each kernel."""
    import subprocess
    import sys
    code = """
import importlib, torch
ob = importlib.import_module("onnx-rs_b200")
ctx = ob.ExecutionContext(ob.Handle(0))
ins = [torch.randn(m, 512, device="cuda").bfloat16() for m in (1, 8, 100, 600)]
w, wt = torch.ones(512, device="cuda").bfloat16(), torch.randn(384, 512, device="cuda")
torch.cuda.synchronize()
def run():
    b, sb = ob.QuantizeBlocks(128).compute([wt], ctx)
    out = []
    for x in ins:
        q, s = ob.RMSNormalization(quantize=True).compute([x, w], ctx)
        out.append(ob.MatMulBlockScaled().compute([q, s, b, sb], ctx)[0])
    return out
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(x, y) and torch.isfinite(x).all() for x, y in zip(got, want))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_handles_on_two_threads(ob):
    """Each thread with a handle and a stream of its own, different sizes at the same time."""
    import threading
    jobs, errors = [], []
    for i, (rows, cols) in enumerate(((3, 40001), (3, 13001))):
        jobs.append((normal((rows, cols), i), normal((cols,), 7 + i), operands(20 + 300 * i, 640, 1024, i)))
    torch.cuda.synchronize()

    def work(x, w, mm):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                with ob.Handle(0) as h:
                    ctx = ob.ExecutionContext(h)
                    for _ in range(20):
                        out = ob.RMSNormalization().compute([x, w], ctx)
                        y = ob.MatMulBlockScaled().compute(list(mm), ctx)[0]
                    h.synchronize()
                    check_norm(out, x, None, w, 1e-5, False)
                    check_mm(y, *mm, None, False, torch.float32)
        except Exception as e:  # noqa: BLE001 -- handed to the test's thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    if errors:
        raise errors[0]


def test_current_device_is_kept(ob, ctx):
    dev = torch.cuda.current_device()
    ob.QuantizeBlocks().compute([normal((2, 256), 1)], ctx)
    assert torch.cuda.current_device() == dev
    if torch.cuda.device_count() > 1:
        with torch.cuda.device(1):
            ob.QuantizeBlocks().compute([normal((2, 256), 1).to("cuda:0")], ctx)
            assert torch.cuda.current_device() == 1
            with pytest.raises(ob.ValidationError):
                ob.QuantizeBlocks().compute([torch.zeros((2, 256), device="cuda:1")], ctx)


def test_long_offsets(ob, ctx):
    """Elements past 2^31: the last rows of a 2.2 G-element matrix."""
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    rows, cols = 70000, 32000
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-3:] = normal((3, cols), 1, torch.bfloat16)
    q, s = ob.QuantizeBlocks().compute([x], ctx)
    qe, se = exact_quantize(x[-3:], 1)
    assert torch.equal(q[-3:].view(torch.uint8).cpu(), qe.view(torch.uint8)) and torch.equal(s[-3:].cpu(), se)
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    y = ob.RMSNormalization().compute([x, w], ctx)[0]
    check_norm([y[-3:]], x[-3:], None, w, 1e-5, False)
    del y, x
    b, sb = operands(1, 300, cols, 3)[2:]
    y = ob.MatMulBlockScaled(dtype=torch.bfloat16).compute([q, s, b, sb], ctx)[0]
    check_mm(y[-3:], q[-3:], s[-3:], b, sb, None, False, torch.bfloat16)
    assert (y[:-3] == 0).all()


@pytest.fixture(params=[True, False], ids=["native_calls", "ctypes"])
def calls(ob, request, monkeypatch):
    """With the module for repeated calls, and without it."""
    if request.param:
        assert ob.ops._calls is not None, "onnx-rs_b200/_calls.so is not built"
    else:
        monkeypatch.setattr(ob.ops, "_calls", None)
    return request.param


def test_repeated_calls(ob, ctx, calls):
    """Layouts in turn through one operator: each call's outputs are its own, and the first's bits."""
    norm, quant = ob.RMSNormalization(1e-6, quantize=True), ob.QuantizeBlocks()
    weights, mm = ob.QuantizeBlocks(128), ob.MatMulBlockScaled(torch.bfloat16, relu=True)
    b, sb = weights.compute([normal((300, 640), 9)], ctx)
    bias = normal((300,), 10)
    seen = {}
    for turn in range(3):
        for i, (lead, res) in enumerate((((1,), True), ((40,), False), ((2, 3), True), ((300,), True))):
            x, r = normal((*lead, 640), i, torch.bfloat16), normal((*lead, 640), 50 + i, torch.bfloat16)
            w = normal((640,), 99, torch.bfloat16)
            out = norm.compute([x, w], ctx, residual=r if res else None)
            check_norm(out, x, r if res else None, w, 1e-6, True)
            out += quant.compute([x[..., :500]], ctx)
            out += mm.compute([out[0], out[1], b, sb] + ([bias] if i % 2 else []), ctx)
            flat = [t.reshape(-1, t.shape[-1]) for t in (out[-1], out[0], out[1])]
            check_mm(*flat, b, sb, bias if i % 2 else None, True, torch.bfloat16)
            layout = [(t.shape, t.stride(), t.dtype) for t in out]
            first = seen.setdefault(i, (out, layout))
            assert layout == first[1]
            if turn:
                for t, f in zip(out, first[0]):
                    assert t.data_ptr() != f.data_ptr()
                    assert torch.equal(t.contiguous().view(torch.uint8), f.contiguous().view(torch.uint8))
    assert bool(norm.__dict__.get("_plans")) == calls


def test_repeated_calls_are_checked(ob, ctx, calls):
    """What differs from the layouts seen before is checked as a first call is."""
    x, w = normal((4, 256), 1), normal((256,), 2)
    norm, mm = ob.RMSNormalization(), ob.MatMulBlockScaled()
    a, sa, b, sb = operands(4, 8, 256, 1)
    for _ in range(2):
        norm.compute([x, w], ctx)
        mm.compute([a, sa, b, sb], ctx)
    for bad in ([x, w[:128]], [x.cpu(), w], [x, w.cpu()], [x.to(torch.int32), w], [x.t().contiguous().t(), w], [x[0, 0], w]):
        with pytest.raises(ob.ValidationError):
            norm.compute(bad, ctx)
    with pytest.raises(ob.ValidationError):
        norm.compute([x, w], ctx, residual=x[:2])
    for bad in ([a, sa[:, :1], b, sb], [a, sa, b[:, :128], sb], [a, sa, b, sb, normal((7,), 1)], [a.float(), sa, b, sb]):
        with pytest.raises(ob.ValidationError):
            mm.compute(bad, ctx)
    out = norm.compute([torch.nn.Parameter(x), torch.nn.Parameter(w)], ctx)[0]
    assert not out.requires_grad
    check_norm([out], x, None, w, 1e-5, False)
    with torch.inference_mode():
        check_norm(norm.compute([x, w], ctx), x, None, w, 1e-5, False)
    h = ob.Handle(0)
    other = ob.ExecutionContext(h)
    check_norm(norm.compute([x, w], other), x, None, w, 1e-5, False)
    h.close()
    with pytest.raises(ob.OnnxB200Error):
        norm.compute([x, w], other)
    check_norm(norm.compute([x, w], ctx), x, None, w, 1e-5, False)


def test_repeated_calls_on_streams(ob, calls):
    """A handle on its own stream, on torch's, and torch on others: always in order with torch's current stream."""
    w = torch.ones(2048, device="cuda")
    for torch_stream in (True, False):
        with ob.Handle(0, torch_stream=torch_stream) as h:
            ctx, norm = ob.ExecutionContext(h), ob.RMSNormalization()
            for stream in (None, torch.cuda.Stream(), None, torch.cuda.Stream()):
                with torch.cuda.stream(stream):
                    x = normal((512, 2048), 3)
                    eye = torch.eye(2048, device="cuda")
                    for _ in range(8):  # a producer that is still running when the call is made
                        x = x @ eye
                    y = norm.compute([x, w], ctx)[0].clone()
                    torch.cuda.current_stream().synchronize()
                    check_norm([y], x, None, w, 1e-5, False)
            torch.cuda.synchronize()


# The error bound of norm_slack holds here too: a thread adds 4 or 8 squares, a shuffle 5 and the row at most 16
# parts, 29 roundings at most of a sum whose square root halves them: 15 U at 4096 columns, where norm_slack has 22,
# 13 at 2048 (18) and 6 at 130 (14.5), with 5 for the division, root and products.
@pytest.mark.parametrize("residual,quantize", [(False, False), (True, True)])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(700, 2), (3, 127), (2, 129), (310, 1025), (2, 2047), (3, 2049), (305, 3001), (2, 3968),
                                       (2, 4095), (3, 4097)])
def test_rmsnorm_off_the_grid(ob, ctx, rows, cols, t, residual, quantize):
    """Rows of every length around what a warp and a thread block hold, none on a 16-byte boundary for long."""
    x = normal((rows, cols + 1), rows + cols, t)[:, 1:]
    r = 3 * normal((rows, cols), 7, t) if residual else None
    w = (1 + 0.3 * normal((cols + 1,), 9)).to(t)[1:]
    out = ob.RMSNormalization(epsilon=1e-5, quantize=quantize).compute([x, w], ctx, residual=r)
    check_norm(out, x, r, w, 1e-5, quantize)


def test_rmsnorm_off_the_grid_non_finite(ob, ctx):
    """As on the grid: a NaN or an infinity stays in its row, a zero row is zero."""
    for cols in (381, 2501):
        x = normal((5, cols), 1)
        x[1] = 0
        x[2, 5] = float("inf")
        x[3, cols - 1] = float("nan")
        w = torch.ones(cols, device="cuda")
        y = ob.RMSNormalization().compute([x, w], ctx)[0]
        assert (y[1] == 0).all() and torch.isnan(y[2, 5]) and (y[2, 6:] == 0).all() and torch.isnan(y[3]).all()
        check_norm([y[[0, 4]]], x[[0, 4]], None, w, 1e-5, False)
        q, s = ob.RMSNormalization(quantize=True).compute([x, w], ctx)
        assert (q[1].float() == 0).all() and torch.isfinite(s[1]).all()
        assert not torch.isfinite(s[2, 0]) and torch.isfinite(s[2, 1:]).all() and not torch.isfinite(s[3]).any()


@pytest.mark.parametrize("m,n,k", [(256, 512, 2560), (100, 1000, 2048), (70, 1700, 4000), (200, 2048, 4096), (129, 2560, 3700),
                                   (512, 2304, 4096), (256, 4200, 3600), (256, 4608, 3600)])
def test_product_with_few_tiles(ob, ctx, m, n, k):
    """Tiles shared by one, two or four pairs of thread blocks, up to and past what runs at once."""
    a, sa, b, sb = operands(m, n, k, m + n)
    bias = normal((n,), 3)
    y = ob.MatMulBlockScaled(torch.float32, relu=True).compute([a, sa, b, sb, bias], ctx)[0]
    check_mm(y, a, sa, b, sb, bias, True, torch.float32)
    assert torch.equal(y, ob.MatMulBlockScaled(torch.float32, relu=True).compute([a, sa, b, sb, bias], ctx)[0])


def test_shared_tiles_first_inside_a_capture():
    """What is asked of the device once, before tiles are shared, may be asked during a capture."""
    import subprocess
    import sys
    code = """
import importlib, torch
ob = importlib.import_module("onnx-rs_b200")
ctx = ob.ExecutionContext(ob.Handle(0))
x, wt = torch.randn(100, 4096, device="cuda"), torch.randn(2000, 4096, device="cuda")
torch.cuda.synchronize()
def run():
    (q, s), (b, sb) = ob.QuantizeBlocks().compute([x], ctx), ob.QuantizeBlocks(128).compute([wt], ctx)
    return ob.MatMulBlockScaled().compute([q, s, b[:400], sb[:4], ], ctx) + ob.MatMulBlockScaled().compute([q, s, b, sb], ctx)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(x, y) and torch.isfinite(x).all() for x, y in zip(got, want))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
