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
