"""GELU (tanh) far left of zero, where its value is small beside its argument: relative to the value itself, in every form of the layer."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8       # half a step of bf16
# The hyperbolic tangent's argument u stays below 13 from -6 on; 2 u log2(e) below 37 is rounded three times, 3 x 37 x 2^-24 x ln 2 = 2^-17.7
# of the exponential, the exponential and the reciprocal add 2^-22 each and the product 2^-24: below 2^-17.  The slope takes it twice, and once
# more for 1 - s and the factor beside it: below 2^-15.
VALUE, SLOPE = 2.0 ** -17, 2.0 ** -15


def _formulas(v):
    """v s and its derivative s + 2 v s (1 - s) u',  s = 1 / (1 + exp(-2 u)), which is (1 + tanh u) / 2 without its cancellation."""
    c = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * c * (v + 0.044715 * v ** 3))
    return v * s, s + 2 * v * s * (1 - s) * c * (1 + 3 * 0.044715 * v * v)


def _arguments():
    return torch.linspace(-6, 3, 1201, dtype=torch.float64).bfloat16().unique()


# rows of the weight past a few rows, a walk over few features, tiles, sums in pieces
@pytest.mark.parametrize("M, N, K", [(4, 72, 64), (8, 264, 264), (333, 264, 16), (333, 264, 64), (1100, 1032, 136), (130, 72, 8192)])
def test_value_and_slope(M, N, K):
    """One feature carries the argument (its weight is one for one column and zero for the rest), so that z is exact."""
    from torchturbo_b200 import kernels as Kn
    from torchturbo_b200.ops import ops

    v = _arguments()
    at = N - 3                                            # the column that sees the argument
    w = torch.zeros(N, K, dtype=torch.bfloat16)
    w[at, K - 1] = 1
    w = w.cuda()
    for first in range(0, v.numel(), M):
        some = v[first:first + M]
        rows = torch.zeros(M, K, dtype=torch.bfloat16)
        rows[:some.numel(), K - 1] = some
        x = rows.cuda().requires_grad_()
        y = ops.linear_bias_act(x, w.detach().requires_grad_(), act="gelu_tanh")
        dy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
        dy[:, at] = 1
        dx, = torch.autograd.grad(y, x, dy)
        value, slope = _formulas(some.double())
        got, grad = y[:some.numel(), at].detach().double().cpu(), dx[:some.numel(), K - 1].double().cpu()
        assert ((got - value).abs() <= value.abs() * (HALF + VALUE * (1 + HALF))).all()
        # the slope crosses zero near -0.75, where its two terms cancel: they are below 0.3 there
        assert ((grad - slope).abs() <= slope.abs() * (HALF + SLOPE) + 0.6 * SLOPE * (some.double() > -2)).all()
    assert Kn.status() == (0, 0)


@pytest.mark.parametrize("M, K", [(4, 64), (40, 16), (140, 64)])
def test_arguments_of_any_size(M, K):
    """Far out the value is the argument or nothing, the slope one or nothing, infinities included."""
    from torchturbo_b200.ops import ops

    inf = float("inf")
    for v, value, slope in ((-40.0, 0.0, 0.0), (-1e10, 0.0, 0.0), (-3e38, 0.0, 0.0), (-inf, 0.0, 0.0), (40.0, None, 1.0), (1e10, None, 1.0), (3e38, None, 1.0),
                            (inf, None, 1.0)):
        x, w = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16).requires_grad_(), torch.zeros(24, K, device="cuda", dtype=torch.bfloat16)
        b = torch.full((24,), v, device="cuda", dtype=torch.bfloat16).requires_grad_()
        y = ops.linear_bias_act(x, w, b, "gelu_tanh")
        assert (y == (b.detach() if value is None else value)).all()
        db, = torch.autograd.grad(y, b, torch.ones_like(y))
        assert (db == M * slope).all()
