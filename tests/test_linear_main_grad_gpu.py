"""Weights with an fp32 accumulation buffer (replicated layers), of few and of many input features, with all that follows the product."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8       # half a step of bf16
ACC = 2.0 ** -15       # fp32 sums: 2^-24 of the summed magnitudes for each of at most 2^9 partial sums


@pytest.mark.parametrize("M, N, K", [(5, 24, 16), (700, 264, 16), (700, 264, 64), (1030, 520, 136)])
def test_against_64_bits(M, N, K):
    from torchturbo_b200.ops import ops
    from torchturbo_b200.ops.dropout import dropout_args, keep_mask

    gen = torch.Generator().manual_seed(M + K)
    x, w, b, dy = ((torch.randn(*s, generator=gen) * 0.5).bfloat16().cuda() for s in ((M, K), (N, K), (N,), (M, N)))
    before = torch.randn(N, K, generator=gen).cuda()
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    w.main_grad = before.clone()
    ops.linear_bias_act(x, w, b, dropout_p=0.25, seed=9).backward(dy)
    assert w.grad is None
    X, W, D = (t.detach().double() for t in (x, w, dy))
    D = D * keep_mask(M, N, dropout_args(0.25, 9), "cpu").double().cuda() * (4 / 3)
    tz = D.abs() * HALF                                    # dropout(dy) is rounded to bf16 before the products
    # the product is added to the buffer in fp32: one rounding of their sum
    got, ref, bound = w.main_grad.double(), before.double() + D.t() @ X, tz.t() @ X.abs() + ACC * (D.t().abs() @ X.abs())
    assert ((got - ref).abs() <= bound + 2.0 ** -23 * (ref.abs() + before.abs())).all()
    for got, ref, bound in ((x.grad, D @ W, tz @ W.abs() + ACC * (D.abs() @ W.abs())), (b.grad, D.sum(0), tz.sum(0) + ACC * D.abs().sum(0))):
        assert ((got.double() - ref).abs() <= ref.abs() * HALF + bound * (1 + HALF)).all()
