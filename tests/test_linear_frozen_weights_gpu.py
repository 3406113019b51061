"""A biased linear layer whose weight is frozen needs its input for nothing in the backward, and does not keep it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(gen, *shape):
    return (torch.randn(*shape, generator=gen) * 0.5).bfloat16().cuda()


@pytest.mark.parametrize("M, N, K, p", [(4096, 1024, 1024, 0.0), (4096, 1024, 1024, 0.2), (65536, 1024, 16, 0.2), (4, 256, 65536, 0.0)])
@pytest.mark.parametrize("train_bias", [False, True])
def test_input_is_let_go(M, N, K, p, train_bias):
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(1)
    src, w, b, dy = (_rand(gen, *s) for s in ((M, K), (N, K), (N,), (M, N)))
    src.requires_grad_()
    b.requires_grad_(train_bias)
    ops.linear_bias_act(src, w, b, dropout_p=p, seed=3).backward(dy)      # what is kept for good is there
    want = [t.grad.clone() for t in (src, b) if t.grad is not None]
    src.grad = b.grad = None
    x = src * 1
    size = x.untyped_storage().nbytes()
    y = ops.linear_bias_act(x, w, b, dropout_p=p, seed=3)
    before = torch.cuda.memory_allocated()
    del x
    assert before - torch.cuda.memory_allocated() >= size
    y.backward(dy)
    for t, ref in zip((t for t in (src, b) if t.grad is not None), want):
        assert torch.equal(t.grad, ref)


@pytest.mark.parametrize("act", [None, "gelu"])
def test_gradient_of_the_gradient_with_a_frozen_weight(act):
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(2)
    x, w, b, dy = _rand(gen, 9, 64).requires_grad_(), _rand(gen, 72, 64), _rand(gen, 72).requires_grad_(), _rand(gen, 9, 72).requires_grad_()
    got = []
    for impl in ("tcgen05_linear_bias_act", "torch_linear_bias_act"):
        y = ops.linear_bias_act(x, w, b, act, dropout_p=0.2, seed=1, impl=impl)
        g = torch.autograd.grad(y, (x, b), dy, create_graph=True)
        second = torch.autograd.grad(sum(v.float().square().sum() for v in g), (dy, x, b), allow_unused=act is None)
        got.append([*g, *(v for v in second if v is not None)])
    assert len(got[0]) == len(got[1]) == (3 if act is None else 5)
    for a, ref in zip(*got):
        assert ref.abs().max() > 0 and torch.equal(a, ref)
