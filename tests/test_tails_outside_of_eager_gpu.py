"""The new operators under function transforms, forward-mode differentiation and tracing: the plain formulation takes over."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _data():
    gen = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=gen).cuda() for s in ((3, 8, 16), (24, 16), (24,)))
    return x.bfloat16(), w.bfloat16(), b.bfloat16(), torch.randint(0, 24, (3, 8), generator=gen).cuda()


def test_vmap():
    from torchturbo_b200.ops import ops

    x, w, b, t = _data()
    y = torch.vmap(lambda v: ops.linear_bias_act(v, w, b, "gelu", dropout_p=0.2, seed=3))(x)
    assert torch.equal(y, torch.stack([ops.linear_bias_act(v, w, b, "gelu", dropout_p=0.2, seed=3, impl="torch_linear_bias_act") for v in x]))
    d = torch.vmap(lambda v: ops.dropout(v, 0.2, 3))(x)
    assert torch.equal(d, torch.stack([ops.dropout(v, 0.2, 3) for v in x]))
    lp = torch.vmap(lambda v, u: ops.linear_logprobs(v, w, u)[0])(x, t)
    assert torch.allclose(lp, torch.stack([ops.linear_logprobs(v, w, u, impl="torch_linear_logprobs")[0] for v, u in zip(x, t)]), atol=1e-5)


def test_forward_mode():
    from torchturbo_b200.ops import ops

    x, w, b, t = _data()
    x = x.float()
    for f in (lambda v: ops.dropout(v, 0.2, 3), lambda v: ops.linear_bias_act(v, w.float(), b.float(), "gelu"),
              lambda v: ops.linear_logprobs(v, w.float(), t)[0]):
        _, tangent = torch.func.jvp(f, (x,), (torch.ones_like(x),))
        eps = 1e-2
        near = (f(x + eps) - f(x - eps)) / (2 * eps)
        assert (tangent - near).norm() <= 1e-2 * near.norm()      # third derivatives times eps^2 / 6, and fp32 differences


def test_traced():
    from torch.fx.experimental.proxy_tensor import make_fx

    from torchturbo_b200.ops import ops

    x, w, b, _ = _data()
    f = make_fx(lambda v: ops.linear_bias_act(v, w, b, "gelu_tanh", dropout_p=0.1, seed=1))(x)
    assert torch.equal(f(x), ops.linear_bias_act(x, w, b, "gelu_tanh", dropout_p=0.1, seed=1, impl="torch_linear_bias_act"))
