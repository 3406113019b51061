"""Both forms of the log-probabilities take the same arguments."""
import inspect

import pytest
import torch


def test_signatures():
    from torchturbo_b200.ops.providers import b200, native

    forms = [inspect.signature(c.__call__).parameters for c in (b200.B200LinearLogprobs, native.TorchLinearLogprobs)]
    assert [(p.name, p.kind, p.default) for p in forms[0].values()] == [(p.name, p.kind, p.default) for p in forms[1].values()]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_a_time(dtype):
    """Of the plain formulation (fp32); the kernels have no use for it."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(1)
    h, w = (torch.randn(*s, generator=gen).to("cuda", dtype) for s in ((7, 16), (24, 16)))
    t = torch.arange(7, device="cuda")
    # fp32 products of 16, in another order
    a, b = (ops.linear_logprobs(h, w, t, want_entropy=True, chunk=c) for c in (3, 1024))
    for u, v in zip(a, b):
        assert torch.allclose(u, v, rtol=1e-5, atol=1e-5)
