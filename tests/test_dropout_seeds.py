"""Where a dropout's seed lives and where one comes from: the same rules in the plain formulation and in the kernels."""
import pytest
import torch

from torchturbo_b200.ops import ops

IMPLS = [("torch_dropout", "torch_linear_bias_act"), (None, None)]


def _calls(x, w, seed, impls):
    one, two = impls
    return (lambda: ops.dropout(x, 0.5, seed, **({"impl": one} if one else {})),
            lambda: ops.linear_bias_act(x, w, dropout_p=0.5, seed=seed, **({"impl": two} if two else {})))


@pytest.mark.parametrize("impls", IMPLS)
@pytest.mark.parametrize("device, other", [("cpu", "meta"), pytest.param("cuda", "cpu", marks=pytest.mark.gpu)])
def test_seed_tensor_on_another_device_is_refused(device, other, impls):
    x, w = torch.ones(6, 16, device=device, dtype=torch.bfloat16), torch.ones(8, 16, device=device, dtype=torch.bfloat16)
    for call in _calls(x, w, torch.zeros(1, dtype=torch.int64, device=other), impls):
        with pytest.raises(AssertionError, match="seed tensor"):
            call()
    for call, same in zip(_calls(x, w, torch.full((1,), 5, device=device), impls), _calls(x, w, 5, impls)):
        assert torch.equal(call(), same())


@pytest.mark.parametrize("impls", IMPLS)
@pytest.mark.parametrize("device, default", [("cpu", "meta"), pytest.param("cuda", "cuda", marks=pytest.mark.gpu)])
def test_seed_from_the_host_whatever_the_default_device_is(device, default, impls):
    x, w = torch.ones(6, 16, device=device, dtype=torch.bfloat16), torch.ones(8, 16, device=device, dtype=torch.bfloat16)
    for call in _calls(x, w, None, impls):
        torch.manual_seed(4)
        want = call()
        torch.manual_seed(4)
        with torch.device(default):
            got = call()
        assert got.device.type == device and torch.equal(got, want)
