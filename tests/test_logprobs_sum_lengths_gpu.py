"""Log-probabilities of long hidden states: the sums behind them are not pulled to zero by more than runs of 512 products are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T, H", [(4096, 2048), (1500, 4096)])
def test_sums_keep_their_size(T, H):
    """A vocabulary of one token of real logits l and of others whose logits are zero: where l is large, -log p of another is l itself, to
    exp(-l).  The tensor cores cut fp32 sums off: 3.1e-7 of their size over runs of 512 products, 6.6e-7 over runs of 1024, always
    towards zero, so that it shows in the mean over rows (whose spread, 1e-7 a row, is below 1e-8 then).  The bound is halfway."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(H)
    h = torch.randn(T, H, generator=gen).bfloat16().cuda()
    w = torch.zeros(8, H, dtype=torch.bfloat16)
    w[0] = (torch.randn(H, generator=gen) * 60 / H ** 0.5).bfloat16()
    w = w.cuda()
    logp, _ = ops.linear_logprobs(h, w, torch.ones(T, dtype=torch.long, device="cuda"))
    l = h.double() @ w[0].double()
    far = l > 25                                   # exp(-25) is 1e-11
    assert far.sum() > T // 8
    off = (-logp.double()[far] - (l + 7 * torch.exp(-l))[far]) / l[far]
    assert off.mean().abs() < 4.8e-7
