"""Adapted layers whose widths the kernels do not take (a rank of 4, an odd output): their products stay in the layer's type, as without
`counter_dropout`, in place of fp32 copies of the operands."""
import pytest
import torch

from torchturbo_b200.engine.peft.lora import LoRALinear, LoraConfig
from torchturbo_b200.ops.dropout import dropout_args, keep_mask

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("inner, outer, rank", [(64, 48, 4), (64, 50, 8), (60, 48, 8), (64, 48, 8)])
@pytest.mark.parametrize("bias", [False, True])
def test_values_gradients_and_types(device, inner, outer, rank, bias):
    gen = torch.Generator().manual_seed(inner + outer + rank)
    layer = LoRALinear(torch.nn.Linear(inner, outer, bias=bias).to(device, torch.bfloat16), LoraConfig(r=rank, lora_alpha=2 * rank, lora_dropout=0.25,
                                                                                                   counter_dropout=True)).train()
    with torch.no_grad():
        layer.lora_B["default"].weight.copy_(torch.randn(outer, rank, generator=gen) * 0.2)
    x = torch.randn(3, 11, inner, generator=gen).to(device, torch.bfloat16).requires_grad_()
    dy = torch.randn(3, 11, outer, generator=gen).to(device, torch.bfloat16)
    wide = []

    class Widened(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if isinstance(out, torch.Tensor) and out.is_floating_point() and out.dtype != torch.bfloat16 and out.numel() >= outer * rank:
                wide.append((func, out.shape))
            return out

    torch.manual_seed(5)
    y = layer(x)
    y.backward(dy)
    weights = [layer.base_layer.weight.shape, layer.lora_A["default"].weight.shape, layer.lora_B["default"].weight.shape]
    with Widened():
        torch.manual_seed(5)
        again = layer(x)
    if device == "cuda" and (inner, outer, rank) != (64, 48, 8):
        assert not [s for _, s in wide if s in weights], "a weight was copied to fp32"
    assert torch.equal(again, y)
    torch.manual_seed(5)
    drop = dropout_args(0.25, int(torch.randint(0, 2 ** 62, (1,))))
    X, W = x.detach().double().cpu(), layer.base_layer.weight.double().cpu()
    b = layer.base_layer.bias.double().cpu() if bias else torch.zeros(outer, dtype=torch.float64)
    A, B = (getattr(layer, n)["default"].weight.detach().double().cpu() for n in ("lora_A", "lora_B"))
    keep = keep_mask(33, inner, drop, "cpu").view(3, 11, inner).double() * 65536 / (65536 - drop.t)
    dropped = X * keep
    want = X @ W.t() + b + 2.0 * dropped @ A.t() @ B.t()
    size = X.abs() @ W.abs().t() + b.abs() + 2.0 * dropped.abs() @ A.abs().t() @ B.abs().t()
    # the dropped input, the rows of A's product, up to two results of products and their sum are rounded to 2^-8 of their size
    unit = 5 * 2.0 ** -8
    assert y.dtype == torch.bfloat16 and ((y.detach().double().cpu() - want).abs() <= unit * size).all()
    D = dy.double().cpu()
    for got, ref, mag in ((x.grad, D @ W + 2.0 * (D @ B @ A) * keep, D.abs() @ W.abs() + 2.0 * (D.abs() @ B.abs() @ A.abs()) * keep),
                          (layer.lora_A["default"].weight.grad, 2.0 * torch.einsum("abr,abk->rk", D @ B, dropped),
                           2.0 * torch.einsum("abr,abk->rk", D.abs() @ B.abs(), dropped.abs())),
                          (layer.lora_B["default"].weight.grad, 2.0 * torch.einsum("abn,abr->nr", D, dropped @ A.t()),
                           2.0 * torch.einsum("abn,abr->nr", D.abs(), dropped.abs() @ A.abs().t()))):
        assert ((got.double().cpu() - ref).abs() <= unit * mag + 1e-12).all()
