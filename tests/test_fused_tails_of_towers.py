"""`fused_linear_tails` of a vision configuration reaches every biased layer behind it: Kimi's tower and projector and Bailing's projector."""
import pytest
import torch

import torchturbo_b200.models.qwen3_vl.modeling as shared
from test_model_families import _build
from test_moonvit import CFG, GRID
from torchturbo_b200.models.bailing_moe_v3_vl.model import _Projector
from torchturbo_b200.models.kimi_k25.vision import MoonViT, MoonViTConfig, PatchMergerMLP, init_moonvit

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture
def calls(monkeypatch):
    """How often the product with a tail is asked for."""
    seen = []
    whole = shared.ops

    class Ops:
        def __getattr__(self, name):
            if name == "linear_bias_act":
                seen.append(name)
            return getattr(whole, name)

    monkeypatch.setattr(shared, "ops", Ops())
    return seen


@pytest.mark.parametrize("device", DEVICES)
def test_kimi_tower_and_projector(device, calls):
    torch.manual_seed(0)
    mods = []
    for fused in (False, True):
        cfg = MoonViTConfig(**CFG, fused_linear_tails=fused)
        mods.append((MoonViT(cfg, torch.float32), PatchMergerMLP(cfg, torch.float32)))
    init_moonvit(*mods[0], 0.05)
    pixels, grid = torch.randn(sum(t * h * w for t, h, w in GRID), 3, 14, 14), torch.tensor(GRID)
    got = []
    for tower, proj in mods:
        for m, ref in zip((tower, proj), mods[0]):
            m.load_state_dict(ref.state_dict())
        # both ways in fp32: operations in another order (on the GPU with the products' own tiles)
        tower, proj = tower.to(device), proj.to(device)
        y = proj(tower(pixels.to(device), grid))
        got.append([y, *torch.autograd.grad(y.square().sum(), [*tower.encoder.parameters(), *proj.parameters()])])
        assert len(calls) == (0 if len(got) == 1 else 4 * CFG["vt_num_hidden_layers"] + 2)
    for a, b in zip(*got):
        assert (a - b).norm() <= 1e-4 * b.norm() + 1e-6


@pytest.mark.parametrize("fused", [False, True])
def test_bailing_projector_takes_the_vision_configuration(fused, calls):
    cls, model = _build("bailing_moe_v3_vl")
    cfg = model.config
    cfg.vision_config.fused_linear_tails = fused
    other = cls(cfg)
    other.load_state_dict(model.state_dict())
    assert isinstance(other.linear_proj, _Projector) and other.linear_proj.fused is fused
    feats = torch.randn(6, other.linear_proj[0].in_features, generator=torch.Generator().manual_seed(1))
    want, y = model.linear_proj(feats), other.linear_proj(feats)
    assert len(calls) == (2 if fused else 0) and torch.allclose(y, want, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("inner, outer", [(64, 50), (60, 48)])
def test_other_widths_keep_their_separate_passes(device, inner, outer, calls):
    """Widths that are no multiple of eight: the operands are not copied to fp32 for a product with a tail."""
    torch.manual_seed(0)
    lin = torch.nn.Linear(inner, outer, device=device, dtype=torch.bfloat16)
    x, r = (torch.randn(9, n, device=device, dtype=torch.bfloat16) for n in (inner, outer))
    got = [shared.linear_tail(fused, x, lin, "gelu", residual=r) for fused in (True, False)]
    assert torch.equal(*got) and not calls
