"""Counter-based dropout of adapters on several ranks, which all draw the same seeds: shards of a sequence have the mask of the whole, ranks
with other data another one, and what every rank of a sequence-parallel group computes alike has the same mask on each."""
import copy

import pytest
import torch

from dist_utils import run_distributed
from test_family_sequence_parallel import CONFIGS
from test_model_families import DSV3
from torchturbo_b200.engine.peft.lora import LoRALinear, LoraConfig

PEFT = {"r": 8, "lora_alpha": 8, "lora_dropout": 0.3, "counter_dropout": True, "target_modules": "all-linear", "target_experts": False}
KIMI = dict(model_type="kimi_k25", text_config=DSV3, media_placeholder_token_id=5,
            vision_config=dict(vt_num_hidden_layers=1, vt_hidden_size=16, vt_num_attention_heads=2, vt_intermediate_size=32, patch_size=2,
                               merge_kernel_size=(2, 2)))


def _layer():
    torch.manual_seed(0)
    layer = LoRALinear(torch.nn.Linear(32, 24), LoraConfig(r=8, lora_dropout=0.4, counter_dropout=True)).train()
    torch.nn.init.normal_(layer.lora_B["default"].weight)
    return layer


def _draw(layer, x):
    torch.manual_seed(7)
    return layer(x)


def test_shards_continue_and_replicas_differ():
    layer, x = _layer(), torch.randn(2, 30, 32, generator=torch.Generator().manual_seed(1))
    whole = _draw(layer, x)
    parts = []
    for shard, rows in enumerate(x.view(60, 32).split(15)):
        layer.shard = shard
        parts.append(_draw(layer, rows))
    assert torch.allclose(torch.cat(parts), whole.view(60, 24), rtol=1e-5, atol=1e-5)
    layer.replica, layer.shard = 1, 0
    other = _draw(layer, x)
    assert ((other - whole).abs() > 1e-3).view(60, 24).any(1).all()


def _w_places(rank, world, config, sp):
    from torchturbo_b200.engine import EngineConfig, TorchTurboEngine

    eng = TorchTurboEngine(EngineConfig.from_dict({"mixed_precision": "fp32", "parallel_plan": {"sp_size": sp, "ep_size": 1}}))
    model = eng.build_model(None, load_weights=False, init_kwargs={"config": copy.deepcopy(config), "seed": 0}, peft_config=dict(PEFT))
    layers = {n: (m.replica, m.shard) for n, m in model.named_modules() if isinstance(m, LoRALinear)}
    dp, shard = (rank, 0) if sp == 1 else (0, rank)
    seen = set()
    for n, place in layers.items():
        kind = next((k for k in ("vision_tower", "mm_projector", "compressor") if f".{k}." in f".{n}."), "rows")
        want = {"vision_tower": (rank, 0), "mm_projector": (dp, 0), "compressor": (dp, 0), "rows": (dp, shard)}[kind]
        assert place == want, (n, place, want)
        seen.add(kind)
    assert seen == ({"vision_tower", "mm_projector", "rows"} if "vision_config" in config else {"compressor", "rows"})


@pytest.mark.parametrize("sp", [1, 2])
@pytest.mark.parametrize("config", [KIMI, CONFIGS["deepseek_v4"]], ids=["kimi_k25", "deepseek_v4"])
def test_ranks_know_their_rows(config, sp):
    run_distributed(_w_places, 2, config, sp, timeout=600)


def _w_steps(rank, world, out):
    from torchturbo_b200.data import PackedCollator, SyntheticPackedDataset
    from torchturbo_b200.engine import EngineConfig, TorchTurboEngine
    from torchturbo_b200.engine.optimizers import OptimizerClassPlan
    from torchturbo_b200.loops import train_step

    eng = TorchTurboEngine(EngineConfig.from_dict({"mixed_precision": "fp32", "parallel_plan": {"sp_size": world, "ep_size": 1},
                                                   "activation_checkpointing": {"enabled": True}}))
    model = eng.build_model(None, load_weights=False, init_kwargs={"config": copy.deepcopy(CONFIGS["deepseek_v4"]), "seed": 0}, peft_config=dict(PEFT))
    opt = eng.prepare_optimizer(model, OptimizerClassPlan(torch.optim.AdamW, lr=1e-2, weight_decay=0.0))
    ds = SyntheticPackedDataset(3, 64, 128, num_docs=3, seed=11)
    hist = [[float(v) for v in train_step(eng, model, opt, [PackedCollator()([ds[i]])])[:2]] for i in range(3)]
    if rank == 0:
        torch.save(torch.tensor(hist), out)


def test_steps_with_two_shards_match_one(tmp_path):
    """Adapters of layers that gather the sequence, recomputed in the backward."""
    for world in (1, 2):
        run_distributed(_w_steps, world, str(tmp_path / f"{world}.pt"), timeout=900)
    a, b = (torch.load(tmp_path / f"{w}.pt") for w in (1, 2))
    assert torch.isfinite(a).all()
    assert torch.allclose(a[:, 0], b[:, 0], rtol=2e-4, atol=2e-5), (a, b)
    assert torch.allclose(a[:, 1], b[:, 1], rtol=5e-3, atol=1e-4), (a, b)
