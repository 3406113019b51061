"""The biased linear layer's tail, counter-based dropout and log-probabilities without logits on the framework's own paths: LoRA, vision
blocks, preference and policy-gradient steps, and a run of them together."""
import pytest
import torch

from dist_utils import run_distributed
from test_dpo_loop import DENSE, _pair_row
from torchturbo_b200.engine import EngineConfig, TorchTurboEngine
from torchturbo_b200.engine.peft.lora import LoRALinear, LoraConfig
from torchturbo_b200.loops.dpo import DPOConfig, dpo_step, sequence_logps
from torchturbo_b200.ops import ops
from torchturbo_b200.ops.dropout import dropout_args, keep_mask

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _engine(device):
    return TorchTurboEngine(EngineConfig.from_dict({"mixed_precision": "fp32" if device == "cpu" else "bf16"}))


@pytest.mark.parametrize("device", DEVICES)
def test_lora_layer_with_counter_dropout(device):
    """Base + B (A dropout(x)) scale, mask by the seed that the host's generator gives; its gradients by the same mask; evaluation merges."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    gen = torch.Generator().manual_seed(0)
    lin = torch.nn.Linear(64, 48).to(device, dtype)
    layer = LoRALinear(lin, LoraConfig(r=8, lora_alpha=16, lora_dropout=0.25, counter_dropout=True)).train()
    with torch.no_grad():
        layer.lora_B["default"].weight.copy_(torch.randn(48, 8, generator=gen) * 0.2)
    x = torch.randn(5, 7, 64, generator=gen).to(device, dtype).requires_grad_()
    torch.manual_seed(3)
    y = layer(x)
    torch.manual_seed(3)
    seed = int(torch.randint(0, 2 ** 62, (1,)))
    drop = dropout_args(0.25, seed)
    X, W, b = x.detach().double().cpu(), lin.weight.double().cpu(), lin.bias.double().cpu()
    A, B = layer.lora_A["default"].weight.double().cpu(), layer.lora_B["default"].weight.double().cpu()
    keep = keep_mask(35, 64, drop, "cpu").view(5, 7, 64).double() * 65536 / (65536 - drop.t)
    dropped = X * keep
    want = X @ W.t() + b + 2.0 * dropped @ A.t() @ B.t()
    # fp32: products of 64; bf16: x, the rows of A's product and both results are rounded to 2^-8 of their size
    size = X.abs() @ W.abs().t() + b.abs() + 2.0 * dropped.abs() @ A.abs().t() @ B.abs().t()
    unit = 2.0 ** -20 if device == "cpu" else 2.0 ** -6
    assert ((y.detach().double().cpu() - want).abs() <= unit * size).all()
    dy = torch.randn(y.shape, generator=gen).to(device, dtype)
    y.backward(dy)
    D = dy.double().cpu()
    for got, ref, mag in ((x.grad, D @ W + 2.0 * (D @ B @ A) * keep, D.abs() @ W.abs() + 2.0 * (D.abs() @ B.abs() @ A.abs()) * keep),
                          (layer.lora_A["default"].weight.grad, 2.0 * torch.einsum("abr,abk->rk", D @ B, dropped),
                           2.0 * torch.einsum("abr,abk->rk", D.abs() @ B.abs(), dropped.abs())),
                          (layer.lora_B["default"].weight.grad, 2.0 * torch.einsum("abn,abr->nr", D, dropped @ A.t()),
                           2.0 * torch.einsum("abn,abr->nr", D.abs(), dropped.abs() @ A.abs().t()))):
        assert ((got.double().cpu() - ref).abs() <= unit * mag + 1e-12).all()
    assert lin.weight.grad is None and lin.bias.grad is None
    layer.eval()
    assert torch.equal(layer(x), torch.nn.functional.linear(x, layer.weight, layer.bias))


def test_lora_layer_keeps_torch_dropout_by_default():
    lin = torch.nn.Linear(16, 8)
    layer = LoRALinear(lin, LoraConfig(r=2, lora_dropout=0.5)).train()
    torch.nn.init.ones_(layer.lora_B["default"].weight)
    x = torch.randn(3, 16)
    torch.manual_seed(1)
    y = layer(x)
    torch.manual_seed(1)
    want = lin(x) + layer.lora_B["default"](layer.lora_A["default"](torch.nn.functional.dropout(x, 0.5))) * layer.cfg.scaling
    assert torch.equal(y, want)


def test_recomputed_forward_draws_the_same_mask():
    from torch.utils.checkpoint import checkpoint

    layer = LoRALinear(torch.nn.Linear(16, 8), LoraConfig(r=2, lora_dropout=0.5, counter_dropout=True)).train()
    torch.nn.init.ones_(layer.lora_B["default"].weight)
    x = torch.randn(3, 16, requires_grad=True)
    grads = []
    for run in (lambda: layer(x), lambda: checkpoint(layer, x, use_reentrant=False)):
        torch.manual_seed(1)
        grads.append(torch.autograd.grad(run().square().sum(), [x, *(p for p in layer.parameters() if p.requires_grad)]))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("device", DEVICES)
def test_vision_block_with_fused_tails(device):
    """The same block and merger both ways: in fp32 alike, in bf16 no further from fp32 than the separate passes."""
    from types import SimpleNamespace

    from torchturbo_b200.models.qwen3_vl.modeling import PatchMerger, VisionBlock, vision_rot_pos

    cfg = dict(hidden_size=128, num_heads=2, intermediate_size=264, spatial_merge_size=2, out_hidden_size=72)
    grid = torch.tensor([[1, 6, 8], [1, 4, 4]])
    cu = torch.tensor([0, 48, 64], dtype=torch.int32)
    gen = torch.Generator().manual_seed(5)
    torch.manual_seed(5)
    mods = [VisionBlock(SimpleNamespace(**cfg)), PatchMerger(SimpleNamespace(**cfg))]
    x0, dy0 = torch.randn(64, 128, generator=gen), torch.randn(16, 72, generator=gen)

    def run(dev, dtype, fused):
        blk, mer = (type(m)(SimpleNamespace(**cfg, fused_linear_tails=fused)).to(dev, dtype) for m in mods)
        for a, b in zip((blk, mer), mods):
            a.load_state_dict(b.state_dict())
        cos, sin = vision_rot_pos(grid, 2, 64, torch.device(dev))
        x = x0.to(dev, dtype).requires_grad_()
        y = mer(blk(x, cos, sin, cu, 48))
        grads = torch.autograd.grad(y, [x, *blk.parameters(), *mer.parameters()], dy0.to(dev, dtype))
        return [t.detach().double().cpu() for t in (y, *grads)]

    want = run("cpu", torch.float32, False)
    if device == "cpu":
        # the same fp32 operations in another order: a few steps of 2^-23 times the sums' lengths
        for a, b in zip(run("cpu", torch.float32, True), want):
            assert (a - b).norm() <= 1e-4 * b.norm() + 1e-6
        return
    for a, b, c in zip(run("cuda", torch.bfloat16, True), run("cuda", torch.bfloat16, False), want):
        # roundings of the same kind in both, fewer in the fused form; 1.25 for the luck of the draw, and key biases have no gradient but roundings
        assert (a - c).norm() <= 1.25 * (b - c).norm() + 2.0 ** -8 * c.norm()


def _on(device, worker):
    """CPU engines set up a process group: in a process of their own."""
    run_distributed(worker, 1, device) if device == "cpu" else worker(0, 1, device)


@pytest.mark.parametrize("device", DEVICES)
def test_preference_step_without_logits(device):
    _on(device, _w_preference)


@pytest.mark.parametrize("device", DEVICES)
def test_policy_gradient_batch_without_logits(device):
    _on(device, _w_policy)


def _w_preference(rank, world, device):
    """Segment log-probabilities with and without logits agree, their gradients too, and a step runs."""
    engine = _engine(device)
    cfg = dict(DENSE) if device == "cpu" else dict(DENSE, head_dim=128, hidden_size=256, intermediate_size=512)
    model = engine.build_model(None, load_weights=False, init_kwargs={"config": cfg})
    batch = _pair_row(0)
    out = {}
    for fused in (False, True):
        sums, counts = sequence_logps(engine, model, dict(batch), DPOConfig(fused_logps=fused), grad=True)
        params = [p for p in model.parameters() if p.requires_grad]
        out[fused] = (sums.detach(), torch.autograd.grad(sums.sum(), params, allow_unused=True))
    tol = 1e-5 if device == "cpu" else 2.0 ** -6      # logits rounded to bf16 in one of them: 2^-9 of up to 1 each, 9 targets a segment
    assert (out[True][0] - out[False][0]).abs().max() <= tol * out[False][0].abs().max()
    for a, b in zip(out[True][1], out[False][1]):
        assert (a is None) == (b is None)
        if a is not None:
            assert (a.float() - b.float()).norm() <= (1e-4 if device == "cpu" else 0.05) * b.float().norm() + 1e-6
    from torchturbo_b200.engine.optimizers import OptimizerClassPlan

    optim = engine.prepare_optimizer(model, OptimizerClassPlan(torch.optim.AdamW, lr=1e-4))
    loss, gnorm, metrics = dpo_step(engine, model, model, optim, dict(batch), DPOConfig(fused_logps=True))
    assert torch.isfinite(loss) and torch.isfinite(gnorm) and abs(float(metrics["rewards/margins"])) < 1e-3


def _w_policy(rank, world, device):
    engine = _engine(device)
    cfg = dict(DENSE) if device == "cpu" else dict(DENSE, head_dim=128, hidden_size=256, intermediate_size=512)
    model = engine.build_model(None, load_weights=False, init_kwargs={"config": cfg})
    gen = torch.Generator().manual_seed(1)
    seqs = [torch.randint(1, 256, (n,), generator=gen) for n in (9, 1, 14)]
    mb = engine.prepare_packed_micro_batch(seqs, {"loss_mask": [torch.ones(len(s)) for s in seqs]})
    plain = engine.compute_logprobs(model, [mb], want_entropy=True)[0]
    fused = engine.compute_logprobs(model, [mb], want_entropy=True, fused=True)[0]
    tol = 1e-5 if device == "cpu" else 2.0 ** -6
    for a, b in zip(fused, plain):
        assert a.shape == b.shape and (a - b).abs().max() <= tol * max(1.0, float(b.abs().max()))
    grads = []
    for f in (False, True):
        model.zero_grad()
        engine.forward_backward_batch(model, [mb], lambda lp, ent, m: -lp - 0.01 * ent, want_entropy=True, fused=f)
        grads.append([p.grad.float().clone() for p in model.parameters() if p.grad is not None])
    assert len(grads[0]) == len(grads[1]) > 0
    for a, b in zip(*grads):
        assert (a - b).norm() <= (1e-4 if device == "cpu" else 0.05) * b.norm() + 1e-6


@pytest.mark.parametrize("device", DEVICES)
def test_a_run_of_them_together(device):
    """A residual block of two biased layers with GELU and dropout, a LoRA branch with dropout and the head's log-probabilities with an
    entropy term, against the same in 64 bits under the same masks."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    gen = torch.Generator().manual_seed(7)
    T, H, I, V = 37, 64, 136, 301
    shapes = dict(x=(T, H), w1=(I, H), b1=(I,), w2=(H, I), b2=(H,), a=(8, H), b=(H, 8), head=(V, H))
    t = {k: (torch.randn(*s, generator=gen) * (1.0 if k == "x" else s[-1] ** -0.5)).to(dtype) for k, s in shapes.items()}
    targets = torch.randint(-1, V, (T,), generator=gen)
    g = torch.randn(T, generator=gen)

    def by_operators(v, tg, gw):
        h = ops.linear_bias_act(v["x"], v["w1"], v["b1"], "gelu", dropout_p=0.1, seed=11)
        y = ops.linear_bias_act(h, v["w2"], v["b2"], residual=v["x"], dropout_p=0.2, seed=12)
        y = ops.linear_bias_act(ops.linear(ops.dropout(y, 0.3, 13), v["a"]), v["b"], residual=y)
        logp, ent = ops.linear_logprobs(y, v["head"], tg, want_entropy=True)
        return (gw * logp).sum() + 0.05 * ent.sum()

    def by_formula(v):
        def keep(cols, p, seed):
            d = dropout_args(p, seed)
            return keep_mask(T, cols, d, "cpu").double() * 65536 / (65536 - d.t)

        h = torch.nn.functional.gelu(v["x"] @ v["w1"].t() + v["b1"]) * keep(I, 0.1, 11)
        y = v["x"] + (h @ v["w2"].t() + v["b2"]) * keep(H, 0.2, 12)
        y = y + (y * keep(H, 0.3, 13)) @ v["a"].t() @ v["b"].t()
        lq = torch.log_softmax(y @ v["head"].t(), -1)
        ok = targets >= 0
        return (g.double() * torch.where(ok, lq.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)).sum() - 0.05 * (lq.exp() * lq).sum()

    leaves = {k: v.to(device).requires_grad_() for k, v in t.items()}
    loss = by_operators(leaves, targets.to(device), g.to(device))
    grads = torch.autograd.grad(loss, list(leaves.values()))
    exact = {k: v.double().requires_grad_() for k, v in t.items()}
    want = by_formula(exact)
    refs = torch.autograd.grad(want, list(exact.values()))
    # about a dozen bf16 roundings between a leaf and the loss and back, each at most 2^-8 in the 2-norm (fp32: 2^-20 with the sums)
    unit = 1e-5 if device == "cpu" else 12 * 2.0 ** -8
    assert abs(float(loss.detach()) - float(want.detach())) <= unit * float(g.abs().sum() * 6)
    for a, b in zip(grads, refs):
        assert (a.double().cpu() - b).norm() <= unit * b.norm()
