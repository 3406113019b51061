"""The operators of an adapter, vision or preference training step around its matrix products: a linear layer with everything
that follows it (bias, activation, dropout, residual), dropout by itself, and per-token log-probabilities of the output head.

A case is a dict of plain values.  `prepare` makes what the caller has in hand, `run` is one call (with its gradients where the
case trains), in plain fp32 torch operations or, with `own`, through the package's operators; `exact` gives the same in 64 bits.

Kinds (sizes are those of this repository's model configurations and of its benchmark):

    linear      y = residual + dropout(act(x W^T + b))
    dropout     y = residual + dropout(x)
    logprobs    log softmax(h W^T)[target] per row, and the entropy of each row's distribution

Dropout masks come from Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011).  Columns 8 g to 8 g + 7 of row i take the eight
16-bit halves (low half first) of the four words drawn for the counter (g, 0, i mod 2^32, i div 2^32) under the seed's two
words; a value stays where its 16 bits are at least t = round(65536 p), times 65536 / (65536 - t).
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

BF16 = torch.bfloat16


def listed() -> list[dict]:
    return [
        # one token through the output projection of a vision merger: latency alone
        dict(name="linear_token", kind="linear", rows=1, k=1152, n=1152, bias=True, act=None, residual=True, p=0.0, train=False),
        # first layer of a ViT block's MLP over a handful of images, training (odd number of patches)
        dict(name="linear_patches", kind="linear", rows=3001, k=1152, n=4304, bias=True, act="gelu_tanh", residual=False, p=0.0,
             train=True),
        # second layer of the same MLP into the residual stream, scoring
        dict(name="linear_residual", kind="linear", rows=3001, k=4304, n=1152, bias=True, act=None, residual=True, p=0.0, train=False),
        # up-projection of a rank-16 adapter onto its layer's output, with dropout on the way: reads and writes are all it is
        dict(name="linear_adapter", kind="linear", rows=8190, k=16, n=4096, bias=False, act=None, residual=True, p=0.05, train=True),
        # a wide biased layer with GELU, dropout and residual over a long packed row, training
        dict(name="linear_wide", kind="linear", rows=8192, k=4096, n=12288, bias=True, act="gelu", residual=True, p=0.1, train=True),
        # adapter dropout of a short preference pair
        dict(name="dropout_short", kind="dropout", rows=61, n=2048, dtype="bf16", residual=False, p=0.05, train=True),
        # the same over a packed row with the residual stream, both directions
        dict(name="dropout_row", kind="dropout", rows=16384, n=4096, dtype="bf16", residual=True, p=0.1, train=True),
        # fp32 features of an odd width
        dict(name="dropout_odd", kind="dropout", rows=4097, n=1003, dtype="fp32", residual=False, p=0.5, train=False),
        # a few dozen answer tokens scored under the benchmark model's head: the weight is read once, little else
        dict(name="logprobs_short", kind="logprobs", rows=61, hidden=2048, vocab=151936, entropy=True, train=False),
        # a packed row scored under the frozen reference of a preference step
        dict(name="logprobs_score", kind="logprobs", rows=4096, hidden=2048, vocab=151936, entropy=False, train=False),
        # the policy's side of the same step: log-probabilities with their gradients
        dict(name="logprobs_train", kind="logprobs", rows=4096, hidden=2048, vocab=151936, entropy=False, train=True),
        # a policy-gradient step with an entropy term, odd row count and an odd vocabulary
        dict(name="logprobs_odd", kind="logprobs", rows=1501, hidden=4096, vocab=32003, entropy=True, train=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "dropout", "logprobs", "logprobs"])
    if kind == "linear":
        limit = 8192 * 4096 * 12288
        while True:
            c = dict(kind=kind, rows=_log(rng, 1, 16384), k=8 * _log(rng, 1, 1024), n=8 * _log(rng, 4, 1536), bias=rng.random() < 0.8,
                     act=rng.choice([None, "gelu", "gelu_tanh"]), residual=rng.random() < 0.6, p=rng.choice([0.0, 0.0, 0.05, 0.3]),
                     train=rng.random() < 0.5)
            if c["rows"] * c["k"] * c["n"] <= limit:
                return c
    if kind == "dropout":
        return dict(kind=kind, rows=_log(rng, 1, 16384), n=_log(rng, 8, 4096), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    residual=rng.random() < 0.4, p=rng.choice([0.05, 0.1, 0.5, 0.9]), train=rng.random() < 0.5)
    limit = 4096 * 2048 * 151936
    while True:
        c = dict(kind=kind, rows=_log(rng, 1, 8192), hidden=8 * _log(rng, 32, 640), vocab=_log(rng, 4000, 160000), entropy=rng.random() < 0.5,
                 train=rng.random() < 0.5)
        if c["rows"] * c["hidden"] * c["vocab"] <= limit:
            return c


class _Maker:
    def __init__(self, seed: int):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=BF16):
        out = torch.empty(*shape, device="cuda", dtype=dtype)
        for part in out.split(8192) if out.dim() == 2 else (out,):       # large weights without an fp32 copy of the whole
            part.copy_(torch.randn(part.shape, generator=self.gen, device="cuda") * std)
        return out

    def seed(self) -> int:
        return int(torch.randint(0, 2 ** 62, (1,), generator=self.gen, device="cuda"))


def prepare(case: dict, seed: int) -> SimpleNamespace:
    make, kind, train = _Maker(seed), case["kind"], case["train"]
    s = SimpleNamespace(case=case, kind=kind, bias=None, residual=None)
    R = case["rows"]
    if kind == "linear":
        K, N = case["k"], case["n"]
        s.x = make.normal(R, K)
        s.w = make.normal(N, K, std=K ** -0.5)
        if case["bias"]:
            s.bias = make.normal(N, std=0.1)
        if case["residual"]:
            s.residual = make.normal(R, N, std=2.0)
        s.dy = make.normal(R, N, std=1e-2) if train else None
        s.leaves = [t for t in (s.x, s.w, s.bias, s.residual) if t is not None]
    elif kind == "dropout":
        dt = BF16 if case["dtype"] == "bf16" else torch.float32
        s.x = make.normal(R, case["n"], dtype=dt)
        if case["residual"]:
            s.residual = make.normal(R, case["n"], std=2.0, dtype=dt)
        s.dy = make.normal(R, case["n"], std=1e-2, dtype=dt) if train else None
        s.leaves = [t for t in (s.x, s.residual) if t is not None]
    else:
        # Logits as of a trained head: a spread of about 2.5, and for most rows a target that stands out by what the row's hidden
        # state shares with the target's weights.  A tenth of the rows are prompt tokens without a target.
        H, V = case["hidden"], case["vocab"]
        s.w = make.normal(V, H, std=2.5 * H ** -0.5)
        s.targets = torch.randint(0, V, (R,), generator=make.gen, device="cuda")
        pull = torch.rand(R, 1, generator=make.gen, device="cuda") * 2.0
        s.x = (make.normal(R, H, dtype=torch.float32) + pull * s.w[s.targets].float()).to(BF16)
        s.targets[torch.rand(R, generator=make.gen, device="cuda") < 0.1] = -100
        s.dlogp = make.normal(R, std=1e-2, dtype=torch.float32) if train else None
        s.dent = make.normal(R, std=1e-3, dtype=torch.float32) if train and case["entropy"] else None
        s.leaves = [s.x, s.w]
    s.seed = make.seed()
    for t in s.leaves:
        t.requires_grad_(train)
    return s


# ------------------------------------------------------------------------------------------------
# plain form
# ------------------------------------------------------------------------------------------------
_M0, _M1, _W0, _W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85


def _draws(rows: int, cols: int, seed: int) -> torch.Tensor:
    """[rows, cols] 16-bit draws as int32.  Words are held in int64: a product of two wraps, its low 64 bits stay right."""
    lo32 = 0xFFFFFFFF
    groups = (cols + 7) // 8
    zero = torch.zeros((rows, groups), dtype=torch.int64, device="cuda")
    c0, c1 = zero + torch.arange(groups, device="cuda"), zero
    c2, c3 = zero + torch.arange(rows, device="cuda")[:, None], zero
    k0, k1 = seed & lo32, seed >> 32
    for _ in range(10):
        a, b = c0 * _M0, c2 * _M1
        c0, c1, c2, c3 = ((b >> 32) & lo32) ^ c1 ^ k0, b & lo32, ((a >> 32) & lo32) ^ c3 ^ k1, a & lo32
        k0, k1 = (k0 + _W0) & lo32, (k1 + _W1) & lo32
    words = torch.stack((c0, c1, c2, c3), -1)
    halves = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, groups * 8)
    return halves[:, :cols].to(torch.int32)


def _factor(rows: int, cols: int, p: float, seed: int) -> torch.Tensor:
    t = round(65536 * p)
    return (_draws(rows, cols, seed) >= t).float() * (65536 / (65536 - t))


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain(s):
    c = s.case
    if s.kind == "linear":
        x, w = s.x.float(), s.w.float()
        z = x @ w.t()
        if s.bias is not None:
            z = z + s.bias.float()
        f = _factor(c["rows"], c["n"], c["p"], s.seed) if c["p"] else None
        y = _act(z, c["act"])
        if f is not None:
            y = y * f
        if s.residual is not None:
            y = y + s.residual.float()
        out = dict(y=y.to(BF16))
        if c["train"]:
            dz = s.dy.float() if f is None else s.dy.float() * f
            if c["act"]:
                dz = dz * _act_slope(z, c["act"])
            out.update(dx=(dz @ w).to(BF16), dw=(dz.t() @ x).to(BF16))
            if s.bias is not None:
                out["dbias"] = dz.sum(0).to(BF16)
            if s.residual is not None:
                out["dresidual"] = s.dy
        return out
    if s.kind == "dropout":
        f = _factor(c["rows"], c["n"], c["p"], s.seed)
        y = s.x.float() * f
        if s.residual is not None:
            y = y + s.residual.float()
        out = dict(y=y.to(s.x.dtype))
        if c["train"]:
            out["dx"] = (s.dy.float() * f).to(s.x.dtype)
            if s.residual is not None:
                out["dresidual"] = s.dy
        return out
    x, w = s.x.float(), s.w.float()
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    has = s.targets >= 0
    at = s.targets.clamp(min=0)[:, None]
    logp = torch.where(has, (logits.gather(1, at) - lse)[:, 0], 0.0)
    out = dict(logp=logp)
    p = e.div_(total)
    logits.sub_(lse)                                   # log-probabilities
    ent = None
    if c["entropy"]:
        ent = out["entropy"] = -(p * logits).sum(1)
    if c["train"]:
        g = torch.where(has, s.dlogp, 0.0)[:, None]
        dl = -g * p
        if c["entropy"]:
            dl -= s.dent[:, None] * p * (logits + ent[:, None])
        dl.scatter_add_(1, at, g)
        out.update(dh=(dl @ w).to(BF16), dw=(dl.t() @ x).to(BF16))
    return out


def run(s):
    """One pass: the call and, where the case trains, the gradients of everything that has one."""
    if not own:
        with torch.no_grad():
            return _plain(s)
    from torchturbo_b200.ops import ops

    c = s.case
    with torch.set_grad_enabled(c["train"]):
        if s.kind == "logprobs":
            logp, ent = ops.linear_logprobs(s.x, s.w, s.targets, want_entropy=c["entropy"])
            out = dict(logp=logp) if ent is None else dict(logp=logp, entropy=ent)
            if c["train"]:
                ys, gs = ((logp,), (s.dlogp,)) if ent is None else ((logp, ent), (s.dlogp, s.dent))
                out["dh"], out["dw"] = torch.autograd.grad(ys, s.leaves, gs)
            return out
        if s.kind == "linear":
            y = ops.linear_bias_act(s.x, s.w, s.bias, c["act"], residual=s.residual, dropout_p=c["p"], seed=s.seed)
            names = ["dx", "dw"] + ["dbias"] * (s.bias is not None)
        else:
            y = ops.dropout(s.x, c["p"], s.seed, residual=s.residual)
            names = ["dx"]
        out = dict(y=y)
        if c["train"]:
            out.update(zip(names + ["dresidual"] * (s.residual is not None), torch.autograd.grad(y, s.leaves, s.dy)))
        return out


def work(case: dict) -> dict:
    R = case["rows"]
    if case["kind"] == "linear":
        K, N = case["k"], case["n"]
        rows, weights = R * K * 2, N * K * 2 + (N * 2 if case["bias"] else 0)
        res = R * N * 2 if case["residual"] else 0
        if case["train"]:                                      # and dy in; dx, dW, db and the residual's gradient (dy itself) out
            return dict(bytes=2 * (rows + weights) + res + 2 * R * N * 2, flops=6 * R * K * N)
        return dict(bytes=rows + weights + res + R * N * 2, flops=2 * R * K * N)
    if case["kind"] == "dropout":
        one = R * case["n"] * (2 if case["dtype"] == "bf16" else 4)
        return dict(bytes=one * (2 + case["residual"] + 2 * case["train"]), flops=2 * R * case["n"] * (1 + case["train"]))
    H, V = case["hidden"], case["vocab"]
    rows, weights, each = R * H * 2, V * H * 2, R * 4 * (2 if case["entropy"] else 1)
    if case["train"]:                                          # the logits are not kept, so that their gradient takes a second product
        return dict(bytes=2 * (rows + weights) + R * 8 + 2 * each, flops=8 * R * H * V)
    return dict(bytes=rows + weights + R * 8 + each, flops=2 * R * H * V)


# ------------------------------------------------------------------------------------------------
# the same in 64 bits
# ------------------------------------------------------------------------------------------------
def _mask64(rows: int, cols: int, p: float, seed: int) -> torch.Tensor:
    """The factors of dropout from 64-bit words on the host, one counter after the other along the last axis."""
    g = -(-cols // 8)
    ctr = np.zeros((4, rows, g), dtype=np.uint64)
    ctr[0] = np.arange(g, dtype=np.uint64)
    ctr[2] = np.arange(rows, dtype=np.uint64)[:, None]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    key = [seed % 2 ** 32, seed // 2 ** 32]
    for i in range(10):
        left, right = ctr[0] * np.uint64(_M0), ctr[2] * np.uint64(_M1)
        k = [np.uint64((key[0] + i * _W0) % 2 ** 32), np.uint64((key[1] + i * _W1) % 2 ** 32)]
        ctr = np.stack((right >> half ^ ctr[1] ^ k[0], right & low, left >> half ^ ctr[3] ^ k[1], left & low))
    u = np.ascontiguousarray(np.moveaxis(ctr, 0, -1).astype("<u4")).view("<u2").reshape(rows, g * 8)[:, :cols]
    t = int(round(p * 2 ** 16))
    return torch.from_numpy((u >= t) / (1 - t / 2 ** 16)).cuda()


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, train = case["kind"], case["train"]
    with torch.no_grad():
        if kind == "logprobs":
            return _exact_logprobs(s)
        x = s.x.double()
        keep = _mask64(case["rows"], case["n"], case["p"], s.seed) if case["p"] else None
        res = 0.0 if s.residual is None else s.residual.double()
        grads = {} if s.residual is None or not train else dict(dresidual=s.dy.double())
        if kind == "dropout":
            out = dict(y=x * keep + res)
            if train:
                out["dx"] = s.dy.double() * keep
            return dict(out, **grads)
        w = s.w.double()
        z = torch.matmul(x, w.T) + (0.0 if s.bias is None else s.bias.double())
        with torch.enable_grad():
            z = z.requires_grad_(train)
            a = z
            if case["act"]:
                a = torch.nn.functional.gelu(z, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
            y = (a if keep is None else a * keep) + res
        out = dict(y=y.detach())
        if train:
            dz, = torch.autograd.grad(y, z, s.dy.double())
            out.update(dx=torch.matmul(dz, w), dw=torch.matmul(dz.T, x))
            if s.bias is not None:
                out["dbias"] = dz.sum(0)
        return dict(out, **grads)


def _exact_logprobs(s):
    """Rows in blocks: 64-bit logits of all of them would not be held."""
    c, w = s.case, s.w.double()
    logps, ents, dhs, dw = [], [], [], torch.zeros_like(w) if s.case["train"] else None
    for a in range(0, c["rows"], 512):
        x, tg = s.x[a:a + 512].double(), s.targets[a:a + 512]
        logq = torch.log_softmax(torch.matmul(x, w.T), 1)
        q, on = torch.exp(logq), torch.nn.functional.one_hot(tg.clamp(min=0), c["vocab"]) * (tg >= 0)[:, None]
        logps.append((logq * on).sum(1))
        ents.append(-(q * logq).sum(1))
        if c["train"]:
            g = s.dlogp[a:a + 512].double() * (tg >= 0)
            d = (on - q) * g[:, None]
            if c["entropy"]:
                d -= s.dent[a:a + 512].double()[:, None] * q * (logq + ents[-1][:, None])
            dhs.append(torch.matmul(d, w))
            dw += torch.matmul(d.T, x)
    out = dict(logp=torch.cat(logps))
    if c["entropy"]:
        out["entropy"] = torch.cat(ents)
    if c["train"]:
        out.update(dh=torch.cat(dhs), dw=dw)
    return out
