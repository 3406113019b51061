"""Counter-based dropout, the biased linear layer with activation, dropout and residual, and per-token log-probabilities of the output
head: plain formulations against the formulas in 64 bits, gradients against differences, and refusals."""
import math

import numpy as np
import pytest
import torch

from torchturbo_b200.ops import ops
from torchturbo_b200.ops.dropout import Dropout, dropout_args, keep_mask, philox


def _draws(rows, cols, seed, first_row=0):
    """[rows, cols] 16-bit draws, one counter at a time in Python integers."""
    out = np.zeros((rows, cols), dtype=np.int64)
    for i in range(rows):
        for g in range((cols + 7) // 8):
            r = first_row + i
            words = philox(g, 0, r % 2 ** 32, r >> 32, seed % 2 ** 32, seed >> 32)
            halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
            n = min(8, cols - 8 * g)
            out[i, 8 * g: 8 * g + n] = halves[:n]
    return torch.from_numpy(out)


# known answers published with the generator
@pytest.mark.parametrize("counter, key, words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_known_answers(counter, key, words):
    assert philox(*counter, *key) == words
    assert tuple(int(w) for w in philox(*(torch.tensor(c) for c in counter), *key)) == words


@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (5, 8), (2, 21), (0, 8)])
@pytest.mark.parametrize("seed", [0, 2 ** 62 + 12345])
@pytest.mark.parametrize("first_row", [0, 2 ** 32 - 1])
def test_mask_by_counter(rows, cols, seed, first_row):
    drop = dropout_args(0.4, seed, first_row)
    assert drop.t == round(0.4 * 65536)
    want = _draws(rows, cols, seed, first_row) >= drop.t
    assert torch.equal(keep_mask(rows, cols, drop, "cpu"), want)
    x = torch.randn(rows, cols, dtype=torch.float64)
    y = ops.dropout(x, 0.4, seed, first_row=first_row)
    assert torch.equal(y, torch.where(want, x * (65536 / (65536 - drop.t)), 0.0))
    tensor = ops.dropout(x, 0.4, torch.tensor([seed]), first_row=first_row)
    assert torch.equal(tensor, y)


def test_shards_and_leading_dimensions():
    x = torch.randn(2, 6, 10)
    whole = ops.dropout(x, 0.3, 7)
    flat = x.view(12, 10)
    parts = [ops.dropout(flat[a:b], 0.3, 7, first_row=a) for a, b in ((0, 5), (5, 6), (6, 12))]
    assert torch.equal(whole.view(12, 10), torch.cat(parts))
    w, b = torch.randn(16, 10), torch.randn(16)
    y = ops.linear_bias_act(x, w, b, "gelu", dropout_p=0.3, seed=9)
    rows = [ops.linear_bias_act(flat[a:c], w, b, "gelu", dropout_p=0.3, seed=9, first_row=a) for a, c in ((0, 7), (7, 12))]
    assert torch.allclose(y.view(12, 16), torch.cat(rows), atol=1e-6)
    assert torch.equal(y == 0, torch.cat(rows).view_as(y) == 0)


def test_share_that_stays():
    """Of n draws with probability q of staying, the count is within six standard deviations; kept values keep the mean."""
    n, p = 1 << 18, 0.1
    kept = keep_mask(1 << 10, 1 << 8, dropout_args(p, 3), "cpu")
    assert abs(int(kept.sum()) - n * (1 - p)) < 6 * math.sqrt(n * p * (1 - p))
    assert abs(float(kept[:, ::2].float().mean() - kept[:, 1::2].float().mean())) < 6 * math.sqrt(4 * p * (1 - p) / n)


def test_nothing_and_everything_dropped():
    x, r = torch.randn(4, 9), torch.randn(4, 9)
    assert torch.equal(ops.dropout(x, 0.0), x) and torch.equal(ops.dropout(x, 0.0, scale=2.0), 2 * x)
    assert torch.equal(ops.dropout(x, 1.0, 1), torch.zeros_like(x)) and torch.equal(ops.dropout(x, 1.0, 1, residual=r), r)
    bad = torch.full((4, 9), float("nan"))
    assert torch.equal(ops.dropout(bad, 1.0, 1), torch.zeros_like(x))


def test_seed_from_the_generator_of_the_host():
    x = torch.ones(64, 64)
    torch.manual_seed(5)
    a, b = ops.dropout(x, 0.5), ops.dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(a, ops.dropout(x, 0.5)) and not torch.equal(a, b)


@pytest.mark.parametrize("bad", [dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(p=float("inf")), dict(p=0.1, seed=-1), dict(p=0.1, seed=2 ** 63), dict(p=0.1, seed=1.0),
                                 dict(p=0.1, seed=True), dict(p=0.1, seed=torch.tensor([1, 2])), dict(p=0.1, seed=torch.tensor(1.0)),
                                 dict(p=0.1, seed=1, first_row=-1)])
def test_refused_dropout_arguments(bad):
    with pytest.raises(ValueError):
        ops.dropout(torch.ones(2, 8), **bad)


def test_refused_shapes():
    x, w = torch.ones(2, 8), torch.ones(4, 8)
    for call in (lambda: ops.dropout(x, 0.1, 1, residual=torch.ones(2, 1)),
                 lambda: ops.dropout(x, 0.1, 1, residual=torch.ones(2, 8, dtype=torch.float64)),
                 lambda: ops.dropout(torch.ones(2, 8, dtype=torch.long), 0.1, 1),
                 lambda: ops.dropout(torch.tensor(1.0), 0.1, 1),
                 lambda: ops.linear_bias_act(x, torch.ones(4, 9)),
                 lambda: ops.linear_bias_act(x, w, torch.ones(1)),
                 lambda: ops.linear_bias_act(x, w, act="relu6"),
                 lambda: ops.linear_bias_act(x, w, residual=torch.ones(4)),
                 lambda: ops.linear_bias_act(x, w, residual=torch.ones(2, 1)),
                 lambda: ops.linear_bias_act(x, w, dropout_p=2.0),
                 lambda: ops.linear_bias_act(x, torch.ones(4, 8, device="meta")),
                 lambda: ops.linear_logprobs(x, torch.ones(4, 9), torch.zeros(2, dtype=torch.long)),
                 lambda: ops.linear_logprobs(x, w, torch.zeros(3, dtype=torch.long)),
                 lambda: ops.linear_logprobs(x, w, torch.zeros(2)),
                 lambda: ops.linear_logprobs(x, torch.ones(0, 8), torch.zeros(2, dtype=torch.long))):
        with pytest.raises(ValueError):
            call()


def _gelu(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh"])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("biased, with_res", [(True, True), (False, False), (True, False)])
def test_linear_against_formula_and_differences(act, p, biased, with_res):
    gen = torch.Generator().manual_seed(2)
    x, w, b, r = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((5, 12), (11, 12), (11,), (5, 11)))
    b, r = b if biased else None, r if with_res else None
    y = ops.linear_bias_act(x, w, b, act, residual=r, dropout_p=p, seed=4)
    z = x @ w.t() + (b if biased else 0)
    keep = keep_mask(5, 11, dropout_args(p, 4), "cpu").double() * 65536 / (65536 - round(65536 * p))
    assert torch.allclose(y, _gelu(z, act) * keep + (r if with_res else 0), atol=1e-12)
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    assert torch.autograd.gradcheck(lambda *_: ops.linear_bias_act(x, w, b, act, residual=r, dropout_p=p, seed=4), leaves)


@pytest.mark.parametrize("want_entropy", [False, True])
def test_logprobs_against_formula_and_differences(want_entropy):
    gen = torch.Generator().manual_seed(3)
    h, w = torch.randn(2, 4, 6, generator=gen, dtype=torch.float64), torch.randn(9, 6, generator=gen, dtype=torch.float64)
    t = torch.tensor([[0, 8, -100, 3], [9, 1, -1, 5]])                 # 9, -1 and -100 are no token
    logp, ent = ops.linear_logprobs(h, w, t, want_entropy=want_entropy)
    q = (h @ w.t()).exp()
    q = q / q.sum(-1, keepdim=True)
    ok = (t >= 0) & (t < 9)
    want = torch.where(ok, q.gather(-1, torch.where(ok, t, 0)[..., None])[..., 0].log(), 0.0)
    assert logp.shape == t.shape and torch.allclose(logp, want, atol=1e-12) and (logp[~ok] == 0).all()
    assert (ent is None) != want_entropy
    if want_entropy:
        assert torch.allclose(ent, -(q * q.log()).sum(-1), atol=1e-12)
    h.requires_grad_(), w.requires_grad_()
    call = lambda *_: tuple(v for v in ops.linear_logprobs(h, w, t, want_entropy=want_entropy, chunk=3) if v is not None)
    assert torch.autograd.gradcheck(call, (h, w))
    if not want_entropy:
        gh, = torch.autograd.grad(ops.linear_logprobs(h, w, t)[0].sum(), h)
        assert (gh[~ok] == 0).all()


def test_no_rows():
    assert ops.dropout(torch.ones(0, 8), 0.1, 1).shape == (0, 8) and ops.dropout(torch.ones(3, 0), 0.1, 1).shape == (3, 0)
    assert ops.linear_bias_act(torch.ones(0, 8), torch.ones(4, 8), dropout_p=0.1, seed=1).shape == (0, 4)
    logp, ent = ops.linear_logprobs(torch.ones(0, 8), torch.ones(4, 8), torch.zeros(0, dtype=torch.long), want_entropy=True)
    assert logp.shape == ent.shape == (0,)


def test_piece_widths():
    from torchturbo_b200.ops.providers.b200 import LinearLogprobsFn as Fn

    for rows, vocab in ((1, 1), (61, 151936), (4096, 151936), (65536, 151936), (4096, 32003), (2 ** 22, 4000), (7, 257)):
        step = Fn.pieces(rows, vocab)
        assert step % 256 == 0 and step > 0
        count = -(-vocab // step)
        assert (count - 1) * step < vocab
        assert rows * min(step, vocab) <= Fn.PIECE + 256 * rows       # never more than a tile's columns over the limit


def test_registry_offers_the_loss_in_pieces_by_name_only():
    from torchturbo_b200.ops.registry import REGISTRY

    names = [c.op_spec().impl_name for c in REGISTRY.list("linear_cross_entropy")]
    assert names.index("tcgen05_linear_cross_entropy") < names.index("tcgen05_linear_cross_entropy_pieces")
    assert isinstance(dropout_args(0.0, None), Dropout)
