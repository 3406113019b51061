"""Biased linear layer with activation, dropout and residual in the product's epilogue: values and gradients against 64 bits at the edges
of its tiles, in all of its forms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8       # half a step of bf16
ACC = 2.0 ** -15       # fp32 sums: 2^-24 of the summed magnitudes for each of at most 2^9 partial sums


def _rand(gen, *shape, std=0.5):
    return (torch.randn(*shape, generator=gen) * std).bfloat16().cuda()


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _slope(z, act):
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(_act(z, act).sum(), z)[0]


def _check(x, w, b, r, act, p, seed, dy=None, first_row=0):
    """The call's result (and gradients for `dy`) against 64 bits.

    The hyperbolic tangent is the hardware's, off by up to 2^-10.98 of its value: of gelu's value |z| / 2 of that, of its slope
    (1 + t) / 2 + z (1 - t^2) c (1 + 0.134 z^2) / 2 at most 2^-11 (1/2 + 0.8 |z| (1 + 0.134 z^2)); rounded up to 2^-10 here.  The
    error function is off by up to 1.5e-7, which is below 2^-22.  The activations' slopes stay below 1.13, their second derivatives below 1.1."""
    from torchturbo_b200.ops import ops
    from torchturbo_b200.ops.dropout import dropout_args, keep_mask

    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(dy is not None)
    y = ops.linear_bias_act(x, w, b, act, residual=r, dropout_p=p, seed=seed, first_row=first_row)
    X, W, B, R = (t.detach().double() if t is not None else None for t in (x, w, b, r))
    z, mag = X @ W.t(), X.abs() @ W.abs().t()
    if b is not None:
        z, mag = z + B, mag + B.abs()
    t = round(65536 * p)
    factor = 65536 / (65536 - t) * keep_mask(x.shape[0], w.shape[0], dropout_args(p, seed, first_row), "cpu").double().cuda()
    approx = 2.0 ** -10 if act == "gelu_tanh" else 2.0 ** -20
    want = _act(z, act) * factor
    tol = factor * (1.13 * ACC * mag + approx * z.abs() / 2 + 2.0 ** -20 * want.abs())
    if r is not None:
        want, tol = want + R, tol + R.abs() * 2.0 ** -23
    assert y.shape == want.shape and y.dtype == torch.bfloat16
    assert ((y.double() - want).abs() <= want.abs() * HALF + tol * (1 + HALF)).all()
    if dy is None:
        return y
    grads = iter(torch.autograd.grad(y, leaves, dy))
    D = dy.double() * factor
    slope = _slope(z, act)
    dz = D * slope
    # pre-activations are kept in bf16
    tz = dz.abs() * HALF
    if act:
        tz = tz + (1 + HALF) * D.abs() * (1.1 * (HALF * z.abs() + ACC * mag) + approx * (0.5 + 0.8 * z.abs() * (1 + 0.134 * z * z)) + 2.0 ** -20)
    if not act and not p:
        tz = torch.zeros_like(tz)
    for got, ref, bound in ((next(grads), dz @ W, tz @ W.abs() + ACC * (dz.abs() @ W.abs())),
                            (next(grads), dz.t() @ X, tz.t() @ X.abs() + ACC * (dz.t().abs() @ X.abs()))):
        assert got.dtype == torch.bfloat16 and ((got.double() - ref).abs() <= ref.abs() * HALF + bound * (1 + HALF) + 1e-30).all()
    if b is not None:
        assert ((next(grads).double() - dz.sum(0)).abs() <= dz.sum(0).abs() * HALF + (tz.sum(0) + ACC * dz.abs().sum(0)) * (1 + HALF) + 1e-30).all()
    if r is not None:
        assert torch.equal(next(grads), dy)
    return y


@pytest.mark.parametrize("M, N", [(1, 8), (1, 1152), (31, 64), (33, 72), (127, 128), (128, 136), (129, 200), (160, 256), (257, 264), (300, 520)])
@pytest.mark.parametrize("K", [8, 64, 136])
@pytest.mark.parametrize("act, p", [(None, 0.0), ("gelu_tanh", 0.0), ("gelu", 0.3)])
def test_edges(M, N, K, act, p):
    from torchturbo_b200 import kernels as Kn

    gen = torch.Generator().manual_seed(M * N + K)
    _check(_rand(gen, M, K), _rand(gen, N, K), _rand(gen, N), _rand(gen, M, N), act, p, 5, _rand(gen, M, N))
    assert Kn.status() == (0, 0)


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh"])
@pytest.mark.parametrize("p", [0.0, 0.05])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("with_res", [False, True])
def test_every_form(act, p, biased, with_res):
    gen = torch.Generator().manual_seed(8)
    x, w, dy = _rand(gen, 140, 72), _rand(gen, 328, 72), _rand(gen, 140, 328)
    b, r = _rand(gen, 328) if biased else None, _rand(gen, 140, 328) if with_res else None
    _check(x, w, b, r, act, p, 2 ** 50 + 1, dy, first_row=2 ** 33)
    _check(x.detach(), w.detach(), b.detach() if biased else None, r.detach() if with_res else None, act, p, 2 ** 50 + 1)


def test_all_dropped():
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(1)
    x, w, b, r = (_rand(gen, *s).requires_grad_() for s in ((40, 64), (72, 64), (72,), (40, 72)))
    y = ops.linear_bias_act(x, w, b, "gelu", residual=r, dropout_p=1.0, seed=1)
    assert torch.equal(y, r)
    grads = torch.autograd.grad(y.float().sum(), (x, w, b, r))
    assert all((g == 0).all() for g in grads[:3]) and (grads[3] == 1).all()


@pytest.mark.parametrize("M, N, K", [(5, 264, 4104), (130, 72, 8192)])
@pytest.mark.parametrize("act, p", [(None, 0.0), ("gelu_tanh", 0.2)])
def test_long_sums_in_pieces(M, N, K, act, p):
    """Few tiles and a long K: the product is formed in pieces, the tail follows their sum."""
    from torchturbo_b200 import kernels as Kn

    assert Kn.gemm_splits(M, N, K, Kn.num_sms()) > 1
    gen = torch.Generator().manual_seed(K)
    _check(_rand(gen, M, K, std=0.1), _rand(gen, N, K, std=0.1), _rand(gen, N), _rand(gen, M, N), act, p, 3, _rand(gen, M, N))
    assert Kn.status() == (0, 0)


@pytest.mark.parametrize("K", [8, 16, 24, 32, 40, 64])
@pytest.mark.parametrize("M, N", [(2, 8), (31, 256), (33, 264), (9511, 24), (99, 21000), (5000, 1032), (700, 4104)])
def test_few_features(M, N, K):
    """Adapters: the backward walks the gradient once, in shares of rows that end inside a step and blocks of columns that are cut."""
    from torchturbo_b200 import kernels as Kn

    gen = torch.Generator().manual_seed(M + N + K)
    for act, p, biased in (("gelu", 0.3, True), (None, 0.0, False), (None, 0.05, False), ("gelu_tanh", 0.0, True)):
        _check(_rand(gen, M, K), _rand(gen, N, K), _rand(gen, N) if biased else None, _rand(gen, M, N), act, p, 5, _rand(gen, M, N), first_row=2 ** 32 - 40)
    assert Kn.status() == (0, 0)


def test_few_features_of_many_rows():
    """More than is walked row by row in the forward."""
    gen = torch.Generator().manual_seed(17)
    M, N = 6200, 4104
    _check(_rand(gen, M, 16), _rand(gen, N, 16), _rand(gen, N), _rand(gen, M, N), None, 0.1, 5, _rand(gen, M, N))


def test_few_features_of_wider_rows():
    """Inputs and weights that are parts of wider matrices, and a seed in memory."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(16)
    x, w, dy = _rand(gen, 90, 48), _rand(gen, 520, 72), _rand(gen, 90, 520)
    got = []
    for xs, ws, seed in ((x[:, 8:32], w[:, 16:40], torch.tensor([9], device="cuda")), (x[:, 8:32].clone(), w[:, 16:40].clone(), 9)):
        leaves = [xs.detach().requires_grad_(), ws.detach().requires_grad_()]
        got.append(torch.autograd.grad(ops.linear_bias_act(*leaves, act="gelu", dropout_p=0.3, seed=seed), leaves, dy))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("N, K", [(8, 8), (24, 264), (2376, 520), (1200, 1032), (4744, 256), (72, 4104)])
def test_few_rows(M, N, K):
    """Rows that the weight streams past: every share of K among warps, one and two columns a warp, ends inside a step."""
    gen = torch.Generator().manual_seed(M + N + K)
    for act, p in (("gelu", 0.3), (None, 0.0), ("gelu_tanh", 0.0)):
        _check(_rand(gen, M, K, std=0.2), _rand(gen, N, K, std=0.2), _rand(gen, N), _rand(gen, M, N), act, p, 5, _rand(gen, M, N))


@pytest.mark.parametrize("M, N, K", [(1500, 1152, 2304), (3001, 4304, 1152), (300, 136, 264), (4200, 520, 1160)])
def test_products_of_the_backward_run_into_one_another(M, N, K):
    """Whatever follows sees both products whole, over many steps in a row and replayed: the same bits as one after the other."""
    from torchturbo_b200 import kernels as Kn
    from torchturbo_b200.ops.dropout import NONE

    gen = torch.Generator().manual_seed(M)
    x, w, dys = _rand(gen, M, K), _rand(gen, N, K), [_rand(gen, M, N) for _ in range(4)]
    z = _rand(gen, M, N, std=2.0)
    want = []
    for dy in dys:
        dz, db = Kn.tail_bwd(dy, z, "gelu", NONE, True, torch.bfloat16)
        want.append((Kn.gemm(dz, w, b_mn=True), Kn.gemm(dz, x, a_mn=True, b_mn=True), db))
    torch.cuda.synchronize()

    def steps():
        got = []
        for dy in dys * 5:
            grads = Kn.linear_tail_bwd(dy, x, w, z, "gelu", NONE, True, True, True)
            got.append([g + 0 for g in grads])
            del grads                   # their memory is the next step's
        return got

    graph = torch.cuda.CUDAGraph()
    eager = steps()
    with torch.cuda.graph(graph):
        replayed = steps()
    graph.replay()
    for got in (eager, replayed):
        for i, grads in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(grads, want[i % 4]))
    assert Kn.status() == (0, 0)


def test_wide_rows():
    gen = torch.Generator().manual_seed(14)
    _check(_rand(gen, 20, 16), _rand(gen, 20000, 16), _rand(gen, 20000), None, "gelu", 0.1, 3, _rand(gen, 20, 20000))


def test_pairs_of_CTAs():
    """Tiles of 256 rows, the last of them with one half empty, and a last tile of columns that is cut."""
    gen = torch.Generator().manual_seed(4)
    M, N, K = 1100, 8264, 520
    _check(_rand(gen, M, K), _rand(gen, N, K), _rand(gen, N), _rand(gen, M, N), "gelu", 0.1, 3, _rand(gen, M, N))


def test_layouts_and_leading_dimensions():
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(6)
    x, w, b, r = _rand(gen, 60, 80), _rand(gen, 96, 80), _rand(gen, 96), _rand(gen, 60, 96)
    want = ops.linear_bias_act(x, w, b, "gelu_tanh", residual=r, dropout_p=0.2, seed=1)
    wide = torch.zeros(60, 160, device="cuda", dtype=torch.bfloat16)
    for off in (0, 8, 3):                                    # rows of a wider matrix, on and off their 16-byte boundary
        wide[:, off:off + 80] = x
        assert torch.equal(ops.linear_bias_act(wide[:, off:off + 80], w, b, "gelu_tanh", residual=r, dropout_p=0.2, seed=1), want)
    wide[:, 5:101] = r
    assert torch.equal(ops.linear_bias_act(x, w, b, "gelu_tanh", residual=wide[:, 5:101], dropout_p=0.2, seed=1), want)
    assert torch.equal(ops.linear_bias_act(x, w.t().contiguous().t(), b, "gelu_tanh", residual=r, dropout_p=0.2, seed=1), want)
    y = ops.linear_bias_act(x.view(3, 20, 80), w, b, "gelu_tanh", residual=r.view(3, 20, 96), dropout_p=0.2, seed=1)
    assert y.shape == (3, 20, 96) and torch.equal(y.view(60, 96), want)
    one = ops.linear_bias_act(x[0], w, b, "gelu_tanh", residual=r[0], dropout_p=0.2, seed=1)
    assert one.shape == (96,) and torch.equal(one, want[0])
    same = ops.linear_bias_act(x[:1].expand(60, 80), w, b)
    assert torch.equal(same, ops.linear_bias_act(x[:1], w, b).expand(60, 96))


def test_gradients_wanted_of_some():
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(7)
    x, w, b, r, dy = _rand(gen, 50, 64), _rand(gen, 72, 64), _rand(gen, 72), _rand(gen, 50, 72), _rand(gen, 50, 72)
    all_ = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(ops.linear_bias_act(*all_[:3], "gelu", residual=all_[3], dropout_p=0.1, seed=1), all_, dy)
    for mask in range(1, 16):
        t = [v.clone().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((x, w, b, r))]
        y = ops.linear_bias_act(*t[:3], "gelu", residual=t[3], dropout_p=0.1, seed=1)
        asked = [v for v in t if v.requires_grad]
        for g, ref in zip(torch.autograd.grad(y, asked, dy), [g for i, g in enumerate(want) if mask >> i & 1]):
            assert torch.equal(g, ref)


def test_main_grad_and_broadcast_gradient():
    """A weight with an fp32 accumulation buffer, and the gradient of a sum, whose rows share their memory."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(9)
    x, w = _rand(gen, 50, 64), _rand(gen, 72, 64).requires_grad_()
    ops.linear_bias_act(x, w, act="gelu").sum().backward()
    v = w.detach().clone().requires_grad_()
    v.main_grad = torch.ones(72, 64, device="cuda")
    ops.linear_bias_act(x, v, act="gelu").sum().backward()
    assert v.grad is None
    assert ((v.main_grad - 1) - w.grad.float()).abs().max() <= HALF * w.grad.float().abs().max() + 1e-5


def test_gradient_of_the_gradient():
    """Where a graph of the gradient is wanted it is formed by separate operations: the same as of the plain formulation."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(13)
    x, w, b = _rand(gen, 8, 16).requires_grad_(), _rand(gen, 24, 16).requires_grad_(), _rand(gen, 24).requires_grad_()
    got = []
    for impl in ("tcgen05_linear_bias_act", "torch_linear_bias_act"):
        y = ops.linear_bias_act(x, w, b, "gelu", dropout_p=0.2, seed=1, impl=impl)
        g = torch.autograd.grad(y.float().sum(), (x, w, b), create_graph=True)
        got.append(torch.autograd.grad(sum(v.float().square().sum() for v in g), (x, w, b)))
    for a, ref in zip(*got):
        assert ref.abs().max() > 0 and torch.equal(a, ref)


def test_captured_step_draws_by_its_seed():
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(10)
    x, w, b = _rand(gen, 130, 64), _rand(gen, 136, 64), _rand(gen, 136)
    dy = _rand(gen, 130, 136)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step(seed):
        y = ops.linear_bias_act(x, w, b, "gelu_tanh", dropout_p=0.3, seed=seed)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = {s: [t.clone() for t in step(s)] for s in (1, 2)}
    seed = torch.tensor([0], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(seed)
    for s, ref in want.items():
        seed.fill_(s)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("M, K", [(3, 64), (130, 64), (5, 4104)])
@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh"])
def test_columns_that_are_not_finite(M, K, act):
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(15)
    x, w, b = _rand(gen, M, K, std=0.1), _rand(gen, 72, K, std=0.1), _rand(gen, 72)
    want = ops.linear_bias_act(x, w, b, act)
    b[3], b[5] = float("inf"), float("nan")
    y = ops.linear_bias_act(x, w, b, act)
    rest = [i for i in range(72) if i not in (3, 5)]
    assert torch.equal(y[:, rest], want[:, rest]) and (y[:, 3] == float("inf")).all() and y[:, 5].isnan().all()
    y = ops.linear_bias_act(x, w, b, act, dropout_p=0.5, seed=1)
    assert ((y[:, 3] == float("inf")) | (y[:, 3] == 0)).all() and ((y[:, 5] == 0) == (y[:, 5] == y[:, 5])).all()


@pytest.mark.parametrize("M, N, K", [(700, 1032, 16), (1500, 1152, 520), (300, 264, 64)])
def test_two_streams_at_once(M, N, K):
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(M)
    sets = [[_rand(gen, *s).requires_grad_() for s in ((M, K), (N, K), (N,), (M, N))] for _ in range(2)]
    dy = _rand(gen, M, N)

    def step(x, w, b, r):
        y = ops.linear_bias_act(x, w, b, "gelu", residual=r, dropout_p=0.1, seed=4)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b, r), dy)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for steps in got[i] for a, b in zip(steps, want[i]))


def test_result_may_be_changed_in_place():
    """The kept pre-activations are no view of the result."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(11)
    x, w = _rand(gen, 16, 64).requires_grad_(), _rand(gen, 72, 64)
    want, = torch.autograd.grad(ops.linear_bias_act(x, w, act="gelu").sum(), x)
    y = ops.linear_bias_act(x, w, act="gelu")
    y.mul_(1.0)
    got, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(got, want)


def test_refusals():
    from torchturbo_b200.ops import ops

    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, w = torch.ones(6, 16, **bf), torch.ones(24, 16, **bf)
    for call in (lambda: ops.linear_bias_act(x, torch.ones(24, 8, **bf)), lambda: ops.linear_bias_act(x, w[0]), lambda: ops.linear_bias_act(x, w, torch.ones(1, **bf)),
                 lambda: ops.linear_bias_act(x, w, torch.ones(24, 1, **bf)), lambda: ops.linear_bias_act(x, w, act="relu6"),
                 lambda: ops.linear_bias_act(x, w, residual=torch.ones(24, **bf)), lambda: ops.linear_bias_act(x, w, residual=torch.ones(1, 24, **bf)),
                 lambda: ops.linear_bias_act(x, w, residual=torch.ones(6, 16, **bf)), lambda: ops.linear_bias_act(x.view(2, 3, 16), w, residual=torch.ones(6, 24, **bf)),
                 lambda: ops.linear_bias_act(x[0, 0], w), lambda: ops.linear_bias_act(x, w.cpu()), lambda: ops.linear_bias_act(x, w, dropout_p=1.5), lambda: ops.linear_bias_act(x, w, dropout_p=0.1, seed=-1)):
        with pytest.raises(ValueError):
            call()


def test_types_and_widths_that_the_kernel_does_not_take():
    """fp32, and widths that are no multiple of eight, take the plain formulation."""
    from torchturbo_b200.ops import ops

    gen = torch.Generator().manual_seed(12)
    for dtype, k, n in ((torch.float32, 16, 24), (torch.bfloat16, 12, 24), (torch.bfloat16, 16, 20)):
        x, w, b = (torch.randn(*s, generator=gen).to(dtype) for s in ((5, k), (n, k), (n,)))
        want = ops.linear_bias_act(x.cuda(), w.cuda(), b.cuda(), "gelu", dropout_p=0.2, seed=1, impl="torch_linear_bias_act")
        assert torch.equal(ops.linear_bias_act(x.cuda(), w.cuda(), b.cuda(), "gelu", dropout_p=0.2, seed=1), want)
    assert ops.linear_bias_act(torch.ones(0, 16, device="cuda", dtype=torch.bfloat16), torch.ones(8, 16, device="cuda", dtype=torch.bfloat16)).shape == (0, 8)
