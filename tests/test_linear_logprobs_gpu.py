"""Log-probabilities and entropies of rows of logits that are not stored, and their gradients, against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8       # half a step of bf16
ACC = 2.0 ** -15       # fp32 sums: 2^-24 of the summed magnitudes for each of at most 2^9 partial sums
EXP = 2.0 ** -20       # an exponential of the hardware and what its argument was rounded to (2^-22 and 2^-23 times up to 4 powers of two)


def _case(T, H, V, seed=0, std=2.5):
    gen = torch.Generator().manual_seed(seed + T + H + V)
    w = (torch.randn(V, H, generator=gen) * std * H ** -0.5).bfloat16()
    t = torch.randint(0, V, (T,), generator=gen)
    h = (torch.randn(T, H, generator=gen) + torch.rand(T, 1, generator=gen) * 2 * w[t].float()).bfloat16()
    t[torch.rand(T, generator=gen) < 0.2] = -100
    return h.cuda(), w.cuda(), t.cuda()


def _exact(h, w, t):
    lg = h.double() @ w.double().t()
    lq = torch.log_softmax(lg, -1)
    p = lq.exp()
    ok = (t >= 0) & (t < w.shape[0])
    on = torch.zeros_like(p)
    rows = ok.nonzero()[:, 0]
    on[rows, t[rows]] = 1.0
    return lg, lq, p, on, ok


def _check(h, w, t, want_entropy, train, call=None):
    from torchturbo_b200.ops import ops

    for x in (h, w):
        x.requires_grad_(train)
    logp, ent = (call or ops.linear_logprobs)(h, w, t, want_entropy=want_entropy)
    with torch.no_grad():
        H, W = h.double(), w.double()
        lg, lq, p, on, ok = _exact(H, W, t)
        err = ACC * (H.abs() @ W.abs().t()) + 2.0 ** -22 * lg.abs()              # of every logit
        worst = err.amax(1)
        lp = (lq * on).sum(1)
        tol = (2 * worst + EXP * (2 + lg.abs().amax(1) + lq.abs().amax(1))) * ok
        assert logp.dtype == torch.float32 and ((logp.double() - lp).abs() <= tol).all() and (logp[~ok] == 0).all()
        H1 = -(p * lq).sum(1)
        if want_entropy:
            # d entropy / d logit = -p (log p + entropy); each exponential, its weight and the join are rounded as well
            bound = (p * (lq + H1[:, None]).abs() * (worst[:, None] + EXP)).sum(1) * 2 + EXP * 4 * (1 + H1.abs() + (p * lq.abs()).sum(1)) \
                + 4 * worst ** 2 * (1 + H1.abs())
            assert ((ent.double() - H1).abs() <= bound).all()
        else:
            assert ent is None
    if not train:
        return logp, ent
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(t.shape, generator=gen).cuda()
    e = torch.randn(t.shape, generator=gen).cuda() * 0.3 if want_entropy else None
    dh, dw = torch.autograd.grad((logp, ent) if want_entropy else logp, (h, w), (g, e) if want_entropy else g)
    with torch.no_grad():
        G = (g.double() * ok)[:, None]
        E = e.double()[:, None] if want_entropy else torch.zeros_like(G)
        s = lq + H1[:, None]
        dl = G * (on - p) - E * p * s
        off = 2 * worst[:, None] + 2 * EXP * (1 + lg.abs())                      # of the logarithm of p
        # of up to 64 rows what the first rounding leaves out goes into the products as well
        tl = dl.abs() * (HALF if t.numel() > 64 else HALF ** 2) + (1 + HALF) * (off * p * (G.abs() + E.abs() * (s.abs() + 2)) + 2.0 ** -22 * G.abs() * on)
        for got, ref, bound in ((dh, dl @ W, tl @ W.abs() + ACC * (dl.abs() @ W.abs())), (dw, dl.t() @ H, tl.t() @ H.abs() + ACC * (dl.t().abs() @ H.abs()))):
            assert got.dtype == torch.bfloat16 and ((got.double() - ref).abs() <= ref.abs() * HALF + bound * (1 + HALF) + 1e-30).all()
    return logp, ent, dh, dw


@pytest.mark.parametrize("T, V", [(1, 1), (1, 7), (1, 4001), (31, 32), (33, 33), (64, 128), (127, 129), (129, 255), (130, 257), (300, 1000)])
@pytest.mark.parametrize("H", [8, 64, 136])
@pytest.mark.parametrize("want_entropy", [False, True])
def test_edges(T, V, H, want_entropy):
    from torchturbo_b200 import kernels as Kn

    _check(*_case(T, H, V), want_entropy, True)
    assert Kn.status() == (0, 0)


@pytest.mark.parametrize("T, H, V", [(61, 2048, 32003), (1100, 512, 16001), (4, 5120, 4000)])
def test_larger(T, H, V):
    _check(*_case(T, H, V), True, True)


@pytest.mark.parametrize("T, share", [(513, 0.0), (600, 0.4), (700, 0.97), (520, 1.0), (1100, 0.5)])
@pytest.mark.parametrize("pieces", [1, 3])
def test_rows_without_a_target_are_left_out(monkeypatch, T, share, pieces):
    """Wide vocabularies: prompts and padding are not computed.  None, some, nearly all and all of the rows; not a number in them stays there."""
    from torchturbo_b200 import kernels as Kn
    from torchturbo_b200.ops import ops
    from torchturbo_b200.ops.providers.b200 import LinearLogprobsFn as Fn

    h, w, t = _case(T, 136, 33003, std=1.0)
    gen = torch.Generator().manual_seed(T)
    t = torch.where(t < 0, 5, t)
    t[(torch.rand(T, generator=gen) < share).cuda()] = -100
    if share == 1.0:
        t[:] = -1
    assert Fn.compact(h, w, False) and not Fn.compact(h, w, True)
    if pieces > 1:
        monkeypatch.setattr(Fn, "PIECE", T * 33003 // 3)
    _check(h, w, t, False, True)
    if 0 < share < 1:
        with torch.no_grad():
            want = ops.linear_logprobs(h, w, t)[0]
            h[t < 0] = float("nan")
        logp, _ = ops.linear_logprobs(h, w, t)
        dh, dw = torch.autograd.grad(logp.sum(), (h, w))
        assert torch.equal(logp, want) and torch.isfinite(dh).all() and torch.isfinite(dw).all() and (dh[t < 0] == 0).all()
        v = w.detach().clone().requires_grad_()
        v.main_grad = torch.ones(33003, 136, device="cuda")
        ops.linear_logprobs(h, v, t)[0].sum().backward()
        assert ((v.main_grad - 1) - dw.float()).abs().max() <= HALF * dw.float().abs().max() + 1e-5
    assert Kn.status() == (0, 0)


@pytest.mark.parametrize("there", [0, 1, 63, 64, 129, 300, 512])
@pytest.mark.parametrize("splits", [0, 2])
def test_products_of_rows_that_the_device_counts(there, splits):
    from torchturbo_b200 import kernels as Kn

    gen = torch.Generator().manual_seed(there)
    K = 4160 if splits else 200
    count = torch.tensor([there], dtype=torch.int32, device="cuda")
    a, b = (torch.randn(*s, generator=gen).bfloat16().cuda() for s in ((512, K), (K, 264)))
    out = torch.full((512, 264), 7.0, dtype=torch.bfloat16, device="cuda")
    Kn.gemm(a, b, b_mn=True, out=out, rows=count, splits=splits)
    assert torch.equal(out[:there], Kn.gemm(a, b, b_mn=True, splits=splits)[:there])
    if not splits:
        assert (out[(there + 255) // 256 * 256:] == 7).all()
    # of the rows of both operands: zeros behind them to the next multiple of 64
    R = 8192 if splits else 512
    x, y = (torch.randn(R, n, generator=gen).bfloat16().cuda() for n in (136, 264))
    x[there:(there + 63) // 64 * 64] = 0
    count.fill_(there)
    want = Kn.gemm(torch.where(torch.arange(R, device="cuda")[:, None] < there, x, 0), y, a_mn=True, b_mn=True, splits=splits)
    assert torch.equal(Kn.gemm(x, y, a_mn=True, b_mn=True, rows=count, splits=splits), want)
    acc = torch.ones(136, 264, device="cuda")
    Kn.gemm(x, y, a_mn=True, b_mn=True, rows=count, out=acc, accumulate=True, splits=splits)
    assert ((acc - 1) - want.float()).abs().max() <= HALF * want.float().abs().max() + 1e-4
    assert Kn.status() == (0, 0)


def test_rows_in_shares():
    """Statistics of more rows than are held at a time (2^26 values of 1188 pieces and three planes: 18688 rows)."""
    from torchturbo_b200.ops import ops

    h, w, t = _case(19001, 8, 151936)
    logp, ent = ops.linear_logprobs(h, w, t, want_entropy=True)
    for a in (0, 18600, 18900):
        parts = ops.linear_logprobs(h[a:a + 101], w, t[a:a + 101], want_entropy=True)
        for x, y in zip((logp, ent), parts):
            assert ((x[a:a + 101] - y).abs() <= 2.0 ** -18 * (1 + y.abs())).all()      # other tiles, other order of the same sums
    _check(h[-64:].clone(), w, t[-64:].clone(), True, False)


@pytest.mark.parametrize("V", [700, 1025])
@pytest.mark.parametrize("want_entropy", [False, True])
def test_several_pieces(monkeypatch, V, want_entropy):
    """A vocabulary in pieces of 256 columns: what is added up over them, and the last one's edge."""
    from torchturbo_b200.ops.providers.b200 import LinearLogprobsFn as Fn

    h, w, t = _case(150, 136, V)
    monkeypatch.setattr(Fn, "PIECE", 150 * 256)
    assert Fn.pieces(150, V) == 256
    _check(h, w, t, want_entropy, True)


def test_targets_outside_of_the_vocabulary():
    """None of them has a log-probability or a gradient through it, at the edge of a tile and of a piece or not."""
    for V in (33, 256, 300):
        h, w, t = _case(40, 64, V)
        t[:8] = torch.tensor([V, V + 1, -1, -100, 2 ** 40, -2 ** 40, V + 31, 511])
        _check(h, w, t, True, True)


def test_all_ignored_and_one_token_vocabulary():
    h, w, t = _case(20, 64, 300)
    t.fill_(-100)
    logp, _, dh, dw = _check(h, w, t, False, True)
    assert (logp == 0).all() and (dh == 0).all() and (dw == 0).all()


def test_peaked_and_flat_rows():
    """A row whose target holds all but 2^-30 of the probability, one whose target has almost none, and one of equal logits."""
    H, V = 64, 500
    w = torch.zeros(V, H, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = torch.linspace(-1, 1, V).bfloat16()
    w[3, 1] = 30.0
    h = torch.zeros(4, H, device="cuda", dtype=torch.bfloat16)
    h[0, 1] = 1.0
    h[1, 1] = 4.0
    h[2, 0] = 2.0
    _check(h, w, torch.tensor([3, 9, 0, 7], device="cuda"), True, True)


def test_rows_that_are_not_finite_stay_by_themselves():
    from torchturbo_b200.ops import ops

    h, w, t = _case(40, 64, 300)
    t[:] = 5
    want, _ = ops.linear_logprobs(h, w, t)
    h[7, 3], h[9, 0] = float("nan"), float("inf")
    got, ent = ops.linear_logprobs(h, w, t, want_entropy=True)
    rest = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(got[rest], want[rest]) and not torch.isfinite(got[[7, 9]]).any() and not torch.isfinite(ent[[7, 9]]).any()
    # without a target their gradient is zero
    t[7] = t[9] = -100
    h.requires_grad_()
    logp, _ = ops.linear_logprobs(h, w, t)
    dh, = torch.autograd.grad(logp.sum(), h)
    assert (logp[[7, 9]] == 0).all() and (dh[[7, 9]] == 0).all() and torch.isfinite(dh).all()


@pytest.mark.parametrize("T", [5, 300])
def test_tokens_that_a_head_rules_out(T):
    """Logits of minus infinity, over whole tiles and inside of one: as if their tokens were not there."""
    from torchturbo_b200.ops import ops

    h, w, t = _case(T, 64, 1100)
    h[:, 0] = 1.0
    t[:] = torch.randint(0, 20, (T,), device="cuda")
    ruled = torch.zeros(1100, dtype=torch.bool, device="cuda")
    ruled[30:40] = ruled[200:1090] = True
    want, _ = ops.linear_logprobs(h, w[~ruled].contiguous(), t)
    w[ruled, 0] = float("-inf")
    got, _ = ops.linear_logprobs(h, w, t)
    # the same sums in other pieces: 2^-24 of the log-sum-exp for each of at most twelve roundings on each side
    assert ((got - want).abs() <= 24 * 2.0 ** -24 * (want.abs() + 12)).all()
    t[0] = 35
    assert ops.linear_logprobs(h, w, t)[0][0] == float("-inf")


def test_layouts_and_gradients_wanted_of_some():
    from torchturbo_b200.ops import ops

    h, w, t = _case(48, 72, 520)
    h.requires_grad_(), w.requires_grad_()
    logp, ent = ops.linear_logprobs(h, w, t, want_entropy=True)
    dh, dw = torch.autograd.grad((logp, ent), (h, w), (torch.ones_like(logp), torch.full_like(ent, 0.1)))
    only, = torch.autograd.grad(ops.linear_logprobs(h, w.detach(), t)[0].sum(), h)
    both, _ = torch.autograd.grad(ops.linear_logprobs(h, w, t)[0].sum(), (h, w))
    assert torch.equal(only, both)
    only, = torch.autograd.grad(ops.linear_logprobs(h.detach(), w, t)[0].sum(), w)
    assert torch.equal(only, torch.autograd.grad(ops.linear_logprobs(h, w, t)[0].sum(), w)[0])
    # one of the two results alone
    a, = torch.autograd.grad(ops.linear_logprobs(h, w, t, want_entropy=True)[0].sum(), h)
    assert torch.equal(a, both)
    b, = torch.autograd.grad(ops.linear_logprobs(h, w, t, want_entropy=True)[1].sum() * 0.1, h)
    assert ((a + b).float() - dh.float()).abs().max() <= 4 * HALF * dh.float().abs().max()
    h3 = h.detach().view(4, 12, 72)
    l3, e3 = ops.linear_logprobs(h3, w.detach(), t.view(4, 12), want_entropy=True)
    assert l3.shape == (4, 12) and torch.equal(l3.flatten(), logp) and torch.equal(e3.flatten(), ent)
    wide = torch.zeros(48, 100, device="cuda", dtype=torch.bfloat16)
    for off in (0, 3):
        wide[:, off:off + 72] = h.detach()
        assert torch.equal(ops.linear_logprobs(wide[:, off:off + 72], w.detach().t().contiguous().t(), t.int())[0], logp)


def test_gradient_of_the_gradient_and_results_changed_in_place():
    from torchturbo_b200.ops import ops

    h, w, t = _case(12, 16, 40)
    h.requires_grad_(), w.requires_grad_()
    got = []
    for impl in ("tcgen05_linear_logprobs", "torch_linear_logprobs"):
        logp, ent = ops.linear_logprobs(h, w, t, want_entropy=True, impl=impl)
        g = torch.autograd.grad(logp.sum() + ent.sum(), (h, w), create_graph=True)
        got.append(torch.autograd.grad(sum(v.float().square().sum() for v in g), (h, w)))
    assert all(ref.abs().max() > 0 and torch.equal(a, ref) for a, ref in zip(*got))
    logp, ent = ops.linear_logprobs(h, w, t, want_entropy=True)
    want = torch.autograd.grad(logp.sum() + ent.sum(), (h, w), retain_graph=True)
    logp, ent = ops.linear_logprobs(h, w, t, want_entropy=True)
    logp.mul_(1.0)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(logp.sum() + ent.sum(), (h, w), retain_graph=True), want))
    ent.mul_(1.0)              # the entropy is part of its own gradient
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(ent.sum(), h)


def test_main_grad():
    from torchturbo_b200.ops import ops

    h, w, t = _case(48, 72, 521)
    w.requires_grad_()
    want, = torch.autograd.grad(ops.linear_logprobs(h, w, t)[0].sum(), w)
    w.main_grad = torch.ones(521, 72, device="cuda")
    ops.linear_logprobs(h, w, t)[0].sum().backward()
    assert w.grad is None and ((w.main_grad - 1) - want.float()).abs().max() <= HALF * want.float().abs().max() + 1e-5


def test_loss_in_pieces_by_name():
    """Selected by name, the loss of the head is what the rows' log-probabilities add up to."""
    from torchturbo_b200.ops import ops

    h, w, t = _case(300, 256, 4001)
    h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t, impl="tcgen05_linear_cross_entropy_pieces")
    lq = torch.log_softmax(h.detach().double() @ w.detach().double().t(), -1)
    ok = t >= 0
    want = -lq[ok, t[ok]].sum()
    assert abs(float(loss.detach()) - float(want)) <= 1e-5 * float(want)
    dh, dw = torch.autograd.grad(loss * 0.5, (h, w))
    d = torch.zeros_like(lq)
    d[ok] = lq[ok].exp()
    d[ok, t[ok]] -= 1
    for got, ref in ((dh, 0.5 * d @ w.detach().double()), (dw, 0.5 * d.t() @ h.detach().double())):
        # rounded to bf16 twice (the logits' gradient, the result): in the 2-norm at most 2^-8 each
        assert (got.double() - ref).norm() <= 2 * HALF * ref.norm()


def test_captured_and_replayed():
    from torchturbo_b200.ops import ops

    h, w, t = _case(70, 64, 1001)
    other = _case(70, 64, 1001, seed=3)
    h.requires_grad_(), w.requires_grad_()
    g = torch.ones(70, device="cuda")

    def step():
        logp, ent = ops.linear_logprobs(h, w, t, want_entropy=True)
        return [logp.detach(), ent.detach(), *torch.autograd.grad((logp, ent), (h, w), (g, g))]

    first = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, first))
    with torch.no_grad():
        for dst, src in zip((h, w, t), other):
            dst.copy_(src)
    graph.replay()
    again = [x.clone() for x in got]
    assert all(torch.equal(a, b) for a, b in zip(again, step()))


def test_two_streams_at_once():
    from torchturbo_b200.ops import ops

    cases = [_case(600, 512, 16001, seed=s) for s in (0, 1)]
    want = [ops.linear_logprobs(*c)[0] for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for c, st in zip(cases, streams):
        with torch.cuda.stream(st):
            got.append(ops.linear_logprobs(*c)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_and_other_types():
    from torchturbo_b200.ops import ops

    h, w, t = _case(6, 64, 40)
    for call in (lambda: ops.linear_logprobs(h, w, t.cpu()), lambda: ops.linear_logprobs(h, w, t[:3]), lambda: ops.linear_logprobs(h, w, t.float()),
                 lambda: ops.linear_logprobs(h, w[:, :32], t), lambda: ops.linear_logprobs(h, w[:0], t)):
        with pytest.raises(ValueError):
            call()
    ref = ops.linear_logprobs(h.float(), w.float(), t, want_entropy=True)                  # plain formulation
    got = ops.linear_logprobs(h, w, t, want_entropy=True)
    assert all((a - b).abs().max() < 1e-4 for a, b in zip(ref, got))
    assert ops.linear_logprobs(h[:0], w, t[:0])[0].shape == (0,)
    narrow = ops.linear_logprobs(h[:, :60].contiguous(), w[:, :60].contiguous(), t)[0]     # rows that are no multiple of 16 bytes
    assert torch.allclose(narrow, ops.linear_logprobs(h[:, :60].float(), w[:, :60].float(), t)[0], atol=1e-5)
