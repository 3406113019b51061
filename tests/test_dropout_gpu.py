"""Dropout kernel: the mask of the host, bit for bit, on rows of any width, in both directions, on slices and streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 8), (3, 7), (2000, 1), (700, 3), (33, 9), (61, 2048), (4097, 1003), (5, 16384), (257, 4104), (1, 100001)]


def _want(x, drop, residual=None):
    from torchturbo_b200.ops.dropout import keep_mask

    keep = keep_mask(x.shape[0], x.shape[1], drop, "cpu").cuda()
    y = torch.where(keep, x.double() * (65536 / (65536 - drop.t)), 0.0)
    return y if residual is None else y + residual.double(), keep


def _near(y, want, size):
    """The factor, the product and the sum are each rounded to fp32 (2^-24 of `size`, three times), the result to its type."""
    half = torch.finfo(y.dtype).eps / 2
    assert ((y.double() - want).abs() <= want.abs() * half + size * 3 * 2.0 ** -24 * (1 + half)).all()


@pytest.mark.parametrize("rows, cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_res", [False, True])
def test_values(rows, cols, dtype, with_res):
    from torchturbo_b200.ops import ops
    from torchturbo_b200.ops.dropout import dropout_args

    gen = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=gen).to(dtype).cuda().requires_grad_()
    res = torch.randn(rows, cols, generator=gen).to(dtype).cuda().requires_grad_() if with_res else None
    drop = dropout_args(0.3, 2 ** 61 + 7, 3)
    y = ops.dropout(x, 0.3, 2 ** 61 + 7, residual=res, first_row=3)
    want, keep = _want(x.detach(), drop, res.detach() if with_res else None)
    _near(y, want, x.detach().double().abs() * 1.5 + (res.detach().double().abs() if with_res else 0))
    if not with_res:
        assert torch.equal(y == 0, ~keep | (x == 0))
    dy = torch.randn(rows, cols, generator=gen).to(dtype).cuda()
    grads = torch.autograd.grad(y, [t for t in (x, res) if t is not None], dy)
    _near(grads[0], _want(dy, drop)[0], dy.double().abs() * 1.5)
    if with_res:
        assert torch.equal(grads[1], dy)


def test_dropped_values_are_zero_whatever_they_were():
    from torchturbo_b200.ops import ops

    for bad in (float("nan"), float("inf")):
        for cols in (64, 13):
            x = torch.full((9, cols), bad, device="cuda", dtype=torch.bfloat16)
            keep = ops.dropout(torch.ones_like(x), 0.5, 1) != 0
            y = ops.dropout(x, 0.5, 1)
            assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    assert (ops.dropout(torch.ones(4, 8, device="cuda"), 1.0, 1) == 0).all()
    x = torch.randn(4, 8, device="cuda")
    assert torch.equal(ops.dropout(x, 0.0), x)


def test_layouts():
    """Slices, transposes, broadcasts and rows off their 16-byte boundary give what the same values without gaps give."""
    from torchturbo_b200.ops import ops

    base = torch.randn(40, 72, device="cuda", dtype=torch.bfloat16)
    for x in (base[:, 8:40], base[:, 1:30], base[::3], base.t(), base[0].expand(5, 72), base.view(-1)[3:3 + 7 * 72].view(7, 72), base.view(4, 10, 72)):
        y = ops.dropout(x, 0.25, 11)
        assert y.shape == x.shape and torch.equal(y, ops.dropout(x.contiguous().clone(), 0.25, 11))


def test_seed_on_the_device_and_replay():
    """A captured call draws by what its seed tensor holds when it is replayed; moving the seed on before the backward is an error."""
    from torchturbo_b200.ops import ops

    x = torch.randn(37, 264, device="cuda", dtype=torch.bfloat16)
    seed = torch.tensor([5], device="cuda")
    eager = {s: ops.dropout(x, 0.4, s) for s in (5, 6, 2 ** 40 + 1)}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.4, seed)
    for s, want in eager.items():
        seed.fill_(s)
        graph.replay()
        assert torch.equal(y, want)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(ValueError, match="captured"):
            ops.dropout(x, 0.4)
        x + 1
    x.requires_grad_()
    z = ops.dropout(x, 0.4, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_streams_and_two_calls_at_once():
    from torchturbo_b200.ops import ops

    xs = [torch.randn(2048, 1024, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    want = [ops.dropout(x, 0.2, i) for i, x in enumerate(xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for i, (x, st) in enumerate(zip(xs, streams)):
        with torch.cuda.stream(st):
            got.append(ops.dropout(x, 0.2, i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradient_of_the_gradient():
    from torchturbo_b200.ops import ops

    x = torch.randn(6, 16, device="cuda", requires_grad=True)
    y = ops.dropout(x, 0.5, 3)
    g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), x)
    keep = (ops.dropout(torch.ones_like(x), 0.5, 3) != 0).float()
    assert torch.allclose(h, 2 * 4 * keep, rtol=1e-6)


def test_refusals():
    from torchturbo_b200.ops import ops

    x = torch.ones(2, 8, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: ops.dropout(x, 0.1, 1, residual=torch.ones(2, 8, dtype=torch.bfloat16)), lambda: ops.dropout(x, 0.1, -1),
                 lambda: ops.dropout(x, 0.1, 1, residual=x.float())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(AssertionError, match="seed tensor"):      # read by the kernel, so it has to be where the rows are
        ops.dropout(x, 0.1, torch.tensor([1]))
