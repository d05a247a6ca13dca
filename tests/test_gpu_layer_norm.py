"""GPU tests of the layer norm and its backward against the formulas in 64 bits.

Bounds: a row's sum is at most 46 additions deep in a lane and its tree (five pieces of eight and six steps; four and
eight waves for the widest rows), so it is within 2^-18 of the sum of magnitudes; with A = mean|x| / sd the normed value n is
off by E = 2^-18 A + 2^-17 |n| at most (the mean; half the variance's error, itself 2^-18 and twice the
mean's; a few roundings of 2^-24). y, dx, dweight and dbias follow from the formulas' terms, plus one
rounding to bf16, 2^-8 of the value. Sums over rows: a term for each row and partial, 2^-24 of the
magnitudes each.
"""

import pytest
import torch

from bongard_amd import fused_mlp, ops
from oracle import int8_oracle as i8

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _inputs(rows, cols, seed, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.logspace(-2, 2, rows)[:, None] + shift
    if cols >= 64:
        x[:, cols // 3] *= 20.0
    x = x.to(BF16)
    w, b = (1 + 0.3 * torch.randn(cols, generator=g)).to(BF16), torch.randn(cols, generator=g).to(BF16)
    return x, w, b, torch.randn(rows, cols, generator=g).to(BF16)


def _within(got, want, tol, what):
    err = (got.cpu().double() - want).abs()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def _check(gpu, x, w, b, dy, eps, checkpoint, shape=None):
    leaves = [t.to(gpu).requires_grad_() for t in (x, w)] + ([] if b is None else [b.to(gpu).requires_grad_()])
    xin = leaves[0] if shape is None else leaves[0].view(shape)
    y = fused_mlp.layer_norm(xin, leaves[1], leaves[2] if b is not None else None, eps, checkpoint=checkpoint)
    assert y.shape == xin.shape and y.dtype == BF16
    grads = torch.autograd.grad(y, leaves, dy.to(gpu).view(y.shape))
    held = i8.restored(*i8.checkpoint(x)) if checkpoint else None
    want, n, mean, sd = i8.layer_norm(x, w, b, eps, held)
    _, n0, _, _ = i8.layer_norm(x, w, b, eps)
    A = x.double().abs().mean(-1, keepdim=True) / sd
    W = w.double().abs()
    E0, E = 2.0 ** -18 * A + 2.0 ** -17 * n0.abs(), 2.0 ** -18 * A + 2.0 ** -17 * n.abs()
    tol = W * E0 + 2.0 ** -23 * (n0.abs() * W + (0 if b is None else b.double().abs())) + 2.0 ** -8 * want.abs()
    _within(y.detach().reshape(x.shape), want, tol, "y")
    dx, dw, db = i8.layer_norm_backward(n, sd, dy, w)
    c = dy.double() * w.double()
    mc, mcn = c.abs().mean(-1, keepdim=True), (c * n).abs().mean(-1, keepdim=True)
    tol = (E * mcn + n.abs() * (c.abs() * E).mean(-1, keepdim=True) + 2.0 ** -17 * (mc + n.abs() * mcn)
           + 2.0 ** -22 * c.abs()) / sd + 2.0 ** -16 * dx.abs() + 2.0 ** -8 * dx.abs()
    _within(grads[0], dx, tol, "dx")
    deep = (x.shape[0] + 32) * 2.0 ** -24
    mag = (dy.double() * n).abs().sum(0)
    _within(grads[1], dw, (dy.double().abs() * E).sum(0) + deep * mag + 2.0 ** -8 * dw.abs(), "dweight")
    if b is not None:
        _within(grads[2], db, deep * dy.double().abs().sum(0) + 2.0 ** -8 * db.abs(), "dbias")


SHAPES = [(1, 8), (1, 2560), (2, 40), (5, 64), (64, 2560), (333, 512), (130, 520), (67, 1032), (1001, 1536),
          (70, 2048), (33, 2568), (501, 4096), (40, 4104), (19, 8192), (7, 8200), (21, 16384), (3001, 2560),
          (601, 2056), (513, 2048), (2100, 1544), (1030, 2560), (300, 5000), (603, 6152), (9, 12288), (520, 12296)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("checkpoint", [False, True])
def test_layer_norm(gpu, rows, cols, checkpoint):
    x, w, b, dy = _inputs(rows, cols, rows + cols)
    _check(gpu, x, w, b, dy, 1e-6, checkpoint)
    _check(gpu, x, w, None, dy, 1e-2, checkpoint)


@pytest.mark.parametrize("checkpoint", [False, True])
def test_rows_far_from_zero(gpu, checkpoint):
    """A mean 50 times the deviation: the variance is of the differences, not of the squares."""
    x, w, b, dy = _inputs(40, 1024, 1)
    x = (x.float() / torch.logspace(-2, 2, 40)[:, None] + 50.0).to(BF16)
    _check(gpu, x, w, b, dy, 1e-6, checkpoint)


def test_shapes_and_strides(gpu):
    """Batched, strided, misaligned and transposed inputs and gradients are read as what they show."""
    x, w, b, dy = _inputs(24, 64, 3)
    _check(gpu, x, w, b, dy, 1e-6, False, shape=(2, 3, 4, 64))
    _check(gpu, x, w, b, dy, 1e-6, True, shape=(24, 1, 64))
    want = ops.layernorm(x.to(gpu), w.to(gpu), b.to(gpu), 1e-6)[0]
    big = torch.zeros(24, 160, dtype=BF16, device=gpu)
    big[:, 3:67] = x.to(gpu)
    assert torch.equal(ops.layernorm(big[:, 3:67], w.to(gpu), b.to(gpu), 1e-6)[0], want)
    assert torch.equal(ops.layernorm(x.t().contiguous().to(gpu).t(), w.to(gpu), b.to(gpu), 1e-6)[0], want)
    ww = torch.zeros(129, dtype=BF16, device=gpu)
    ww[1::2] = w.to(gpu)
    assert torch.equal(ops.layernorm(x.to(gpu), ww[1::2], b.to(gpu), 1e-6)[0], want)
    leaf = x.to(gpu).requires_grad_()
    y = fused_mlp.layer_norm(leaf, w.to(gpu))
    (g1,) = torch.autograd.grad(y, leaf, dy.to(gpu), retain_graph=True)
    (g2,) = torch.autograd.grad(y, leaf, dy.t().contiguous().to(gpu).t(), retain_graph=True)
    (g3,) = torch.autograd.grad(y.sum(), leaf)  # an expanded gradient
    assert torch.equal(g1, g2) and g3.shape == g1.shape
    flat = torch.zeros(24 * 64 + 1, dtype=BF16, device=gpu)
    flat[1:] = dy.to(gpu).flatten()
    (g4,) = torch.autograd.grad(fused_mlp.layer_norm(leaf, w.to(gpu)), leaf, flat[1:].view(24, 64))
    assert torch.equal(g1, g4)


def test_checkpoint_is_the_quantizers(gpu):
    for rows, cols in ((5, 40), (300, 2560), (40, 4104), (9, 16384)):
        x, w, b, _ = (t.to(gpu) for t in _inputs(rows, cols, cols))
        y, mean, rstd, q = ops.layernorm(x, w, b, 1e-6, want_stats=True, checkpoint=True)
        want = ops.quantize_mxint8(x)
        assert torch.equal(q.data, want.data) and torch.equal(q.exps, want.exps)
        plain = ops.layernorm(x, w, b, 1e-6, want_stats=True)
        assert torch.equal(y, plain[0]) and torch.equal(mean, plain[1]) and torch.equal(rstd, plain[2])
        assert ops.layernorm(x, w, b, 1e-6)[1:] == (None, None, None)


def test_gradients_are_the_differences(gpu):
    """Central differences of the layer norm in 64 bits against the kernel's gradient, along random
    directions: second order in the step (1e-4), and the gradients' rounding to bf16, 2^-8 of each term."""
    x, w, b, dy = _inputs(12, 48, 5)
    leaves = [t.to(gpu).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(fused_mlp.layer_norm(*leaves, 1e-3), leaves, dy.to(gpu))
    g = torch.Generator().manual_seed(0)

    def f(x, w, b):
        return (torch.nn.functional.layer_norm(x, (48,), w, b, 1e-3) * dy.double()).sum()
    base = [t.double() for t in (x, w, b)]
    for k in range(3):
        for _ in range(4):
            d = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
            if k == 0:  # in units of each row's deviation
                d = d * base[0].std(-1, keepdim=True)
            up, down = [[t + s * 1e-4 * d if i == k else t for i, t in enumerate(base)] for s in (1, -1)]
            diff = (f(*up) - f(*down)) / 2e-4
            terms = grads[k].cpu().double() * d
            assert abs(diff - terms.sum()) <= 2.0 ** -8 * terms.abs().sum() + 1e-6 * abs(diff)


def test_special_rows(gpu):
    """A constant row is the bias; a row with NaN or inf is NaN, the others keep theirs, in the gradient of
    x too; eps 0 on a row of one value gives NaN as the formula does."""
    x, w, b, dy = _inputs(20, 256, 7)
    x[3], x[4] = 2.5, 0.0
    y = ops.layernorm(x.to(gpu), w.to(gpu), b.to(gpu), 1e-6)[0].cpu()
    assert torch.equal(y[3], b) and torch.equal(y[4], b)
    bad = x.clone()
    bad[7, 9], bad[11, 0] = float("nan"), float("inf")
    for checkpoint in (False, True):
        got = []
        for t in (x, bad):
            leaf = t.to(gpu).requires_grad_()
            y = fused_mlp.layer_norm(leaf, w.to(gpu), b.to(gpu), checkpoint=checkpoint)
            got.append((y.detach().cpu(), torch.autograd.grad(y, leaf, dy.to(gpu))[0].cpu()))
        rows = [i for i in range(20) if i not in (7, 11)]
        for a, c in zip(*got):
            assert torch.equal(a[rows], c[rows]) and bool(torch.isnan(c[[7, 11]]).all())
    assert bool(torch.isnan(ops.layernorm(x[3:4].to(gpu), w.to(gpu), b.to(gpu), 0.0)[0]).all())


def test_parts_of_the_gradient_and_no_rows(gpu):
    x, w, b, dy = (t.to(gpu) for t in _inputs(300, 520, 2))
    for q in (False, True):
        _, mean, rstd, c = ops.layernorm(x, w, b, 1e-6, want_stats=True, checkpoint=q)
        held = c if q else x
        every = ops.layernorm_backward(held, dy, w, mean, rstd)
        for needs in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
            got = ops.layernorm_backward(held, dy, w, mean, rstd, needs=needs)
            for n, g, e in zip(needs, got, every):
                assert torch.equal(g, e) if n else g is None
        # the same bits every time
        assert all(torch.equal(a, e) for a, e in zip(ops.layernorm_backward(held, dy, w, mean, rstd), every))
    leaves = [t.detach().clone().requires_grad_() for t in (x[:0], w, b)]
    for q in (False, True):
        y = fused_mlp.layer_norm(*leaves, checkpoint=q)
        grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
        assert tuple(y.shape) == (0, 520) and tuple(grads[0].shape) == (0, 520)
        assert not bool(grads[1].any()) and not bool(grads[2].any())


def test_past_32_bit_offsets(gpu):
    rows, cols, tail = (1 << 31) // 16384 + 70, 16384, 50
    x, w, b, dy = (t.to(gpu) for t in _inputs(tail, cols, 4))
    big = torch.zeros(rows, cols, dtype=BF16, device=gpu)
    big[-tail:] = x
    d = torch.zeros(rows, cols, dtype=BF16, device=gpu)
    d[-tail:] = dy
    y, mean, rstd, q = ops.layernorm(big, w, b, 1e-6, want_stats=True, checkpoint=True)
    y2, mean2, rstd2, q2 = ops.layernorm(x, w, b, 1e-6, want_stats=True, checkpoint=True)
    assert torch.equal(y[-tail:], y2) and torch.equal(q.data[-tail:], q2.data)
    assert torch.equal(q.exps[-tail:], q2.exps) and torch.equal(mean[-tail:], mean2)
    del y
    for held, held2 in ((big, x), (q, q2)):
        dx = ops.layernorm_backward(held, d, w, mean, rstd, needs=(True, False, False))[0]
        assert torch.equal(dx[-tail:], ops.layernorm_backward(held2, dy, w, mean2, rstd2)[0])


def test_refusals(gpu):
    x, w, b, dy = (t.to(gpu) for t in _inputs(6, 64, 1))
    with pytest.raises(Exception, match="cols % 8"):
        ops.layernorm(x[:, :12], w[:12], None, 1e-6)
    with pytest.raises(ValueError, match="weight must be"):
        ops.layernorm(x, w[:32], None, 1e-6)
    with pytest.raises(ValueError, match="bias must be"):
        ops.layernorm(x, w, b.float(), 1e-6)
    with pytest.raises(TypeError, match="bfloat16"):
        ops.layernorm(x.float(), w, b, 1e-6)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.layernorm(x.cpu(), w.cpu(), None, 1e-6)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.layernorm(x, w.cpu(), None, 1e-6)
    _, mean, rstd, q = ops.layernorm(x, w, b, 1e-6, want_stats=True, checkpoint=True)
    with pytest.raises(ValueError, match="x must be"):
        ops.layernorm_backward(x[:3], dy, w, mean, rstd)
    with pytest.raises(ValueError, match="checkpoint must be"):
        ops.layernorm_backward(q, dy[:, :32], w[:32], mean, rstd)
    with pytest.raises(ValueError, match="mean must be"):
        ops.layernorm_backward(x, dy, w, mean[:3], rstd)
