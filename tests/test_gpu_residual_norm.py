"""GPU tests of the residual norm (bf8_rmsnorm_residual_bf16 and its backward) against the
formulas in 64 bits on the same bf16 inputs.

Bounds, counted before the first run: a bf16 result is off by its own rounding, 2^-8 of the
value, and by the fp32 arithmetic before it. A row sum of squares of n terms in any order is off by
n * 2^-24 of itself at most and the reciprocal root by half that and a few roundings: (n + 16) *
2^-24 of each product bounds it. A mean over the row of terms t is off by n * 2^-24 * mean|t|, so
the gradients are bounded with the sums of their terms' magnitudes, and the weights' gradients, sums over rows,
by one more rounding per row. y is compared with the norm of the kernel's own rounded out.
"""

import pytest
import torch
from torch.autograd import forward_ad

from bongard_amd import fused_mlp, linear, ops
from oracle import mxfp4_oracle as mx4

pytestmark = pytest.mark.gpu
U, B16 = 2.0 ** -24, 2.0 ** -8
EPS = 1e-6


def _inputs(rows, cols, seed, gate):
    g = torch.Generator().manual_seed(seed)
    def r(*s, std=1.0):
        return (torch.randn(*s, generator=g) * std).to(torch.bfloat16)
    t = dict(h=r(rows, cols, std=0.3), res=r(rows, cols), post=r(cols, std=0.2), pre=r(cols, std=0.2),
             gate=r(cols) if gate else None, dout=r(rows, cols, std=1e-2), dy=r(rows, cols, std=1e-2))
    t["res"][:, cols // 2] *= 30.0
    if rows > 3:
        t["h"][1] = 0.0
        t["h"][2] *= 1e4
        t["res"][3] = 0.0
        t["h"][3] = 0.0  # a row of zeros all the way
    return t


def _formulas(t, scale, z, out):
    """(results, bounds) of forward and backward in fp64, from the kernel's out."""
    d = {k: v.double() for k, v in t.items() if v is not None}
    h, res, post, pre, dout, dy = (d[k] for k in ("h", "res", "post", "pre", "dout", "dy"))
    gate = d.get("gate", torch.ones_like(post))
    rows, cols = h.shape
    r1 = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    r2 = 1 / (out.square().mean(-1, keepdim=True) + EPS).sqrt()
    n1, n2 = h * r1, out * r2
    n = gate * n1 * (z + post)
    ref, tol = {}, {}
    ref["out"] = scale * res + n
    tol["out"] = B16 * ref["out"].abs() + (cols + 16) * U * n.abs() + 4 * U * (scale * res).abs()
    ref["y"] = n2 * (z + pre)
    tol["y"] = (B16 + (cols + 16) * U) * ref["y"].abs()
    c = dy * (z + pre)
    g = dout + r2 * (c - n2 * (c * n2).mean(-1, keepdim=True))
    g_abs = dout.abs() + r2 * (c.abs() + n2.abs() * (c * n2).abs().mean(-1, keepdim=True))
    ref["dres"] = scale * g
    tol["dres"] = B16 * ref["dres"].abs() + (3 * cols + 32) * U * abs(scale) * g_abs
    w = (gate * (z + post)).abs()
    e = g * gate * (z + post)
    ref["dh"] = r1 * (e - n1 * (e * n1).mean(-1, keepdim=True))
    bound = r1 * (w * g_abs + n1.abs() * (w * g_abs * n1.abs()).mean(-1, keepdim=True))
    tol["dh"] = B16 * ref["dh"].abs() + (6 * cols + 64) * U * bound
    S, S_abs = (g * n1).sum(0), (g_abs * n1.abs()).sum(0)
    P, P_abs = (dy * n2).sum(0), (dy * n2).abs().sum(0)
    k = (rows + 4 * cols + 64) * U
    ref["dpost"], tol["dpost"] = gate * S, k * gate.abs() * S_abs
    ref["dpre"], tol["dpre"] = P, k * P_abs
    ref["dgate"], tol["dgate"] = (z + post) * S, k * (z + post).abs() * S_abs
    for name in ("dpost", "dpre", "dgate"):
        tol[name] = tol[name] + B16 * ref[name].abs()
    return ref, tol


SHAPES = [(1, 8), (5, 64), (33, 520), (64, 2560), (700, 1000), (3001, 256), (130, 2568), (7, 4096),
          (65, 5120), (9, 8192), (5, 16384), (4099, 2560)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("gate,scale,zero_centered", [(False, 1.0, True), (True, 0.5, True),
                                                      (True, -1.25, False)])
def test_matches_the_formulas(gpu, rows, cols, gate, scale, zero_centered):
    t = _inputs(rows, cols, rows + cols, gate)
    dev = {k: None if v is None else v.to(gpu) for k, v in t.items()}
    kw = dict(gate=dev["gate"], residual_scale=scale, zero_centered=zero_centered)
    out, y = ops.rmsnorm_residual(dev["h"], dev["res"], dev["post"], dev["pre"], EPS, **kw)
    grads = ops.rmsnorm_residual_backward(dev["h"], out, dev["dout"], dev["dy"], dev["post"], dev["pre"],
                                          EPS, **kw)
    ref, tol = _formulas(t, scale, 1.0 if zero_centered else 0.0, out.cpu().double())
    got = dict(out=out, y=y, **dict(zip(("dh", "dres", "dpost", "dpre", "dgate"), grads)))
    assert (got["dgate"] is None) == (not gate)
    for name, v in got.items():
        if v is not None:
            worst = ((v.cpu().double() - ref[name]).abs() / tol[name].clamp(min=1e-300)).max().item()
            assert worst <= 1.0, f"{name}: {worst:.3g} of the bound"
    again = ops.rmsnorm_residual_backward(dev["h"], out, dev["dout"], dev["dy"], dev["post"], dev["pre"],
                                          EPS, **kw)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("given", ["dout", "dy"])
def test_one_gradient_alone(gpu, given):
    """A missing gradient counts as zeros; what is not asked for is not computed and the rest is
    the same."""
    t = {k: v.to(gpu) for k, v in _inputs(40, 512, 3, True).items()}
    out, _ = ops.rmsnorm_residual(t["h"], t["res"], t["post"], t["pre"], EPS, gate=t["gate"])
    zero = torch.zeros_like(t["dy"])
    args = dict(dout=zero, dy=zero)
    args[given] = t[given]
    want = ops.rmsnorm_residual_backward(t["h"], out, args["dout"], args["dy"], t["post"], t["pre"], EPS,
                                         gate=t["gate"])
    args = dict(dout=None, dy=None)
    args[given] = t[given]
    got = ops.rmsnorm_residual_backward(t["h"], out, args["dout"], args["dy"], t["post"], t["pre"], EPS,
                                        gate=t["gate"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for k in range(5):
        needs = [i == k for i in range(5)]
        one = ops.rmsnorm_residual_backward(t["h"], out, args["dout"], args["dy"], t["post"], t["pre"],
                                            EPS, gate=t["gate"], needs=needs)
        assert [v is not None for v in one] == needs and torch.equal(one[k], want[k])


def test_autograd_and_differences(gpu):
    """residual_norm's gradients are the backward op's, also where one result goes unused, and its
    forward moves as they say: along the gradient of <out, u> + <y, v>, a central difference of the bf16
    results, whose rounding noise (2^-8 of each of the results, uncorrelated) is far below the step."""
    t = {k: v.to(gpu) for k, v in _inputs(96, 640, 11, True).items()}
    names = ("h", "res", "post", "pre", "gate")
    shaped = {k: (v.view(2, 48, 640) if v.dim() == 2 else v) for k, v in t.items()}
    leaves = [shaped[n].clone().requires_grad_() for n in names]
    out, y = fused_mlp.residual_norm(*leaves[:4], EPS, gate=leaves[4], residual_scale=0.7)
    assert out.shape == y.shape == (2, 48, 640)
    grads = torch.autograd.grad([out, y], leaves, [shaped["dout"], shaped["dy"]], retain_graph=True)
    want = ops.rmsnorm_residual_backward(t["h"], out.detach().view(96, 640), t["dout"], t["dy"], t["post"],
                                         t["pre"], EPS, gate=t["gate"], residual_scale=0.7)
    for a, b in zip(grads, want):
        assert torch.equal(a.reshape(b.shape), b)
    only = torch.autograd.grad(out, leaves, shaped["dout"], allow_unused=True, retain_graph=True)
    assert only[3] is None or bool((only[3] == 0).all())
    x = {n: t[n].cpu().double() for n in names}
    u, v = t["dout"].cpu().double(), t["dy"].cpu().double()

    def f(move):
        o, w = ops.rmsnorm_residual(*[(x[n] + move.get(n, 0)).to(torch.bfloat16).to(gpu)
                                      for n in names[:4]], EPS,
                                    gate=(x["gate"] + move.get("gate", 0)).to(torch.bfloat16).to(gpu),
                                    residual_scale=0.7)
        return (o.cpu().double() * u).sum() + (w.cpu().double() * v).sum()

    for n, g in zip(names, want):
        g = g.cpu().double()
        step = {"h": 0.02, "res": 0.05}.get(n, 0.05) * g.sign()
        if n == "h":
            step[1:4] = 0.0  # rows of zeros and of 1e4: not smooth, not moved
        if n == "res":
            step[3] = 0.0
        lo, hi = ((x[n] + s * step).to(torch.bfloat16).double() for s in (-1, 1))
        told = (g * (hi - lo)).sum()
        diff = f({n: hi - x[n]}) - f({n: lo - x[n]})
        assert abs(diff - told) <= 0.05 * abs(told), (n, diff.item(), told.item())


def test_rows_past_32_bit_offsets(gpu):
    """Tensors of more than 4 GiB: every row's results are those of a call on a few rows."""
    cols, few = 2560, 64
    t = {k: v.to(gpu) for k, v in _inputs(few, cols, 7, True).items()}
    rows = few * 13200
    many = {k: (v.repeat(rows // few, 1) if v.dim() == 2 else v) for k, v in t.items()}
    assert many["h"].numel() * 2 > 1 << 32
    kw = dict(gate=t["gate"], residual_scale=0.5)
    out, y = ops.rmsnorm_residual(many["h"], many["res"], t["post"], t["pre"], EPS, **kw)
    want = ops.rmsnorm_residual(t["h"], t["res"], t["post"], t["pre"], EPS, **kw)
    grads = ops.rmsnorm_residual_backward(many["h"], out, many["dout"], many["dy"], t["post"], t["pre"],
                                          EPS, **kw, needs=(True, True, False, False, False))
    told = ops.rmsnorm_residual_backward(t["h"], want[0], t["dout"], t["dy"], t["post"], t["pre"], EPS, **kw)
    for a, b in zip((out, y, *grads[:2]), (*want, *told[:2])):
        assert bool((a.view(-1, few, cols) == b).all())


def test_rows_as_they_come(gpu):
    """Strided and misaligned inputs, no rows, and NaN or inf rows that leave the others alone."""
    t = {k: v.to(gpu) for k, v in _inputs(64, 256, 5, False).items() if v is not None}
    want = ops.rmsnorm_residual(t["h"], t["res"], t["post"], t["pre"], EPS)
    wide = torch.zeros(64, 300, dtype=torch.bfloat16, device=gpu)
    wide[:, 3:259] = t["h"]
    flat = torch.zeros(64 * 256 + 1, dtype=torch.bfloat16, device=gpu)
    flat[1:] = t["res"].flatten()
    got = ops.rmsnorm_residual(wide[:, 3:259], flat[1:].view(64, 256), t["post"], t["pre"], EPS)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    h = t["h"].clone()
    h[4, 7], h[9, 0] = float("nan"), float("inf")
    out, y = ops.rmsnorm_residual(h, t["res"], t["post"], t["pre"], EPS)
    rows = [i for i in range(64) if i not in (4, 9)]
    assert torch.equal(out[rows], want[0][rows]) and torch.equal(y[rows], want[1][rows])
    assert bool(torch.isnan(y[4]).all()) and bool(torch.isnan(out[9, 0]))
    none = torch.empty(0, 256, dtype=torch.bfloat16, device=gpu)
    out, y = ops.rmsnorm_residual(none, none, t["post"], t["pre"], EPS)
    assert out.shape == y.shape == (0, 256)
    grads = ops.rmsnorm_residual_backward(none, none, none, none, t["post"], t["pre"], EPS)
    assert bool((grads[2] == 0).all()) and bool((grads[3] == 0).all()) and grads[0].shape == (0, 256)


def test_refusals(gpu):
    t = {k: v.to(gpu) for k, v in _inputs(8, 64, 5, True).items()}
    f = lambda **kw: ops.rmsnorm_residual(*[{**t, **kw}[n] for n in ("h", "res", "post", "pre")], EPS,  # noqa: E731
                                          gate=kw.get("gate"))
    with pytest.raises(ValueError, match="residual must be"):
        f(res=t["res"][:4])
    with pytest.raises(ValueError, match="post_weight"):
        f(post=t["post"][:32])
    with pytest.raises(ValueError, match="pre_weight"):
        f(pre=t["pre"].float())
    with pytest.raises(ValueError, match="gate"):
        f(gate=t["gate"][:8])
    with pytest.raises(TypeError, match="bfloat16"):
        f(h=t["h"].float())
    with pytest.raises(RuntimeError, match="HIP device"):
        f(h=t["h"].cpu())
    with pytest.raises(Exception, match="cols"):
        f(h=t["h"][:, :12], res=t["res"][:, :12], post=t["post"][:12], pre=t["pre"][:12])
    with pytest.raises(Exception, match="16384"):
        z = torch.zeros(1, 16392, dtype=torch.bfloat16, device=gpu)
        ops.rmsnorm_residual(z, z, z[0], z[0], EPS)
    with pytest.raises(ValueError, match="no gradient"):
        ops.rmsnorm_residual_backward(t["h"], t["res"], None, None, t["post"], t["pre"], EPS)


@pytest.mark.parametrize("mode", ["no_grad", "nothing_trained", "compiled"])
def test_every_way_of_calling_gives_the_same(gpu, mode):
    """residual_norm without gradients, and from code under torch.compile (which leaves it out of its
    graphs), against a recorded call."""
    t = {k: v.to(gpu) for k, v in _inputs(9, 264, 5, True).items()}

    def call(h, res, post, pre, gate):
        out, y = fused_mlp.residual_norm(h, res, post, pre, EPS, gate=gate, residual_scale=0.5)
        return out + 0.0, y + 0.0

    args = [t[k].clone().requires_grad_(True) for k in ("h", "res", "post", "pre", "gate")]
    want = call(*args)
    if mode == "compiled":
        got = torch.compile(call, backend="eager")(*args)
        grads = [torch.autograd.grad(r, args, (t["dout"], t["dy"])) for r in (got, want)]
        assert all(torch.equal(a, b) for a, b in zip(*grads))
    elif mode == "no_grad":
        with torch.no_grad():
            got = call(*args)
    else:
        got = call(*(a.detach() for a in args))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(a.requires_grad == (mode == "compiled") for a in got)


def test_forward_mode(gpu):
    """A dual tensor is refused by residual_norm and by the layers around it, in and out of no_grad, and no
    call returns results without its tangent; calls that hold none are as ever, beside it and after."""
    t = {k: v.to(gpu) for k, v in _inputs(9, 256, 5, True).items()}
    names = ("h", "res", "post", "pre")
    want = fused_mlp.residual_norm(*[t[n] for n in names], EPS, gate=t["gate"])
    w = torch.zeros(256, 256, dtype=torch.bfloat16, device=gpu)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            got = fused_mlp.residual_norm(*[t[n] for n in names], EPS, gate=t["gate"])
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            for name in (*names, "gate"):
                d = {**t, name: forward_ad.make_dual(t[name], torch.ones_like(t[name]))}
                with pytest.raises(NotImplementedError, match="jvp"):
                    fused_mlp.residual_norm(*[d[n] for n in names], EPS, gate=d["gate"])
            d = forward_ad.make_dual(t["h"], t["h"])
            with pytest.raises(NotImplementedError, match="jvp"):
                linear.Mxfp4LinearFunction.apply(d, w, None)
            with pytest.raises(NotImplementedError, match="jvp"):
                linear.Mxfp4GegluMlpFunction.apply(d, w, w[:, :128].contiguous(), None, None, 128)
    got = fused_mlp.residual_norm(*[t[n] for n in names], EPS, gate=t["gate"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows,cols", [(2100, 2568), (2100, 4104), (2100, 8200)])
def test_blocks_that_take_several_wide_rows(gpu, rows, cols):
    """Rows of a block each (past 2560 columns, every width's kernel), more of them than the forward's and the
    backward's blocks: a block's next row, its sums over rows, and the partials of the whole grid."""
    t = _inputs(rows, cols, rows + cols, True)
    dev = {k: v.to(gpu) for k, v in t.items()}
    kw = dict(gate=dev["gate"], residual_scale=0.5)

    def call():
        out, y = ops.rmsnorm_residual(dev["h"], dev["res"], dev["post"], dev["pre"], EPS, **kw)
        return dict(zip(("out", "y", "dh", "dres", "dpost", "dpre", "dgate"),
                        (out, y, *ops.rmsnorm_residual_backward(dev["h"], out, dev["dout"], dev["dy"],
                                                                dev["post"], dev["pre"], EPS, **kw))))

    got, again = call(), call()
    ref, tol = _formulas(t, 0.5, 1.0, got["out"].cpu().double())
    for name, v in got.items():
        worst = ((v.cpu().double() - ref[name]).abs() / tol[name].clamp(min=1e-300)).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3g} of the bound"
        assert torch.equal(v, again[name]), name


@pytest.mark.parametrize("rows,cols,gate,scale,z", [(65, 2560, True, 0.5, 1.0), (33, 4096, False, -1.25, 0.0)])
def test_forward_against_the_oracle(gpu, rows, cols, gate, scale, z):
    """out, and y as the norm of that out (a normed h of zeros added to it)."""
    t = _inputs(rows, cols, 13, gate)
    dev = {k: None if v is None else v.to(gpu) for k, v in t.items()}
    out, y = (v.cpu().double() for v in ops.rmsnorm_residual(
        dev["h"], dev["res"], dev["post"], dev["pre"], EPS, gate=dev["gate"], residual_scale=scale,
        zero_centered=bool(z)))
    d = {k: None if v is None else v.double() for k, v in t.items()}
    ref, _ = mx4.residual_norm(d["h"], d["res"], d["post"], d["pre"], EPS, d["gate"], scale, z)
    n = (ref - scale * d["res"]).abs()
    tol = B16 * ref.abs() + (cols + 16) * U * n + 4 * U * (scale * d["res"]).abs()
    assert bool(((out - ref).abs() <= tol).all())
    _, ref = mx4.residual_norm(0 * d["h"], out, d["post"], d["pre"], EPS, d["gate"], 1.0, z)
    assert bool(((y - ref).abs() <= (B16 + (cols + 16) * U) * ref.abs()).all())
