"""GPU tests of the MXFP4 path against the CPU oracle.

  * quantize: codes and scale planes equal to the oracle's, bit for bit, either copy;
  * read-back: exactly the codes' values (bf16 holds them);
  * product: the terms are exact, so an fp32 sum of K of them in any order, each addition off by
    an ulp at most, is within K * 2^-23 * sum|a b|; a bf16 result is off by its rounding more,
    2^-8 of the value;
  * the gated MLP and the modules: every step equals the separate ops on the same inputs, bit for
    bit, and on inputs the format holds exactly the gradients are the differences.
"""

import threading
import types

import pytest
import torch
from torch import nn

from bongard_amd import _lib, fused_mlp, linear, ops, te_linear
from oracle import fp8_oracle as orc
from oracle import mxfp4_oracle as mx4

pytestmark = pytest.mark.gpu


def _x(rows, cols, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if spread:
        x *= torch.logspace(-8, 8, rows)[:, None]
        x[:, cols // 3] *= 300.0
        x[rows // 2, : min(cols, 32)] = 0.0
    return x.to(torch.bfloat16)


def _special(rows, cols, seed):
    """Blocks holding inf, NaN, the largest and the smallest magnitudes."""
    x = _x(rows, cols, seed, spread=False)
    x[0, cols - 1], x[rows - 1, 0], x[rows // 2, cols // 2] = float("inf"), float("nan"), -float("inf")
    x[rows // 3, :8] = 3.38e38
    x[rows - 1, cols // 2:] = 1e-39
    return x


def _check(q, x, rowwise, colwise):
    if rowwise:
        codes, e = mx4.quantize(x)
        assert torch.equal(q.planes.cpu(), mx4.planes(e))
        assert torch.equal(q.data.cpu(), codes)
        back = ops.dequant_mxfp4(q).cpu().double()
        assert torch.equal(torch.nan_to_num(back, 1e30), torch.nan_to_num(
            mx4.values(codes, e).to(torch.bfloat16).double(), 1e30))
    if colwise:
        codes, e = mx4.quantize(x, 0)
        assert torch.equal(q.planes_t.cpu(), mx4.planes(e))
        assert torch.equal(q.data_t.cpu(), codes)
        back = ops.dequant_mxfp4(q, transpose=True).cpu().double()
        assert tuple(back.shape) == (x.shape[1], x.shape[0])
        assert torch.equal(torch.nan_to_num(back, 1e30), torch.nan_to_num(
            mx4.values(codes, e).to(torch.bfloat16).double(), 1e30)[:, :x.shape[0]])


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (33, 160), (64, 2560), (95, 256), (257, 512),
                                       (500, 2048), (2001, 1056), (4100, 2592)])
@pytest.mark.parametrize("make", [_x, _special])
def test_quantize_bit_exact(gpu, rows, cols, make):
    x = make(rows, cols, rows + cols)
    for rowwise, colwise in ((True, False), (False, True), (True, True)):
        _check(ops.quantize_mxfp4(x.to(gpu), rowwise=rowwise, colwise=colwise), x, rowwise, colwise)


@pytest.mark.parametrize("rows,cols", [(32, 8), (40, 24), (1, 40), (130, 1000)])
def test_quantize_columns_alone_of_any_width(gpu, rows, cols):
    x = _x(rows, cols, rows * cols)
    _check(ops.quantize_mxfp4(x.to(gpu), rowwise=False, colwise=True), x, False, True)


def test_quantize_every_mantissa_under_every_scale(gpu):
    """For each exponent of a block's largest value, every bf16 magnitude from it down to where
    all codes are 0: the conversions round as the oracle at every tie and every scale."""
    blocks = []
    for top in list(range(0, 0x7F80, 0x80)) + list(range(0x40, 0x7F80, 0x80)) + list(range(0x41, 0x7F80, 0x80)):
        low = max(0, top - 5 * 128)
        keys = torch.arange(low, top + 1, dtype=torch.int32)
        keys = torch.nn.functional.pad(keys, (0, -len(keys) % 31))
        k = keys.reshape(-1, 31)
        k = torch.cat([torch.full((k.shape[0], 1), top, dtype=torch.int32), k], 1)
        sign = (torch.arange(k.numel()).reshape(k.shape) % 3 == 1).int() << 15
        blocks.append(k | sign)
    keys = torch.cat(blocks)
    x = torch.where(keys >= 0x8000, keys - 0x10000, keys).to(torch.int16).view(torch.bfloat16)
    x = x.reshape(-1, 32)
    _check(ops.quantize_mxfp4(x.to(gpu)), x, True, False)


def test_quantize_views_and_strides(gpu):
    """Strided, transposed, misaligned and batched inputs are read as what they show."""
    big = _x(70, 300, 3).to(gpu)
    for view in (big[:, 4:292], big[1::2, :64], big.t()[:64, :64], big[3:67].reshape(2, 32, 300)[..., :96],
                 big.flatten()[1:1 + 64 * 64].view(64, 64)):
        flat = view.reshape(-1, view.shape[-1]).contiguous().cpu()
        _check(ops.quantize_mxfp4(view, colwise=True), flat, True, True)


def test_quantize_empty_and_large_offsets(gpu):
    q = ops.quantize_mxfp4(torch.empty(0, 64, dtype=torch.bfloat16, device=gpu), colwise=True)
    assert tuple(q.data.shape) == (0, 32) and tuple(q.data_t.shape) == (64, 0)
    assert tuple(ops.dequant_mxfp4(q).shape) == (0, 64)
    # element offsets past 2^31: the last rows are quantized as by themselves
    rows, cols = (1 << 31) // 16384 + 70, 16384
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=gpu)
    x[:-100].zero_()
    tail = _x(100, cols, 9)
    x[-100:] = tail.to(gpu)
    q = ops.quantize_mxfp4(x)
    codes, e = mx4.quantize(tail)
    assert torch.equal(q.data[-100:].cpu(), codes)
    assert torch.equal(q.planes[:, -100:].cpu(), mx4.planes(e))
    assert torch.equal(ops.dequant_mxfp4(q)[-100:].cpu().double(), mx4.values(codes, e))


def _operand(rows, K, seed, gpu, spread=True):
    x = _x(rows, K, seed, spread)
    q = ops.quantize_mxfp4(x.to(gpu))
    return q, mx4.quantize(x)


def _check_product(y, ref, mag, K, dtype):
    err = (y.cpu().double() - ref).abs()
    tol = K * 2.0 ** -23 * mag
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} of the bound"


PRODUCTS = [(1, 8, 32), (1, 2048, 2560), (7, 40, 96), (33, 64, 160), (64, 1024, 2560), (129, 264, 224),
            (256, 256, 512), (500, 2560, 2048), (300, 520, 5152), (2001, 640, 1056), (520, 1032, 10240)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(gpu, M, N, K):
    a, ra = _operand(M, K, M + K, gpu)
    b, rb = _operand(N, K, N + K, gpu, spread=False)
    ref, mag = mx4.mm(ra, rb)
    bias = _x(1, N, 5, spread=False)[0].to(gpu)
    y32 = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32)
    _check_product(y32, ref, mag, K, torch.float32)
    y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes)
    _check_product(y, ref, mag, K, torch.bfloat16)
    yb = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, bias=bias, out_dtype=torch.float32)
    full = ref + bias.cpu().double()
    _check_product(yb, full, mag + full.abs() + bias.cpu().double().abs(), K, torch.float32)
    # the same inputs again: the same bits
    assert torch.equal(y32, ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32))


def test_product_strides_and_out(gpu):
    """Operands whose rows are longer than K, an out whose rows are longer than N and whose other
    columns keep what they held."""
    M, N, K = 70, 136, 320
    a, ra = _operand(M, K, 1, gpu)
    b, rb = _operand(N, K, 2, gpu, spread=False)
    wide_a = torch.full((M, K // 2 + 64), 0x77, dtype=torch.uint8, device=gpu)
    wide_b = torch.full((N, K // 2 + 32), 0x77, dtype=torch.uint8, device=gpu)
    wide_a[:, :K // 2], wide_b[:, :K // 2] = a.data, b.data
    ref, mag = mx4.mm(ra, rb)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((M + 2, N + 24), 7.0, dtype=dtype, device=gpu)
        y = ops.gemm_mxfp4(wide_a[:, :K // 2], a.planes, wide_b[:, :K // 2], b.planes, out_dtype=dtype,
                           out=out[:M, :N])
        assert y.data_ptr() == out.data_ptr()
        _check_product(y, ref, mag, K, dtype)
        assert bool((out[M:] == 7).all()) and bool((out[:, N:] == 7).all())
    empty = ops.gemm_mxfp4(a.data[:0], a.planes[:, :0].contiguous(), b.data, b.planes)
    assert tuple(empty.shape) == (0, N)


def test_product_special_blocks(gpu):
    """A NaN block makes its row's products NaN, whatever the other operand holds there; the rows
    beside it keep theirs. Codes of zero under the largest and smallest scales stay zero."""
    M, N, K = 40, 48, 128
    xa, xb = _x(M, K, 3, spread=False), _x(N, K, 4, spread=False)
    xa[5, 70] = float("nan")
    xa[7, 32:64] = 0.0
    xb[9] = 0.0
    a, b = ops.quantize_mxfp4(xa.to(gpu)), ops.quantize_mxfp4(xb.to(gpu))
    y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32).cpu()
    ref, mag = mx4.mm(mx4.quantize(xa), mx4.quantize(xb))
    rows = [i for i in range(M) if i != 5]
    assert bool(torch.isnan(y[5]).all())
    _check_product(y[rows], ref[rows], mag[rows], K, torch.float32)
    assert bool((y[rows][:, 9] == 0).all())
    # tiny and huge blocks: 2^-60 and 2^60 in every combination that fp32 holds
    sa = torch.where(torch.arange(M) % 2 == 0, 2.0 ** 60, 2.0 ** -60)[:, None]
    xa = (_x(M, K, 6, spread=False).float() * sa).to(torch.bfloat16)
    a = ops.quantize_mxfp4(xa.to(gpu))
    y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32)
    ref, mag = mx4.mm(mx4.quantize(xa), mx4.quantize(xb))
    _check_product(y, ref, mag, K, torch.float32)


def _mlp_inputs(M, K, I, seed, gpu):
    g = torch.Generator().manual_seed(seed)
    def r(*s, std=1.0):
        return (torch.randn(*s, generator=g) * std).to(torch.bfloat16).to(gpu)
    return r(M, K), r(2 * I, K, std=0.05), r(K, I, std=0.05), r(M, K, std=1e-2)


@pytest.mark.parametrize("M,K,I", [(1, 32, 128), (33, 96, 128), (64, 256, 384), (300, 320, 640),
                                   (517, 512, 1024), (1030, 256, 2560)])
@pytest.mark.parametrize("colwise,keep", [(False, False), (True, True)])
def test_gated_product(gpu, M, K, I, colwise, keep):
    """GU is the product (as the separate op gives it within the order of its sums), and H's copies
    are the quantizer's of the gated GELU of that GU, bit for bit."""
    x, w, _, _ = _mlp_inputs(M, K, I, M + K + I, gpu)
    xq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    hq, GU = ops.gemm_geglu_mxfp4(xq.data, xq.planes, wq.data, wq.planes, I, colwise=colwise,
                                  keep_gu=True)
    ref, mag = mx4.mm(mx4.quantize(x.cpu()), mx4.quantize(w.cpu()))
    _check_product(GU, ref, mag, K, torch.bfloat16)
    H, _ = ops.geglu(GU)
    want = ops.quantize_mxfp4(H, colwise=colwise)
    assert torch.equal(hq.data, want.data) and torch.equal(hq.planes, want.planes)
    if colwise:
        assert torch.equal(hq.data_t, want.data_t) and torch.equal(hq.planes_t, want.planes_t)
    if not keep:
        h2, none = ops.gemm_geglu_mxfp4(xq.data, xq.planes, wq.data, wq.planes, I, colwise=colwise)
        assert none is None and torch.equal(h2.data, hq.data) and torch.equal(h2.planes, hq.planes)


@pytest.mark.parametrize("M,I", [(1, 128), (31, 256), (64, 640), (257, 384), (2001, 2560), (2304, 4096)])
def test_gated_backward(gpu, M, I):
    """dGU's copies are the quantizer's of the separate gated-GELU backward's output, bit for bit."""
    g = torch.Generator().manual_seed(M + I)
    dH = (torch.randn(M, I, generator=g) * 1e-2).to(torch.bfloat16).to(gpu)
    GU = torch.randn(M, 2 * I, generator=g).to(torch.bfloat16).to(gpu)
    GU[0, :3] = torch.tensor([12.0, -12.0, 1e-20])
    dGU, _ = ops.geglu_bwd(dH, GU)
    want = ops.quantize_mxfp4(dGU, colwise=True)
    for rowwise, colwise in ((True, True), (True, False), (False, True)):
        q = ops.geglu_bwd_mxfp4(dH, GU, rowwise=rowwise, colwise=colwise)
        if rowwise:
            assert torch.equal(q.data, want.data) and torch.equal(q.planes, want.planes)
        if colwise:
            assert torch.equal(q.data_t, want.data_t) and torch.equal(q.planes_t, want.planes_t)


@pytest.mark.parametrize("M,N,K", [(1, 32, 64), (50, 96, 128), (500, 256, 320), (1000, 1024, 512)])
def test_linear_function(gpu, M, N, K):
    """Forward, dX and dW against the oracle's products of the oracle's copies."""
    x, w, dy = _x(M, K, 1, False), _x(N, K, 2, False), _x(M, N, 3, False)
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    y = linear.Mxfp4LinearFunction.apply(xg, wg, None)
    y.backward(dy.to(gpu))
    for got, a, b, k in ((y.detach(), mx4.quantize(x), mx4.quantize(w), K),
                         (xg.grad, mx4.quantize(dy), mx4.quantize(w, 0), N),
                         (wg.grad, mx4.quantize(dy, 0), mx4.quantize(x, 0), M)):
        ref, mag = mx4.mm(a, b)
        _check_product(got, ref, mag, (k + 31) // 32 * 32, torch.bfloat16)


def test_linear_gradients_are_the_differences(gpu):
    """On values the format holds exactly (grid values, a 6 in every block either way) the layer is
    bilinear: y(x + d) - y(x) is exactly what the gradient says."""
    M, N, K = 64, 96, 128
    g = torch.Generator().manual_seed(0)
    grid = torch.tensor([-4., -3., -2., -1., 0., 1., 2., 3., 4.])
    def exact(*shape):
        t = grid[torch.randint(0, 9, shape, generator=g)]
        for k in range(0, shape[0], 32):  # a 6 for each block of rows and of columns
            for j in range(0, shape[1], 32):
                t[k + torch.arange(32), j + torch.randperm(32, generator=g)] = 6.0
        return t.to(torch.bfloat16)
    x, w, dy = exact(M, K), exact(N, K), exact(M, N)
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    linear.Mxfp4LinearFunction.apply(xg, wg, None).backward(dy.to(gpu))
    for name, base, grad in (("x", x, xg.grad), ("w", w, wg.grad)):
        step = torch.where((base != 6) & (torch.rand(base.shape, generator=g) < 0.3),
                           (base == 0).to(torch.bfloat16), torch.zeros_like(base))  # 0 -> 1
        moved = (base + step).to(gpu)
        args = (moved, w.to(gpu)) if name == "x" else (x.to(gpu), moved)
        qs = [ops.quantize_mxfp4(t) for t in args]
        q0 = [ops.quantize_mxfp4(t.to(gpu)) for t in (x, w)]
        f = lambda q: ops.gemm_mxfp4(q[0].data, q[0].planes, q[1].data, q[1].planes,  # noqa: E731
                                     out_dtype=torch.float32).cpu().double()
        diff = ((f(qs) - f(q0)) * dy.double()).sum()
        # the gradients are integers; bf16 keeps each within 2^-8 of itself
        told = (grad.cpu().double() * step.double()).sum()
        slack = 2.0 ** -8 * (grad.cpu().double().abs() * step.double()).sum()
        assert abs(diff - told) <= slack and diff != 0


@pytest.mark.parametrize("M,K,I", [(37, 96, 256), (512, 256, 384)])
def test_mlp_function_is_its_ops(gpu, M, K, I):
    x, w_gu, w_d, dy = _mlp_inputs(M, K, I, 5, gpu)
    leaves = [t.requires_grad_() for t in (x, w_gu, w_d)]
    y = linear.Mxfp4GegluMlpFunction.apply(*leaves, None, None, I)
    grads = torch.autograd.grad(y, leaves, dy)
    Q = lambda t: ops.quantize_mxfp4(t.detach(), colwise=True)  # noqa: E731
    xq, gq, dq = Q(x), Q(w_gu), Q(w_d)
    hq, GU = ops.gemm_geglu_mxfp4(xq.data, xq.planes, gq.data, gq.planes, I, colwise=True, keep_gu=True)
    mm = ops.gemm_mxfp4
    assert torch.equal(y, mm(hq.data, hq.planes, dq.data, dq.planes))
    yq = Q(dy)
    dH = mm(yq.data, yq.planes, dq.data_t, dq.planes_t)
    uq = ops.geglu_bwd_mxfp4(dH, GU, colwise=True)
    assert torch.equal(grads[0], mm(uq.data, uq.planes, gq.data_t, gq.planes_t))
    assert torch.equal(grads[1], mm(uq.data_t, uq.planes_t, xq.data_t, xq.planes_t))
    assert torch.equal(grads[2], mm(yq.data_t, yq.planes_t, hq.data_t, hq.planes_t))
    with torch.no_grad():
        assert torch.equal(linear.Mxfp4GegluMlpFunction.apply(x, w_gu, w_d, gq, dq, I), y)


class _Mlp(nn.Module):
    def __init__(self, hidden, inter):
        super().__init__()
        self.config = types.SimpleNamespace(hidden_activation="gelu_pytorch_tanh")
        self.hidden_size, self.intermediate_size = hidden, inter
        self.gate_proj, self.up_proj = (nn.Linear(hidden, inter, bias=False) for _ in range(2))
        self.down_proj = nn.Linear(inter, hidden, bias=False)
        self.dropout = nn.Dropout(0.0)


@pytest.mark.parametrize("split", [False, True])
def test_modules_run_the_recipe(gpu, monkeypatch, split):
    """TELinear, TEMLP (fused or split gate and up) and FusedMLP under 'mxfp4': ragged rows, cached
    weights, gradients equal to the functions' on the same tensors."""
    monkeypatch.setenv("BONGARD_TE_SPLIT_GATE_UP", "1" if split else "0")
    torch.manual_seed(0)
    H, I, M = 128, 256, 75
    x, dy = _x(M, H, 8, False).to(gpu), _x(M, H, 9, False).to(gpu)
    lin = te_linear.TELinear([nn.Linear(H, H, bias=False)], "mxfp4").to(gpu).train()
    xl = x.clone().requires_grad_()
    for _ in range(2):
        y = lin(xl.view(1, M, H))
    assert lin.counts["weight_quantizations"] == 1 and lin.counts["cached_weights"] == 1
    y.backward(dy.view(1, M, H))
    x2, w2 = x.clone().requires_grad_(), lin.weight.detach().clone().requires_grad_()
    linear.Mxfp4LinearFunction.apply(x2, w2, None).backward(dy)
    assert torch.equal(xl.grad, x2.grad) and torch.equal(lin.weight.grad, w2.grad)
    mlp = te_linear.TEMLP(_Mlp(H, I), "mxfp4").to(gpu).train()
    xm = x.clone().requires_grad_()
    ym = mlp(xm)
    ym.backward(dy)
    w_gu = mlp._gate_up_weight().detach().clone().requires_grad_()
    w_d = mlp.down.weight.detach().clone().requires_grad_()
    x2 = x.clone().requires_grad_()
    y2 = linear.Mxfp4GegluMlpFunction.apply(x2, w_gu, w_d, None, None, I)
    y2.backward(dy)
    assert torch.equal(ym, y2) and torch.equal(xm.grad, x2.grad)
    got = (torch.cat([mlp.gate_proj.weight.grad, mlp.up_proj.weight.grad]) if split
           else mlp.gate_up.weight.grad)
    assert torch.equal(got, w_gu.grad) and torch.equal(mlp.down.weight.grad, w_d.grad)
    if split:
        return
    norm = nn.Module()
    norm.weight, norm.eps = nn.Parameter(torch.randn(H).to(torch.bfloat16) * 0.1), 1e-6
    fused = fused_mlp.FusedMLP(_Mlp(H, I), norm, "mxfp4").to(gpu).train()
    xf = x.clone().requires_grad_()
    yf = fused(xf)
    yf.backward(dy)
    normed, _, _ = ops.rmsnorm(x, fused.layer_norm_weight.detach(), 1e-6)
    y2 = linear.Mxfp4GegluMlpFunction.apply(normed, fused.fc1_weight.detach(), fused.fc2_weight.detach(),
                                            None, None, I)
    assert torch.equal(yf, y2)
    assert all(p.grad is not None for p in fused.parameters()) and xf.grad.shape == x.shape


def test_layer_together_in_a_graph(gpu):
    """Residual norm, MLP and the next residual norm, forward and backward, captured once and
    replayed on new inputs beside eager work: every replay gives the eager bits. Two graphs of one
    stream own their workspaces."""
    H, I = 256, 512
    torch.manual_seed(1)
    w_gu = (torch.randn(2 * I, H, device=gpu) * 0.05).to(torch.bfloat16)
    w_d = (torch.randn(H, I, device=gpu) * 0.05).to(torch.bfloat16)
    ws = [(torch.randn(H, device=gpu) * 0.1).to(torch.bfloat16) for _ in range(4)]

    def step(h, res, dres, dy):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in (h, res, w_gu, w_d, *ws)]
            out, y = fused_mlp.residual_norm(leaves[0], leaves[1], leaves[4], leaves[5])
            m = linear.Mxfp4GegluMlpFunction.apply(y, leaves[2], leaves[3], None, None, I)
            out, y = fused_mlp.residual_norm(m, out, leaves[6], leaves[7])
            grads = torch.autograd.grad([out, y], leaves, [dres, dy])
        return [out.detach(), y.detach(), *grads]

    graphs = []
    for M in (70, 513):
        ins = [torch.randn(M, H, device=gpu).to(torch.bfloat16) for _ in range(4)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*ins)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*ins)
        graphs.append((graph, ins, outs))
    for rep in range(3):
        for graph, ins, outs in graphs:
            for t in ins:
                t.copy_(torch.randn_like(t))
            want = [t.clone() for t in step(*ins)]
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b), f"replay {rep}"


def test_products_past_32_bit_offsets(gpu):
    """Results of more than 4 GiB: the rows at the end are those of a call on them alone, which differ in no
    sum (the same plan's K order), and so are the gated product's and its backward's."""
    M, N, K, tail = 70016, 32768, 64, 512
    a, b = _x(tail, K, 1, spread=False).to(gpu), ops.quantize_mxfp4(_x(N, K, 2, spread=False).to(gpu))
    big = torch.zeros(M, K, dtype=torch.bfloat16, device=gpu)
    big[-tail:] = a
    q, small = ops.quantize_mxfp4(big), ops.quantize_mxfp4(a)
    y = ops.gemm_mxfp4(q.data, q.planes, b.data, b.planes)
    assert y.numel() * 2 > 1 << 32
    assert torch.equal(y[-tail:], ops.gemm_mxfp4(small.data, small.planes, b.data, b.planes))
    assert not bool(y[:-tail].any())
    del y
    hq, GU = ops.gemm_geglu_mxfp4(q.data, q.planes, b.data, b.planes, N // 2, colwise=True, keep_gu=True)
    h2, GU2 = ops.gemm_geglu_mxfp4(small.data, small.planes, b.data, b.planes, N // 2, colwise=True,
                                   keep_gu=True)
    assert torch.equal(GU[-tail:], GU2) and torch.equal(hq.data[-tail:], h2.data)
    assert torch.equal(hq.data_t[:, -tail // 2:], h2.data_t)
    assert torch.equal(hq.planes[:, -tail:], h2.planes) and torch.equal(hq.planes_t[-4:], h2.planes_t)
    dH = torch.zeros(M, N // 2, dtype=torch.bfloat16, device=gpu)
    dH[-tail:] = _x(tail, N // 2, 3, spread=False).to(gpu)
    d = ops.geglu_bwd_mxfp4(dH, GU, colwise=True)
    d2 = ops.geglu_bwd_mxfp4(dH[-tail:], GU2, colwise=True)
    assert torch.equal(d.data[-tail:], d2.data) and torch.equal(d.planes[:, -tail:], d2.planes)
    assert torch.equal(d.data_t[:, -tail // 2:], d2.data_t) and torch.equal(d.planes_t[-4:], d2.planes_t)


def test_two_graphs_at_once(gpu):
    """Calls with a workspace (a product in K pieces, the norm's backward) captured into two graphs,
    replayed side by side on two streams: neither touches the other's."""
    M, N, K = 96, 256, 16384
    assert _lib.lib().bf8_gemm_mxfp4_workspace(M, N, K) > 0
    post, pre = _x(1, 512, 3).to(gpu)[0], _x(1, 512, 4).to(gpu)[0]

    def work(a, b, h, dy):
        y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32)
        out, _ = ops.rmsnorm_residual(h, dy, post, pre, 1e-6)
        return [y, *ops.rmsnorm_residual_backward(h, out, dy, dy, post, pre, 1e-6)[:4]]

    sides, ins = [], []
    for k in range(2):
        ins.append((ops.quantize_mxfp4(_x(M, K, 10 + k).to(gpu)), ops.quantize_mxfp4(_x(N, K, 20 + k).to(gpu)),
                    _x(700, 512, 30 + k).to(gpu), _x(700, 512, 40 + k).to(gpu)))
    want = [[t.clone() for t in work(*i)] for i in ins]
    torch.cuda.synchronize()
    for i in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work(*i)
        sides.append((torch.cuda.Stream(), graph, outs))
    for rep in range(5):
        for _, _, outs in sides:
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()
        for stream, graph, _ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, outs), w in zip(sides, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w)), f"replay {rep}"


def test_one_tensor_as_both_operands(gpu):
    """A Gram matrix: symmetric to the bit, and the product of two equal tensors."""
    q = ops.quantize_mxfp4(_x(300, 2080, 9).to(gpu))
    y = ops.gemm_mxfp4(q.data, q.planes, q.data[:296], q.planes[:, :296].contiguous(),
                       out_dtype=torch.float32)
    z = ops.gemm_mxfp4(q.data, q.planes, q.data.clone()[:296], q.planes[:, :296].contiguous(),
                       out_dtype=torch.float32)
    assert torch.equal(y, z)


def test_second_derivatives_are_refused(gpu):
    x = _x(40, 64, 1).to(gpu).requires_grad_()
    w = _x(32, 64, 2).to(gpu).requires_grad_()
    n = _x(1, 64, 3).to(gpu)[0].requires_grad_()
    results = [linear.Mxfp4LinearFunction.apply(x, w, None), fused_mlp.residual_norm(x, x, n, n)[1],
               linear.Mxfp4GegluMlpFunction.apply(x, _x(256, 64, 4).to(gpu).requires_grad_(),
                                                  _x(64, 128, 5).to(gpu), None, None, 128)]
    for y in results:
        for dy, told in ((torch.ones_like(y), "does not require grad"), (2 * y, "once_differentiable")):
            (g,) = torch.autograd.grad(y, x, dy, create_graph=True)
            with pytest.raises(RuntimeError, match=told):
                g.float().square().sum().backward()


def test_another_stream(gpu):
    x, w = _x(300, 512, 1).to(gpu), _x(256, 512, 2).to(gpu)
    def f():
        a, b = ops.quantize_mxfp4(x, colwise=True), ops.quantize_mxfp4(w)
        return ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes)
    want = f()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f()
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(gpu):
    x = torch.zeros(64, 64, dtype=torch.bfloat16, device=gpu)
    q = ops.quantize_mxfp4(x)
    with pytest.raises(ValueError, match="cols % 32"):
        ops.quantize_mxfp4(x[:, :40])
    with pytest.raises(Exception, match="cols % 8"):
        ops.quantize_mxfp4(x[:, :12], rowwise=False, colwise=True)
    with pytest.raises(TypeError, match="bfloat16"):
        ops.quantize_mxfp4(x.float())
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.quantize_mxfp4(x.cpu())
    with pytest.raises(ValueError, match="nothing"):
        ops.quantize_mxfp4(x, rowwise=False)
    with pytest.raises(ValueError, match="columnwise"):
        ops.dequant_mxfp4(q, transpose=True)
    mm = ops.gemm_mxfp4
    with pytest.raises(ValueError, match="inner dims"):
        mm(q.data, q.planes, *[getattr(ops.quantize_mxfp4(torch.cat([x, x], 1)), n) for n in ("data", "planes")])
    with pytest.raises(ValueError, match="a_planes"):
        mm(q.data, q.planes[:, :32], q.data, q.planes)
    with pytest.raises(TypeError, match="uint8"):
        mm(q.data.view(torch.int8), q.planes, q.data, q.planes)
    with pytest.raises(ValueError, match="contiguous rows"):
        mm(q.data.t().contiguous().t(), q.planes, q.data, q.planes)
    with pytest.raises(ValueError, match="bias"):
        mm(q.data, q.planes, q.data, q.planes, bias=x[0, :32].contiguous())
    with pytest.raises(TypeError, match="out_dtype"):
        mm(q.data, q.planes, q.data, q.planes, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="out must be"):
        mm(q.data, q.planes, q.data, q.planes, out=x.float())
    with pytest.raises(Exception, match="N % 8"):
        mm(q.data, q.planes, q.data[:4], q.planes[:, :4].contiguous())
    with pytest.raises(ValueError, match="128"):
        ops.gemm_geglu_mxfp4(q.data, q.planes, q.data, q.planes, 32)
    with pytest.raises(ValueError, match="rows"):
        ops.gemm_geglu_mxfp4(q.data, q.planes, q.data, q.planes, 128)
    with pytest.raises(ValueError, match="multiples of 32"):
        linear.Mxfp4LinearFunction.apply(x, torch.zeros(40, 64, dtype=torch.bfloat16, device=gpu,
                                                        requires_grad=True), None)


TILES = ["256x160", "160x256", "128x128", "192x256", "128x64", "64x128", "256x256w8", "128x128o2",
         "128x64:3", "256x256w8:2", "256x128"]  # (the last has no FP4 variant: the plan's own)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("M,N,K", [(5, 24, 32), (300, 328, 1312), (517, 1040, 4128)])
def test_product_on_every_tile(gpu, monkeypatch, tile, M, N, K):
    """Every tile's FP4 variant: partial tiles, a last step of 32, 160 and 32 K-values, one step and
    many, K pieces."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    a, ra = _operand(M, K, M + K, gpu)
    b, rb = _operand(N, K, N + K, gpu, spread=False)
    ref, mag = mx4.mm(ra, rb)
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=dtype)
        _check_product(y, ref, mag, K, dtype)


@pytest.mark.parametrize("tile", ["128x64", "64x128"])
@pytest.mark.parametrize("M,N,K", [(1040, 2056, 2208), (70, 136, 2080), (130, 72, 1792), (33, 520, 2048)])
def test_product_of_few_and_many_small_tiles(gpu, monkeypatch, tile, M, N, K):
    """The small tiles with more of them than CUs, and with fewer on either side of the eight K steps from
    which two groups of waves share a tile's steps (even and odd numbers of them)."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    a, ra = _operand(M, K, M + K, gpu)
    b, rb = _operand(N, K, N + K, gpu, spread=False)
    ref, mag = mx4.mm(ra, rb)
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=dtype)
        _check_product(y, ref, mag, K, dtype)


def test_tail_split(gpu, monkeypatch):
    """Whole tiles in full rounds, the last round's tiles in K pieces."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", "256x256w8:t")
    M, N, K = 4160, 3848, 4128
    a, ra = _operand(M, K, 1, gpu, spread=False)
    b, rb = _operand(N, K, 2, gpu, spread=False)
    y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32)
    rows = torch.cat([torch.arange(0, 64), torch.arange(M - 80, M)])
    ref = mx4.values(ra[0][rows], ra[1][rows]) @ mx4.values(*rb).t()
    mag = mx4.values(ra[0][rows], ra[1][rows]).abs() @ mx4.values(*rb).abs().t()
    _check_product(y[rows.to(gpu)], ref, mag, K, torch.float32)


@pytest.mark.parametrize("tile", ["256x256w8", "160x256", "64x128", "192x256"])
@pytest.mark.parametrize("M,K,I", [(1, 32, 128), (45, 288, 256), (290, 544, 640)])
def test_gated_product_on_every_tile(gpu, monkeypatch, tile, M, K, I):
    """The gated-GELU epilogue of every tile: H's copies from its own GU, one K step and several, ragged
    rows, a NaN and an inf among the inputs of the last case."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    x, w, _, _ = _mlp_inputs(M, K, I, M + K + I, gpu)
    if M == 290:
        x[M - 1, 5], x[7, 40] = float("nan"), 3e38
    xq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    hq, GU = ops.gemm_geglu_mxfp4(xq.data, xq.planes, wq.data, wq.planes, I, colwise=True, keep_gu=True)
    rows = [i for i in range(M) if M != 290 or i not in (7, M - 1)]
    ref, mag = mx4.mm(mx4.quantize(x.cpu()), mx4.quantize(w.cpu()))
    _check_product(GU[rows], ref[rows], mag[rows], K, torch.bfloat16)
    want = ops.quantize_mxfp4(ops.geglu(GU)[0], colwise=True)
    assert torch.equal(hq.planes, want.planes) and torch.equal(hq.data, want.data)
    assert torch.equal(hq.planes_t, want.planes_t) and torch.equal(hq.data_t, want.data_t)


@pytest.mark.parametrize("rows,cols", [(3300, 2560), (8193, 1096), (13000, 2592), (16416, 2080)])
def test_quantize_both_copies_of_large_tensors(gpu, rows, cols):
    """The block tilings of large tensors (past 8M and 32M elements): ragged rows and columns, special
    blocks; the copies alone are the same."""
    x = _special(rows, cols, 7)
    rowwise = cols % 32 == 0
    q = ops.quantize_mxfp4(x.to(gpu), rowwise=rowwise, colwise=True)
    if rowwise:
        codes, e = mx4.quantize(x)
        assert torch.equal(q.planes.cpu(), mx4.planes(e)) and torch.equal(q.data.cpu(), codes)
    codes, e = mx4.quantize(x, 0)
    assert torch.equal(q.planes_t.cpu(), mx4.planes(e)) and torch.equal(q.data_t.cpu(), codes)
    only = ops.quantize_mxfp4(x.to(gpu), rowwise=False, colwise=True)
    assert torch.equal(only.data_t, q.data_t) and torch.equal(only.planes_t, q.planes_t)


def test_gated_backward_takes_every_gate(gpu):
    """Gates outside the gelu tables (zeros, tiny, 8 and above, inf, NaN) in some rows and all of them."""
    g = torch.Generator().manual_seed(3)
    for M, I in ((70, 256), (3300, 2560)):
        GU = torch.randn(M, 2 * I, generator=g).to(torch.bfloat16)
        GU[::7, :I] = 0.0
        GU[3, :8] = torch.tensor([8.0, -8.0, 100.0, -100.0, float("inf"), -float("inf"), float("nan"), 1e-38])
        GU[5, : I // 2] *= 1e-6
        dH = (torch.randn(M, I, generator=g) * 1e-2).to(torch.bfloat16)
        GU, dH = GU.to(gpu), dH.to(gpu)
        want = ops.quantize_mxfp4(ops.geglu_bwd(dH, GU)[0], colwise=True)
        q = ops.geglu_bwd_mxfp4(dH, GU, colwise=True)
        assert torch.equal(q.data, want.data) and torch.equal(q.planes, want.planes)
        assert torch.equal(q.data_t, want.data_t) and torch.equal(q.planes_t, want.planes_t)


def test_gram_matrix_is_symmetric(gpu):
    """One tensor as both operands: y is the oracle's product, and y[i, j] and y[j, i], sums of the same
    terms, differ by no more than two sums of them may."""
    K, n = 2080, 296
    a, ra = _operand(n, K, 9, gpu)
    y = ops.gemm_mxfp4(a.data, a.planes, a.data, a.planes, out_dtype=torch.float32)
    ref, mag = mx4.mm(ra, ra)
    _check_product(y, ref, mag, K, torch.float32)
    y = y.cpu().double()
    assert bool(((y - y.t()).abs() <= 2 * K * 2.0 ** -23 * mag).all())


@pytest.mark.parametrize("tile,has", [("256x256w8", True), ("160x256", True), ("64x128", True),
                                      ("192x256", False)])
def test_gated_product_runs_the_tile_that_is_named(gpu, monkeypatch, capfd, tile, has):
    """A named tile is the one that runs where it has a gated FP4 variant (192x256 has none: the plan's own
    choice, which is printed where it is made), and gives the product and its copies."""
    M, K, I = 290, 544, 640
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    monkeypatch.setenv("BONGARD_FP8_GEMM_DEBUG", "1")
    x, w, _, _ = _mlp_inputs(M, K, I, 7, gpu)
    xq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    capfd.readouterr()
    hq, GU = ops.gemm_geglu_mxfp4(xq.data, xq.planes, wq.data, wq.planes, I, colwise=True, keep_gu=True)
    assert ("bf8 plan geglu mx" in capfd.readouterr().err) == (not has)
    ref, mag = mx4.mm(mx4.quantize(x.cpu()), mx4.quantize(w.cpu()))
    _check_product(GU, ref, mag, K, torch.bfloat16)
    want = ops.quantize_mxfp4(ops.geglu(GU)[0], colwise=True)
    assert torch.equal(hq.planes, want.planes) and torch.equal(hq.data, want.data)
    assert torch.equal(hq.planes_t, want.planes_t) and torch.equal(hq.data_t, want.data_t)


def test_product_with_every_workspace(gpu):
    """The C entry with its workspace, with less and with none: other plans, each within the product's bound,
    what lies behind the bytes it was given left alone, and the same bits whenever the bytes are the same."""
    M, N, K = 96, 256, 16384
    L = _lib.lib()
    need = L.bf8_gemm_mxfp4_workspace(M, N, K)
    assert need > 512
    a, ra = _operand(M, K, 1, gpu)
    b, rb = _operand(N, K, 2, gpu, spread=False)
    ref, mag = mx4.mm(ra, rb)
    stream = torch.cuda.current_stream(gpu).cuda_stream

    def call(given):
        ws = torch.full((need,), 0x5A, dtype=torch.uint8, device=gpu)
        y = torch.full((M, N), 7.0, device=gpu)
        rc = L.bf8_gemm_mxfp4(a.data.data_ptr(), K // 2, a.planes.data_ptr(), b.data.data_ptr(), K // 2,
                              b.planes.data_ptr(), M, N, K, None, y.data_ptr(), ops.OUT_F32, N,
                              ws.data_ptr() if given else None, given, stream)
        assert rc == 0, L.bf8_last_error()
        torch.cuda.synchronize()
        assert bool((ws[given:] == 0x5A).all())
        _check_product(y, ref, mag, K, torch.float32)
        return y

    sizes = (0, 256, need // 2 // 256 * 256, need - 256, need)
    first = [call(s) for s in sizes]
    for s, y in zip(sizes[::-1], first[::-1]):
        assert torch.equal(call(s), y), s
    assert torch.equal(ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32), first[-1])


def test_one_row_of_any_stride(gpu):
    """A single row is contiguous whatever its row stride says: operands and results of one row."""
    x, b = ops.quantize_mxfp4(_x(1, 64, 1).to(gpu)), ops.quantize_mxfp4(_x(256, 64, 2).to(gpu))
    row = x.data.reshape(-1, 1).t()
    assert row.stride() == (1, 1) and row.is_contiguous()
    want = ops.gemm_mxfp4(x.data, x.planes, b.data, b.planes)
    out = torch.empty(256, 1, dtype=torch.bfloat16, device=gpu).t()
    assert torch.equal(ops.gemm_mxfp4(row, x.planes, b.data, b.planes, out=out), want)
    h, gu = ops.gemm_geglu_mxfp4(row, x.planes, b.data, b.planes, 128, keep_gu=True)
    h2, gu2 = ops.gemm_geglu_mxfp4(x.data, x.planes, b.data, b.planes, 128, keep_gu=True)
    assert torch.equal(gu, gu2) and torch.equal(h.data, h2.data) and torch.equal(h.planes, h2.planes)


def test_modules_train_on_no_rows(gpu):
    """A step on an empty batch: empty results, gradients of zeros."""
    H, I = 128, 256
    torch.manual_seed(0)
    norm = nn.Module()
    norm.weight, norm.eps = nn.Parameter(torch.randn(H).to(torch.bfloat16) * 0.1), 1e-6
    for mod in (te_linear.TELinear([nn.Linear(H, H, bias=False)], "mxfp4"),
                te_linear.TEMLP(_Mlp(H, I), "mxfp4"), fused_mlp.FusedMLP(_Mlp(H, I), norm, "mxfp4")):
        mod = mod.to(gpu).train()
        x = torch.empty(0, H, dtype=torch.bfloat16, device=gpu, requires_grad=True)
        y = mod(x)
        y.sum().backward()
        assert y.shape == x.grad.shape == (0, H)
        assert all(bool((p.grad == 0).all()) for p in mod.parameters())


def test_two_threads_on_one_stream(gpu):
    """Calls of several launches with a workspace between them (a product in K pieces, the norms' backwards),
    issued by two threads on one stream: each gets its own results."""
    M, N, K = 96, 256, 16384
    w = _x(1, 512, 3).to(gpu)[0]

    def work(a, b, h, dy):
        y = ops.gemm_mxfp4(a.data, a.planes, b.data, b.planes, out_dtype=torch.float32)
        out, _ = ops.rmsnorm_residual(h, dy, w, w, 1e-6)
        return [y, *ops.rmsnorm_residual_backward(h, out, dy, dy, w, w, 1e-6)[:4],
                *ops.rmsnorm_backward(h, dy, w, 1e-6)]

    ins = [(ops.quantize_mxfp4(_x(M, K, 10 + k).to(gpu)), ops.quantize_mxfp4(_x(N, K, 20 + k).to(gpu)),
            _x(700, 512, 30 + k).to(gpu), _x(700, 512, 40 + k).to(gpu)) for k in range(2)]
    want = [work(*i) for i in ins]
    torch.cuda.synchronize()
    got, start = [[], []], threading.Barrier(2)

    def run(k):
        start.wait(30)
        for _ in range(40):
            got[k].append(work(*ins[k]))

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        assert len(got[k]) == 40
        assert all(torch.equal(a, b) for outs in got[k] for a, b in zip(outs, want[k]))
