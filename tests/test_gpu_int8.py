"""GPU tests of the int8 path and its checkpoints against the CPU oracle.

  * quantize and checkpoints: codes, scales and exponents equal to the oracle's, bit for bit; read-backs
    are the values rounded once (a checkpoint's exactly);
  * product: the sum is exact. It is rounded to fp32, multiplied by the product of two scales and the
    bias added: at most four roundings of 2^-24 of the product, one of the result, and for bf16 its
    rounding more, 2^-8 of it;
  * the gated product, the MLP and the modules: every step equals the separate ops on the same inputs, bit
    for bit, and on inputs the format holds exactly the gradients are the differences.
"""

import types

import pytest
import torch
from torch import nn

from bongard_amd import _lib, fused_mlp, linear, ops, te_linear
from oracle import int8_oracle as i8

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _x(rows, cols, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if spread:
        x *= torch.logspace(-8, 8, rows)[:, None]
        x[:, cols // 3] *= 300.0
        x[rows // 2] = 0.0
    return x.to(BF16)


def _special(rows, cols, seed):
    """Rows holding inf, NaN, the largest and the smallest magnitudes."""
    x = _x(rows, cols, seed, spread=False)
    x[0, cols - 1], x[rows - 1, 0], x[rows // 2, cols // 2] = float("inf"), float("nan"), -float("inf")
    x[rows // 3, :8] = torch.finfo(BF16).min
    x[rows - 1, cols // 2:] = 1e-39
    return x


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.cpu().double(), 1e30), torch.nan_to_num(b.double(), 1e30))


def _check(q, x, rowwise, colwise):
    if rowwise:
        codes, s = i8.quantize(x)
        assert torch.equal(q.data.cpu(), codes) and _same(q.row_scale, s)
        assert _same(ops.dequant_int8(q), (codes.float() * s[:, None]).to(BF16))
    if colwise:
        codes, s = i8.quantize(x, 0)
        assert torch.equal(q.data_t.cpu(), codes) and _same(q.col_scale, s)
        back = ops.dequant_int8(q, transpose=True)
        assert tuple(back.shape) == (x.shape[1], x.shape[0])
        assert _same(back, (codes.float() * s[:, None]).to(BF16)[:, :x.shape[0]])


@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 16), (3, 96), (33, 168), (64, 2560), (95, 256), (257, 512),
                                       (500, 2048), (2001, 1056), (4100, 2592), (37, 4104), (70, 10240),
                                       (9, 16384), (5, 16392), (130, 20480), (3, 32768)])
@pytest.mark.parametrize("make", [_x, _special])
def test_quantize_bit_exact(gpu, rows, cols, make):
    x = make(rows, cols, rows + cols)
    for rowwise, colwise in ((True, False), (False, True), (True, True)):
        _check(ops.quantize_int8(x.to(gpu), rowwise=rowwise, colwise=colwise), x, rowwise, colwise)


def test_quantize_every_magnitude_under_every_largest(gpu):
    """For each of the 128 mantissas of a row's largest value (at three exponents, the floor's among them),
    every bf16 magnitude from it down to where all codes are 0."""
    for top in (0x3F80, 0x0080, 0x7F00, 0x2B80 - 0x80):  # 1, 2^-126, 2^127, below 2^-40
        heads = torch.arange(top, top + 128, dtype=torch.int32)
        keys = torch.arange(10 * 128, dtype=torch.int32)
        k = (heads[:, None] - keys).clamp(min=0)
        k = k | ((torch.arange(k.numel()).reshape(k.shape) % 3 == 1).int() << 15)
        x = torch.where(k >= 0x8000, k - 0x10000, k).to(torch.int16).view(BF16)
        _check(ops.quantize_int8(x.to(gpu), colwise=True), x, True, True)


def test_quantize_views_and_strides(gpu):
    """Strided, transposed, misaligned and batched inputs are read as what they show."""
    big = _x(70, 300, 3).to(gpu)
    for view in (big[:, 4:292], big[1::2, :64], big.t()[:64, :64], big[3:67].reshape(2, 32, 300)[..., :96],
                 big.flatten()[1:1 + 64 * 64].view(64, 64)):
        flat = view.reshape(-1, view.shape[-1]).contiguous().cpu()
        _check(ops.quantize_int8(view, colwise=True), flat, True, True)


def test_quantize_empty_and_large_offsets(gpu):
    q = ops.quantize_int8(torch.empty(0, 64, dtype=BF16, device=gpu), colwise=True)
    assert tuple(q.data.shape) == (0, 64) and tuple(q.data_t.shape) == (64, 0)
    assert bool((q.col_scale == q.col_scale[0]).all()) and q.col_scale[0].item() == i8.quantize(torch.zeros(1, 8))[1]
    assert tuple(ops.dequant_int8(q).shape) == (0, 64)
    # element offsets past 2^31: the last rows are quantized as by themselves
    rows, cols = (1 << 31) // 16384 + 70, 16384
    x = torch.empty(rows, cols, dtype=BF16, device=gpu)
    x[:-100].zero_()
    tail = _x(100, cols, 9)
    x[-100:] = tail.to(gpu)
    q = ops.quantize_int8(x, colwise=True)
    codes, s = i8.quantize(tail)
    assert torch.equal(q.data[-100:].cpu(), codes) and _same(q.row_scale[-100:], s)
    assert torch.equal(q.data_t[:, rows - 100:rows].cpu(), i8.quantize(tail, 0)[0][:, :100])
    assert _same(ops.dequant_int8(q)[-100:], (codes.float() * s[:, None]).to(BF16))
    c = ops.quantize_mxint8(x)
    codes, e = i8.checkpoint(tail)
    assert torch.equal(c.data[-100:].cpu(), codes) and torch.equal(c.exps[-100:].cpu(), e)
    assert _same(ops.dequant_mxint8(c)[-100:], i8.restored(codes, e))


def _operand(rows, K, seed, gpu, spread=True):
    x = _x(rows, K, seed, spread)
    return ops.quantize_int8(x.to(gpu)), i8.quantize(x)


def _check_product(y, ref, full, dtype):
    """ref: the product, full: with the bias."""
    tol = 2.0 ** -22 * ref.abs() + 2.0 ** -24 * full.abs()
    if dtype == BF16:
        tol = tol + 2.0 ** -8 * full.abs()
    err = (y.cpu().double() - full).abs()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} of the bound"


PRODUCTS = [(1, 8, 16), (1, 2048, 2560), (7, 40, 96), (33, 64, 160), (64, 1024, 2560), (129, 264, 224),
            (256, 256, 512), (500, 2560, 2048), (300, 520, 5152), (2001, 640, 1056), (520, 1032, 10240)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(gpu, M, N, K):
    a, ra = _operand(M, K, M + K, gpu)
    b, rb = _operand(N, K, N + K, gpu, spread=False)
    ref, _ = i8.mm(ra, rb)
    bias = _x(1, N, 5, spread=False)[0]
    full = ref + bias.double()
    for dtype in (F32, BF16):
        y = ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, out_dtype=dtype)
        _check_product(y, ref, ref, dtype)
        yb = ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, bias=bias.to(gpu), out_dtype=dtype)
        _check_product(yb, ref, full, dtype)
        assert torch.equal(y, ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, out_dtype=dtype))


TILES = ["256x160", "160x256", "128x128", "192x256", "128x64", "64x128", "256x256w8", "256x256w8x",
         "192x128o2", "128x128o2", "128x64k2", "64x128k2", "128x64:3", "256x256w8:2", "256x128"]


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("M,N,K", [(5, 24, 16), (300, 328, 1312), (517, 1040, 4128)])
def test_product_on_every_tile(gpu, monkeypatch, tile, M, N, K):
    """Partial tiles, a last step of 16 and 32 K-values, one step and many, K pieces (256x128 has no int8
    variant: the plan's own)."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    a, ra = _operand(M, K, M + K, gpu)
    b, rb = _operand(N, K, N + K, gpu, spread=False)
    ref, _ = i8.mm(ra, rb)
    bias = _x(1, N, 5, spread=False)[0]
    for dtype in (F32, BF16):
        y = ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, bias=bias.to(gpu), out_dtype=dtype)
        _check_product(y, ref, ref + bias.double(), dtype)


def test_tail_split(gpu, monkeypatch):
    """Whole tiles in full rounds, the last round's tiles in K pieces."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", "256x256w8:t")
    M, N, K = 4160, 3848, 4128
    a, ra = _operand(M, K, 1, gpu, spread=False)
    b, rb = _operand(N, K, 2, gpu, spread=False)
    rows = torch.cat([torch.arange(0, 64), torch.arange(M - 80, M)])
    ref, _ = i8.mm((ra[0][rows], ra[1][rows]), rb)
    for dtype in (F32, BF16):
        y = ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, out_dtype=dtype)
        _check_product(y[rows.to(gpu)], ref, ref, dtype)


@pytest.mark.parametrize("tile", ["", "256x256w8", "128x64:8"])
def test_product_of_the_longest_sums(gpu, monkeypatch, tile):
    """K = 133,120 of the largest codes: sums next to 2^31, of either sign."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    M, N, K = 24, 16, 133120
    a = torch.full((M, K), 127, dtype=torch.int8, device=gpu)
    a[1::2] = -127
    b = torch.full((N, K), 127, dtype=torch.int8, device=gpu)
    one = torch.ones(M, device=gpu)
    y = ops.gemm_int8(a, one, b, one[:N], out_dtype=F32)
    want = torch.where(torch.arange(M) % 2 == 0, 1.0, -1.0)[:, None] * torch.full((M, N), 127.0 * 127.0 * K)
    assert torch.equal(y.cpu(), want)
    with pytest.raises(_lib.Fp8LibError, match="133120"):
        ops.gemm_int8(torch.zeros(8, K + 16, dtype=torch.int8, device=gpu), one[:8],
                      torch.zeros(8, K + 16, dtype=torch.int8, device=gpu), one[:8])


def test_product_strides_and_out(gpu):
    """Operands whose rows are longer than K, an out whose rows are longer than N and whose other
    columns keep what they held; scales that start off 16 bytes."""
    M, N, K = 70, 136, 320
    a, ra = _operand(M, K, 1, gpu)
    b, rb = _operand(N, K, 2, gpu, spread=False)
    wide_a = torch.full((M, K + 64), 0x77, dtype=torch.int8, device=gpu)
    wide_b = torch.full((N, K + 32), 0x77, dtype=torch.int8, device=gpu)
    wide_a[:, :K], wide_b[:, :K] = a.data, b.data
    s = torch.empty(M + N + 2, device=gpu)
    s[1:M + 1], s[M + 1:-1] = a.row_scale, b.row_scale
    ref, _ = i8.mm(ra, rb)
    for dtype in (BF16, F32):
        out = torch.full((M + 2, N + 24), 7.0, dtype=dtype, device=gpu)
        y = ops.gemm_int8(wide_a[:, :K], s[1:M + 1], wide_b[:, :K], s[M + 1:-1], out_dtype=dtype, out=out[:M, :N])
        assert y.data_ptr() == out.data_ptr()
        _check_product(y, ref, ref, dtype)
        assert bool((out[M:] == 7).all()) and bool((out[:, N:] == 7).all())
    empty = ops.gemm_int8(a.data[:0], a.row_scale[:0], b.data, b.row_scale)
    assert tuple(empty.shape) == (0, N)
    # an empty sum is the bias; a single row of any stride
    none = torch.empty(3, 0, dtype=torch.int8, device=gpu)
    bias = _x(1, 8, 4, spread=False)[0].to(gpu)
    y = ops.gemm_int8(none, s[:3], torch.empty(8, 0, dtype=torch.int8, device=gpu), s[:8], bias=bias)
    assert torch.equal(y, bias.expand(3, 8))
    one = torch.as_strided(a.data, (1, K), (K + 8, 1))
    assert torch.equal(ops.gemm_int8(one, a.row_scale[:1], b.data, b.row_scale)[0],
                       ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale)[0])


def test_product_special_rows(gpu):
    """A row that held NaN or inf makes its products NaN and no others."""
    M, N, K = 40, 48, 128
    xa, xb = _x(M, K, 3, spread=False), _x(N, K, 4, spread=False)
    xa[5, 70], xa[8, 1], xb[9] = float("nan"), float("inf"), 0.0
    a, b = ops.quantize_int8(xa.to(gpu)), ops.quantize_int8(xb.to(gpu))
    y = ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, out_dtype=F32).cpu()
    ref, _ = i8.mm(i8.quantize(xa), i8.quantize(xb))
    rows = [i for i in range(M) if i not in (5, 8)]
    assert bool(torch.isnan(y[[5, 8]]).all())
    _check_product(y[rows], ref[rows], ref[rows], F32)
    assert bool((y[rows][:, 9] == 0).all())


@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 15, 16, 17, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("N,K", [(2048, 2560), (40, 16), (2560, 10240), (1032, 272), (8, 4112), (4104, 5120),
                                 (200, 20496), (6160, 640)])
def test_tokens_through_a_linear(gpu, M, N, K):
    """x quantized in the call: the product of the quantizer's codes, whichever kernel runs it."""
    x, b = _x(M, K, M + K), _operand(N, K, N, gpu, spread=False)
    bias = _x(1, N, 7, spread=False)[0]
    ref, _ = i8.mm(i8.quantize(x), b[1])
    for dtype in (F32, BF16):
        y = ops.linear_int8(x.to(gpu), b[0].data, b[0].row_scale, out_dtype=dtype)
        _check_product(y, ref, ref, dtype)
        yb = ops.linear_int8(x.to(gpu).view(M, 1, K), b[0].data, b[0].row_scale, bias=bias.to(gpu), out_dtype=dtype)
        assert tuple(yb.shape) == (M, 1, N)
        _check_product(yb.view(M, N), ref, ref + bias.double(), dtype)
    x[M - 1, K - 1] = float("inf")  # that token's row alone
    y = ops.linear_int8(x.to(gpu), b[0].data, b[0].row_scale)
    assert bool(torch.isnan(y[M - 1]).all()) and not bool(torch.isnan(y[:M - 1]).any())


def test_linear_of_no_tokens_and_wide_rows_of_weights(gpu):
    b, rb = _operand(72, 320, 1, gpu, spread=False)
    assert tuple(ops.linear_int8(torch.empty(0, 320, dtype=BF16, device=gpu), b.data, b.row_scale).shape) == (0, 72)
    wide = torch.full((72, 400), 99, dtype=torch.int8, device=gpu)
    wide[:, :320] = b.data
    for M in (1, 20, 40):
        x = _x(M, 320, M, spread=False)
        y = ops.linear_int8(x.to(gpu), wide[:, :320], b.row_scale, out_dtype=F32)
        ref, _ = i8.mm(i8.quantize(x), rb)
        _check_product(y, ref, ref, F32)


@pytest.mark.parametrize("M", [1, 2, 5, 15, 16, 17, 32, 33, 200])
@pytest.mark.parametrize("I,K", [(128, 16), (256, 1792), (10240, 2560), (128, 8208), (384, 272), (4608, 4096),
                                 (128, 20496)])
def test_tokens_through_a_gated_projection(gpu, M, I, K):
    """The gated product of the quantizer's codes, bit for bit, whichever kernel runs it: small and large gates, zeros,
    a token of inf."""
    x, w = _x(M, K, M + I, spread=False), _x(2 * I, K, K, spread=False)
    w[:I] *= torch.logspace(-6, 2, I)[:, None].to(BF16)
    w[3] = 0
    wq = ops.quantize_int8(w.to(gpu))
    for bad in (False, True):
        if bad:
            x[M - 1, K // 2] = float("inf")
        q = ops.quantize_int8(x.to(gpu))
        want, _ = ops.gemm_geglu_int8(q.data, q.row_scale, wq.data, wq.row_scale, I)
        got = ops.linear_geglu_int8(x.to(gpu).view(M, 1, K), wq.data, wq.row_scale)
        assert tuple(got.shape) == (M, 1, I)
        assert torch.equal(got.view(M, I).view(torch.int16), want.view(torch.int16))
        assert bool(torch.isnan(got[M - 1]).all()) == bad
    wide = torch.full((2 * I, K + 16), 99, dtype=torch.int8, device=gpu)
    wide[:, :K] = wq.data
    assert torch.equal(ops.linear_geglu_int8(x[:M - 1].to(gpu), wide[:, :K], wq.row_scale), want[:M - 1])
    with pytest.raises(ValueError, match="multiple of 128"):
        ops.linear_geglu_int8(x.to(gpu), wq.data[:64], wq.row_scale[:64])
    with pytest.raises(ValueError, match="inner dims"):
        ops.linear_geglu_int8(x.to(gpu)[:, :8], wq.data, wq.row_scale)


# ---- checkpoints -------------------------------------------------------------------------------
def _check_ckpt(q, x):
    codes, e = i8.checkpoint(x)
    assert torch.equal(q.exps.cpu(), e)
    ok = e.repeat_interleave(32, 1)[:, :x.shape[1]] != 255
    assert torch.equal(q.data.cpu()[ok], codes[ok])
    assert _same(ops.dequant_mxint8(q), i8.restored(codes, e))


@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 32), (3, 40), (64, 2560), (33, 136), (2001, 1056)])
@pytest.mark.parametrize("make", [_x, _special])
def test_checkpoint_bit_exact(gpu, rows, cols, make):
    x = make(rows, cols, rows + cols)
    _check_ckpt(ops.quantize_mxint8(x.to(gpu)), x)


def test_checkpoint_every_magnitude_under_every_exponent(gpu):
    for off in (0, 1, 126, 127):
        heads = torch.arange(0, 0x7F80, 0x80, dtype=torch.int32) + off
        keys = torch.cat([torch.zeros(1, dtype=torch.int32), torch.randperm(9 * 128, generator=torch.Generator().manual_seed(off))[:31].int()])
        for shift in range(0, 9 * 128, 31):
            k = (heads[:, None] - (keys + shift) % (9 * 128) * (keys > 0)).clamp(min=0)
            k = k | ((torch.arange(k.numel()).reshape(k.shape) % 3 == 1).int() << 15)
            x = torch.where(k >= 0x8000, k - 0x10000, k).to(torch.int16).view(BF16)
            if shift % (31 * 6) == 0:
                _check_ckpt(ops.quantize_mxint8(x.to(gpu)), x)


def _gu(M, I, seed, gpu):
    g = torch.Generator().manual_seed(seed)
    GU = torch.randn(M, 2 * I, generator=g).to(BF16)
    GU[0, :3] = torch.tensor([12.0, -12.0, 1e-20])
    GU[-1, I:I + 32] = 0.0
    dH = (torch.randn(M, I, generator=g) * 1e-2).to(BF16)
    return GU.to(gpu), dH.to(gpu)


@pytest.mark.parametrize("M,I", [(1, 32), (31, 96), (64, 640), (257, 384), (2001, 2560), (3, 10272), (4100, 544),
                                 (1024, 32), (1031, 288), (1100, 10272)])
def test_gated_gelu_from_a_checkpoint(gpu, M, I):
    """H is the gated GELU's, the checkpoint the quantizer's and the gradient the separate backward's at
    the values read back, bit for bit."""
    GU, dH = _gu(M, I, M + I, gpu)
    H, q = ops.geglu_mxint8(GU)
    assert torch.equal(H, ops.geglu(GU)[0])
    want = ops.quantize_mxint8(GU)
    assert torch.equal(q.data, want.data) and torch.equal(q.exps, want.exps)
    dGU = ops.geglu_bwd_mxint8(dH, q)
    assert torch.equal(dGU, ops.geglu_bwd(dH, ops.dequant_mxint8(q))[0])
    # its int8 copies (from 1024 rows on by the maxima that the backward leaves)
    for rowwise, colwise in ((True, True), (True, False), (False, True)):
        got = ops.geglu_bwd_mxint8(dH, q, rowwise=rowwise, colwise=colwise)
        want = ops.quantize_int8(dGU, rowwise=rowwise, colwise=colwise)
        for name in ("data", "row_scale", "data_t", "col_scale"):
            a, b = getattr(got, name), getattr(want, name)
            assert (a is None and b is None) or torch.equal(a, b), name
    leaf = GU.clone().requires_grad_()
    h = fused_mlp.gated_gelu(leaf.view(1, M, 2 * I), checkpoint=True)
    h.backward(dH.view(1, M, I))
    assert torch.equal(h[0], H) and torch.equal(leaf.grad, dGU)
    leaf.grad = None
    h = fused_mlp.gated_gelu(leaf)
    h.backward(dH)
    assert torch.equal(h, H) and torch.equal(leaf.grad, ops.geglu_bwd(dH, GU)[0])
    with torch.no_grad():
        assert torch.equal(fused_mlp.gated_gelu(leaf, checkpoint=True), H)


def test_gated_gelu_gradient_is_the_difference(gpu):
    """At pre-activations the checkpoint holds exactly, central differences of the function in 64 bits:
    second order in the step (2^-7; the third derivative of gelu is below 2, so off by under
    2^-14 * 2 / 6 * |u dh|), and the chain's three roundings to bf16 (2^-8 each) and the activation's."""
    g = torch.Generator().manual_seed(2)
    M, I = 16, 64
    GU = torch.randint(-96, 97, (M, 2 * I), generator=g).float() / 32
    GU[:, ::32] = 96 / 32  # each block's largest: steps of 2^-5
    GU = GU.to(BF16)
    assert torch.equal(i8.restored(*i8.checkpoint(GU)), GU.double())
    dH = torch.randn(M, I, generator=g).to(BF16)
    leaf = GU.to(gpu).requires_grad_()
    fused_mlp.gated_gelu(leaf, checkpoint=True).backward(dH.to(gpu))
    f = lambda v: nn.functional.gelu(v[:, :I], approximate="tanh") * v[:, I:] * dH.double()  # noqa: E731
    v, h = GU.double(), 2.0 ** -7
    for half in (0, 1):
        step = torch.zeros_like(v)
        step[:, half * I:(half + 1) * I] = h
        diff = (f(v + step) - f(v - step)) / (2 * h)
        got = leaf.grad[:, half * I:(half + 1) * I].cpu().double()
        scale = (v[:, I:] if half == 0 else nn.functional.gelu(v[:, :I], approximate="tanh")) * dH.double()
        assert bool(((got - diff).abs() <= 3 * 2.0 ** -8 * diff.abs() + 2.0 ** -14 * scale.abs() + 2.0 ** -20).all())


def test_codes_of_a_nonfinite_gradient(gpu):
    """Rows and columns of dGU that hold an inf or a NaN: the quantizer's NaN scales and zero codes, also where the
    backward leaves the maxima."""
    GU, dH = _gu(1100, 544, 7, gpu)
    dH[3, 9], dH[1099, 543], dH[700, 64] = float("nan"), float("inf"), -float("inf")
    _, q = ops.geglu_mxint8(GU)
    got = ops.geglu_bwd_mxint8(dH, q, rowwise=True, colwise=True)
    want = ops.quantize_int8(ops.geglu_bwd_mxint8(dH, q), rowwise=True, colwise=True)
    assert torch.isnan(want.row_scale).nonzero().flatten().tolist() == [3, 700, 1099]
    for name in ("data", "row_scale", "data_t", "col_scale"):
        a, b = getattr(got, name), getattr(want, name)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


def test_gated_gelu_of_nonfinite_blocks(gpu):
    """inf or NaN in a block makes that block's gradient NaN and no other's, but for a gate from 2^64 on, at
    which torch's gelu has a NaN gradient itself (its square is inf); H is the gated GELU's."""
    GU, dH = _gu(8, 64, 1, gpu)
    GU[2, 5], GU[4, 64 + 40], GU[6, 33] = float("inf"), float("nan"), torch.finfo(BF16).min
    H, q = ops.geglu_mxint8(GU)
    want = ops.geglu(GU)[0]
    assert torch.equal(H.view(torch.int16), want.view(torch.int16))
    dGU = ops.geglu_bwd_mxint8(dH, q)
    bad = torch.isnan(ops.dequant_mxint8(q))
    assert bad.sum().item() == 64
    want = bad[:, :64] | bad[:, 64:]
    want[6, 33] = True
    leaf = GU[6, 33].cpu().requires_grad_()
    assert bool(torch.isnan(torch.autograd.grad(nn.functional.gelu(leaf, approximate="tanh"), leaf)[0]))
    assert torch.equal(torch.isnan(dGU)[:, :64], want)
    assert not bool(torch.isnan(dGU[[0, 1, 3, 5, 7]]).any())


# ---- the gated product, the MLP, the modules --------------------------------------------------------
def _mlp_inputs(M, K, I, seed, gpu):
    g = torch.Generator().manual_seed(seed)

    def r(*s, std=1.0):
        return (torch.randn(*s, generator=g) * std).to(BF16).to(gpu)
    return r(M, K), r(2 * I, K, std=0.05), r(K, I, std=0.05), r(M, K, std=1e-2)


def _check_gated(gpu, M, K, I):
    x, w, _, _ = _mlp_inputs(M, K, I, M + K + I, gpu)
    xq, wq = ops.quantize_int8(x), ops.quantize_int8(w)
    H, q = ops.gemm_geglu_int8(xq.data, xq.row_scale, wq.data, wq.row_scale, I, keep_gu=True)
    GU = ops.gemm_int8(xq.data, xq.row_scale, wq.data, wq.row_scale)
    assert torch.equal(H, ops.geglu(GU)[0])
    want = ops.quantize_mxint8(GU)
    assert torch.equal(q.data, want.data) and torch.equal(q.exps, want.exps)
    h2, none = ops.gemm_geglu_int8(xq.data, xq.row_scale, wq.data, wq.row_scale, I)
    assert none is None and torch.equal(h2, H)


@pytest.mark.parametrize("M,K,I", [(1, 16, 128), (33, 96, 128), (64, 256, 384), (300, 320, 640),
                                   (517, 512, 1024), (1030, 256, 2560)])
def test_gated_product(gpu, M, K, I):
    """H and the checkpoint are those of the separate product's bf16 result, bit for bit (the sums are exact,
    the scaling is the same)."""
    _check_gated(gpu, M, K, I)


@pytest.mark.parametrize("tile", ["256x256w8", "160x256", "64x128", "192x256", "128x128"])
@pytest.mark.parametrize("M,K,I", [(1, 16, 128), (45, 288, 256), (530, 160, 640)])
def test_gated_product_on_every_tile(gpu, monkeypatch, tile, M, K, I):
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    _check_gated(gpu, M, K, I)


def test_gated_product_of_nonfinite_rows(gpu):
    """A token that held inf: its H is NaN and its checkpoint reads back as NaN, the others keep theirs."""
    M, K, I = 70, 64, 128
    x, w, _, _ = _mlp_inputs(M, K, I, 3, gpu)
    bad = x.clone()
    bad[7, 3] = float("inf")
    wq = ops.quantize_int8(w)
    got = []
    for t in (x, bad):
        xq = ops.quantize_int8(t)
        got.append(ops.gemm_geglu_int8(xq.data, xq.row_scale, wq.data, wq.row_scale, I, keep_gu=True))
    (H, q), (Hb, qb) = got
    assert bool(torch.isnan(Hb[7]).all()) and bool((qb.exps[7] == 255).all())
    rows = [i for i in range(M) if i != 7]
    assert torch.equal(H[rows], Hb[rows]) and torch.equal(q.data[rows], qb.data[rows])


@pytest.mark.parametrize("M,N,K", [(1, 32, 64), (50, 96, 128), (500, 256, 320), (1000, 1024, 512)])
def test_linear_function(gpu, M, N, K):
    """Forward, dX, dW and the bias' gradient against the oracle's products of the oracle's copies."""
    x, w, dy = _x(M, K, 1, False), _x(N, K, 2, False), _x(M, N, 3, False)
    bias = _x(1, N, 4, False)[0]
    leaves = [t.to(gpu).requires_grad_() for t in (x, w, bias)]
    y = linear.Int8LinearFunction.apply(*leaves, None)
    y.backward(dy.to(gpu))
    ref, _ = i8.mm(i8.quantize(x), i8.quantize(w))
    _check_product(y.detach(), ref, ref + bias.double(), BF16)
    for got, a, b in ((leaves[0].grad, i8.quantize(dy), i8.quantize(w, 0)),
                      (leaves[1].grad, i8.quantize(dy, 0), i8.quantize(x, 0))):
        ref, _ = i8.mm(a, b)
        _check_product(got, ref, ref, BF16)
    want = dy.double().sum(0)
    tol = 2.0 ** -8 * want.abs() + (M + 64) * 2.0 ** -24 * dy.double().abs().sum(0)
    assert bool(((leaves[2].grad.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("M", [1, 20, 100])
def test_functions_without_gradients(gpu, M):
    """Under no_grad with cached weights few tokens take the kernels of serving: the values of the forward that
    keeps for a backward. A bias that alone is trained has its gradient."""
    x, w, w_gu, w_d = (_x(*s, 7, False).to(gpu) for s in ((M, 256), (96, 256), (512, 256), (64, 256)))
    bias = _x(1, 96, 4, False)[0].to(gpu).requires_grad_()
    wq, gq, dq = (linear.quantize_weight_int8(t) for t in (w, w_gu, w_d))
    leaf = x.clone().requires_grad_()
    want = linear.Int8LinearFunction.apply(leaf, w, bias, wq)
    mlp = linear.Int8GegluMlpFunction.apply(leaf, w_gu, w_d, gq, dq, 256)
    with torch.no_grad():
        assert torch.equal(linear.Int8LinearFunction.apply(leaf, w, bias, wq), want)
        assert torch.equal(linear.Int8GegluMlpFunction.apply(leaf, w_gu, w_d, gq, dq, 256), mlp)
    y = linear.Int8LinearFunction.apply(x, w, bias, wq)
    assert torch.equal(y, want)
    y.backward(torch.ones_like(y))
    assert torch.equal(bias.grad, torch.full_like(bias, M))


@pytest.mark.parametrize("M,N,K", [(1, 16, 8), (17, 32, 264), (333, 4112, 40), (1000, 1024, 512), (2049, 64, 2048),
                                   (64, 8208, 72), (37, 272, 80), (1100, 4112, 2576)])
def test_linear_calls_are_their_parts(gpu, M, N, K):
    """The forward in one call, both gradients in one and each alone: the quantizer's copies through the products, bit
    for bit."""
    x, w, dy = (_x(*s, 7, False).to(gpu) for s in ((M, K), (N, K), (M, N)))
    xq, wq = (ops.quantize_int8(t, rowwise=False, colwise=True) for t in (x, w))
    if K % 16 == 0:  # the forward, with either copy, both and none
        rows = [ops.quantize_int8(t) for t in (x, w)]
        bias = _x(1, N, 4, False)[0].to(gpu)
        want = ops.gemm_int8(rows[0].data, rows[0].row_scale, rows[1].data, rows[1].row_scale, bias=bias)
        for keep_x, keep_w in ((True, True), (True, False), (False, True), (False, False)):
            y, *kept = ops.linear_int8_forward(x, w, bias=bias, keep_x=keep_x, keep_w=keep_w)
            assert torch.equal(y, want)
            for got, q, keep in ((kept[:2], xq, keep_x), (kept[2:], wq, keep_w)):
                if keep:
                    assert torch.equal(got[0], q.data_t) and torch.equal(got[1], q.col_scale)
                else:
                    assert got == [None, None]
        y, *kept = ops.linear_int8_forward(x[:0], w, keep_x=True, keep_w=True)
        assert y.shape == (0, N) and kept[0].shape == (K, 0) and torch.equal(kept[2], wq.data_t)
        with pytest.raises(ValueError, match="inner dims"):
            ops.linear_int8_forward(x, w[:, :-16])
    q = ops.quantize_int8(dy, colwise=True)
    dx = ops.gemm_int8(q.data, q.row_scale, wq.data_t, wq.col_scale)
    dw = ops.gemm_int8(q.data_t, q.col_scale, xq.data_t, xq.col_scale)
    wt, xt = (wq.data_t, wq.col_scale), (xq.data_t, xq.col_scale)
    got = ops.linear_int8_backward(dy, *wt, *xt)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    wide = torch.zeros(M, N + 8, dtype=BF16, device=gpu)[:, 8:].copy_(dy)  # (its rows are copied)
    got = ops.linear_int8_backward(wide, *wt)
    assert torch.equal(got[0], dx) and got[1] is None
    got = ops.linear_int8_backward(dy, x_t=xt[0], x_t_scale=xt[1])
    assert got[0] is None and torch.equal(got[1], dw)
    far = torch.empty(K + 1, device=gpu)[1:].copy_(wt[1])  # (off its alignment)
    rows = torch.zeros(K, N + 16, dtype=torch.int8, device=gpu)[:, 16:].copy_(wt[0])
    got = ops.linear_int8_backward(dy, rows, far, x_t_scale=far)
    assert torch.equal(got[0], dx) and got[1] is None
    with pytest.raises(ValueError, match="w_t must be"):
        ops.linear_int8_backward(dy, wq.data_t[:, :-8], wt[1])
    with pytest.raises(ValueError, match="w_t_scale"):
        ops.linear_int8_backward(dy, wt[0], wt[1][1:])
    with pytest.raises(ValueError, match="x_t needs x_t_scale"):
        ops.linear_int8_backward(dy, *wt, xt[0], None)
    with pytest.raises(ValueError, match="nothing requested"):
        ops.linear_int8_backward(dy)
    dx, dw = ops.linear_int8_backward(dy[:0], *wt, xt[0][:, :0].contiguous(), xt[1])
    assert dx.shape == (0, K) and not bool(dw.any()) and dw.shape == (N, K)


def test_linear_gradients_are_the_differences(gpu):
    """On whole values up to 127 with a 127 in every row and column the layer is exactly bilinear:
    y(x + d) - y(x) is what the gradient says."""
    M, N, K = 64, 96, 128
    g = torch.Generator().manual_seed(0)

    def exact(*shape):
        t = torch.randint(-4, 5, shape, generator=g).float()
        for k in range(max(shape)):
            t[k % shape[0], k % shape[1]] = 127.0
        return t.to(BF16)
    x, w, dy = exact(M, K), exact(N, K), exact(M, N)
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    linear.Int8LinearFunction.apply(xg, wg, None, None).backward(dy.to(gpu))
    for name, base, grad in (("x", x, xg.grad), ("w", w, wg.grad)):
        step = torch.where((base != 127) & (torch.rand(base.shape, generator=g) < 0.3), 1.0, 0.0).to(BF16)
        moved = (base + step).to(gpu)
        args = (moved, w.to(gpu)) if name == "x" else (x.to(gpu), moved)

        def f(a, b):
            q, r = ops.quantize_int8(a), ops.quantize_int8(b)
            return ops.gemm_int8(q.data, q.row_scale, r.data, r.row_scale, out_dtype=F32).cpu().double()
        diff = ((f(*args) - f(x.to(gpu), w.to(gpu))) * dy.double()).sum()
        # the gradients are whole numbers; bf16 keeps each within 2^-8 of itself
        told = (grad.cpu().double() * step.double()).sum()
        slack = 2.0 ** -8 * (grad.cpu().double().abs() * step.double()).sum()
        assert abs(diff - told) <= slack and diff != 0


@pytest.mark.parametrize("M,K,I", [(1, 32, 128), (37, 96, 256), (512, 256, 384), (1023, 48, 128), (1100, 320, 640)])
def test_mlp_function_is_its_ops(gpu, M, K, I):
    x, w_gu, w_d, dy = _mlp_inputs(M, K, I, 5, gpu)
    leaves = [t.requires_grad_() for t in (x, w_gu, w_d)]
    y = linear.Int8GegluMlpFunction.apply(*leaves, None, None, I)
    grads = torch.autograd.grad(y, leaves, dy)
    Q = lambda t: ops.quantize_int8(t.detach(), colwise=True)  # noqa: E731
    mm = ops.gemm_int8
    xq, gq, dq = Q(x), Q(w_gu), Q(w_d)
    H, gu = ops.gemm_geglu_int8(xq.data, xq.row_scale, gq.data, gq.row_scale, I, keep_gu=True)
    hq = Q(H)
    assert torch.equal(y, mm(hq.data, hq.row_scale, dq.data, dq.row_scale))
    yq = Q(dy)
    dH = mm(yq.data, yq.row_scale, dq.data_t, dq.col_scale)
    uq = Q(ops.geglu_bwd_mxint8(dH, gu))
    assert torch.equal(grads[0], mm(uq.data, uq.row_scale, gq.data_t, gq.col_scale))
    assert torch.equal(grads[1], mm(uq.data_t, uq.col_scale, xq.data_t, xq.col_scale))
    assert torch.equal(grads[2], mm(yq.data_t, yq.col_scale, hq.data_t, hq.col_scale))
    with torch.no_grad():
        assert torch.equal(linear.Int8GegluMlpFunction.apply(x, w_gu, w_d, gq, dq, I), y)
        assert torch.equal(ops.geglu_mlp_int8(x.view(1, M, K), gq.data, gq.row_scale, dq.data, dq.row_scale)[0], y)
    for i in range(3):  # each gradient by itself
        one = [t.detach().requires_grad_(i == k) for k, t in enumerate(leaves)]
        (g,) = torch.autograd.grad(linear.Int8GegluMlpFunction.apply(*one, None, None, I), one[i], dy)
        assert torch.equal(g, grads[i])
    none = torch.empty(0, K, dtype=BF16, device=gpu, requires_grad=True)
    y = linear.Int8GegluMlpFunction.apply(none, w_gu, w_d, None, None, I)
    grads = torch.autograd.grad(y, [none, w_gu, w_d], dy[:0])
    assert y.shape == dy[:0].shape and [g.shape for g in grads] == [none.shape, w_gu.shape, w_d.shape]
    assert not any(bool(g.any()) for g in grads)


def test_a_plan_named_after_a_layer_has_run(gpu, monkeypatch):
    """The products of a layer's calls are as asked for by then, or without the K pieces that the workspace cannot
    hold: the same values."""
    M, K, I = 140, 1152, 1280
    x, w_gu, w_d, dy = _mlp_inputs(M, K, I, 8, gpu)
    leaves = [t.requires_grad_() for t in (x, w_gu, w_d)]

    def f():
        y = linear.Int8LinearFunction.apply(leaves[0], leaves[1], None, None)
        z = linear.Int8GegluMlpFunction.apply(*leaves, None, None, I)
        return [y, z, *torch.autograd.grad(y, leaves[:2], torch.ones_like(y)), *torch.autograd.grad(z, leaves, dy)]
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", "256x256w8")
    want = f()
    for tile in ("128x64:8", "64x128:4", "", "256x256w8:2"):
        monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
        for a, b in zip(f(), want):
            assert torch.equal(a, b), tile


@pytest.mark.parametrize("tile", ["256x256w8", "128x128", ""])
@pytest.mark.parametrize("M,K,I", [(1, 32, 128), (129, 96, 256), (513, 256, 384), (1100, 320, 640)])
def test_copies_of_h_in_the_mlps_forward(gpu, monkeypatch, tile, M, K, I):
    """H's columnwise codes and the result from the maxima that the eight-wave tile leaves, and where none does: the
    quantizer's of the product's H, a token of inf among them."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    x, w_gu, w_d, _ = _mlp_inputs(M, K, I, 6, gpu)
    for bad in (False, True):
        if bad:
            x[M // 2, 3] = float("inf")
        xq, gq, dq = (ops.quantize_int8(t) for t in (x, w_gu, w_d))
        H, gu = ops.gemm_geglu_int8(xq.data, xq.row_scale, gq.data, gq.row_scale, I, keep_gu=True)
        hq = ops.quantize_int8(H, colwise=True)
        want = ops.gemm_int8(hq.data, hq.row_scale, dq.data, dq.row_scale)
        y, gu8, exps, x_t, x_s, h_t, h_s = ops._geglu_mlp_int8_forward(x, I, gq, dq, True, False, True)
        assert x_t is None and x_s is None
        same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # noqa: E731
        assert same(y, want) and same(gu8, gu.data) and same(exps, gu.exps)
        assert torch.equal(h_t, hq.data_t) and same(h_s, hq.col_scale)
        assert bool(torch.isnan(h_s).all()) == bad
        y, *kept = ops._geglu_mlp_int8_forward(x, I, gq, dq, False, False, False)
        assert same(y, want) and kept == [None] * 6


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
    """TELinear, TEMLP (fused or split gate and up) and FusedMLP under 'int8': ragged rows, cached
    weights, gradients equal to the functions' on the same tensors."""
    monkeypatch.setenv("BONGARD_TE_SPLIT_GATE_UP", "1" if split else "0")
    torch.manual_seed(0)
    H, I, M = 128, 256, 75
    x, dy = _x(M, H, 8, False).to(gpu), _x(M, H, 9, False).to(gpu)
    lin = te_linear.TELinear([nn.Linear(H, H, bias=False)], "int8").to(gpu).train()
    xl = x.clone().requires_grad_()
    for _ in range(2):
        y = lin(xl.view(1, M, H))
    assert lin.counts["weight_quantizations"] == 1 and lin.counts["cached_weights"] == 1
    y.backward(dy.view(1, M, H))
    x2, w2 = x.clone().requires_grad_(), lin.weight.detach().clone().requires_grad_()
    linear.Int8LinearFunction.apply(x2, w2, None, None).backward(dy)
    assert torch.equal(xl.grad, x2.grad) and torch.equal(lin.weight.grad, w2.grad)
    mlp = te_linear.TEMLP(_Mlp(H, I), "int8").to(gpu).train()
    xm = x.clone().requires_grad_()
    for _ in range(2):
        ym = mlp(xm)
    ym.backward(dy)
    w_gu = mlp._gate_up_weight().detach().clone().requires_grad_()
    w_d = mlp.down.weight.detach().clone().requires_grad_()
    x2 = x.clone().requires_grad_()
    y2 = linear.Int8GegluMlpFunction.apply(x2, w_gu, w_d, None, None, I)
    y2.backward(dy)
    assert torch.equal(ym, y2) and torch.equal(xm.grad, x2.grad)
    got = (torch.cat([mlp.gate_proj.weight.grad, mlp.up_proj.weight.grad]) if split
           else mlp.gate_up.weight.grad)
    assert torch.equal(got, w_gu.grad) and torch.equal(mlp.down.weight.grad, w_d.grad)
    state = te_linear.restore_hf_layout(nn.ModuleDict({"mlp": mlp}), nn.ModuleDict({"mlp": mlp}).state_dict())
    assert set(state) == {f"mlp.{n}_proj.weight" for n in ("gate", "up", "down")}
    if split:
        return
    norm = nn.Module()
    norm.weight, norm.eps = nn.Parameter(torch.randn(H).to(BF16) * 0.1), 1e-6
    fused = fused_mlp.FusedMLP(_Mlp(H, I), norm, "int8").to(gpu).train()
    xf = x.clone().requires_grad_()
    yf = fused(xf)
    yf.backward(dy)
    normed, _, _ = ops.rmsnorm(x, fused.layer_norm_weight.detach(), 1e-6)
    y2 = linear.Int8GegluMlpFunction.apply(normed, fused.fc1_weight.detach(), fused.fc2_weight.detach(),
                                           None, None, I)
    assert torch.equal(yf, y2)
    assert all(p.grad is not None for p in fused.parameters()) and xf.grad.shape == x.shape


@pytest.mark.parametrize("rows,cols", [(1, 8), (7, 264), (600, 2560), (5000, 1032)])
def test_column_sums(gpu, rows, cols):
    x = _x(rows, cols, 1, False)
    got, want = ops.column_sums(x.to(gpu)).cpu().double(), x.double().sum(0)
    tol = 2.0 ** -8 * want.abs() + (rows + 64) * 2.0 ** -24 * x.double().abs().sum(0)
    assert bool(((got - want).abs() <= tol).all())
    assert not bool(ops.column_sums(x.to(gpu)[:0]).any())


def test_layer_together_in_a_graph(gpu):
    """Layer norm (checkpointed), int8 projection, gated GELU from a checkpoint, another layer norm and the
    int8 MLP, forward and backward, captured once and replayed on new inputs beside eager work: every
    replay gives the eager bits."""
    H, I = 256, 512
    torch.manual_seed(1)
    ws = [(torch.randn(*s, device=gpu) * 0.05).to(BF16) for s in
          ((2 * H, H), (2 * I, H), (H, I), (H,), (H,), (H,), (2 * H,))]

    def step(x, dy):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in (x, *ws)]
            n = fused_mlp.layer_norm(leaves[0], leaves[4], leaves[5], checkpoint=True)
            gu = linear.Int8LinearFunction.apply(n, leaves[1], leaves[7], None)
            h = fused_mlp.gated_gelu(gu, checkpoint=True)
            n = fused_mlp.layer_norm(h, leaves[6])
            y = linear.Int8GegluMlpFunction.apply(n, leaves[2], leaves[3], None, None, I)
            grads = torch.autograd.grad(y, leaves, dy)
        return [y.detach(), *grads]

    graphs = []
    for M in (70, 513):
        ins = [torch.randn(M, H, device=gpu).to(BF16) for _ in range(2)]
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
            for k, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), f"replay {rep}, result {k}"


def test_decoding_and_a_long_batch_in_a_graph(gpu):
    """Serving of 1, 20 and 100 tokens (one kernel, one kernel a product, the quantizer and the GEMM) through a norm, a
    projection and the MLP, and the MLP's training at rows whose gradient leaves its maxima, captured and replayed
    on new inputs beside eager work: every replay gives the eager bits."""
    H, I = 256, 512
    torch.manual_seed(2)
    w, w_gu, w_d, nw = ((torch.randn(*s, device=gpu) * 0.05).to(BF16) for s in ((H, H), (2 * I, H), (H, I), (H,)))
    q, gq, dq = (linear.quantize_weight_int8(t) for t in (w, w_gu, w_d))

    def serve(x):
        n = ops.linear_int8(fused_mlp.layer_norm(x, nw), q.data, q.row_scale)
        return [n, ops.geglu_mlp_int8(n, gq.data, gq.row_scale, dq.data, dq.row_scale)]

    def train(x):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in (x, w_gu, w_d)]
            y = linear.Int8GegluMlpFunction.apply(*leaves, None, None, I)
            return [y.detach(), *torch.autograd.grad(y, leaves, x)]
    graphs = []
    for M, f in ((1, serve), (20, serve), (100, serve), (1100, train)):
        x = torch.randn(M, H, device=gpu).to(BF16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = f(x)
        graphs.append((graph, x, f, outs))
    for rep in range(3):
        for graph, x, f, outs in graphs:
            x.copy_(torch.randn_like(x))
            want = [t.clone() for t in f(x)]
            graph.replay()
            torch.cuda.synchronize()
            for k, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), f"replay {rep} of {x.shape[0]} rows, result {k}"


def test_two_graphs_at_once(gpu):
    """Calls with a workspace (a product in K pieces, columns' scales, the norm's backward, sums of
    columns) captured into two graphs, replayed side by side on two streams: neither touches the other's."""
    M, N, K = 96, 256, 16384
    assert _lib.lib().bf8_gemm_int8_workspace(M, N, K) > 0
    w = _x(1, 512, 3, False).to(gpu)[0]

    def work(a, b, h, dy):
        y = ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale, out_dtype=F32)
        q = ops.quantize_int8(h, colwise=True)
        _, mean, rstd, _ = ops.layernorm(h, w, None, 1e-6, want_stats=True)
        return [y, q.data_t, q.col_scale, *ops.layernorm_backward(h, dy, w, mean, rstd), ops.column_sums(dy)]

    sides, ins = [], []
    for k in range(2):
        ins.append((ops.quantize_int8(_x(M, K, 10 + k).to(gpu)), ops.quantize_int8(_x(N, K, 20 + k).to(gpu)),
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
        for (_, _, outs), v in zip(sides, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, v)), f"replay {rep}"


def test_products_past_32_bit_offsets(gpu):
    """Results of more than 4 GiB: the rows at the end are those of a call on them alone, and so are the gated
    product's, its checkpoint's and the backward's from it."""
    M, N, K, tail = 70016, 32768, 64, 512
    a, b = _x(tail, K, 1, spread=False).to(gpu), ops.quantize_int8(_x(N, K, 2, spread=False).to(gpu))
    big = torch.zeros(M, K, dtype=BF16, device=gpu)
    big[-tail:] = a
    q, small = ops.quantize_int8(big), ops.quantize_int8(a)
    y = ops.gemm_int8(q.data, q.row_scale, b.data, b.row_scale)
    assert y.numel() * 2 > 1 << 32
    assert torch.equal(y[-tail:], ops.gemm_int8(small.data, small.row_scale, b.data, b.row_scale))
    assert not bool(y[:-tail].any())
    del y
    H, gu = ops.gemm_geglu_int8(q.data, q.row_scale, b.data, b.row_scale, N // 2, keep_gu=True)
    H2, gu2 = ops.gemm_geglu_int8(small.data, small.row_scale, b.data, b.row_scale, N // 2, keep_gu=True)
    assert torch.equal(H[-tail:], H2) and torch.equal(gu.data[-tail:], gu2.data)
    assert torch.equal(gu.exps[-tail:], gu2.exps)
    dH = torch.zeros(M, N // 2, dtype=BF16, device=gpu)
    dH[-tail:] = _x(tail, N // 2, 3, spread=False).to(gpu)
    d, d2 = ops.geglu_bwd_mxint8(dH, gu), ops.geglu_bwd_mxint8(dH[-tail:], gu2)
    assert torch.equal(d[-tail:], d2)
    h, c = ops.geglu_mxint8(d)
    h2, c2 = ops.geglu_mxint8(d2)
    assert torch.equal(h[-tail:], h2) and torch.equal(c.data[-tail:], c2.data) and torch.equal(c.exps[-tail:], c2.exps)


def test_one_tensor_as_both_operands(gpu):
    """A Gram matrix: symmetric to the bit, and the product of two equal tensors."""
    q = ops.quantize_int8(_x(296, 2080, 9).to(gpu))
    y = ops.gemm_int8(q.data, q.row_scale, q.data, q.row_scale, out_dtype=F32)
    assert torch.equal(y, y.t())
    assert torch.equal(y, ops.gemm_int8(q.data, q.row_scale, q.data.clone(), q.row_scale.clone(), out_dtype=F32))


def test_second_derivatives_are_refused(gpu):
    x = _x(40, 64, 1).to(gpu).requires_grad_()
    w = _x(32, 64, 2).to(gpu).requires_grad_()
    n = _x(1, 64, 3).to(gpu)[0].requires_grad_()
    results = [linear.Int8LinearFunction.apply(x, w, None, None), fused_mlp.layer_norm(x, n),
               fused_mlp.gated_gelu(x, checkpoint=True),
               linear.Int8GegluMlpFunction.apply(x, _x(256, 64, 4).to(gpu).requires_grad_(),
                                                 _x(64, 128, 5).to(gpu), None, None, 128)]
    for y in results:
        for dy, told in ((torch.ones_like(y), "does not require grad"), (2 * y, "once_differentiable")):
            (g,) = torch.autograd.grad(y, x, dy, create_graph=True)
            with pytest.raises(RuntimeError, match=told):
                g.float().square().sum().backward()


def test_another_stream(gpu):
    x, w = _x(300, 512, 1).to(gpu), _x(256, 512, 2).to(gpu)

    def f():
        a, b = ops.quantize_int8(x, colwise=True), ops.quantize_int8(w)
        return ops.gemm_int8(a.data, a.row_scale, b.data, b.row_scale)
    want = f()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f()
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(gpu):
    x = torch.zeros(64, 64, dtype=BF16, device=gpu)
    q = ops.quantize_int8(x)
    with pytest.raises(_lib.Fp8LibError, match="cols % 8"):
        ops.quantize_int8(x[:, :12])
    with pytest.raises(TypeError, match="bfloat16"):
        ops.quantize_int8(x.float())
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.quantize_int8(x.cpu())
    with pytest.raises(ValueError, match="nothing"):
        ops.quantize_int8(x, rowwise=False)
    with pytest.raises(ValueError, match="columnwise"):
        ops.dequant_int8(q, transpose=True)
    mm, s = ops.gemm_int8, q.row_scale
    two = ops.quantize_int8(torch.cat([x, x], 1))
    with pytest.raises(ValueError, match="inner dims"):
        mm(q.data, s, two.data, two.row_scale)
    with pytest.raises(ValueError, match="a_scale"):
        mm(q.data, s[:32], q.data, s)
    with pytest.raises(ValueError, match="b_scale"):
        mm(q.data, s, q.data, s.double())
    with pytest.raises(TypeError, match="int8"):
        mm(q.data.view(torch.uint8), s, q.data, s)
    with pytest.raises(ValueError, match="contiguous rows"):
        mm(q.data.t().contiguous().t(), s, q.data, s)
    with pytest.raises(ValueError, match="bias"):
        mm(q.data, s, q.data, s, bias=x[0, :32].contiguous())
    with pytest.raises(TypeError, match="out_dtype"):
        mm(q.data, s, q.data, s, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="out must be"):
        mm(q.data, s, q.data, s, out=x.float())
    with pytest.raises(_lib.Fp8LibError, match="N % 8"):
        mm(q.data, s, q.data[:4], s[:4])
    with pytest.raises(ValueError, match="inner dims"):
        ops.linear_int8(x, two.data, two.row_scale)
    with pytest.raises(ValueError, match="128"):
        ops.gemm_geglu_int8(q.data, s, q.data, s, 32)
    with pytest.raises(ValueError, match="rows"):
        ops.gemm_geglu_int8(q.data, s, q.data, s, 128)
    with pytest.raises(ValueError, match="multiples of 16"):
        linear.Int8LinearFunction.apply(x, torch.zeros(40, 64, dtype=BF16, device=gpu, requires_grad=True),
                                        None, None)
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.geglu_mxint8(x[:, :48])
    with pytest.raises(ValueError, match="checkpoint must be"):
        ops.geglu_bwd_mxint8(x, ops.quantize_mxint8(x))
    with pytest.raises(ValueError, match="checkpoint must be"):
        ops.dequant_mxint8(ops.MxInt8Tensor(q.data, q.data))


@pytest.mark.parametrize("shape", [(3, 7, 32), (1, 300, 32), (32,), (0, 4, 32)])
def test_functions_of_batched_rows(gpu, shape):
    """x of any number of dimensions: the values and the gradients of its rows, in its shape (x longer than K among
    them, whose rows the backward must not take for K)."""
    I, N = 128, 48
    M = torch.Size(shape[:-1]).numel()
    x = _x(M + 1, 32, 1, False)[:M].to(gpu).view(shape)
    w, w_gu, w_d = (_x(*s, 7, False).to(gpu) for s in ((N, 32), (2 * I, 32), (N, I)))
    copies = [linear.quantize_weight_int8(t) for t in (w, w_gu, w_d)]
    for cached in (False, True):
        wq, gq, dq = copies if cached else (None,) * 3
        for f, weights in ((lambda t, a: linear.Int8LinearFunction.apply(t, a, None, wq), (w,)),
                           (lambda t, a, b: linear.Int8GegluMlpFunction.apply(t, a, b, gq, dq, I), (w_gu, w_d))):
            leaves = [t.detach().requires_grad_() for t in (x, *weights)]
            rows = [t.detach().requires_grad_() for t in (x.reshape(-1, 32), *weights)]
            y, want = f(*leaves), f(*rows)
            assert y.shape == (*shape[:-1], N) and torch.equal(y.reshape(-1, N), want)
            dy = torch.ones_like(want)
            got = torch.autograd.grad(y, leaves, dy.view(y.shape))
            for a, b in zip(got, torch.autograd.grad(want, rows, dy)):
                assert torch.equal(a.reshape(b.shape), b)
            assert got[0].shape == x.shape
            with torch.no_grad():
                assert torch.equal(f(*leaves), y)


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("lead", [(5,), (0,), (2, 3), (0, 3), (2, 0)])
def test_gated_gelu_of_no_rows_and_of_any_alignment(gpu, checkpoint, lead):
    """Recorded or not, an empty batch and pre-activations (and their gradient) whose storage starts off 16 bytes."""
    I = 64
    n = torch.Size(lead).numel()
    GU, dH = _x(n + 1, 2 * I, 3, False)[:n], _x(n + 1, I, 4, False)[:n]

    def off(t, shape):
        for k in (1, 4):
            store = torch.zeros(t.numel() + 8, dtype=BF16, device=gpu)
            yield store[k:k + t.numel()].copy_(t.flatten()).view(shape)
    want = ops.geglu(GU.to(gpu))[0] if n else torch.empty(0, I, dtype=BF16, device=gpu)
    for gu, dh in zip(off(GU, (*lead, 2 * I)), off(dH, (*lead, I))):
        with torch.no_grad():
            h = fused_mlp.gated_gelu(gu, checkpoint=checkpoint)
        assert h.shape == (*lead, I) and torch.equal(h.reshape(n, I), want)
        leaf = gu.detach().requires_grad_()
        assert leaf.data_ptr() == gu.data_ptr()
        h = fused_mlp.gated_gelu(leaf, checkpoint=checkpoint)
        assert torch.equal(h.detach().reshape(n, I), want)
        (grad,) = torch.autograd.grad(h, leaf, dh)
        assert grad.shape == leaf.shape
        if n:
            held = ops.dequant_mxint8(ops.quantize_mxint8(GU.to(gpu))) if checkpoint else GU.to(gpu)
            assert torch.equal(grad.reshape(n, 2 * I), ops.geglu_bwd(dH.to(gpu), held)[0])


def test_elementwise_gated_gelu_of_no_rows_leaves_maxima_of_zero(gpu):
    """No rows through the plain entries: partials of 0 that a cast may read."""
    none = torch.empty(0, 128, dtype=BF16, device=gpu)
    parts = torch.full((4,), 7, dtype=torch.int32, device=gpu)
    H, p = ops.geglu(none, partials=parts)
    assert tuple(H.shape) == (0, 64) and not bool(p.any())
    parts.fill_(7)
    dGU, p = ops.geglu_bwd(H, none, partials=parts)
    assert tuple(dGU.shape) == (0, 128) and not bool(p.any())


def test_gated_gelu_launches_on_its_tensors_device(gpu, monkeypatch):
    """Where another device is the current one, the tensors' is made it for the launch, with a checkpoint and without."""
    real, made = ops.torch.cuda.device, []

    def device(idx):
        made.append(idx)
        return real(idx)
    GU, dH = _gu(4, 64, 1, gpu)
    monkeypatch.setattr(ops.torch.cuda, "device", device)
    for checkpoint in (False, True):
        leaf = GU.detach().requires_grad_()
        monkeypatch.setattr(ops.torch._C, "_cuda_getDevice", lambda: 7)
        h = fused_mlp.gated_gelu(leaf, checkpoint=checkpoint)
        assert made == [0]
        torch.autograd.grad(h, leaf, dH)
        assert made == [0, 0]
        monkeypatch.undo()
        monkeypatch.setattr(ops.torch.cuda, "device", device)
        made.clear()


def test_read_back_of_codes_off_their_alignment(gpu):
    """Codes whose storage starts anywhere, as the other entries take them."""
    q = ops.quantize_int8(_x(20, 64, 1).to(gpu), colwise=True)
    for k in (1, 4, 7):
        store = torch.zeros(20 * 64 + 8, dtype=torch.int8, device=gpu)
        off = store[k:k + 20 * 64].copy_(q.data.flatten()).view(20, 64)
        got = ops.dequant_int8(ops.Int8Tensor(off, q.row_scale, None, None, 20, 64))
        assert torch.equal(got, ops.dequant_int8(q))
        off = store[k:k + 32 * 32].copy_(q.data_t[:32].flatten()).view(32, 32)
        got = ops.dequant_int8(ops.Int8Tensor(None, None, off, q.col_scale[:32], 20, 32), transpose=True)
        assert torch.equal(got, ops.dequant_int8(q, transpose=True)[:32])


@pytest.mark.parametrize("tile,has", [("256x256w8", True), ("160x256", True), ("64x128", True), ("128x128", True),
                                      ("192x256", False)])
@pytest.mark.parametrize("M,K,I", [(1, 16, 128), (290, 544, 640)])
def test_gated_product_runs_the_tile_that_is_named(gpu, monkeypatch, capfd, tile, has, M, K, I):
    """A named tile is the one that runs where it has a gated int8 variant (192x256 has none: the plan's own choice,
    which is printed where it is made), and gives the product's H and checkpoint."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    monkeypatch.setenv("BONGARD_FP8_GEMM_DEBUG", "1")
    x, w, _, _ = _mlp_inputs(M, K, I, 7, gpu)
    xq, wq = ops.quantize_int8(x), ops.quantize_int8(w)
    capfd.readouterr()
    H, gu = ops.gemm_geglu_int8(xq.data, xq.row_scale, wq.data, wq.row_scale, I, keep_gu=True)
    assert ("bf8 plan geglu" in capfd.readouterr().err) == (not has)
    GU = ops.gemm_int8(xq.data, xq.row_scale, wq.data, wq.row_scale)
    want = ops.quantize_mxint8(GU)
    assert torch.equal(H, ops.geglu(GU)[0]) and torch.equal(gu.data, want.data) and torch.equal(gu.exps, want.exps)


@pytest.mark.parametrize("shape", [(48,), (1, 48)])
def test_a_bias_of_any_shape_has_its_gradient(gpu, shape):
    """The forward takes N values; their gradient comes back in the bias' shape, with others and alone."""
    x, w, dy = (_x(*s, 7, False).to(gpu) for s in ((20, 32), (48, 32), (20, 48)))
    bias = _x(1, 48, 3, False).to(gpu).view(shape).requires_grad_()
    for leaf in (x.clone().requires_grad_(), x):
        linear.Int8LinearFunction.apply(leaf, w, bias, None).backward(dy)
        assert bias.grad.shape == shape and torch.equal(bias.grad.flatten(), ops.column_sums(dy))
        bias.grad = None


@pytest.mark.parametrize("M", [0, 1, 37, 1030])
def test_codes_of_a_wide_gradient(gpu, M):
    """Rows of dGU wider than the quantizer takes: the oracle's codes and scales whatever the number of rows."""
    I = 16416
    GU, dH = _gu(M + 1, I, 5, gpu)
    _, q = ops.geglu_mxint8(GU[:M])
    dGU = ops.geglu_bwd_mxint8(dH[:M], q)
    got = ops.geglu_bwd_mxint8(dH[:M], q, rowwise=True, colwise=True)
    assert tuple(got.data.shape) == (M, 2 * I) and tuple(got.data_t.shape) == (2 * I, (M + 15) // 16 * 16)
    if M:
        _check(got, dGU.cpu(), True, True)
        for rowwise, colwise in ((True, False), (False, True)):
            _check(ops.geglu_bwd_mxint8(dH[:M], q, rowwise=rowwise, colwise=colwise), dGU.cpu(), rowwise, colwise)


def test_product_of_codes_of_minus_128(gpu):
    """No quantizer writes them; their sums stay exact up to K 131,056 (* 128^2 < 2^31)."""
    M, N, K = 8, 16, 131056
    a = torch.full((M, K), -128, dtype=torch.int8, device=gpu)
    b = torch.full((N, K), -128, dtype=torch.int8, device=gpu)
    b[1::2] = 127
    one = torch.ones(N, device=gpu)
    y = ops.gemm_int8(a, one[:M], b, one, out_dtype=F32).cpu().double()
    want = torch.where(torch.arange(N) % 2 == 0, 128.0, -127.0).double() * 128 * K
    assert bool(((y - want).abs() <= 2.0 ** -24 * want.abs()).all())


def test_gated_gelu_of_the_widest_rows(gpu):
    """Rows of 2^22 and more, which the forward takes, have their gradient."""
    I = (1 << 22) + 32
    g = torch.Generator(device=gpu).manual_seed(0)
    GU, dH = (torch.randn(1, n, generator=g, device=gpu).to(BF16) for n in (2 * I, I))
    leaf = GU.clone().requires_grad_()
    fused_mlp.gated_gelu(leaf, checkpoint=True).backward(dH)
    assert torch.equal(leaf.grad, ops.geglu_bwd(dH, ops.dequant_mxint8(ops.quantize_mxint8(GU)))[0])
    with pytest.raises(_lib.Fp8LibError, match="too large"):
        ops.geglu_bwd_mxint8(dH, ops.quantize_mxint8(GU), rowwise=True)
