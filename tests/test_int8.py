"""CPU tests of the int8 and layer-norm oracle (against values worked out by hand) and of the refusals of
the int8, checkpoint and layer-norm entries, before any launch."""

import ctypes
import re
from fractions import Fraction

import pytest
import torch
from torch.autograd import forward_ad

from bongard_amd import _lib, fused_mlp, linear, ops, te_linear
from oracle import int8_oracle as i8


def test_codes_and_scales_of_hand_worked_rows():
    x = torch.tensor([[127.0, 63.5, 0.5, 1.5, -2.5, -127.0, 0.25, 64.0],   # steps of 1: ties to even
                      [254.0, 1.0, 3.0, 5.0, -7.0, 127.0, 0.0, 2.0],       # steps of 2
                      [1.0, 0.5, -0.5, 0.0, -1.0, 0.25, 0.0078125, 0.00390625],
                      [0.0] * 8]).to(torch.bfloat16)
    codes, scale = i8.quantize(x)
    assert codes[0].tolist() == [127, 64, 0, 2, -2, -127, 0, 64]
    assert codes[1].tolist() == [127, 0, 2, 2, -4, 64, 0, 1]
    # 127 x: 63.5 is a tie, to 64; 31.75; 0.9921875; 0.49609375
    assert codes[2].tolist() == [127, 64, -64, 0, -127, 32, 1, 0]
    assert codes[3].tolist() == [0] * 8
    assert scale.tolist()[:2] == [1.0, 2.0]
    assert scale[2].item() == torch.tensor(1 / 127, dtype=torch.float64).float().item()
    assert scale[3].item() == torch.tensor(2.0 ** -40 / 127, dtype=torch.float64).float().item()
    x[0, 3] = float("inf")
    x[2, 0] = float("nan")
    codes, scale = i8.quantize(x)
    assert torch.isnan(scale).tolist() == [True, False, True, False]
    assert not codes[0].any() and not codes[2].any()


def test_codes_are_the_nearest_of_the_exact_quotient():
    """Against rational arithmetic, rows of every seventh mantissa of their largest value."""
    g = torch.Generator().manual_seed(0)
    for m in range(128, 256, 7):
        x = torch.randint(-m, m + 1, (1, 24), generator=g).float() * 2.0 ** torch.randint(-9, 1, (1, 24), generator=g)
        x[0, 0], x[0, 1] = m, m / 2
        x = x.to(torch.bfloat16)
        codes, _ = i8.quantize(x)
        for c, v in zip(codes[0].tolist(), x[0].tolist()):
            q = Fraction(v) * 127 / Fraction(x.double().abs().max().item())
            assert c == round(q), (m, v)  # Python's round: ties to even


def test_columns_are_the_rows_of_the_transpose():
    x = torch.randn(21, 24).to(torch.bfloat16)
    codes, scale = i8.quantize(x, 0)
    want, ws = i8.quantize(x.t().contiguous())
    assert codes.shape == (24, 32) and torch.equal(codes[:, :21], want) and not codes[:, 21:].any()
    assert torch.equal(scale, ws)


@pytest.mark.parametrize("amax,e", [(127.0, 133), (127.5, 134), (64.0, 133), (63.5, 132), (1.0, 127),
                                    (1.984375, 127), (1.9921875, 128), (2.0 ** -126, 7), (2.0 ** -133, 7),
                                    (0.0, 7), (3.3895e38, 254), (float("inf"), 255), (float("nan"), 255)])
def test_checkpoint_exponents(amax, e):
    x = torch.zeros(1, 40)
    x[0, 3], x[0, 5] = amax, -amax / 2 if amax == amax else 0.0
    codes, exps = i8.checkpoint(x.to(torch.bfloat16))
    assert exps.tolist() == [[e, 7]]
    if amax == 3.3895e38:
        assert codes[0, 3] == 127  # 127.5 steps of the last power of two
    elif 7 < e < 255:
        assert codes.abs().max() >= 64 and i8.restored(codes, exps)[0, 3] == pytest.approx(amax, rel=1 / 128)


def test_checkpoint_codes_are_the_nearest_and_bf16_holds_the_values():
    x = torch.randn(9, 72).to(torch.bfloat16)
    codes, e = i8.checkpoint(x)
    v = i8.restored(codes, e)
    step = torch.ldexp(torch.ones(()), e.int() - 133).double().repeat_interleave(32, 1)[:, :72]
    assert bool(((v - x.double()).abs() <= step / 2).all())
    assert torch.equal(v.to(torch.bfloat16).double(), v)
    x = torch.zeros(1, 32)
    x[0, :5] = torch.tensor([64.0, 0.5, 1.5, -2.5, 63.5])
    assert i8.checkpoint(x.to(torch.bfloat16))[0][0, :5].tolist() == [64, 0, 2, -2, 64]


def test_layer_norm_of_hand_worked_rows():
    x = torch.tensor([[1.0, 3.0, 1.0, 3.0], [5.0, 5.0, 5.0, 5.0], [0.0, 0.0, 0.0, 8.0]])
    w, b = torch.tensor([1.0, 2.0, 3.0, 4.0]), torch.tensor([0.0, 1.0, 0.0, -1.0])
    y, n, mean, sd = i8.layer_norm(x, w, b, 0.0)
    assert mean.flatten().tolist() == [2, 5, 2] and sd[0].item() == 1 and sd[2].item() == 12 ** 0.5
    assert y[0].tolist() == [-1, 3, -3, 3]
    y, _, _, sd = i8.layer_norm(x, w, b, 9.0)
    assert sd[1].item() == 3 and y[1].tolist() == b.tolist()
    # the gradients are autograd's of the formula
    x = torch.randn(5, 8, dtype=torch.float64, requires_grad=True)
    w, b, dy = (torch.randn(s, dtype=torch.float64) for s in ((8,), (8,), (5, 8)))
    w.requires_grad_(), b.requires_grad_()
    want = torch.autograd.grad(torch.nn.functional.layer_norm(x, (8,), w, b, 1e-5), [x, w, b], dy)
    _, n, _, sd = i8.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5)
    for a, v in zip(i8.layer_norm_backward(n, sd, dy, w.detach()), want):
        assert torch.allclose(a, v, rtol=1e-12, atol=1e-13)


def test_recipe_is_offered():
    assert "int8" in te_linear.RECIPES
    t = te_linear.TELinear([torch.nn.Linear(64, 32, bias=False)], "int8")
    assert t.get_extra_state().numel() == 0 and t.recipe.checkpoint_block == 32
    with pytest.raises(ValueError, match="multiples of 16"):
        linear._check_int8("layer", 64, 40)


def _calls(L):
    null = ctypes.c_void_p(0)
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    q, d, g, h = L.bf8_quantize_int8_bf16, L.bf8_dequant_int8, L.bf8_gemm_int8, L.bf8_gemm_geglu_int8
    m, dm, cs = L.bf8_quantize_mxint8_bf16, L.bf8_dequant_mxint8, L.bf8_column_sums_bf16
    f, b = L.bf8_geglu_mxint8, L.bf8_geglu_bwd_mxint8
    t, qm = L.bf8_linear_int8, L.bf8_quantize_int8_maxima_bf16
    n, nb = L.bf8_layernorm_bf16, L.bf8_layernorm_bwd_bf16
    lb, mb = L.bf8_linear_int8_backward, 1 << 20
    lg, lf = L.bf8_linear_geglu_int8, L.bf8_linear_int8_forward
    gb, kept, big = L.bf8_geglu_mlp_int8_backward, (p,) * 10, 1 << 30
    gf, w4 = L.bf8_geglu_mlp_int8_forward, (p,) * 4
    return [
        (gf, (p, 0, 16, 128, 16, *w4, p, p, p, p, p, p, p, p, big, null), "empty"),
        (gf, (p, 4, 24, 128, 16, *w4, p, p, p, p, p, p, p, p, big, null), "K % 16"),
        (gf, (p, 4, 16, 96, 16, *w4, p, p, p, p, p, p, p, p, big, null), "I % 128"),
        (gf, (p, 4, 16, 128, 12, *w4, p, p, p, p, p, p, p, p, big, null), "N % 8"),
        (gf, (p, 4, 16, 128, 16, *w4, null, p, p, p, p, p, p, p, big, null), "NULL"),
        (gf, (p, 4, 16, 128, 16, *w4, p, p, null, p, p, p, p, p, big, null), "NULL"),
        (gf, (p, 4, 16, 128, 16, *w4, p, p, p, p, p, p, null, p, big, null), "NULL"),
        (gf, (p, 4, 16, 128, 16, *w4, p, p, p, p, p, p, p, p, 64, null), "workspace needs"),
        (gb, (p, 0, 16, 32, 16, *kept, p, p, p, p, big, null), "empty"),
        (gb, (p, 4, 16, 24, 16, *kept, p, p, p, p, big, null), "I % 32"),
        (gb, (p, 4, 16, 16416, 16, *kept, p, p, p, p, big, null), "16384"),
        (gb, (p, 4, 16, 32, 24, *kept, p, p, p, p, big, null), "N % 16"),
        (gb, (p, 4, 12, 32, 16, *kept, p, p, p, p, big, null), "K % 8"),
        (gb, (p, 4, 16, 32, 16, *kept, null, null, null, p, big, null), "nothing requested"),
        (gb, (p, 4, 16, 32, 16, null, *kept[1:], p, p, p, p, big, null), "NULL"),
        (gb, (p, 4, 16, 32, 16, *kept[:2], null, *kept[3:], null, p, null, p, big, null), "NULL"),
        (gb, (p, 133121, 16, 32, 16, *kept, p, p, p, p, big, null), "133120"),
        (gb, (p, 4, 16, 32, 16, *kept, p, p, p, p, 64, null), "workspace needs"),
        (lf, (p, p, 0, 16, 16, null, p, p, p, p, p, p, mb, null), "empty"),
        (lf, (p, p, 4, 16, 24, null, p, p, p, p, p, p, mb, null), "K % 16"),
        (lf, (p, p, 4, 12, 16, null, p, p, p, p, p, p, mb, null), "N % 8"),
        (lf, (p, p, 4, 16, 32784, null, p, p, p, p, p, p, mb, null), "32768"),
        (lf, (p, p, 4, 16, 16, null, p, p, null, p, p, p, mb, null), "NULL"),
        (lf, (p, null, 4, 16, 16, null, p, p, p, p, p, p, mb, null), "NULL"),
        (lf, (p, p, 4, 16, 16, null, p, p, odd, p, p, p, mb, null), "16-byte"),
        (lf, (p, p, 70000, 16, 32768, null, p, p, p, p, p, p, mb, null), "2 GiB"),
        (lf, (p, p, 4, 16, 16, null, p, p, p, p, p, p, 64, null), "workspace needs"),
        (lg, (p, p, 32, p, 4, 64, 32, p, null, 0, null), "I % 128"),
        (lg, (p, p, 24, p, 4, 128, 24, p, null, 0, null), "K % 16"),
        (lg, (p, p, 32784, p, 4, 128, 32784, p, null, 0, null), "32768"),
        (lg, (p, p, 16, p, 4, 128, 32, p, null, 0, null), "row stride"),
        (lg, (odd, p, 32, p, 4, 128, 32, p, null, 0, null), "16-byte"),
        (lg, (p, null, 32, p, 4, 128, 32, p, null, 0, null), "NULL"),
        (lg, (p, p, 32, p, 4, 128, 0, p, null, 0, null), "K == 0"),
        (lg, (p, p, 32, p, 40, 128, 32, p, null, 0, null), "workspace needs"),
        (lb, (p, 0, 16, 16, p, p, p, p, p, p, p, mb, null), "empty"),
        (lb, (p, 4, 24, 16, p, p, p, p, p, p, p, mb, null), "N % 16"),
        (lb, (p, 4, 32784, 16, p, p, p, p, p, p, p, mb, null), "32768"),
        (lb, (p, 4, 16, 12, p, p, p, p, p, p, p, mb, null), "K % 8"),
        (lb, (p, 133121, 16, 16, p, p, p, p, p, p, p, mb, null), "133120"),
        (lb, (p, 4, 16, 16, p, p, p, p, null, null, p, mb, null), "nothing requested"),
        (lb, (p, 4, 16, 16, null, p, p, p, p, p, p, mb, null), "NULL"),
        (lb, (p, 4, 16, 16, p, p, p, null, p, p, p, mb, null), "NULL"),
        (lb, (p, 4, 16, 16, p, p, p, odd, p, p, p, mb, null), "16-byte"),
        (lb, (p, 66000, 32768, 16, p, p, null, null, p, null, p, mb, null), "2 GiB"),
        (lb, (p, 100000, 32768, 16, p, p, p, p, p, p, p, mb, null), "2 GiB"),
        (lb, (p, 4, 16, 16, p, p, p, p, p, p, p, 64, null), "workspace needs"),
        (lb, (p, 4, 16, 16, p, p, p, p, p, p, null, 0, null), "workspace needs"),
        (q, (p, 4, 12, p, p, null, null, null, 0, null), "cols % 8"),
        (q, (p, 4, 32776, p, p, null, null, null, 0, null), "32768"),
        (q, (p, -1, 16, p, p, null, null, null, 0, null), "bad shape"),
        (q, (p, 4, 16, null, null, null, null, null, 0, null), "give out"),
        (q, (p, 4, 16, p, null, null, null, null, 0, null), "give out"),
        (q, (p, 4, 16, null, null, p, null, p, 1 << 20, null), "give out"),
        (q, (null, 4, 16, p, p, null, null, null, 0, null), "x is NULL"),
        (q, (odd, 4, 16, p, p, null, null, null, 0, null), "16-byte"),
        (q, (p, 4, 16, odd, p, null, null, null, 0, null), "8-byte"),
        (q, (p, 4, 16, null, null, p, p, null, 0, null), "workspace needs"),
        (q, (p, 4, 16, null, null, p, p, p, 8, null), "workspace needs"),
        (d, (p, p, 4, 12, p, null), "cols % 8"),
        (d, (p, null, 4, 16, p, null), "NULL"),
        (d, (p, p, 4, 16, odd, null), "16-byte"),
        (g, (p, 32, p, p, 32, p, 4, 8, 24, null, p, 0, 8, null, 0, null), "K % 16"),
        (g, (p, 133136, p, p, 133136, p, 4, 8, 133136, null, p, 0, 8, null, 0, null), "133120"),
        (g, (p, 32, p, p, 32, p, 4, 9, 32, null, p, 0, 12, null, 0, null), "N % 8"),
        (g, (p, 32, p, p, 32, p, 4, 8, 32, null, p, 0, 4, null, 0, null), "ldc"),
        (g, (p, 16, p, p, 32, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "row stride"),
        (g, (p, 40, p, p, 32, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "row stride"),
        (g, (p, 32, odd, p, 32, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "16-byte"),
        (g, (p, 32, p, p, 32, null, 4, 8, 32, null, p, 0, 8, null, 0, null), "B or its scales"),
        (g, (p, 32, p, p, 32, p, 4, 8, 32, null, p, 2, 8, null, 0, null), "out_dtype"),
        (g, (p, 32, p, p, 32, p, 4, 8, 32, odd, p, 0, 8, null, 0, null), "bias"),
        (g, (p, 32, p, p, 32, p, 4, 8, 32, null, null, 0, 8, null, 0, null), "C is NULL"),
        (g, (p, 32, p, p, 32, p, 4, 8, 32, null, p, 0, 8, odd, 64, null), "workspace"),
        (g, (p, 32, p, p, 32, p, 4, 8, 0, null, p, 0, 8, null, 0, null), "K == 0"),
        (g, (p, 1 << 20, p, p, 32, p, 1 << 11, 8, 32, null, p, 0, 8, null, 0, null), "2 GiB"),
        (t, (p, p, 32, p, 4, 8, 24, null, p, 0, 8, null, 0, null), "K % 16"),
        (t, (p, p, 32784, p, 4, 8, 32784, null, p, 0, 8, null, 0, null), "32768"),
        (t, (p, p, 32, p, 4, 12, 32, null, p, 0, 12, null, 0, null), "N % 8"),
        (t, (p, p, 16, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "row stride"),
        (t, (odd, p, 32, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "16-byte"),
        (t, (p, p, 32, p, 4, 8, 32, odd, p, 0, 8, null, 0, null), "8-byte"),
        (t, (p, p, 32, null, 4, 8, 32, null, p, 0, 8, null, 0, null), "NULL"),
        (t, (p, p, 32, p, 4, 8, 32, null, p, 3, 8, null, 0, null), "out_dtype"),
        (t, (p, p, 32, p, 4, 8, 0, null, p, 0, 8, null, 0, null), "K == 0"),
        (t, (p, p, 32, p, 400, 8, 32, null, p, 0, 8, null, 0, null), "workspace needs"),
        (h, (p, 32, p, p, 32, p, 4, 96, 32, p, null, null, null), "multiple of 128"),
        (h, (p, 32, p, p, 32, p, 4, 128, 40, p, null, null, null), "K % 16"),
        (h, (p, 32, p, p, 32, p, 4, 128, 0, p, null, null, null), "K == 0"),
        (h, (p, 32, p, p, 32, p, 4, 128, 32, null, null, null, null), "H is NULL"),
        (h, (p, 32, p, p, 32, p, 4, 128, 32, p, p, null, null), "exponents"),
        (h, (p, 32, p, p, 32, p, 4, 128, 32, p, odd, p, null), "8-byte"),
        (h, (p, 32, null, p, 32, p, 4, 128, 32, p, null, null, null), "X or its scales"),
        (m, (p, 4, 12, p, p, null), "cols % 8"),
        (m, (p, 4, 16, p, null, null), "NULL"),
        (m, (odd, 4, 16, p, p, null), "16-byte"),
        (dm, (odd, p, 4, 16, p, null), "8-byte"),
        (dm, (p, p, 4, 16, null, null), "NULL"),
        (f, (p, 4, 40, p, p, p, null), "I % 32"),
        (f, (p, 4, 64, p, p, null, null), "NULL"),
        (f, (odd, 4, 64, p, p, p, null), "16-byte"),
        (b, (p, p, p, 4, 24, p, null, 0, null), "I % 32"),
        (b, (p, null, p, 4, 32, p, null, 0, null), "NULL"),
        (b, (p, odd, p, 4, 32, p, null, 0, null), "8-byte"),
        (b, (p, p, p, 4, 32, p, p, 8, null), "maxima need"),
        (qm, (p, 4, 24, 2, p, p, null, null, p, 1 << 20, null), "cols % 8"),
        (qm, (p, 4, 32, 3, p, p, null, null, p, 1 << 20, null), "parts"),
        (qm, (p, 4, 32, 2, p, p, null, null, p, 8, null), "bytes of maxima"),
        (qm, (p, 4, 32, 2, p, p, null, null, null, 1 << 20, null), "bytes of maxima"),
        (qm, (p, 4, 32, 2, p, null, null, null, p, 1 << 20, null), "give out"),
        (qm, (odd, 4, 32, 2, p, p, null, null, p, 1 << 20, null), "16-byte"),
        (cs, (p, 0, 16, p, p, 1 << 20, null), "rows > 0"),
        (cs, (p, 4, 12, p, p, 1 << 20, null), "cols % 8"),
        (cs, (p, 4, 16, null, p, 1 << 20, null), "must be given"),
        (cs, (p, 4, 16, p, p, 8, null), "workspace of 8 bytes"),
        (n, (p, 4, 12, p, null, 1e-6, p, null, null, null, null, null), "cols % 8"),
        (n, (p, 4, 16392, p, null, 1e-6, p, null, null, null, null, null), "16384"),
        (n, (p, 4, 16, null, null, 1e-6, p, null, null, null, null, null), "NULL"),
        (n, (p, 4, 16, p, odd, 1e-6, p, null, null, null, null, null), "16-byte"),
        (n, (p, 4, 16, p, p, 1e-6, p, p, null, null, null, null), "mean and rstd"),
        (n, (p, 4, 16, p, p, 1e-6, p, p, p, p, null, null), "go together"),
        (nb, (p, null, null, p, 0, 16, p, p, p, p, null, null, null, 0, null), "no rows"),
        (nb, (p, p, p, p, 4, 16, p, p, p, p, null, null, null, 0, null), "give x or"),
        (nb, (null, null, null, p, 4, 16, p, p, p, p, null, null, null, 0, null), "give x or"),
        (nb, (p, null, null, p, 4, 16, p, p, null, p, null, null, null, 0, null), "NULL"),
        (nb, (p, null, null, p, 4, 16, p, p, p, null, null, null, null, 0, null), "nothing"),
        (nb, (p, null, null, p, 4, 16, p, p, p, p, p, null, p, 8, null), "workspace of 8 bytes"),
        (nb, (p, null, null, odd, 4, 16, p, p, p, p, null, null, null, 0, null), "16-byte"),
    ]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are no memory: the host checks alone")
def test_entries_refuse_before_any_launch():
    L = _lib.lib()
    for fn, args, message in _calls(L):
        assert fn(*args) == 1, (fn.__name__, args)
        told = L.bf8_last_error().decode()
        assert told.startswith(fn.__name__ + ":") and message in told, (message, told)


def test_a_weight_gradient_of_too_many_tokens():
    """More terms than an int32 sum holds are refused where the forward could still be told."""
    x, w = torch.empty(133121, 16, dtype=torch.bfloat16), torch.empty(16, 16, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="133120 tokens"):
        linear.Int8LinearFunction.apply(x, w, None, None)
    down = torch.empty(16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="133120 tokens"):
        linear.Int8GegluMlpFunction.apply(x, torch.empty(256, 16, dtype=torch.bfloat16, requires_grad=True), down,
                                          None, None, 128)


def test_sizes_of_nothing():
    """Empty calls return without a launch or a pointer; the workspaces of nothing are empty."""
    L = _lib.lib()
    null, p = ctypes.c_void_p(0), ctypes.c_void_p(4096)
    assert L.bf8_quantize_int8_bf16(null, 0, 64, p, p, null, null, null, 0, null) == 0
    assert L.bf8_dequant_int8(null, null, 0, 64, null, null) == 0
    assert L.bf8_gemm_int8(null, 64, null, null, 64, null, 0, 8, 64, null, null, 0, 8, null, 0, null) == 0
    assert L.bf8_gemm_geglu_int8(null, 64, null, null, 64, null, 0, 128, 64, null, null, null, null) == 0
    assert L.bf8_quantize_mxint8_bf16(null, 0, 64, null, null, null) == 0
    assert L.bf8_dequant_mxint8(null, null, 3, 0, null, null) == 0
    assert L.bf8_geglu_mxint8(null, 0, 32, null, null, null, null) == 0
    assert L.bf8_geglu_bwd_mxint8(null, null, null, 0, 32, null, null, 0, null) == 0
    assert L.bf8_layernorm_bf16(null, 0, 64, null, null, 1e-6, null, null, null, null, null, null) == 0
    assert L.bf8_quantize_int8_workspace(0, 64, 0) == 0 and L.bf8_quantize_int8_workspace(3, 64, 0) >= 64 * 6
    assert L.bf8_quantize_int8_workspace(3, 64, 1) == 0 and L.bf8_quantize_int8_workspace(5000, 64, 1) >= 64 * 6
    for ws in (L.bf8_column_sums_workspace, L.bf8_layernorm_bwd_workspace):
        assert ws(0, 64) == 0 and ws(3, 64) >= 64 * 4
    assert L.bf8_gemm_int8_workspace(0, 8, 64) == 0


@pytest.mark.parametrize("tile", ["256x160", "160x256", "128x128", "192x256", "128x64", "64x128", "256x256w8",
                                  "256x256w8x", "192x128o2", "128x128o2", "128x64k2", "64x128k2", "128x64:3",
                                  "256x256w8:2"])
def test_a_named_tile_is_the_plan(monkeypatch, capfd, tile):
    """Every tile of the int8 product can be named, in as many pieces; 256x128, 256x256 and 128x128k2 have
    no such variant (a plan of the planner's own is printed)."""
    L = _lib.lib()
    M, N, K = 517, 1040, 8224
    monkeypatch.setenv("BONGARD_FP8_GEMM_DEBUG", "1")
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    pieces = int(tile.partition(":")[2] or 1)
    assert L.bf8_gemm_int8_workspace(M, N, K) == (4 * pieces * M * N if pieces > 1 else 0)
    assert "bf8 plan" not in capfd.readouterr().err
    for none in ("256x128", "256x256", "128x128k2"):
        monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", none)
        L.bf8_gemm_int8_workspace(M, N, K)
        assert "bf8 plan gemm" in capfd.readouterr().err


@pytest.mark.parametrize("M,N,K,tiles,splits", [
    (2001, 2560, 10240, {"128x128o2", "192x128o2", "256x160", "160x256"}, [1]),  # in two pieces 91 us, unsplit 70-80
    (4096, 2560, 10240, {"256x160", "256x256w8x"}, [1]),  # 106 us, in two pieces 159
    (64, 2048, 2560, {"128x64", "128x64k2"}, range(1, 8)),
])
def test_planner_picks_int8(monkeypatch, capfd, M, N, K, tiles, splits):
    """Its partials cost more than FP8's: fewer products run in K pieces."""
    monkeypatch.delenv("BONGARD_FP8_GEMM_TILE", raising=False)
    monkeypatch.setenv("BONGARD_FP8_GEMM_DEBUG", "1")
    _lib.lib().bf8_gemm_int8_workspace(M, N, K)
    tile, pieces = re.search(r"tile (\S+) splits (\d+)", capfd.readouterr().err).groups()
    assert tile in tiles and int(pieces) in splits


def test_layer_norm_refuses_forward_mode_tangents(monkeypatch):
    """No tangent is dropped, whether gradients are recorded or not."""
    monkeypatch.setattr(ops, "_layernorm", lambda x, *a, **k: (torch.zeros_like(x), None, None))
    args = dict(x=torch.ones(4, 16), weight=torch.ones(16), bias=torch.ones(16))
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            assert fused_mlp.layer_norm(**args).shape == (4, 16)
            for name in args:
                dual = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
                with pytest.raises(NotImplementedError, match="jvp"):
                    fused_mlp.layer_norm(**{**args, name: dual})


def _copy_of(rows, cols):
    """An int8 weight's cached copies, as the functions take them."""
    z = lambda *s: torch.zeros(*s, dtype=torch.int8)  # noqa: E731
    return ops.Int8Tensor(z(rows, cols), torch.ones(rows), z(cols, (rows + 15) // 16 * 16), torch.ones(cols), rows, cols)


def test_weights_and_their_copies_must_fit():
    """The backward's sizes are the weights' and x's, its operands the cached copies: others would run it past their
    ends. Refused by the forward, before any tensor is read."""
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, requires_grad=True)  # noqa: E731
    x, w = z(4, 32), z(48, 32)
    for q in (_copy_of(64, 32), _copy_of(48, 16), _copy_of(32, 48)):
        with pytest.raises(ValueError, match="wq is the copy"):
            linear.Int8LinearFunction.apply(x, w, None, q)
    gu, down = z(256, 32), z(16, 128)
    apply = linear.Int8GegluMlpFunction.apply
    for args in ((z(512, 32), down, None, None), (gu, z(16, 256), None, None), (z(256, 64), down, None, None),
                 (gu, z(16, 256), _copy_of(256, 32), _copy_of(16, 128))):
        with pytest.raises(ValueError, match="intermediate size 128"):
            apply(x, *args, 128)
    with pytest.raises(ValueError, match="gu_q is the copy"):
        apply(x, gu, down, _copy_of(512, 32), _copy_of(16, 128), 128)
    with pytest.raises(ValueError, match="down_q is the copy"):
        apply(x, gu, down, _copy_of(256, 32), _copy_of(32, 128), 128)


def test_functions_see_x_as_rows(monkeypatch):
    """x of any number of dimensions reaches the int8 calls as [M, K] and its gradient comes back in its shape: the
    backward's K is x's last size, not its second."""
    seen = []

    def forward(x, I, gu_q, down_q, *keep):
        seen.append(tuple(x.shape))
        return (torch.zeros(x.shape[0], down_q.rows, dtype=torch.bfloat16), *[None] * 6)

    def backward(dy, K, I, needs, *kept):
        seen.append((dy.reshape(-1, dy.shape[-1]).shape[0], K, I))
        return torch.ones(dy.reshape(-1, dy.shape[-1]).shape[0], K, dtype=torch.bfloat16), None, None
    monkeypatch.setattr(ops, "_geglu_mlp_int8_forward", forward)
    monkeypatch.setattr(ops, "_geglu_mlp_int8_backward", backward)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    for shape in ((6, 32), (2, 3, 32), (1, 64, 32), (32,), (2, 1, 2, 32)):
        rows, x = z(*shape).numel() // 32, z(*shape).requires_grad_()
        y = linear.Int8GegluMlpFunction.apply(x, z(256, 32), z(16, 128), _copy_of(256, 32), _copy_of(16, 128), 128)
        assert y.shape == (*shape[:-1], 16)
        y.backward(torch.ones_like(y))
        assert x.grad.shape == x.shape and seen[-2:] == [(rows, 32), (rows, 32, 128)]


def _refusal(entry, *args):
    """What an entry says of sizes and no memory: nothing of the sizes where it is the workspace that it misses."""
    L = _lib.lib()
    assert getattr(L, entry)(*args) == 1
    told = L.bf8_last_error().decode()
    return None if "workspace needs" in told else told


def _ctypes(flags, *given):
    p, null = ctypes.c_void_p(4096), ctypes.c_void_p(0)
    return [p if flags[k] else null for k in given]


SIZES = [(4, 32, 32768), (4, 32, 32784), (104857, 2560, 20480), (104858, 2560, 20480), (104848, 2560, 20480),
         (133120, 32, 16128), (133120, 32, 16144), (133121, 32, 32), (66000, 32784, 32), (65535, 16, 32768),
         (65536, 16, 32768), (65519, 16, 32768), (1, 65536, 32768), (1, 65520, 32768), (16384, 131072, 16)]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are no memory: the host checks alone")
@pytest.mark.parametrize("dx,dw", [(True, False), (False, True), (True, True)])
def test_a_linears_forward_refuses_what_its_backward_does(dx, dw):
    """The same sizes on both sides of every limit: rows, features, tokens, 2 GiB."""
    seen = set()
    for M, K, N in SIZES:
        told = _refusal("bf8_linear_int8_backward", ctypes.c_void_p(4096), M, N, K, *_ctypes((dx, dw), 0, 0, 1, 1, 0, 1),
                        ctypes.c_void_p(4096), 64, ctypes.c_void_p(0))
        try:
            linear._check_int8_backward("layer", M, K, N, dx, dw)
            assert told is None, (M, K, N, told)
        except ValueError as e:
            assert told is not None, (M, K, N, e)
        seen.add(told is None)
    assert seen == {True, False}


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are no memory: the host checks alone")
@pytest.mark.parametrize("needs", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1), (1, 0, 1), (0, 1, 1)])
def test_a_gated_mlps_forward_refuses_what_its_backward_does(monkeypatch, needs):
    """As its autograd function checks: intermediate sizes, output features, tokens, [gate | up] of 2 GiB."""
    monkeypatch.setattr(linear, "_check_int8_weight", lambda *a: None)
    z = lambda r, c, n: torch.empty(1, 1, dtype=torch.bfloat16).expand(r, c).requires_grad_(bool(n))  # noqa: E731
    seen = set()
    for M, K, I, N in [(4, 16, 16384, 16), (4, 16, 16512, 16), (4, 16, 128, 32768), (4, 16, 128, 32784),
                       (104848, 16, 10240, 16), (104849, 16, 10240, 16), (104858, 16, 10240, 16), (133120, 16, 128, 16),
                       (133121, 16, 128, 16), (65536, 16, 256, 32768), (65520, 16, 256, 32768)]:
        dh = needs[0] or needs[1]
        flags = (dh, needs[1], needs[2], needs[0])
        told = _refusal("bf8_geglu_mlp_int8_backward", ctypes.c_void_p(4096), M, K, I, N,
                        *_ctypes(flags, 0, 0, 1, 1, 2, 2, 3, 3, 0, 0, 3, 1, 2), ctypes.c_void_p(4096), 64,
                        ctypes.c_void_p(0))
        args = z(M, K, needs[0]), z(2 * I, K, needs[1]), z(N, I, needs[2])
        try:
            linear.Int8GegluMlpFunction.apply(*args, None, None, I)
        except ValueError as e:
            assert told is not None and "gradient" in str(e), (M, K, I, N, e)
        except RuntimeError:  # (past the checks: these tensors are on no GPU)
            assert told is None, (M, K, I, N, told)
        with torch.no_grad(), pytest.raises(RuntimeError):
            linear.Int8GegluMlpFunction.apply(*args, None, None, I)
        seen.add(told is None)
    assert seen == {True, False}


@pytest.mark.parametrize("M,N", [(4, 32784), (104858, 20480)])
def test_an_int8_linear_refuses_in_its_forward(M, N):
    z = lambda r, c: torch.empty(1, 1, dtype=torch.bfloat16).expand(r, c)  # noqa: E731
    with pytest.raises(ValueError, match="gradients take"):
        linear.Int8LinearFunction.apply(z(M, 2560).requires_grad_(), z(N, 2560), None, None)
    with torch.no_grad(), pytest.raises(RuntimeError):  # (past the checks)
        linear.Int8LinearFunction.apply(z(M, 2560).requires_grad_(), z(N, 2560), None, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are no memory: the host checks alone")
def test_a_gated_mlps_backward_refuses_before_its_first_launch():
    """Sizes and alignments that only its last products read."""
    p, odd, null = ctypes.c_void_p(4096), ctypes.c_void_p(4100), ctypes.c_void_p(0)
    f, big = _lib.lib().bf8_geglu_mlp_int8_backward, 1 << 40
    for M, args, message in ((104864, [p] * 13, "2 GiB"), (65536, [p] * 13, None),
                             *((4, [p] * k + [odd] + [p] * (12 - k), "aligned") for k in range(13) if k != 1)):
        I = 10240
        assert f(p, M, 16, I, 16, *args, p, 64 if message is None else big, null) == 1
        told = _lib.lib().bf8_last_error().decode()
        assert told.startswith("bf8_geglu_mlp_int8_backward:") and (message or "workspace needs") in told, (M, told)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are no memory: the host checks alone")
@pytest.mark.parametrize("tile", ["", "256x256w8"])
def test_a_gated_mlps_forward_refuses_before_its_first_launch(monkeypatch, tile):
    """Whichever plan runs the products: H's columnwise codes off 16 bytes (one of two quantizations writes them),
    operands of 2 GiB that only the down product reads."""
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    L = _lib.lib()
    p, odd, null = ctypes.c_void_p(4096), ctypes.c_void_p(4100), ctypes.c_void_p(0)
    f, big = L.bf8_geglu_mlp_int8_forward, 1 << 40
    # (W_gu, its scale, W_down, its scale, Y, GU8, its exponents, Xt, its scale, Ht, its scale)
    cases = [(4, 128, 16, [p] * k + [odd] + [p] * (10 - k), "aligned") for k in range(11) if k != 6]
    cases += [(4, 128, 16, [p] * 11, None), (65536, 32768, 16, [p] * 11, "2 GiB"), (65535, 32768, 16, [p] * 11, None),
              (4, 32768, 65536, [p] * 11, "2 GiB"), (4, 32768, 65528, [p] * 11, None)]
    for M, I, N, args, message in cases:
        assert f(p, M, 16, I, N, *args, p, big if message else 64, null) == 1
        told = L.bf8_last_error().decode()
        assert told.startswith("bf8_geglu_mlp_int8_forward:") and (message or "workspace needs") in told, (M, N, told)
    assert f(odd, 4, 16, 128, 16, *[p] * 11, p, big, null) == 1 and "aligned" in L.bf8_last_error().decode()
