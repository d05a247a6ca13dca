"""CPU tests of the MXFP4 oracle (against values worked out by hand and against a search over the
grid) and of the refusals of the MXFP4 and residual-norm entries, before any launch."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from bongard_amd import _lib, fused_mlp, linear, ops, te_linear
from oracle import fp8_oracle as orc
from oracle import mxfp4_oracle as mx4

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def _block(*head):
    x = torch.zeros(1, 32)
    x[0, :len(head)] = torch.tensor(head)
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("amax,e", [(6.0, 127), (6.03125, 128), (5.0, 127), (3.0, 126), (3.015625, 127),
                                    (12.0, 128), (1.0, 125), (2.0 ** -126, 0), (2.0 ** -133, 0),
                                    (0.0, 0), (3.3895e38, 253), (float("inf"), 254), (float("nan"), 255)])
def test_scale_is_the_smallest_that_clips_nothing(amax, e):
    x = _block(amax, -amax / 2 if amax == amax else 0.0)
    assert mx4.exponents(x).item() == e
    if 0 < e < 254:
        s = 2.0 ** (e - 127)
        assert x.double().abs().max() <= 6 * s and x.double().abs().max() > 3 * s


def test_codes_are_the_nearest_and_ties_go_to_the_even_code():
    ticks = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.2, 0.26, 4.9, 5.1])
    packed, e = mx4.quantize(_block(*ticks.tolist(), -0.75))
    v = mx4.values(packed, e)[0]
    assert v[:13].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, 0.5, 4, 6, -1]
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 96, generator=g).to(torch.bfloat16)
    packed, e = mx4.quantize(x)
    s = torch.ldexp(torch.ones((), dtype=torch.float64), e.int() - 127).repeat_interleave(32, 1)
    err = (mx4.values(packed, e) - x.double()).abs() / s
    best = (x.double().abs()[..., None] / s[..., None] - GRID).abs().amin(-1)
    assert torch.equal(err, best)


def test_planes_and_columns():
    x = torch.randn(40, 160).to(torch.bfloat16)
    packed, e = mx4.quantize(x, 0)
    assert packed.shape == (160, 32) and e.shape == (160, 2)
    assert bool((mx4.values(packed, e)[:, 40:] == 0).all())
    p = mx4.planes(e)
    assert p.shape == (1, 160) and bool(((p >> 16) == 0x7F7F).all())


def test_recipe_is_offered():
    assert "mxfp4" in te_linear.RECIPES
    t = te_linear.TELinear([torch.nn.Linear(64, 32, bias=False)], "mxfp4")
    assert t.get_extra_state().numel() == 0 and t.recipe.block_size == 32
    with pytest.raises(ValueError, match="multiples of 32"):
        linear._check_mxfp4("layer", 64, 40)


def _calls(L):
    null = ctypes.c_void_p(0)
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    q, g = L.bf8_quantize_mxfp4_bf16, L.bf8_gemm_mxfp4
    n, b = L.bf8_rmsnorm_residual_bf16, L.bf8_rmsnorm_residual_bwd_bf16
    deq = L.bf8_dequant_mxfp4
    h, d = L.bf8_gemm_geglu_mxfp4, L.bf8_geglu_bwd_mxfp4
    return [
        (h, (p, 16, p, p, 16, p, 4, 96, 32, p, p, null, null, null, null), "multiple of 128"),
        (h, (p, 16, p, p, 16, p, 4, 128, 48, p, p, null, null, null, null), "32-element"),
        (h, (p, 16, p, p, 16, p, 4, 128, 0, p, p, null, null, null, null), "K == 0"),
        (h, (p, 16, p, p, 16, p, 4, 128, 32, null, p, null, null, null, null), "NULL"),
        (h, (p, 16, p, p, 16, p, 4, 128, 32, p, p, p, null, null, null), "H4t needs"),
        (h, (p, 16, p, p, 16, p, 4, 128, 32, p, p, null, null, odd, null), "16-byte"),
        (h, (p, 16, null, p, 16, p, 4, 128, 32, p, p, null, null, null, null), "X or its scale"),
        (h, (p, 16, p, p, 8, p, 4, 128, 32, p, p, null, null, null, null), "row stride"),
        (h, (p, 16, p, p, 16, p, 1 << 20, 1 << 12, 32, p, p, null, null, null, null), "2 Gi"),
        (d, (p, p, 4, 64, p, p, null, null, null), "I % 128"),
        (d, (p, p, 4, 128, null, null, null, null, null), "give out"),
        (d, (odd, p, 4, 128, p, p, null, null, null), "16-byte"),
        (d, (p, null, 4, 128, p, p, null, null, null), "must be given"),
        (q, (p, 32, 40, p, p, null, null, null), "cols % 32"),
        (q, (p, 32, 12, null, null, p, p, null), "cols % 8"),
        (q, (p, -1, 32, p, p, null, null, null), "negative"),
        (q, (p, 32, 32, null, null, null, null, null), "give out"),
        (q, (p, 32, 32, p, null, null, null, null), "give out"),
        (q, (p, 32, 32, null, null, odd, p, null), "16-byte"),
        (q, (odd, 32, 32, p, p, null, null, null), "16-byte"),
        (q, (null, 32, 32, p, p, null, null, null), "x must be given"),
        (deq, (p, p, 4, 40, p, null), "cols % 32"),
        (deq, (p, null, 4, 32, p, null), "NULL"),
        (deq, (p, p, 4, 32, odd, null), "16-byte"),
        (g, (p, 16, p, p, 16, p, 4, 8, 48, null, p, 0, 8, null, 0, null), "32-element"),
        (g, (p, 16, p, p, 16, p, 4, 9, 32, null, p, 0, 12, null, 0, null), "N % 8"),
        (g, (p, 16, p, p, 16, p, 4, 8, 64, null, p, 0, 8, null, 0, null), "row stride"),
        (g, (p, 24, p, p, 16, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "row stride"),
        (g, (odd, 16, p, p, 16, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "16-byte"),
        (g, (p, 16, ctypes.c_void_p(4098), p, 16, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "planes"),
        (g, (p, 16, null, p, 16, p, 4, 8, 32, null, p, 0, 8, null, 0, null), "NULL"),
        (g, (p, 16, p, p, 16, p, 4, 8, 32, null, p, 2, 8, null, 0, null), "out_dtype"),
        (g, (p, 16, p, p, 16, p, 4, 8, 32, null, p, 0, 8, odd, 64, null), "workspace"),
        (g, (p, 16, p, p, 16, p, 4, 8, 0, null, p, 0, 8, null, 0, null), "K == 0"),
        (g, (p, 1 << 20, p, p, 16, p, 1 << 12, 8, 32, null, p, 0, 8, null, 0, null), "2 GiB"),
        (n, (p, p, 4, 12, p, p, null, 1.0, 1e-6, 1, p, p, null), "cols % 8"),
        (n, (p, p, 4, 16392, p, p, null, 1.0, 1e-6, 1, p, p, null), "16384"),
        (n, (p, null, 4, 16, p, p, null, 1.0, 1e-6, 1, p, p, null), "NULL"),
        (n, (p, p, 4, 16, p, p, odd, 1.0, 1e-6, 1, p, p, null), "16-byte"),
        (b, (p, p, p, p, 0, 16, p, p, null, 1.0, 1e-6, 1, p, p, null, null, null, null, 0, null), "no rows"),
        (b, (p, p, null, null, 4, 16, p, p, null, 1.0, 1e-6, 1, p, p, null, null, null, null, 0, null), "NULL"),
        (b, (p, p, p, p, 4, 16, p, p, null, 1.0, 1e-6, 1, null, null, null, null, null, null, 0, null), "nothing"),
        (b, (p, p, p, p, 4, 16, p, p, null, 1.0, 1e-6, 1, p, p, null, null, p, p, 1 << 20, null), "without a gate"),
        (b, (p, p, p, p, 4, 16, p, p, null, 1.0, 1e-6, 1, p, p, p, null, null, p, 8, null), "workspace of 8 bytes"),
        (b, (p, p, p, p, 4, 16, p, p, null, 1.0, 1e-6, 1, odd, p, p, null, null, p, 8, null), "16-byte"),
    ]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are no memory: the host checks alone")
def test_entries_refuse_before_any_launch():
    L = _lib.lib()
    for fn, args, message in _calls(L):
        assert fn(*args) == 1, (fn.__name__, args)
        told = L.bf8_last_error().decode()
        assert told.startswith(fn.__name__ + ":") and message in told, (message, told)


def test_sizes_of_nothing():
    """Empty calls return without a launch or a pointer; the workspaces of nothing are empty."""
    L = _lib.lib()
    null = ctypes.c_void_p(0)
    p = ctypes.c_void_p(4096)
    assert L.bf8_quantize_mxfp4_bf16(null, 0, 64, p, p, null, null, null) == 0
    assert L.bf8_dequant_mxfp4(null, null, 0, 64, null, null) == 0
    assert L.bf8_gemm_mxfp4(null, 32, null, null, 32, null, 0, 8, 64, null, null, 0, 8, null, 0, null) == 0
    assert L.bf8_rmsnorm_residual_bf16(null, null, 0, 64, null, null, null, 1.0, 1e-6, 1, null, null, null) == 0
    assert L.bf8_gemm_mxfp4_workspace(0, 8, 64) == 0
    assert L.bf8_rmsnorm_residual_bwd_workspace(0, 64) == 0
    assert L.bf8_rmsnorm_residual_bwd_workspace(3, 64) >= 2 * 64 * 4


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["h", "residual", "post_weight", "pre_weight", "gate"])
def test_residual_norm_refuses_forward_mode_tangents(monkeypatch, name, grad):
    """No tangent is dropped: a dual argument is refused, whether gradients are recorded or not, while
    a call that holds none goes through, also beside a level of forward mode."""
    monkeypatch.setattr(ops, "rmsnorm_residual",
                        lambda h, residual, *a, **k: (torch.zeros_like(h), torch.zeros_like(h)))
    args = dict(h=torch.ones(4, 16), residual=torch.ones(4, 16), post_weight=torch.ones(16),
                pre_weight=torch.ones(16), gate=torch.ones(16))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        out, y = fused_mlp.residual_norm(**args)
        assert out.shape == y.shape == (4, 16)
        dual = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(NotImplementedError, match="jvp"):
            fused_mlp.residual_norm(**{**args, name: dual})
    x = args["h"]
    told = torch.func.jvp(lambda t: t + fused_mlp.residual_norm(**args)[0], (x,), (x,))
    assert torch.equal(told[1], x)  # what the transform does not touch is called as ever


def test_residual_norm_refuses_a_scale_that_wants_a_gradient(monkeypatch):
    """The residual's scale is a number, for which no gradient is computed: a tensor that asks for one (or
    holds a tangent) is refused, one that does not is taken as the number it holds."""
    seen = []

    def record(h, residual, *a, residual_scale, **k):
        seen.append(residual_scale)
        return torch.zeros_like(h), torch.zeros_like(h)

    monkeypatch.setattr(ops, "rmsnorm_residual", record)
    h, w = torch.ones(4, 16), torch.ones(16)
    scale = torch.tensor(0.5, requires_grad=True)
    with pytest.raises(ValueError, match="residual_scale"):
        fused_mlp.residual_norm(h, h, w, w, residual_scale=scale)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="residual_scale"):
        dual = forward_ad.make_dual(torch.tensor(0.5), torch.tensor(1.0))
        fused_mlp.residual_norm(h, h, w, w, residual_scale=dual)
    fused_mlp.residual_norm(h, h, w, w, residual_scale=scale.detach())
    with torch.no_grad():
        fused_mlp.residual_norm(h, h, w, w, residual_scale=scale)
    assert seen == [0.5, 0.5]


@pytest.mark.parametrize("tile", ["256x160", "160x256", "128x128", "192x256", "128x64", "64x128", "256x256w8",
                                  "128x128o2", "128x64:3", "256x256w8:2"])
def test_a_named_tile_is_the_plan(monkeypatch, capfd, tile):
    """Every tile of the linear FP4 product can be named (a plan of the planner's own is printed), in as many
    pieces; 256x128 and 256x256 have no such variant."""
    L = _lib.lib()
    M, N, K = 517, 1040, 8224
    monkeypatch.setenv("BONGARD_FP8_GEMM_DEBUG", "1")
    monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", tile)
    pieces = int(tile.partition(":")[2] or 1)
    assert L.bf8_gemm_mxfp4_workspace(M, N, K) == (4 * pieces * M * N if pieces > 1 else 0)
    assert "bf8 plan" not in capfd.readouterr().err
    for none in ("256x128", "256x256"):
        monkeypatch.setenv("BONGARD_FP8_GEMM_TILE", none)
        L.bf8_gemm_mxfp4_workspace(M, N, K)
        assert "bf8 plan gemm mx" in capfd.readouterr().err


def test_oracle_residual_norm_of_hand_worked_rows():
    """Rows whose root mean squares are whole: |h| = 2 and |h| = 3, sums of |4| and |2|; a row of zeros."""
    h = torch.tensor([[2., -2., 2., 2.], [3., 3., -3., 3.], [0., 0., 0., 0.]], dtype=torch.float64)
    post = torch.tensor([0.5, 0.0, 1.0, -0.5], dtype=torch.float64)
    gate = torch.tensor([2.0, 1.0, -1.0, 4.0], dtype=torch.float64)
    pre = torch.tensor([0.0, 1.0, -0.5, -1.0], dtype=torch.float64)
    # normed h times 1 + post and the gate: [3, -1, -2, 2], [3, 1, 2, 2], zeros
    res = torch.tensor([[2., 10., -4., 4.], [-2., -6., -8., 0.], [4., 4., -4., 4.]], dtype=torch.float64)
    out, y = mx4.residual_norm(h, res, post, pre, 1e-300, gate=gate, scale=0.5)
    assert out.tolist() == [[4., 4., -4., 4.], [2., -2., -2., 2.], [2., 2., -2., 2.]]
    assert y.tolist() == [[1., 2., -0.5, 0.]] + [[1., -2., -0.5, 0.], [1., 2., -0.5, 0.]]
    out, y = mx4.residual_norm(h[:2], res[:2], post, pre, 0.0, scale=1.0, z=0.0)
    assert out.tolist() == [[2.5, 10., -3., 3.5], [-1.5, -6., -9., -0.5]]
    r = (out.square().sum(-1, keepdim=True) / 4).sqrt()
    assert torch.allclose(y, out / r * pre, rtol=1e-15, atol=0)
    # eps counts in the mean of squares: a row of ones under eps 3 is halved
    one = torch.ones(1, 4, dtype=torch.float64)
    out, _ = mx4.residual_norm(one, 0 * one, 0 * post, pre, 3.0)
    assert out.tolist() == [[0.5] * 4]


def test_a_call_has_its_workspace_to_itself():
    """Two calls at once (of two threads on one stream, of two graphs) never share one."""
    like = torch.empty(0)
    a, b = ops._call_workspace(1 << 16, like), ops._call_workspace(1 << 16, like)
    assert a[1] == b[1] == a[0].numel() == 1 << 16
    assert a[0].data_ptr() != b[0].data_ptr() and a[0].device == like.device
