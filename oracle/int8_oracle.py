"""CPU restatement of the 8-bit integer formats and the layer norm in 64 bits (test infrastructure only)."""

import torch

FLOOR = 2.0 ** -40


def _nearest_even(n, d):
    """n / d to the nearest integer, ties to even, of whole numbers given in float64 (exact below 2^53):
    by the remainder, so that no quotient is rounded."""
    q = torch.floor(n / d)
    r = n - q * d
    q = torch.where(r < 0, q - 1, torch.where(r >= d, q + 1, q))
    r = n - q * d
    up = (2 * r > d) | ((2 * r == d) & (q % 2 != 0))
    return torch.where(up, q + 1, q)


def quantize(x, dim=-1):
    """(codes int8, scales fp32) of bf16 x [rows, cols], one scale a row, or with dim 0 one a column (the
    copy transposed and filled up with zeros to whole 16)."""
    x = x.double()
    if dim == 0:
        x = torch.nn.functional.pad(x.t(), (0, (-x.shape[0]) % 16))
    amax = x.abs().amax(-1, keepdim=True) if x.shape[1] else x.new_zeros(x.shape[0], 1)
    bad = ~torch.isfinite(amax)
    a = torch.where(bad, torch.ones_like(amax), amax.clamp(min=FLOOR))
    x = torch.where(bad, torch.zeros_like(x), x)
    # both are 8-bit significands (a power of two at the least) times powers of two: over 2^(k - 60), with
    # 2^k about a, the two are whole numbers, and what lies below is far under half a code
    k = torch.frexp(a)[1].long()
    unit = ((k - 60 + 1023) << 52).view(torch.float64)
    codes = _nearest_even((x * 127 / unit).round(), a / unit)
    scale = (a / 127).float()
    scale[bad] = float("nan")
    return codes.to(torch.int8), scale.flatten()


def values(codes, scale):
    return codes.double() * scale.double()[:, None]


def mm(a, b):
    """(product, sum of magnitudes) of two quantized operands in 64 bits (whole sums, exact)."""
    s = a[1].double()[:, None] * b[1].double()
    x, y = a[0].double(), b[0].double()
    return (x @ y.t()) * s, (x.abs() @ y.abs().t()) * s


def checkpoint(x):
    """(codes int8 [rows, cols], exponents uint8 [rows, blocks]) of bf16 x."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.double(), (0, (-cols) % 32)).reshape(rows, -1, 32)
    amax = b.abs().amax(-1)
    e = torch.full(amax.shape, 7, dtype=torch.long)
    for k in range(8, 255):  # the least 2^(k - 133) within whose 127 steps the block's largest lies
        e[amax > 127 * 2.0 ** (k - 1 - 133)] = k
    e[~torch.isfinite(amax)] = 255
    step = torch.ldexp(torch.ones((), dtype=torch.float64), (e - 133))[..., None]
    codes = torch.round(torch.nan_to_num(b / step, 0.0, 0.0, 0.0)).clamp(-127, 127)
    codes[e == 255] = 0
    return codes.reshape(rows, -1)[:, :cols].to(torch.int8), e.to(torch.uint8)


def restored(codes, e):
    rows, cols = codes.shape
    step = torch.ldexp(torch.ones((), dtype=torch.float64), e.long() - 133)
    step[e == 255] = float("nan")
    return codes.double() * step.repeat_interleave(32, 1)[:, :cols]


def layer_norm(x, weight, bias, eps, held=None):
    """(y, n, mean, sd) in 64 bits; n of the values `held` (x's own where None)."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    sd = ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    y = (x - mean) / sd * weight.double() + (0 if bias is None else bias.double())
    return y, ((x if held is None else held) - mean) / sd, mean, sd


def layer_norm_backward(n, sd, dy, weight):
    """(dx, dweight, dbias) in 64 bits."""
    dy = dy.double()
    c = dy * weight.double()
    dx = (c - c.mean(-1, keepdim=True) - n * (c * n).mean(-1, keepdim=True)) / sd
    return dx, (dy * n).sum(0), dy.sum(0)
