"""CPU restatement of the MXFP4 path and of the residual norm (test infrastructure only).

MXFP4 (OCP Microscaling Formats v1.0): blocks of 32 e2m1 codes under an E8M0 scale. The scale here is
the smallest power of two 2^(e - 127) with max|x| <= 6 * 2^(e - 127), e >= 0; a block with inf has
e = 254, with NaN e = 255 and codes 0. Codes round to nearest, ties to the even code, and keep the
sign of what they stand for. Parity unpinned: the reference has no MXFP4 path.
"""

import torch

from . import fp8_oracle as orc


def exponents(x):
    """Biased exponents uint8 [rows, cols / 32] of bf16 x, in integers: amax = 1.f * 2^(E - 127),
    6 = 1.5 * 2^2."""
    key = x.reshape(x.shape[0], -1, 32).view(torch.int16).int() & 0x7FFF
    nan = (key > 0x7F80).any(-1)
    top = key.amax(-1)
    e = ((top >> 7) - 2 + ((top & 0x7F) > 64).int()).clamp(min=0)
    e = torch.where(top == 0x7F80, torch.full_like(e, 254), e)
    return torch.where(nan, torch.full_like(e, 255), e).to(torch.uint8)


def quantize(x, axis=-1):
    """(packed codes uint8 [., . / 2], exponents uint8 [., . / 32]) of bf16 x along ``axis`` (0: the
    copy of x^T, its last block filled up with zeros)."""
    if axis == 0:
        x = x.t().contiguous()
        x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32))
    e = exponents(x)
    scale = torch.ldexp(torch.ones((), dtype=torch.float64), e.int() - 127)
    p = x.double().reshape(*e.shape, 32) / scale[..., None]
    code = torch.where((e == 255)[..., None], torch.zeros_like(p, dtype=torch.uint8),
                       orc.e2m1_code(p)).reshape(x.shape)
    return code[:, ::2] | (code[:, 1::2] << 4), e


def values(packed, e):
    """fp64 values of codes and exponents."""
    codes = torch.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)
    scale = torch.ldexp(torch.ones((), dtype=torch.float64), e.int() - 127)
    scale = torch.where(e == 255, torch.full_like(scale, float("nan")), scale)
    return orc.e2m1_decode(codes).double() * scale.repeat_interleave(32, 1)


def planes(e):
    """int32 [ceil(blocks / 4), rows]: a dword of four blocks' exponents, absent ones 127."""
    e = torch.nn.functional.pad(e, (0, -e.shape[1] % 4), value=127)
    return e.contiguous().view(torch.int32).t().contiguous()


def mm(a, b):
    """(fp64 A @ B^T, sum |a b|) of (packed, exponents) operands."""
    a, b = values(*a), values(*b)
    return a @ b.t(), a.abs() @ b.abs().t()


def residual_norm(h, res, post, pre, eps, gate=None, scale=1.0, z=1.0):
    """out and y in the inputs' precision, y from out as it is."""
    def norm(x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (z + w)

    n = norm(h, post)
    out = scale * res + (n if gate is None else n * gate)
    return out, norm(out, pre)
