"""Tensor-level FP8 ops on top of libbongard_fp8.so (gfx950 HIP kernels).

Every op runs on the caller's current HIP stream, allocates its outputs with PyTorch's
caching allocator, and never synchronises with the host. Inputs must be CUDA (HIP)
tensors; there is no CPU path.

Quantized tensors are returned as :class:`Fp8Tensor`: fp8 payload(s) plus a 4-float
device "meta" record ``{amax, scale, scale_inv, 0}`` with
``scale = fp32(fp8_max / max(f64(amax), 1e-12))`` and ``q = fp8(clamp(x * scale))``,
the semantics of torchao's tensorwise recipe (tensor_to_amax / amax_to_scale /
to_fp8_saturated) behind bongard/float8_training.py:22 and of TE's
Float8CurrentScaling behind bongard/te_linear.py:38-39,73-74.
"""

import ctypes
import functools
import os
from dataclasses import dataclass, field
from typing import Optional, Sequence

import torch

from . import _lib

E4M3 = 0
E5M2 = 1
FP8_MAX = {E4M3: 448.0, E5M2: 57344.0}
TORCH_FP8 = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}
OUT_BF16 = 0
OUT_F32 = 1
SCALE_POW2 = 0x10  # OR'ed into fmt: round the scale down to a power of two


@dataclass
class Fp8Tensor:
    """A per-tensor-scaled FP8 tensor: ``data`` [rows, cols] and/or ``data_t`` [cols, rows]."""

    data: Optional[torch.Tensor]
    data_t: Optional[torch.Tensor]
    meta: torch.Tensor  # float32 [4] (or a view into a larger buffer)
    fmt: int
    rows: int
    cols: int

    @property
    def scale(self):
        return self.meta[1]

    @property
    def scale_inv(self):
        return self.meta[2]

    @property
    def amax(self):
        return self.meta[0]


# Host cost matters at small shapes (eager forwards of a few microseconds of GPU work):
# pointers and streams go to the C ABI as plain integers (ctypes converts them for the
# void* parameters), the current stream is read through torch's raw-handle accessor, and
# the plan-dependent counts are cached per shape.
def _ptr(t):
    return t.data_ptr() if t is not None else None


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _dev_index(device=None):
    if device is None:
        return torch.cuda.current_device()
    if not isinstance(device, torch.device):
        device = torch.device(device)
    return device.index if device.index is not None else torch.cuda.current_device()


def _stream(device=None):
    """The caller's current HIP stream on ``device`` as an integer handle."""
    idx = _dev_index(device)
    if _raw_stream is not None:
        return _raw_stream(idx)
    return torch.cuda.current_stream(idx).cuda_stream


def _stream_key(device):
    idx = _dev_index(device)
    return idx, _stream(idx)


def _tile_override():
    # the GEMM planner reads this variable on every call; cached counts follow it
    return os.environ.get("BONGARD_FP8_GEMM_TILE", "")


@functools.lru_cache(maxsize=4096)
def _amax_partials_cached(n):
    return int(_lib.lib().bf8_amax_partials(n))


@functools.lru_cache(maxsize=4096)
def _many_partials_cached(sizes):
    return int(_lib.lib().bf8_quantize_many_partials(
        len(sizes), (ctypes.c_int64 * len(sizes))(*sizes)))


@functools.lru_cache(maxsize=4096)
def _gemm_ws_cached(M, N, K, override):
    return int(_lib.lib().bf8_gemm_workspace(M, N, K))


@functools.lru_cache(maxsize=4096)
def _geglu_partials_cached(M, I, override):
    return int(_lib.lib().bf8_geglu_partials(M, I))


def _require_gpu(*tensors):
    for t in tensors:
        if t is not None and t.device.type != "cuda":
            raise RuntimeError("bongard_amd FP8 ops need tensors on the HIP device (no CPU path)")


def _byte_matrix(who, **tensors):
    """FP8 payloads and E8M0 scale arrays reach the kernels as row-major byte matrices
    (row stride = stride(0), elements contiguous within a row): reject anything else
    rather than let the kernel read a transposed view's bytes in the wrong order."""
    for name, t in tensors.items():
        if t is None:
            continue
        if t.dim() != 2 or t.element_size() != 1 or (t.shape[1] > 1 and t.stride(1) != 1):
            raise ValueError(f"{who}: {name} must be a 2-D one-byte tensor with contiguous rows "
                             f"(got {t.dtype} {tuple(t.shape)} strides {t.stride()})")


def _out_matrix(who, out, shape, dtype):
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or (shape[1] > 1 and out.stride(1) != 1):
        raise ValueError(f"{who}: out must be {dtype} {tuple(shape)} with contiguous rows")


def _check_cast_outputs(who, out, out_t, rows, cols):
    """Caller-supplied cast outputs: contiguous one-byte [rows, cols] / [cols, rows]."""
    for name, t, shape in (("out", out, (rows, cols)), ("out_t", out_t, (cols, rows))):
        if t is not None and (tuple(t.shape) != shape or t.element_size() != 1
                              or not t.is_contiguous()):
            raise ValueError(f"{who}: {name} must be a contiguous one-byte tensor of shape "
                             f"{shape} (got {t.dtype} {tuple(t.shape)})")


def _gu_operand(who, GU, M, I):
    """The forward's saved [gate | up] pre-activations: bf16 [M, 2I], contiguous."""
    if GU.dtype != torch.bfloat16 or tuple(GU.shape) != (M, 2 * I):
        raise ValueError(f"{who}: GU must be bf16 [{M}, {2 * I}] (got {GU.dtype} {tuple(GU.shape)})")
    return GU.contiguous()


def _bf16_2d(x):
    if x.dtype != torch.bfloat16:
        raise TypeError(f"expected a bfloat16 tensor, got {x.dtype}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if not x.is_contiguous():
        x = x.contiguous()
    return x


def amax_partials_count(n):
    return _amax_partials_cached(int(n))


def new_meta(device, count=1):
    """Uninitialised meta record(s): float32 [count, 4] (or [4] when count == 1); the
    kernels that produce a meta write all four words."""
    return torch.empty((count, 4) if count > 1 else (4,), dtype=torch.float32, device=device)


# Per-(device, stream) scratch for amax partials, reused in stream order.
_PARTIALS = {}


def partials_buffer(count, device):
    key = _stream_key(device)
    buf = _PARTIALS.get(key)
    if buf is None or buf.numel() < count:
        buf = torch.empty(max(int(count), 4096), dtype=torch.int32, device=device)
        _PARTIALS[key] = buf
    return buf


# Per-(device, stream) split-K workspace of bf8_gemm (fp32 partial sums), reused in
# stream order.
_GEMM_WS = {}


def gemm_workspace(nbytes, device):
    key = _stream_key(device)
    buf = _GEMM_WS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=device)
        _GEMM_WS[key] = buf
    return buf


def quantize(x, fmt=E4M3, *, rowwise=True, transpose=False, meta=None, out=None, out_t=None,
             pow2=False):
    """Current-scaling quantization of a bf16 tensor (flattened to 2-D [rows, cols]).

    Returns an :class:`Fp8Tensor` whose ``data`` is [rows, cols] (if ``rowwise``) and
    ``data_t`` [cols, rows] (if ``transpose``), both as torch float8 tensors. ``pow2``
    rounds the scale down to a power of two (torchao round_scales_to_power_of_2).
    """
    _require_gpu(x)
    x = _bf16_2d(x)
    rows, cols = x.shape
    dev = x.device
    if meta is None:
        meta = new_meta(dev)
    if rowwise and out is None:
        out = torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=dev)
    if transpose and out_t is None:
        out_t = torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=dev)
    _check_cast_outputs("quantize", out if rowwise else None, out_t if transpose else None,
                        rows, cols)
    L = _lib.lib()
    parts = partials_buffer(_amax_partials_cached(rows * cols), dev)
    _lib.check(L.bf8_quantize_bf16(_ptr(x), rows, cols, fmt | (SCALE_POW2 if pow2 else 0),
                                   _ptr(out if rowwise else None),
                                   _ptr(out_t if transpose else None), _ptr(meta),
                                   _ptr(parts), _stream(dev)), "bf8_quantize_bf16")
    return Fp8Tensor(out if rowwise else None, out_t if transpose else None, meta, fmt, rows, cols)


def quantize_many(xs, fmts=None, *, pow2=False, metas=None):
    """:func:`quantize` (rowwise output, current scaling) of up to 8 bf16 tensors in two
    launches: one amax pass over all of them, one cast pass. Each result equals that
    tensor's own ``quantize(x, fmt, pow2=pow2)``, bytes and meta. ``fmts``: one format
    for all tensors or one per tensor (default e4m3); ``metas``: optional meta rows to
    write (as ``quantize(meta=...)``)."""
    xs = [_bf16_2d(x) for x in xs]
    count = len(xs)
    if not 1 <= count <= 8:
        raise ValueError(f"quantize_many: {count} tensors (1 to 8 supported)")
    _require_gpu(*xs)
    dev = xs[0].device
    if any(x.device != dev for x in xs):
        raise ValueError("quantize_many: tensors on different devices")
    if fmts is None or isinstance(fmts, int):
        fmts = [E4M3 if fmts is None else fmts] * count
    if len(fmts) != count:
        raise ValueError("quantize_many: one format per tensor")
    if metas is None:
        metas = new_meta(dev, count).unbind(0) if count > 1 else (new_meta(dev),)
    outs = [torch.empty(x.shape, dtype=TORCH_FP8[f], device=dev) for x, f in zip(xs, fmts)]
    L = _lib.lib()
    sizes = tuple(x.numel() for x in xs)
    n = (ctypes.c_int64 * count)(*sizes)
    parts = partials_buffer(max(1, _many_partials_cached(sizes)), dev)
    flag = SCALE_POW2 if pow2 else 0
    _lib.check(L.bf8_quantize_many_bf16(
        count, (ctypes.c_void_p * count)(*[x.data_ptr() for x in xs]), n,
        (ctypes.c_int * count)(*[f | flag for f in fmts]),
        (ctypes.c_void_p * count)(*[o.data_ptr() for o in outs]),
        (ctypes.c_void_p * count)(*[m.data_ptr() for m in metas]), _ptr(parts), _stream(dev)),
        "bf8_quantize_many_bf16")
    return [Fp8Tensor(o, None, m, f, x.shape[0], x.shape[1])
            for x, o, m, f in zip(xs, outs, metas, fmts)]


def amax(x):
    """Per-block partial amax keys (int32 view of fp32 bits) of a bf16 tensor."""
    _require_gpu(x)
    x = _bf16_2d(x)
    partials = torch.empty(amax_partials_count(x.numel()), dtype=torch.int32, device=x.device)
    _lib.check(_lib.lib().bf8_amax_bf16(_ptr(x), x.numel(), _ptr(partials), _stream(x.device)),
               "bf8_amax_bf16")
    return partials


def scale_from_partials(partials, fmt, meta=None):
    if meta is None:
        meta = new_meta(partials.device)
    _lib.check(_lib.lib().bf8_scale_from_partials(_ptr(partials), partials.numel(), fmt,
                                                  _ptr(meta), _stream(partials.device)),
               "bf8_scale_from_partials")
    return meta


def cast_partials(x, partials, fmt=E4M3, *, rowwise=True, transpose=False):
    """Cast whose scale comes from amax partials (as returned by ``gemm_geglu`` /
    ``geglu_bwd``); returns the Fp8Tensor with its freshly written meta."""
    _require_gpu(x, partials)
    x = _bf16_2d(x)
    rows, cols = x.shape
    meta = new_meta(x.device)
    out = torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=x.device) if rowwise else None
    out_t = torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=x.device) if transpose else None
    _lib.check(_lib.lib().bf8_cast_partials_bf16(_ptr(x), rows, cols, _ptr(partials),
                                                 partials.numel(), fmt, _ptr(meta), _ptr(out),
                                                 _ptr(out_t), _stream(x.device)),
               "bf8_cast_partials_bf16")
    return Fp8Tensor(out, out_t, meta, fmt, rows, cols)


def cast(x, meta, fmt=E4M3, *, rowwise=True, transpose=False, out=None, out_t=None):
    """Cast with an existing scale (``meta[1]``), e.g. delayed scaling."""
    _require_gpu(x, meta)
    x = _bf16_2d(x)
    rows, cols = x.shape
    if rowwise and out is None:
        out = torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=x.device)
    if transpose and out_t is None:
        out_t = torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=x.device)
    _check_cast_outputs("cast", out if rowwise else None, out_t if transpose else None,
                        rows, cols)
    scale_ptr = ctypes.c_void_p(meta.data_ptr() + 4)
    _lib.check(_lib.lib().bf8_cast_bf16(_ptr(x), rows, cols, scale_ptr, fmt,
                                        _ptr(out if rowwise else None),
                                        _ptr(out_t if transpose else None), _stream(x.device)),
               "bf8_cast_bf16")
    return Fp8Tensor(out if rowwise else None, out_t if transpose else None, meta, fmt, rows, cols)


def _sinv_ptr(meta):
    return meta.data_ptr() + 8


def gemm(a, a_fmt, a_meta, b, b_fmt, b_meta, *, out_dtype=torch.bfloat16, bias=None,
         seg_ends: Optional[Sequence[int]] = None, b_meta_stride=4, out=None):
    """``C = (a @ b.T) * a_scale_inv * b_scale_inv (+ bias)`` on fp8 operands.

    a: fp8 [M, K], b: fp8 [N, K] (row-major, K contiguous). ``b_meta`` is the meta of b,
    or for ``seg_ends`` (fused projections) the first of ``len(seg_ends)`` meta records
    ``b_meta_stride`` floats apart.
    """
    _require_gpu(a, b, a_meta, b_meta)
    _byte_matrix("gemm", a=a, b=b)
    M, K = a.shape
    N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"gemm: inner dims differ ({K} vs {Kb})")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("gemm: out_dtype must be bfloat16 or float32")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    _out_matrix("gemm", out, (M, N), out_dtype)
    n_seg = 1
    seg = None
    if seg_ends is not None:
        n_seg = len(seg_ends)
        seg = (ctypes.c_int64 * n_seg)(*[int(s) for s in seg_ends])
    if bias is not None:
        if bias.dtype != torch.bfloat16:
            raise TypeError("gemm: bias must be bfloat16")
        bias = bias.contiguous()
    L = _lib.lib()
    ws_bytes = _gemm_ws_cached(M, N, K, _tile_override())
    ws = gemm_workspace(ws_bytes, a.device) if ws_bytes else None
    ws_bytes = ws.numel() if ws is not None else 0
    _lib.check(L.bf8_gemm(_ptr(a), a_fmt, a.stride(0), _ptr(b), b_fmt, b.stride(0), M, N, K,
                          _sinv_ptr(a_meta), _sinv_ptr(b_meta), b_meta_stride, seg, n_seg,
                          _ptr(bias), _ptr(out), OUT_BF16 if out_dtype == torch.bfloat16 else OUT_F32,
                          out.stride(0), _ptr(ws), ws_bytes, _stream(a.device)), "bf8_gemm")
    return out


@functools.lru_cache(maxsize=256)
def _gemm_kmajor_ws_cached(M, N, K, override):
    return int(_lib.lib().bf8_gemm_kmajor_workspace(M, N, K))


def gemm_kmajor(a, a_fmt, a_meta, b_t, b_fmt, b_meta, *, a_kmajor=False,
                out_dtype=torch.bfloat16, out=None, accumulate=False):
    """:func:`gemm` with B given as ``b_t`` = B^T [K, N] (and, when ``a_kmajor``, A as ``a``
    = A^T [K, M]): the backward's dgrad and wgrad GEMMs on the fp8 tensors as their
    producers wrote them, no transposed copies (bf8_gemm_kmajor; e5m2 x e4m3). Same
    products and fp32 sums as :func:`gemm` on the transposed operands. ``accumulate``: the
    bf16 result is added to ``out`` (one rounding of the sum of the two bf16 values, as
    ``out + result`` rounds it)."""
    _require_gpu(a, b_t, a_meta, b_meta)
    _byte_matrix("gemm_kmajor", a=a, b_t=b_t)
    if a_kmajor:
        K, M = a.shape
    else:
        M, K = a.shape
    Kb, N = b_t.shape
    if K != Kb:
        raise ValueError(f"gemm_kmajor: inner dims differ ({K} vs {Kb})")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("gemm_kmajor: out_dtype must be bfloat16 or float32")
    if accumulate and (out is None or out_dtype != torch.bfloat16):
        raise ValueError("gemm_kmajor: accumulate needs a bfloat16 out")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    _out_matrix("gemm_kmajor", out, (M, N), out_dtype)
    ws_bytes = _gemm_kmajor_ws_cached(M, N, K, _tile_override())
    ws = gemm_workspace(ws_bytes, a.device) if ws_bytes else None
    ws_bytes = ws.numel() if ws is not None else 0
    L = _lib.lib()
    entry = L.bf8_gemm_kmajor_add if accumulate else L.bf8_gemm_kmajor
    _lib.check(entry(
        _ptr(a), a_fmt, a.stride(0), int(bool(a_kmajor)), _ptr(b_t), b_fmt, b_t.stride(0), M, N,
        K, _sinv_ptr(a_meta), _sinv_ptr(b_meta), _ptr(out),
        OUT_BF16 if out_dtype == torch.bfloat16 else OUT_F32, out.stride(0), _ptr(ws), ws_bytes,
        _stream(a.device)), "bf8_gemm_kmajor")
    return out


@dataclass
class AxisFp8Tensor:
    """An axiswise-scaled FP8 tensor (torchao AXISWISE granularity) of x [rows, cols]:
    ``data`` [rows, cols] with one scale per row (``row_sinv`` fp32 [rows], the inverse
    scales) and/or ``data_t`` [cols, rows] with one scale per column of x (``col_sinv``
    fp32 [cols])."""

    data: Optional[torch.Tensor]
    row_sinv: Optional[torch.Tensor]
    data_t: Optional[torch.Tensor]
    col_sinv: Optional[torch.Tensor]
    fmt: int
    rows: int
    cols: int


_AXIS_WS = {}


def quantize_axiswise(x, fmt=E4M3, *, rowwise=True, colwise=False, pow2=True):
    """Per-row (``rowwise``, torchao axiswise_dim=-1) and/or per-column (``colwise``,
    axiswise_dim=0, stored transposed) quantization of a bf16 tensor; ``pow2`` rounds the
    scales down to powers of two as torchao's rowwise recipes do."""
    _require_gpu(x)
    x = _bf16_2d(x)
    rows, cols = x.shape
    dev = x.device
    if not (rowwise or colwise):
        raise ValueError("quantize_axiswise: nothing requested")
    out = torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=dev) if rowwise else None
    rs = torch.empty(rows, dtype=torch.float32, device=dev) if rowwise else None
    out_t = torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=dev) if colwise else None
    cs = torch.empty(cols, dtype=torch.float32, device=dev) if colwise else None
    L = _lib.lib()
    ws, nbytes = None, 0
    if colwise:
        nbytes = int(L.bf8_axiswise_workspace(rows, cols))
        key = _stream_key(dev)
        ws = _AXIS_WS.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
            _AXIS_WS[key] = ws
        nbytes = ws.numel()
    _lib.check(L.bf8_quantize_axiswise_bf16(_ptr(x), rows, cols, fmt | (SCALE_POW2 if pow2 else 0),
                                            _ptr(out), _ptr(rs), _ptr(out_t), _ptr(cs), _ptr(ws),
                                            nbytes, _stream(dev)), "bf8_quantize_axiswise_bf16")
    return AxisFp8Tensor(out, rs, out_t, cs, fmt, rows, cols)


def gemm_axiswise(a, a_fmt, a_sinv, b, b_fmt, b_sinv, *, out_dtype=torch.bfloat16, bias=None,
                  out=None):
    """``C[m, n] = (a @ b.T)[m, n] * a_sinv[m] * b_sinv[n] (+ bias[n])`` on fp8 operands.

    a: fp8 [M, K], b: fp8 [N, K]. ``a_sinv`` is fp32 [M] (one inverse scale per row of a)
    or a single value (1-element tensor, e.g. a meta's ``scale_inv``); likewise ``b_sinv``
    with [N]."""
    _require_gpu(a, b, a_sinv, b_sinv)
    _byte_matrix("gemm_axiswise", a=a, b=b)
    M, K = a.shape
    N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"gemm_axiswise: inner dims differ ({K} vs {Kb})")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("gemm_axiswise: out_dtype must be bfloat16 or float32")

    def vec_flag(sv, n, what):
        if sv.dtype != torch.float32 or not sv.is_contiguous():
            raise TypeError(f"gemm_axiswise: {what} must be contiguous float32")
        if sv.numel() == n and n != 1:
            return 1
        if sv.numel() == 1:
            return 0
        raise ValueError(f"gemm_axiswise: {what} must have 1 or {n} elements")

    a_vec = vec_flag(a_sinv, M, "a_sinv")
    b_vec = vec_flag(b_sinv, N, "b_sinv")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    _out_matrix("gemm_axiswise", out, (M, N), out_dtype)
    if bias is not None:
        if bias.dtype != torch.bfloat16:
            raise TypeError("gemm_axiswise: bias must be bfloat16")
        bias = bias.contiguous()
    L = _lib.lib()
    ws_bytes = _gemm_ws_cached(M, N, K, _tile_override())
    ws = gemm_workspace(ws_bytes, a.device) if ws_bytes else None
    ws_bytes = ws.numel() if ws is not None else 0
    _lib.check(L.bf8_gemm_axiswise(_ptr(a), a_fmt, a.stride(0), _ptr(b), b_fmt, b.stride(0), M, N,
                                   K, _ptr(a_sinv), a_vec, _ptr(b_sinv), b_vec, _ptr(bias),
                                   _ptr(out), OUT_BF16 if out_dtype == torch.bfloat16 else OUT_F32,
                                   out.stride(0), _ptr(ws), ws_bytes, _stream(a.device)),
               "bf8_gemm_axiswise")
    return out


@dataclass
class MxFp8Tensor:
    """An MXFP8 tensor of x [rows, cols] (32-element blocks, one E8M0 byte each):
    ``data`` [rows, cols] with ``scales`` [rows, mx_scale_ld(cols)] (blocks along rows)
    and/or ``data_t`` [cols, rows] with ``scales_t`` [cols, mx_scale_ld(rows)] (blocks along
    columns of x, stored transposed). ``planes`` int32 [ceil(cols / 128), rows] and
    ``planes_t`` [ceil(rows / 128), cols] hold the same scales as one plane of dwords per 128
    K-values, which the GEMMs load in whole lines (``gemm_mx(..., a_planes=, b_planes=)``)."""

    data: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]
    data_t: Optional[torch.Tensor]
    scales_t: Optional[torch.Tensor]
    fmt: int
    rows: int
    cols: int
    planes: Optional[torch.Tensor] = None
    planes_t: Optional[torch.Tensor] = None

    def scale_planes(self, transpose=False):
        """``planes`` (``planes_t``), made from the scale rows for a tensor that has only
        those, as one put together from bf8_quantize_mx_bf16's outputs does; None without a
        copy of that direction."""
        planes, scales = ((self.planes_t, self.scales_t) if transpose
                          else (self.planes, self.scales))
        if planes is not None or scales is None:
            return planes
        ld = mx_scale_ld(self.rows if transpose else self.cols)
        return scales[:, :ld].contiguous().view(torch.int32).t().contiguous()


def mx_scale_ld(K):
    return (int(K) + 127) // 128 * 4


def _new_planes(K, rows, device):
    """Scale planes of an operand [rows, K]."""
    return torch.empty(((K + 127) // 128, rows), dtype=torch.int32, device=device)


def _mx_planes(who, rows, K, **planes):
    for name, t in planes.items():
        if t.dtype != torch.int32 or tuple(t.shape) != ((K + 127) // 128, rows[name]) \
                or not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be contiguous int32 "
                             f"[{(K + 127) // 128}, {rows[name]}] (got {t.dtype} {tuple(t.shape)})")


def quantize_mx(x, fmt=E4M3, *, rowwise=True, colwise=False, scale_rows=True):
    """MXFP8 quantization of a bf16 tensor (TE MXFP8BlockScaling arithmetic). ``scale_rows``
    False: the scales as planes only (``scales`` and ``scales_t`` None), for a tensor that
    only feeds the GEMMs."""
    _require_gpu(x)
    x = _bf16_2d(x)
    rows, cols = x.shape
    dev = x.device
    if not (rowwise or colwise):
        raise ValueError("quantize_mx: nothing requested")
    out = sc = pl = out_t = sc_t = pl_t = None
    if rowwise:
        out = torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=dev)
        if scale_rows:
            sc = torch.empty((rows, mx_scale_ld(cols)), dtype=torch.uint8, device=dev)
        pl = _new_planes(cols, rows, dev)
    if colwise:
        out_t = torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=dev)
        if scale_rows:
            sc_t = torch.empty((cols, mx_scale_ld(rows)), dtype=torch.uint8, device=dev)
        pl_t = _new_planes(rows, cols, dev)
    _lib.check(_lib.lib().bf8_quantize_mx_planes_bf16(
        _ptr(x), rows, cols, fmt, _ptr(out), _ptr(sc), _ptr(pl), _ptr(out_t), _ptr(sc_t),
        _ptr(pl_t), _stream(dev)), "bf8_quantize_mx_planes_bf16")
    return MxFp8Tensor(out, sc, out_t, sc_t, fmt, rows, cols, pl, pl_t)


def geglu_bwd_mx(dH, GU, fmt=E4M3, *, rowwise=True, colwise=False):
    """:func:`geglu_bwd` and the :func:`quantize_mx` of its dGU [M, 2I] in one pass (planes
    only, the same bytes and scales; the bf16 dGU is not written). I must be a multiple of 128."""
    _require_gpu(dH, GU)
    dH = dH.contiguous()
    M, I = dH.shape
    GU = _gu_operand("geglu_bwd_mx", GU, M, I)
    dev = dH.device
    if not (rowwise or colwise):
        raise ValueError("geglu_bwd_mx: nothing requested")
    out = pl = out_t = pl_t = None
    if rowwise:
        out = torch.empty((M, 2 * I), dtype=TORCH_FP8[fmt], device=dev)
        pl = _new_planes(2 * I, M, dev)
    if colwise:
        out_t = torch.empty((2 * I, M), dtype=TORCH_FP8[fmt], device=dev)
        pl_t = _new_planes(M, 2 * I, dev)
    _lib.check(_lib.lib().bf8_geglu_bwd_mx_planes(
        _ptr(dH), _ptr(GU), M, I, fmt, _ptr(out), _ptr(pl), _ptr(out_t), _ptr(pl_t),
        _stream(dev)), "bf8_geglu_bwd_mx_planes")
    return MxFp8Tensor(out, None, out_t, None, fmt, M, 2 * I, pl, pl_t)


def quantize_mx_many(xs, fmts=None, *, scale_rows=True):
    """Rowwise :func:`quantize_mx` of up to 8 bf16 tensors in one launch; each result
    equals that tensor's own ``quantize_mx(x, fmt)`` (bytes and scales). ``fmts``: one
    format for all or one per tensor (default e4m3)."""
    xs = [_bf16_2d(x) for x in xs]
    count = len(xs)
    if not 1 <= count <= 8:
        raise ValueError(f"quantize_mx_many: {count} tensors (1 to 8 supported)")
    _require_gpu(*xs)
    dev = xs[0].device
    if any(x.device != dev for x in xs):
        raise ValueError("quantize_mx_many: tensors on different devices")
    if fmts is None or isinstance(fmts, int):
        fmts = [E4M3 if fmts is None else fmts] * count
    if len(fmts) != count:
        raise ValueError("quantize_mx_many: one format per tensor")
    outs = [torch.empty(x.shape, dtype=TORCH_FP8[f], device=dev) for x, f in zip(xs, fmts)]
    scs = [torch.empty((x.shape[0], mx_scale_ld(x.shape[1])), dtype=torch.uint8, device=dev)
           if scale_rows else None for x in xs]
    pls = [_new_planes(x.shape[1], x.shape[0], dev) for x in xs]
    _lib.check(_lib.lib().bf8_quantize_mx_many_planes_bf16(
        count, (ctypes.c_void_p * count)(*[x.data_ptr() for x in xs]),
        (ctypes.c_int64 * count)(*[x.shape[0] for x in xs]),
        (ctypes.c_int64 * count)(*[x.shape[1] for x in xs]), (ctypes.c_int * count)(*fmts),
        (ctypes.c_void_p * count)(*[o.data_ptr() for o in outs]),
        (ctypes.c_void_p * count)(*[_ptr(c) for c in scs]),
        (ctypes.c_void_p * count)(*[c.data_ptr() for c in pls]), _stream(dev)),
        "bf8_quantize_mx_many_planes_bf16")
    return [MxFp8Tensor(o, c, None, None, f, x.shape[0], x.shape[1], pl)
            for x, o, c, f, pl in zip(xs, outs, scs, fmts, pls)]


@functools.lru_cache(maxsize=4096)
def _gemm_mx_ws_cached(M, N, K, override):
    return int(_lib.lib().bf8_gemm_mx_workspace(M, N, K))


def gemm_mx(a, a_scales, b, b_scales, *, out_dtype=torch.bfloat16, bias=None, out=None,
            a_planes=None, b_planes=None):
    """``C = a @ b.T`` on MXFP8 (e4m3) operands a [M, K], b [N, K] with their E8M0 block
    scales [M, >= mx_scale_ld(K)], [N, ...], or with both operands' scale planes (the scale
    rows are then not read and may be None; the same result, faster)."""
    by_planes = a_planes is not None and b_planes is not None
    if by_planes:
        _require_gpu(a, b, a_planes, b_planes)
        _byte_matrix("gemm_mx", a=a, b=b)
    else:
        _require_gpu(a, b, a_scales, b_scales)
        _byte_matrix("gemm_mx", a=a, b=b, a_scales=a_scales, b_scales=b_scales)
    M, K = a.shape
    N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"gemm_mx: inner dims differ ({K} vs {Kb})")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("gemm_mx: out_dtype must be bfloat16 or float32")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    _out_matrix("gemm_mx", out, (M, N), out_dtype)
    if bias is not None:
        if bias.dtype != torch.bfloat16:
            raise TypeError("gemm_mx: bias must be bfloat16")
        bias = bias.contiguous()
    L = _lib.lib()
    ws_bytes = _gemm_mx_ws_cached(M, N, K, _tile_override())
    ws = gemm_workspace(ws_bytes, a.device) if ws_bytes else None
    ws_bytes = ws.numel() if ws is not None else 0
    if by_planes:
        _mx_planes("gemm_mx", {"a_planes": M, "b_planes": N}, K, a_planes=a_planes,
                   b_planes=b_planes)
        _lib.check(L.bf8_gemm_mx_planes(
            _ptr(a), a.stride(0), _ptr(a_planes), _ptr(b), b.stride(0), _ptr(b_planes), M, N, K,
            _ptr(bias), _ptr(out), OUT_BF16 if out_dtype == torch.bfloat16 else OUT_F32,
            out.stride(0), _ptr(ws), ws_bytes, _stream(a.device)), "bf8_gemm_mx_planes")
        return out
    _lib.check(L.bf8_gemm_mx(_ptr(a), a.stride(0), _ptr(a_scales), a_scales.stride(0), _ptr(b),
                             b.stride(0), _ptr(b_scales), b_scales.stride(0), M, N, K, _ptr(bias),
                             _ptr(out), OUT_BF16 if out_dtype == torch.bfloat16 else OUT_F32,
                             out.stride(0), _ptr(ws), ws_bytes, _stream(a.device)), "bf8_gemm_mx")
    return out


def gemm_geglu_mx(x8, x_scales, w8, w_scales, intermediate, *, keep_gu=False):
    """Gate/up GEMM + gated GELU on MXFP8 operands; returns ``(H bf16 [M, I], GU or None)``."""
    _require_gpu(x8, x_scales, w8, w_scales)
    _byte_matrix("gemm_geglu_mx", x8=x8, w8=w8, x_scales=x_scales, w_scales=w_scales)
    M, K = x8.shape
    I = int(intermediate)
    if w8.shape != (2 * I, K):
        raise ValueError(f"gemm_geglu_mx: W must be [{2 * I}, {K}]")
    H = torch.empty((M, I), dtype=torch.bfloat16, device=x8.device)
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=x8.device) if keep_gu else None
    _lib.check(_lib.lib().bf8_gemm_geglu_mx(_ptr(x8), x8.stride(0), _ptr(x_scales),
                                            x_scales.stride(0), _ptr(w8), w8.stride(0),
                                            _ptr(w_scales), w_scales.stride(0), M, I, K, _ptr(H),
                                            H.stride(0), _ptr(GU), _stream(x8.device)),
               "bf8_gemm_geglu_mx")
    return H, GU


def gemm_geglu_mx_quant(x8, x_scales, w8, w_scales, intermediate, *, colwise=False,
                        keep_gu=False, keep_h=False):
    """:func:`gemm_geglu_mx` with H's MXFP8 (e4m3) quantization done in the GEMM epilogue.

    Returns ``(hq, GU or None, H or None)``: ``hq`` an :class:`MxFp8Tensor` of H with the
    rowwise copy and, if ``colwise`` (needs M % 32 == 0), the columnwise one, byte for byte
    what :func:`quantize_mx` gives for the bf16 H; ``H`` the bf16 H when ``keep_h``."""
    _require_gpu(x8, x_scales, w8, w_scales)
    _byte_matrix("gemm_geglu_mx_quant", x8=x8, w8=w8, x_scales=x_scales, w_scales=w_scales)
    M, K = x8.shape
    I = int(intermediate)
    if w8.shape != (2 * I, K):
        raise ValueError(f"gemm_geglu_mx_quant: W must be [{2 * I}, {K}]")
    dev = x8.device
    fp8 = TORCH_FP8[E4M3]
    h8 = torch.empty((M, I), dtype=fp8, device=dev)
    h8_sc = torch.empty((M, mx_scale_ld(I)), dtype=torch.uint8, device=dev)
    h8t = h8t_sc = None
    if colwise:
        h8t = torch.empty((I, M), dtype=fp8, device=dev)
        h8t_sc = torch.empty((I, mx_scale_ld(M)), dtype=torch.uint8, device=dev)
    H = torch.empty((M, I), dtype=torch.bfloat16, device=dev) if keep_h else None
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=dev) if keep_gu else None
    _lib.check(_lib.lib().bf8_gemm_geglu_mx_quant(
        _ptr(x8), x8.stride(0), _ptr(x_scales), x_scales.stride(0), _ptr(w8), w8.stride(0),
        _ptr(w_scales), w_scales.stride(0), M, I, K, _ptr(H), I, _ptr(h8), _ptr(h8_sc),
        h8_sc.stride(0), _ptr(h8t), _ptr(h8t_sc), h8t_sc.stride(0) if colwise else 0, _ptr(GU),
        _stream(dev)), "bf8_gemm_geglu_mx_quant")
    return MxFp8Tensor(h8, h8_sc, h8t, h8t_sc, E4M3, M, I), GU, H


def gemm_geglu_mx_planes(x8, x_planes, w8, w_planes, intermediate, *, colwise=False,
                         keep_gu=False):
    """:func:`gemm_geglu_mx_quant` on scale planes, H's scales written as planes: ``(hq, GU
    or None)``, ``hq`` an :class:`MxFp8Tensor` with ``planes`` / ``planes_t`` and no scale
    rows; the same bytes and scale values."""
    who = "gemm_geglu_mx_planes"
    _require_gpu(x8, x_planes, w8, w_planes)
    _byte_matrix(who, x8=x8, w8=w8)
    M, K = x8.shape
    I = int(intermediate)
    if w8.shape != (2 * I, K):
        raise ValueError(f"{who}: W must be [{2 * I}, {K}]")
    _mx_planes(who, {"x_planes": M, "w_planes": 2 * I}, K, x_planes=x_planes, w_planes=w_planes)
    dev = x8.device
    fp8 = TORCH_FP8[E4M3]
    h8 = torch.empty((M, I), dtype=fp8, device=dev)
    hp = _new_planes(I, M, dev)
    h8t = torch.empty((I, M), dtype=fp8, device=dev) if colwise else None
    hpt = _new_planes(M, I, dev) if colwise else None
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=dev) if keep_gu else None
    _lib.check(_lib.lib().bf8_gemm_geglu_mx_planes(
        _ptr(x8), x8.stride(0), _ptr(x_planes), _ptr(w8), w8.stride(0), _ptr(w_planes), M, I, K,
        None, I, _ptr(h8), _ptr(hp), _ptr(h8t), _ptr(hpt), _ptr(GU), _stream(dev)),
        "bf8_gemm_geglu_mx_planes")
    return MxFp8Tensor(h8, None, h8t, None, E4M3, M, I, hp, hpt), GU


def geglu_partials_count(M, intermediate):
    return _geglu_partials_cached(int(M), int(intermediate), _tile_override())


def gemm_geglu(x8, x_meta, w8, w_meta, intermediate, *, w_meta_stride=0, keep_gu=False,
               partials=None):
    """Gate/up GEMM with the gated-GELU epilogue.

    x8: fp8 e4m3 [M, K]; w8: fp8 e4m3 [2I, K] (gate rows then up rows). Returns
    ``(H bf16 [M, I], GU bf16 [M, 2I] or None, h_partials int32 [tiles])``; the per-tile
    amax partials of |H| feed ``cast_partials`` (or a delayed scaler). ``partials``: an
    optional caller-owned buffer of at least ``geglu_partials_count(M, I)`` entries.
    """
    _require_gpu(x8, w8, x_meta, w_meta)
    _byte_matrix("gemm_geglu", x8=x8, w8=w8)
    M, K = x8.shape
    I = int(intermediate)
    if w8.shape != (2 * I, K):
        raise ValueError(f"gemm_geglu: weight must be [{2 * I}, {K}], got {tuple(w8.shape)}")
    L = _lib.lib()
    H = torch.empty((M, I), dtype=torch.bfloat16, device=x8.device)
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=x8.device) if keep_gu else None
    count = _geglu_partials_cached(M, I, _tile_override())
    if partials is None:
        parts = torch.empty(count, dtype=torch.int32, device=x8.device)
    else:
        if partials.numel() < count or partials.dtype != torch.int32:
            raise ValueError(f"gemm_geglu: partials must be int32 with >= {count} entries")
        parts = partials[:count]
    _lib.check(L.bf8_gemm_geglu(_ptr(x8), x8.stride(0), _ptr(w8), w8.stride(0), M, I, K,
                                _sinv_ptr(x_meta), _sinv_ptr(w_meta), w_meta_stride, _ptr(H),
                                H.stride(0), _ptr(GU), _ptr(parts), _stream(x8.device)),
               "bf8_gemm_geglu")
    return H, GU, parts


def gemm_geglu_quant(x8, x_meta, w8, w_meta, intermediate, h_meta, *, w_meta_stride=0,
                     transpose=False, keep_gu=False, keep_h=False, partials=None):
    """:func:`gemm_geglu` with H cast to e4m3 in the epilogue with the scale ``h_meta[1]``
    (a device meta record, e.g. from :func:`delayed_scale_fold`), byte for byte what
    :func:`cast` gives for the bf16 H. Returns ``(hq, GU or None, H or None, h_partials)``:
    ``hq`` the :class:`Fp8Tensor` of H (``data`` [M, I], ``data_t`` [I, M] when
    ``transpose``, which needs M % 32 == 0) with meta ``h_meta``."""
    _require_gpu(x8, w8, x_meta, w_meta, h_meta)
    _byte_matrix("gemm_geglu_quant", x8=x8, w8=w8)
    M, K = x8.shape
    I = int(intermediate)
    if w8.shape != (2 * I, K):
        raise ValueError(f"gemm_geglu_quant: weight must be [{2 * I}, {K}], got {tuple(w8.shape)}")
    dev = x8.device
    L = _lib.lib()
    h8 = torch.empty((M, I), dtype=TORCH_FP8[E4M3], device=dev)
    h8t = torch.empty((I, M), dtype=TORCH_FP8[E4M3], device=dev) if transpose else None
    H = torch.empty((M, I), dtype=torch.bfloat16, device=dev) if keep_h else None
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=dev) if keep_gu else None
    count = _geglu_partials_cached(M, I, _tile_override())
    if partials is None:
        parts = torch.empty(count, dtype=torch.int32, device=dev)
    else:
        if partials.numel() < count or partials.dtype != torch.int32:
            raise ValueError(f"gemm_geglu_quant: partials must be int32 with >= {count} entries")
        parts = partials[:count]
    _lib.check(L.bf8_gemm_geglu_quant(
        _ptr(x8), x8.stride(0), _ptr(w8), w8.stride(0), M, I, K, _sinv_ptr(x_meta),
        _sinv_ptr(w_meta), w_meta_stride, ctypes.c_void_p(h_meta.data_ptr() + 4), _ptr(H), I,
        _ptr(h8), _ptr(h8t), _ptr(GU), _ptr(parts), _stream(dev)), "bf8_gemm_geglu_quant")
    return Fp8Tensor(h8, h8t, h_meta, E4M3, M, I), GU, H, parts


def delayed_scale_fold(state, length, pos, prev_partials, fmt=E4M3, meta_out=None):
    """The scale step of :func:`cast_delayed` alone: pushes ``prev_partials`` (the previous
    step's amax partials, or None) into history slot ``pos``, derives this step's scale and
    returns it as a meta record (``meta_out``, allocated when None)."""
    _require_gpu(state)
    if meta_out is None:
        meta_out = new_meta(state.device)
    n_prev = 0 if prev_partials is None else prev_partials.numel()
    _lib.check(_lib.lib().bf8_delayed_scale_fold(_ptr(state), int(length), int(pos),
                                                 _ptr(prev_partials), n_prev, fmt,
                                                 _ptr(meta_out), _stream(state.device)),
               "bf8_delayed_scale_fold")
    return meta_out


def geglu(GU, *, partials=None):
    """H bf16 [M, I] = gelu_tanh(gate) * up from the bf16 pre-activations GU [M, 2I]
    (gate | up), bit for bit the reference's bf16 chain, and the per-block amax partials
    of |H| (for ``cast_partials``)."""
    _require_gpu(GU)
    if GU.dtype != torch.bfloat16 or GU.dim() != 2 or GU.shape[1] % 2:
        raise ValueError(f"geglu: GU must be bf16 [M, 2I] (got {GU.dtype} {tuple(GU.shape)})")
    GU = _rows_bf16(GU)
    M, I = GU.shape[0], GU.shape[1] // 2
    L = _lib.lib()
    H = torch.empty((M, I), dtype=torch.bfloat16, device=GU.device)
    count = int(L.bf8_geglu_partials_elementwise(M, I))
    if partials is None:
        parts = torch.empty(count, dtype=torch.int32, device=GU.device)
    else:
        if partials.numel() < count or partials.dtype != torch.int32:
            raise ValueError(f"geglu: partials must be int32 with >= {count} entries")
        parts = partials[:count]
    _call("bf8_geglu_bf16", GU.get_device(), L.bf8_geglu_bf16, _ptr(GU), M, I, _ptr(H), _ptr(parts))
    return H, parts


def geglu_bwd_partials_count(M, intermediate):
    return int(_lib.lib().bf8_geglu_bwd_partials(int(M), int(intermediate)))


def geglu_bwd(dH, GU, *, partials=None):
    """dGU bf16 [M, 2I] (d_gate | d_up) from dH [M, I] and the forward's GU, and the
    per-block amax partials of |dGU| (for ``cast_partials`` or a delayed scaler;
    ``partials``: an optional caller-owned buffer)."""
    _require_gpu(dH, GU)
    dH = _rows_bf16(dH)
    M, I = dH.shape
    GU = _rows_bf16(_gu_operand("geglu_bwd", GU, M, I))
    L = _lib.lib()
    dGU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=dH.device)
    count = int(L.bf8_geglu_bwd_partials(M, I))
    if partials is None:
        parts = torch.empty(count, dtype=torch.int32, device=dH.device)
    else:
        if partials.numel() < count or partials.dtype != torch.int32:
            raise ValueError(f"geglu_bwd: partials must be int32 with >= {count} entries")
        parts = partials[:count]
    _call("bf8_geglu_bwd", dH.get_device(), L.bf8_geglu_bwd, _ptr(dH), _ptr(GU), M, I, _ptr(dGU), _ptr(parts))
    return dGU, parts


RMSNORM_MAX_COLS = 4096


def rmsnorm_supported(cols):
    """Whether the fused RMSNorm kernel takes rows of ``cols`` elements."""
    return cols % 8 == 0 and 0 < cols <= RMSNORM_MAX_COLS


def rmsnorm_partials_count(rows):
    return int(_lib.lib().bf8_rmsnorm_partials(int(rows)))


def rmsnorm(x, weight, eps, *, zero_centered=True, want_rstd=False, partials=None):
    """RMSNorm of bf16 rows (HF T5Gemma2RMSNorm arithmetic) fused with the amax of its output.

    Returns ``(y bf16 [rows, cols], rstd fp32 [rows] or None, partials int32)``; pass the
    partials to :func:`cast_partials` (current scaling) to quantize y without an amax pass.
    ``partials``: an optional caller-owned buffer of at least ``rmsnorm_partials_count``
    entries (e.g. a delayed scaler's producer buffer).
    """
    _require_gpu(x, weight)
    x = _bf16_2d(x)
    rows, cols = x.shape
    if weight.dtype != torch.bfloat16 or weight.numel() != cols:
        raise ValueError(f"rmsnorm: weight must be bf16 [{cols}]")
    weight = weight.contiguous()
    L = _lib.lib()
    y = torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_rstd else None
    count = int(L.bf8_rmsnorm_partials(rows))
    if partials is None:
        parts = torch.empty(count, dtype=torch.int32, device=x.device)
    else:
        if partials.numel() < count or partials.dtype != torch.int32:
            raise ValueError(f"rmsnorm: partials must be int32 with >= {count} entries")
        parts = partials[:count]
    _lib.check(L.bf8_rmsnorm_bf16(_ptr(x), rows, cols, _ptr(weight), float(eps),
                                  int(bool(zero_centered)), _ptr(y), _ptr(rstd), _ptr(parts),
                                  _stream(x.device)), "bf8_rmsnorm_bf16")
    return y, rstd, parts


def rmsnorm_backward(x, dy, weight, eps, *, zero_centered=True, need_dx=True, need_dw=True):
    """Gradients (dx bf16 [rows, cols] or None, dweight bf16 [cols] or None) of
    :func:`rmsnorm` for the bf16 gradient dy of its output."""
    _require_gpu(x, dy, weight)
    x = _bf16_2d(x)
    dy = _bf16_2d(dy)
    rows, cols = x.shape
    if tuple(dy.shape) != (rows, cols):
        raise ValueError(f"rmsnorm_backward: dy must be [{rows}, {cols}]")
    if weight.dtype != torch.bfloat16 or weight.numel() != cols:
        raise ValueError(f"rmsnorm_backward: weight must be bf16 [{cols}]")
    if not (need_dx or need_dw):
        return None, None
    weight = weight.contiguous()
    L = _lib.lib()
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty(cols, dtype=torch.bfloat16, device=x.device) if need_dw else None
    if rows == 0:  # a sum over no rows
        return dx, dw if dw is None else dw.zero_()
    ws, nbytes = None, 0
    if need_dw:
        ws, nbytes = _call_workspace(int(L.bf8_rmsnorm_bwd_workspace(rows, cols)), x)
    _lib.check(L.bf8_rmsnorm_bwd_bf16(_ptr(x), _ptr(dy), rows, cols, _ptr(weight), float(eps),
                                      int(bool(zero_centered)), _ptr(dx), _ptr(dw), _ptr(ws),
                                      nbytes, _stream(x.device)), "bf8_rmsnorm_bwd_bf16")
    return dx, dw


def geglu_bwd_delayed_partials_count(M, intermediate):
    return int(_lib.lib().bf8_geglu_bwd_delayed_partials(int(M), int(intermediate)))


def geglu_bwd_delayed(dH, GU, state, length, pos, prev_partials, fmt=E5M2, *, rowwise=True,
                      transpose=False, partials_out, meta_out=None):
    """dGU of the gated GELU quantized at once with a delayed scale (``cast_delayed``
    semantics for state / pos / prev_partials / meta_out); returns the :class:`Fp8Tensor`
    of dGU [M, 2I] (``data`` and/or ``data_t``). ``partials_out`` receives this step's
    amax partials (``geglu_bwd_delayed_partials_count`` entries)."""
    _require_gpu(dH, GU, state)
    dH = dH.contiguous()
    M, I = dH.shape
    GU = _gu_operand("geglu_bwd_delayed", GU, M, I)
    dev = dH.device
    if meta_out is None:
        meta_out = new_meta(dev)
    out = torch.empty((M, 2 * I), dtype=TORCH_FP8[fmt], device=dev) if rowwise else None
    out_t = torch.empty((2 * I, M), dtype=TORCH_FP8[fmt], device=dev) if transpose else None
    n_prev = 0 if prev_partials is None else prev_partials.numel()
    _lib.check(_lib.lib().bf8_geglu_bwd_delayed(
        _ptr(dH), _ptr(GU), M, I, _ptr(state), int(length), int(pos), _ptr(prev_partials),
        n_prev, fmt, _ptr(meta_out), _ptr(out), _ptr(out_t), _ptr(partials_out), _stream(dev)),
        "bf8_geglu_bwd_delayed")
    return Fp8Tensor(out, out_t, meta_out, fmt, M, 2 * I)


def new_delayed_state(length, device):
    """Delayed-scaling state: float32 [length + 4] = history, {amax, scale, scale_inv, pos}."""
    st = torch.zeros(length + 4, dtype=torch.float32, device=device)
    st[length + 1] = 1.0
    st[length + 2] = 1.0
    return st


def delayed_scale_begin(state, length, fmt):
    _lib.check(_lib.lib().bf8_delayed_scale_begin(_ptr(state), length, fmt,
                                                  _stream(state.device)),
               "bf8_delayed_scale_begin")
    return state[length:length + 4]


def delayed_scale_end(state, length, partials):
    _lib.check(_lib.lib().bf8_delayed_scale_end(_ptr(state), length, _ptr(partials),
                                                partials.numel(), _stream(state.device)),
               "bf8_delayed_scale_end")


def cast_amax_partials_count(rows, cols, transpose):
    return int(_lib.lib().bf8_cast_amax_partials(int(rows), int(cols), int(bool(transpose))))


def cast_delayed(x, state, length, pos, prev_partials, fmt=E4M3, *, rowwise=True,
                 transpose=False, partials_out=None, meta_out=None):
    """One-pass delayed-scaling cast (bf8_cast_delayed_bf16).

    ``prev_partials``: the previous step's amax partials (None on the first step), pushed
    into history slot ``pos`` before the scale is derived. ``partials_out``: buffer for
    this step's amax partials of |x| (``cast_amax_partials_count`` entries), or None when
    the producer of x wrote them. Returns an :class:`Fp8Tensor` whose meta is
    ``meta_out`` (a fresh record if None): {history max, scale, scale_inv, 0}.
    """
    _require_gpu(x, state)
    x = _bf16_2d(x)
    rows, cols = x.shape
    dev = x.device
    if meta_out is None:
        meta_out = new_meta(dev)
    out = torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=dev) if rowwise else None
    out_t = torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=dev) if transpose else None
    n_prev = 0 if prev_partials is None else prev_partials.numel()
    _lib.check(_lib.lib().bf8_cast_delayed_bf16(
        _ptr(x), rows, cols, _ptr(state), int(length), int(pos), _ptr(prev_partials), n_prev,
        fmt, _ptr(meta_out), _ptr(out), _ptr(out_t), _ptr(partials_out), _stream(dev)),
        "bf8_cast_delayed_bf16")
    return Fp8Tensor(out, out_t, meta_out, fmt, rows, cols)


def cast_delayed_many(jobs):
    """Several :func:`cast_delayed` calls in one launch (bf8_cast_delayed_many_bf16).

    ``jobs``: up to 8 dicts with the keys x, state, length, pos, prev_partials, fmt,
    rowwise, transpose, partials_out, meta_out (the arguments of :func:`cast_delayed`).
    Returns one :class:`Fp8Tensor` per job; bytes, metas, histories and partials equal
    those of the calls made one by one in order."""
    count = len(jobs)
    if not 1 <= count <= 8:
        raise ValueError(f"cast_delayed_many: {count} tensors (1 to 8 supported)")
    fields = {k: [] for k in ("x", "rows", "cols", "state", "len", "pos", "prev", "n_prev",
                              "fmt", "meta", "out", "out_t", "parts")}
    results = []
    dev = None
    for j in jobs:
        x = _bf16_2d(j["x"])
        _require_gpu(x, j["state"])
        dev = x.device if dev is None else dev
        if x.device != dev:
            raise ValueError("cast_delayed_many: tensors on different devices")
        rows, cols = x.shape
        fmt = j.get("fmt", E4M3)
        meta = j.get("meta_out")
        if meta is None:
            meta = new_meta(dev)
        out = (torch.empty((rows, cols), dtype=TORCH_FP8[fmt], device=dev)
               if j.get("rowwise", True) else None)
        out_t = (torch.empty((cols, rows), dtype=TORCH_FP8[fmt], device=dev)
                 if j.get("transpose", False) else None)
        prev = j.get("prev_partials")
        for key, val in (("x", _ptr(x)), ("rows", rows), ("cols", cols),
                         ("state", _ptr(j["state"])), ("len", int(j["length"])),
                         ("pos", int(j["pos"])), ("prev", _ptr(prev)),
                         ("n_prev", 0 if prev is None else prev.numel()), ("fmt", fmt),
                         ("meta", _ptr(meta)), ("out", _ptr(out)), ("out_t", _ptr(out_t)),
                         ("parts", _ptr(j.get("partials_out")))):
            fields[key].append(val)
        results.append(Fp8Tensor(out, out_t, meta, fmt, rows, cols))
    P = ctypes.c_void_p * count
    I64 = ctypes.c_int64 * count
    I32 = ctypes.c_int * count
    _lib.check(_lib.lib().bf8_cast_delayed_many_bf16(
        count, P(*fields["x"]), I64(*fields["rows"]), I64(*fields["cols"]), P(*fields["state"]),
        I32(*fields["len"]), I32(*fields["pos"]), P(*fields["prev"]), I64(*fields["n_prev"]),
        I32(*fields["fmt"]), P(*fields["meta"]), P(*fields["out"]), P(*fields["out_t"]),
        P(*fields["parts"]), _stream(dev)), "bf8_cast_delayed_many_bf16")
    return results


# ---- NVFP4 (e2m1 in 16-blocks, e4m3 block scales, fp32 tensor scale) -------------------
@dataclass
class NvFp4Tensor:
    """An NVFP4 tensor of x [rows, cols]: ``data`` uint8 [rows, cols / 2] (two e2m1 codes a
    byte) with ``scales`` uint8 e4m3 [rows, cols / 16] (blocks along cols) and/or the
    columnwise copy ``data_t`` [cols, rows / 2] with ``scales_t`` [cols, rows / 16] (blocks
    along rows), and ``meta`` fp32 [4] = {amax, S_enc, S_dec, 0}. ``cache_dequant``: keep
    the exact bf16 dequantization of each copy on the object after its first use (a weight
    cached across microbatches: 2 bytes per element per copy, no dequantization pass per
    GEMM afterwards)."""

    data: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]
    data_t: Optional[torch.Tensor]
    scales_t: Optional[torch.Tensor]
    meta: torch.Tensor
    rows: int
    cols: int
    cache_dequant: bool = False
    _deq: Optional[torch.Tensor] = field(default=None, repr=False)
    _deq_t: Optional[torch.Tensor] = field(default=None, repr=False)


def nvfp4_dequant(q, *, transpose=False):
    """bf16 = e2m1(code) * s of ``q``'s rowwise copy (or with ``transpose`` its columnwise
    copy), exact and without S_dec; kept on ``q`` when ``q.cache_dequant`` is set, or
    written by the quantizer itself (``quantize_nvfp4(dequant_rows=True)``)."""
    attr = "_deq_t" if transpose else "_deq"
    if getattr(q, attr) is None and not q.cache_dequant:
        return dequant_nvfp4(q.data_t, q.scales_t) if transpose else dequant_nvfp4(q.data, q.scales)
    d = getattr(q, attr)
    if d is None:
        d = dequant_nvfp4(q.data_t, q.scales_t) if transpose else dequant_nvfp4(q.data, q.scales)
        setattr(q, attr, d)
    return d


def quantize_nvfp4(x, *, rowwise=True, colwise=False, partials=None, dequant_rows=False,
                   dequant_cols=False):
    """NVFP4 quantization of a bf16 tensor (flattened to 2-D): an amax pass and the block
    quantization (rowwise needs cols % 16 == 0, columnwise rows % 16 == 0). ``partials``:
    the amax partials of |x| its producer wrote (int32 / uint32 fp32 bits: ``geglu_bwd``'s,
    the fused RMSNorm's, the gated-GELU GEMM's); the amax pass is then skipped
    (bf8_quantize_nvfp4_partials_bf16, the same outputs bit for bit). ``dequant_rows``: the
    rowwise copy is kept only as its exact bf16 dequantization (``nvfp4_dequant(q)``; data
    and scales None), for a tensor whose rowwise copy only feeds the next GEMM
    (bf8_quantize_nvfp4_dequant_bf16); ``dequant_cols``: the columnwise copy likewise
    (``nvfp4_dequant(q, transpose=True)``; cols % 8 == 0)."""
    _require_gpu(x, partials)
    x = _bf16_2d(x)
    rows, cols = x.shape
    dev = x.device
    meta = new_meta(dev)
    u8 = torch.uint8
    codes = rowwise and not dequant_rows
    codes_t = colwise and not dequant_cols
    out = torch.empty((rows, cols // 2), dtype=u8, device=dev) if codes else None
    sc = torch.empty((rows, cols // 16), dtype=u8, device=dev) if codes else None
    out_t = torch.empty((cols, rows // 2), dtype=u8, device=dev) if codes_t else None
    sc_t = torch.empty((cols, rows // 16), dtype=u8, device=dev) if codes_t else None
    L = _lib.lib()
    if partials is not None:
        if partials.dtype != torch.int32 or partials.dim() != 1 or partials.numel() < 1:
            raise ValueError("quantize_nvfp4: partials must be a non-empty 1-D int32 tensor")
    if (dequant_rows and rowwise) or (dequant_cols and colwise):
        if codes:
            raise ValueError("quantize_nvfp4: dequant_cols with rowwise codes is not supported")
        deq = torch.empty((rows, cols), dtype=torch.bfloat16, device=dev) if rowwise else None
        deq_t = (torch.empty((cols, rows), dtype=torch.bfloat16, device=dev)
                 if colwise and dequant_cols else None)
        if partials is not None:
            parts, n_parts = partials.contiguous(), partials.numel()
        else:
            parts, n_parts = partials_buffer(max(1, _amax_partials_cached(rows * cols)), dev), 0
        _lib.check(L.bf8_quantize_nvfp4_dequant2_bf16(
            _ptr(x), rows, cols, _ptr(parts), n_parts, _ptr(deq), _ptr(deq_t), _ptr(out_t),
            _ptr(sc_t), _ptr(meta), _stream(dev)), "bf8_quantize_nvfp4_dequant2_bf16")
        return NvFp4Tensor(None, None, out_t, sc_t, meta, rows, cols, _deq=deq, _deq_t=deq_t)
    if partials is not None:
        _lib.check(L.bf8_quantize_nvfp4_partials_bf16(
            _ptr(x), rows, cols, _ptr(partials.contiguous()), partials.numel(), _ptr(out),
            _ptr(sc), _ptr(out_t), _ptr(sc_t), _ptr(meta), _stream(dev)),
            "bf8_quantize_nvfp4_partials_bf16")
        return NvFp4Tensor(out, sc, out_t, sc_t, meta, rows, cols)
    parts = partials_buffer(max(1, int(L.bf8_amax_partials(rows * cols))), dev)
    _lib.check(L.bf8_quantize_nvfp4_bf16(_ptr(x), rows, cols, _ptr(out), _ptr(sc), _ptr(out_t),
                                         _ptr(sc_t), _ptr(meta), _ptr(parts), _stream(dev)),
               "bf8_quantize_nvfp4_bf16")
    return NvFp4Tensor(out, sc, out_t, sc_t, meta, rows, cols)


def dequant_nvfp4(data, scales):
    """bf16 [rows, 2 * data cols] = e2m1(code) * s per element (exact, without S_dec)."""
    _require_gpu(data, scales)
    rows, half = data.shape
    out = torch.empty((rows, 2 * half), dtype=torch.bfloat16, device=data.device)
    _lib.check(_lib.lib().bf8_dequant_nvfp4(_ptr(data.contiguous()), _ptr(scales.contiguous()),
                                            rows, 2 * half, _ptr(out), _stream(data.device)),
               "bf8_dequant_nvfp4")
    return out


def gemm_bf16(a, b, a_sinv, b_sinv, *, out_dtype=torch.bfloat16):
    """``C = (a @ b.T accumulated in fp32) * a_sinv * b_sinv`` on bf16 a [M, K], b [N, K]
    (row-major) with the bf16 MFMA; a_sinv, b_sinv: device fp32 scalars."""
    _require_gpu(a, b, a_sinv, b_sinv)
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise TypeError("gemm_bf16: a and b must be bfloat16")
    if a.stride(1) != 1 or b.stride(1) != 1:
        raise ValueError("gemm_bf16: a and b must be row-major")
    M, K = a.shape
    N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"gemm_bf16: inner dims differ ({K} vs {Kb})")
    out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    L = _lib.lib()
    ws_bytes = int(L.bf8_gemm_bf16_workspace(M, N, K))
    ws = gemm_workspace(ws_bytes, a.device) if ws_bytes else None
    ws_bytes = ws.numel() if ws is not None else 0
    _lib.check(L.bf8_gemm_bf16(_ptr(a), a.stride(0), _ptr(b), b.stride(0), M, N, K,
                               _ptr(a_sinv), _ptr(b_sinv), _ptr(out),
                               OUT_BF16 if out_dtype == torch.bfloat16 else OUT_F32,
                               out.stride(0), _ptr(ws), ws_bytes, _stream(a.device)),
               "bf8_gemm_bf16")
    return out


def gemm_geglu_bf16(a, b, a_sinv, b_sinv, intermediate, *, keep_gu=False, partials=None):
    """:func:`gemm_geglu` on bf16 operands a [M, K], b [2I, K] (gate rows then up rows) with
    device fp32 scalars a_sinv, b_sinv applied to the sums (bf8_gemm_geglu_bf16). Returns
    ``(H bf16 [M, I], GU bf16 [M, 2I] or None, h_partials int32)``."""
    _require_gpu(a, b, a_sinv, b_sinv)
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise TypeError("gemm_geglu_bf16: a and b must be bfloat16")
    if a.stride(1) != 1 or b.stride(1) != 1:
        raise ValueError("gemm_geglu_bf16: a and b must be row-major")
    M, K = a.shape
    I = int(intermediate)
    if tuple(b.shape) != (2 * I, K):
        raise ValueError(f"gemm_geglu_bf16: weight must be [{2 * I}, {K}], got {tuple(b.shape)}")
    H = torch.empty((M, I), dtype=torch.bfloat16, device=a.device)
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=a.device) if keep_gu else None
    count = _geglu_partials_cached(M, I, _tile_override())
    if partials is None:
        parts = torch.empty(count, dtype=torch.int32, device=a.device)
    else:
        if partials.numel() < count or partials.dtype != torch.int32:
            raise ValueError(f"gemm_geglu_bf16: partials must be int32 with >= {count} entries")
        parts = partials[:count]
    _lib.check(_lib.lib().bf8_gemm_geglu_bf16(
        _ptr(a), a.stride(0), _ptr(b), b.stride(0), M, I, K, _ptr(a_sinv), _ptr(b_sinv),
        _ptr(H), H.stride(0), _ptr(GU), _ptr(parts), _stream(a.device)), "bf8_gemm_geglu_bf16")
    return H, GU, parts


def gemm_geglu_nvfp4(a_data, a_scales, a_meta, b_data, b_scales, b_meta, intermediate, *,
                     keep_gu=False, a_deq=None, b_deq=None):
    """The NVFP4 gate/up projection with the gated GELU in its epilogue: both operands
    dequantized exactly to bf16, then :func:`gemm_geglu_bf16` with the two S_dec.
    ``a_deq`` / ``b_deq``: an operand's bf16 dequantization when the caller holds it."""
    a = a_deq if a_deq is not None else dequant_nvfp4(a_data, a_scales)
    b = b_deq if b_deq is not None else dequant_nvfp4(b_data, b_scales)
    return gemm_geglu_bf16(a, b, a_meta[2:3], b_meta[2:3], intermediate, keep_gu=keep_gu)


def gemm_nvfp4(a_data, a_scales, a_meta, b_data, b_scales, b_meta, *, out_dtype=torch.bfloat16,
               a_deq=None, b_deq=None):
    """``C = (A^ @ B^.T) * S_dec(a) * S_dec(b)`` for NVFP4 operands A [M, K], B [N, K]
    (blocks along K): both dequantized exactly to bf16, then the bf16 MFMA GEMM.
    ``a_deq`` / ``b_deq``: an operand's bf16 dequantization when the caller holds it."""
    a = a_deq if a_deq is not None else dequant_nvfp4(a_data, a_scales)
    b = b_deq if b_deq is not None else dequant_nvfp4(b_data, b_scales)
    return gemm_bf16(a, b, a_meta[2:3], b_meta[2:3], out_dtype=out_dtype)


# ---- MXFP4: e2m1 codes in blocks of 32 under a power of two ---------------------------------
# The ops below run in training steps and decoding loops of small tensors, where a call's host time is
# what it takes: their checks read the tensors' fields once, and tensors that are as the
# kernels want them (2-D, contiguous, aligned) pass without a call.
def _index_of(who, first, *rest):
    """The device index of the tensors (None among ``rest`` is skipped), which must be one."""
    idx = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != idx:
            _require_gpu(first, t)
            raise ValueError(f"{who}: tensors on different devices ({first.device} and {t.device})")
    if idx < 0:
        _require_gpu(first)
    return idx


def _call(what, idx, fn, *args):
    """Calls a library entry on the current stream of device ``idx`` (made the current one for the
    launch where it is not) and checks its status."""
    if idx == torch._C._cuda_getDevice():
        rc = fn(*args, _stream_of(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _stream_of(idx))
    if rc:
        _lib.check(rc, what)


def _stream_of(idx):
    return _raw_stream(idx) if _raw_stream is not None else torch.cuda.current_stream(idx).cuda_stream


def _call_workspace(nbytes, like):
    """``(workspace, its bytes)`` of a call, its own: two threads may launch on one stream by turns, and
    two graphs captured on one may replay side by side. It is free for the stream's next call where this one
    returns. (0.2-0.3 us of host time over a workspace that the stream's calls share, 12-16 us a call.)"""
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device), nbytes


def _rows_bf16(t):
    """``t`` as the kernels read it: bf16 [rows, cols], contiguous and 16-byte aligned, copied or
    flattened where it is not."""
    if t.dtype is not torch.bfloat16 or t.dim() != 2 or not t.is_contiguous():
        t = _bf16_2d(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


@dataclass
class Mxfp4Tensor:
    """An MXFP4 tensor of x [rows, cols] (32-element blocks of e2m1 codes under one E8M0 scale):
    ``data`` uint8 [rows, cols / 2] (two codes a byte, the even element in the low nibble) with
    ``planes`` int32 [ceil(cols / 128), rows] (blocks along rows), and/or ``data_t`` uint8
    [cols, R / 2] with ``planes_t`` int32 [ceil(rows / 128), cols] (blocks along columns of x,
    stored transposed; R is ``rows`` rounded up to 32, the codes past ``rows`` 0). A plane holds
    a dword of four scale bytes for every row."""

    data: Optional[torch.Tensor]
    planes: Optional[torch.Tensor]
    data_t: Optional[torch.Tensor]
    planes_t: Optional[torch.Tensor]
    rows: int
    cols: int


def _new_mxfp4(rows, cols, rowwise, colwise, device):
    out = pl = out_t = pl_t = None
    if rowwise:
        if cols % 32:
            raise ValueError(f"MXFP4 blocks along rows need cols % 32 == 0 (got {cols})")
        out = torch.empty((rows, cols // 2), dtype=torch.uint8, device=device)
        pl = torch.empty(((cols + 127) // 128, rows), dtype=torch.int32, device=device)
    if colwise:
        out_t = torch.empty((cols, (rows + 31) // 32 * 16), dtype=torch.uint8, device=device)
        pl_t = torch.empty(((rows + 127) // 128, cols), dtype=torch.int32, device=device)
    return Mxfp4Tensor(out, pl, out_t, pl_t, rows, cols)


def quantize_mxfp4(x, *, rowwise=True, colwise=False):
    """MXFP4 quantization of a bf16 tensor (flattened to [rows, cols]) as a :class:`Mxfp4Tensor`:
    per block of 32 the smallest power of two s with max|x| <= 6 s, the values x / s rounded to
    the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code). ``rowwise``: blocks
    along rows (cols a multiple of 32); ``colwise``: along columns, any number of rows (cols a
    multiple of 8). Both copies come from one pass over x."""
    idx = _index_of("quantize_mxfp4", x)
    x = _rows_bf16(x)
    rows, cols = x.shape
    if not (rowwise or colwise):
        raise ValueError("quantize_mxfp4: nothing requested")
    q = _new_mxfp4(rows, cols, rowwise, colwise, x.device)
    if rows and cols:
        _call("bf8_quantize_mxfp4_bf16", idx, _lib.lib().bf8_quantize_mxfp4_bf16, x.data_ptr(), rows,
              cols, _ptr(q.data), _ptr(q.planes), _ptr(q.data_t), _ptr(q.planes_t))
    return q


def _mxfp4_operand(who, name, codes, planes):
    """(rows, K) of an MXFP4 operand, checked."""
    if codes.dtype is not torch.uint8:
        raise TypeError(f"{who}: {name} must be uint8 codes (got {codes.dtype})")
    if codes.dim() != 2 or (codes.stride(1) != 1 and codes.shape[1] > 1):
        _byte_matrix(who, **{name: codes})
    rows, half = codes.shape
    if (planes.dtype is not torch.int32 or planes.shape != ((half + 63) // 64, rows)
            or not planes.is_contiguous()):
        _mx_planes(who, {f"{name}_planes": rows}, 2 * half, **{f"{name}_planes": planes})
    return rows, 2 * half


def dequant_mxfp4(q, *, transpose=False):
    """The values of a :class:`Mxfp4Tensor` as bf16 [rows, cols], or with ``transpose`` those of
    its columnwise copy, [cols, rows] (a view of rows padded to 32 where rows is not a multiple).
    Exact: a code times its block's power of two is a bf16 value."""
    who = "dequant_mxfp4"
    codes, planes = (q.data_t, q.planes_t) if transpose else (q.data, q.planes)
    if codes is None:
        raise ValueError(f"{who}: the tensor has no {'columnwise' if transpose else 'rowwise'} copy")
    idx = _index_of(who, codes, planes)
    rows, cols = _mxfp4_operand(who, "codes", codes, planes)
    codes = codes.contiguous()
    out = torch.empty((rows, cols), dtype=torch.bfloat16, device=codes.device)
    if rows and cols:
        _call("bf8_dequant_mxfp4", idx, _lib.lib().bf8_dequant_mxfp4, codes.data_ptr(),
              planes.data_ptr(), rows, cols, out.data_ptr())
    return out[:, :q.rows] if transpose and q.rows != cols else out


def gemm_mxfp4(a, a_planes, b, b_planes, *, bias=None, out_dtype=torch.bfloat16, out=None):
    """``C = A @ B.T (+ bias)`` of MXFP4 operands A [M, K] and B [N, K] (codes and scale planes as
    :func:`quantize_mxfp4` writes them) on the block-scaled FP4 MFMA, sums in fp32."""
    who = "gemm_mxfp4"
    idx = _index_of(who, a, a_planes, b, b_planes, bias, out)
    M, K = _mxfp4_operand(who, "a", a, a_planes)
    N, Kb = _mxfp4_operand(who, "b", b, b_planes)
    if K != Kb:
        raise ValueError(f"{who}: inner dims differ ({K} vs {Kb})")
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise TypeError(f"{who}: out_dtype must be bfloat16 or float32")
    if out is None:
        out, ldc = torch.empty((M, N), dtype=out_dtype, device=a.device), N
    else:
        _out_matrix(who, out, (M, N), out_dtype)
        ldc = out.stride(0) if M > 1 else N
    if bias is not None:
        if bias.dtype != torch.bfloat16 or bias.numel() != N:
            raise ValueError(f"{who}: bias must be bfloat16 [{N}] (got {bias.dtype} {tuple(bias.shape)})")
        bias = bias.contiguous()
        if bias.data_ptr() % 8:
            bias = bias.clone()
    if K == 0:  # an empty sum
        return out.zero_() if bias is None else out.copy_(bias.reshape(1, N).expand(M, N))
    L, ws = _lib.lib(), None
    ws_bytes = L.bf8_gemm_mxfp4_workspace(M, N, K)
    if ws_bytes:
        ws, ws_bytes = _call_workspace(ws_bytes, a)
    # (a single row's stride(0) may be anything)
    _call("bf8_gemm_mxfp4", idx, L.bf8_gemm_mxfp4, a.data_ptr(), a.stride(0) if M > 1 else K // 2,
          a_planes.data_ptr(), b.data_ptr(), b.stride(0), b_planes.data_ptr(), M, N, K, _ptr(bias),
          out.data_ptr(), OUT_BF16 if out_dtype is torch.bfloat16 else OUT_F32, ldc, _ptr(ws), ws_bytes)
    return out


def gemm_geglu_mxfp4(x, x_planes, w, w_planes, intermediate, *, colwise=False, keep_gu=False):
    """Gate/up product of MXFP4 operands X [M, K] and W [2I, K] (gate rows then up rows) with the
    gated GELU: ``(hq, GU or None)``, ``hq`` the :class:`Mxfp4Tensor` of H = gelu_tanh(gate) *
    up [M, I] (gate, up, the activation and H rounded to bf16, as :func:`geglu` does; with
    ``colwise`` the columnwise copy as well) and ``GU`` the bf16 pre-activations when
    ``keep_gu``. I must be a multiple of 128."""
    who = "gemm_geglu_mxfp4"
    idx = _index_of(who, x, x_planes, w, w_planes)
    I = int(intermediate)
    M, K = _mxfp4_operand(who, "x", x, x_planes)
    N, Kw = _mxfp4_operand(who, "w", w, w_planes)
    if N != 2 * I or K != Kw:
        raise ValueError(f"{who}: w must have {2 * I} rows of {K} values (got {N} of {Kw})")
    if I % 128:
        raise ValueError(f"{who}: the intermediate size must be a multiple of 128 (got {I})")
    if K == 0:
        raise ValueError(f"{who}: K must not be 0")
    hq = _new_mxfp4(M, I, True, colwise, x.device)
    GU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=x.device) if keep_gu else None
    if M and I:
        _call("bf8_gemm_geglu_mxfp4", idx, _lib.lib().bf8_gemm_geglu_mxfp4, x.data_ptr(),
              x.stride(0) if M > 1 else K // 2,
              x_planes.data_ptr(), w.data_ptr(), w.stride(0), w_planes.data_ptr(), M, I, K,
              hq.data.data_ptr(), hq.planes.data_ptr(), _ptr(hq.data_t), _ptr(hq.planes_t), _ptr(GU))
    return hq, GU


def geglu_bwd_mxfp4(dH, GU, *, rowwise=True, colwise=False):
    """:func:`geglu_bwd` and the :func:`quantize_mxfp4` of its dGU [M, 2I] in one pass (the same
    codes and planes; the bf16 dGU is not written). I must be a multiple of 128."""
    who = "geglu_bwd_mxfp4"
    idx = _index_of(who, dH, GU)
    dH = _rows_bf16(dH)
    M, I = dH.shape
    GU = _rows_bf16(_gu_operand(who, GU, M, I))
    if not (rowwise or colwise):
        raise ValueError(f"{who}: nothing requested")
    if I % 128:
        raise ValueError(f"{who}: the intermediate size must be a multiple of 128 (got {I})")
    q = _new_mxfp4(M, 2 * I, rowwise, colwise, dH.device)
    if M and I:
        _call("bf8_geglu_bwd_mxfp4", idx, _lib.lib().bf8_geglu_bwd_mxfp4, dH.data_ptr(), GU.data_ptr(),
              M, I, _ptr(q.data), _ptr(q.planes), _ptr(q.data_t), _ptr(q.planes_t))
    return q


# ---- the norms on either side of a residual connection ---------------------------------------
def _norm_weight(who, name, t, cols):
    if t.dtype is not torch.bfloat16 or t.shape != (cols,):
        raise ValueError(f"{who}: {name} must be bf16 [{cols}] (got {t.dtype} {tuple(t.shape)})")
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.contiguous().clone()


def _norm_weights(who, cols, post_weight, pre_weight, gate):
    return (_norm_weight(who, "post_weight", post_weight, cols),
            _norm_weight(who, "pre_weight", pre_weight, cols),
            None if gate is None else _norm_weight(who, "gate", gate, cols))


def rmsnorm_residual(h, residual, post_weight, pre_weight, eps, *, gate=None, residual_scale=1.0,
                     zero_centered=True):
    """The norm of a block's output ``h``, its addition to the residual stream and the norm of the
    sum for the next block, in one kernel (bf16 tensors [..., cols], fp32 arithmetic):
    ``out = residual_scale * residual + gate * rmsnorm(h, post_weight)`` and
    ``y = rmsnorm(out, pre_weight)``; returns ``(out, y)``. ``gate``: bf16 [cols] or None (1). cols: a
    multiple of 8, 16384 at most. No gradients (:func:`bongard_amd.fused_mlp.residual_norm` has them)."""
    who = "rmsnorm_residual"
    idx = _index_of(who, h, residual, post_weight, pre_weight, gate)
    shape = h.shape
    if residual.shape != shape:
        raise ValueError(f"{who}: residual must be {tuple(shape)} (got {tuple(residual.shape)})")
    post, pre, gate = _norm_weights(who, shape[-1], post_weight, pre_weight, gate)
    h, residual = _rows_bf16(h), _rows_bf16(residual)
    rows, cols = h.shape
    out, y = torch.empty_like(h), torch.empty_like(h)
    if rows:
        _call("bf8_rmsnorm_residual_bf16", idx, _lib.lib().bf8_rmsnorm_residual_bf16, h.data_ptr(),
              residual.data_ptr(), rows, cols, post.data_ptr(), pre.data_ptr(), _ptr(gate),
              residual_scale, eps, 1 if zero_centered else 0, out.data_ptr(), y.data_ptr())
    return (out, y) if len(shape) == 2 else (out.view(shape), y.view(shape))


@functools.lru_cache(maxsize=4096)
def _residual_norm_ws_cached(rows, cols):
    return int(_lib.lib().bf8_rmsnorm_residual_bwd_workspace(rows, cols))


def rmsnorm_residual_backward(h, out, dout, dy, post_weight, pre_weight, eps, *, gate=None,
                              residual_scale=1.0, zero_centered=True,
                              needs=(True, True, True, True, True)):
    """Gradients ``(dh, dresidual, dpost, dpre, dgate)`` of :func:`rmsnorm_residual` from its ``h``
    and ``out`` and the gradients ``dout`` and ``dy`` of its results (one of them may be None: zero).
    ``needs``: which to compute (the others are None; ``dgate`` is None without a gate)."""
    who = "rmsnorm_residual_backward"
    if dout is None and dy is None:
        raise ValueError(f"{who}: no gradient given")
    idx = _index_of(who, h, out, dout, dy, post_weight, pre_weight, gate)
    shape = h.shape
    for name, t in (("out", out), ("dout", dout), ("dy", dy)):
        if t is not None and t.shape != shape:
            raise ValueError(f"{who}: {name} must be {tuple(shape)} (got {tuple(t.shape)})")
    post, pre, gate = _norm_weights(who, shape[-1], post_weight, pre_weight, gate)
    h, out = _rows_bf16(h), _rows_bf16(out)
    dout = dout if dout is None else _rows_bf16(dout)
    dy = dy if dy is None else _rows_bf16(dy)
    rows, cols = h.shape
    dh = torch.empty_like(h) if needs[0] else None
    dres = torch.empty_like(h) if needs[1] else None
    weights = [needs[2], needs[3], needs[4] and gate is not None]
    dpost, dpre, dgate = [torch.empty_like(post) if n else None for n in weights]
    if rows == 0:
        for g in (dpost, dpre, dgate):
            if g is not None:
                g.zero_()
    elif needs[0] or needs[1] or any(weights):
        ws, nbytes = None, 0
        if any(weights):
            ws, nbytes = _call_workspace(_residual_norm_ws_cached(rows, cols), h)
        _call("bf8_rmsnorm_residual_bwd_bf16", idx, _lib.lib().bf8_rmsnorm_residual_bwd_bf16,
              h.data_ptr(), out.data_ptr(), _ptr(dout), _ptr(dy), rows, cols, post.data_ptr(),
              pre.data_ptr(), _ptr(gate), residual_scale, eps, 1 if zero_centered else 0, _ptr(dh),
              _ptr(dres), _ptr(dpost), _ptr(dpre), _ptr(dgate), _ptr(ws), nbytes)
    if len(shape) != 2:
        dh, dres = (g if g is None else g.view(shape) for g in (dh, dres))
    return dh, dres, dpost, dpre, dgate


# ---- int8: codes under one scale for each row, checkpoints in blocks of 32 ----------------------
@dataclass
class Int8Tensor:
    """An int8 tensor of x [rows, cols]: ``data`` [rows, cols] with ``row_scale`` fp32 [rows] (x ~
    data * row_scale[:, None]), and/or ``data_t`` [cols, R], one scale for each column of x in
    ``col_scale`` fp32 [cols] (R is ``rows`` rounded up to 16, the codes past ``rows`` 0)."""

    data: Optional[torch.Tensor]
    row_scale: Optional[torch.Tensor]
    data_t: Optional[torch.Tensor]
    col_scale: Optional[torch.Tensor]
    rows: int
    cols: int


def _new_int8(rows, cols, rowwise, colwise, device):
    out = scale = out_t = scale_t = None
    if rowwise:
        out = torch.empty((rows, cols), dtype=torch.int8, device=device)
        scale = torch.empty(rows, dtype=torch.float32, device=device)
    if colwise:
        out_t = torch.empty((cols, (rows + 15) // 16 * 16), dtype=torch.int8, device=device)
        scale_t = torch.empty(cols, dtype=torch.float32, device=device)
    return Int8Tensor(out, scale, out_t, scale_t, rows, cols)


@functools.lru_cache(maxsize=4096)
def _quantize_int8_ws_cached(rows, cols, both):
    return int(_lib.lib().bf8_quantize_int8_workspace(rows, cols, both))


def quantize_int8(x, *, rowwise=True, colwise=False):
    """int8 quantization of a bf16 tensor (flattened to [rows, cols]) as an :class:`Int8Tensor`: of each
    row the scale a / 127, a = max(max|x|, 2^-40), and the codes 127 x / a to nearest (ties to even);
    ``colwise``: of each column likewise, stored transposed. A row (column) that holds inf or NaN has the
    scale NaN and codes 0. cols: a multiple of 8 (16 for a product), 32768 at most."""
    who = "quantize_int8"
    idx = _index_of(who, x)
    x = _rows_bf16(x)
    rows, cols = x.shape
    if not (rowwise or colwise):
        raise ValueError(f"{who}: nothing requested")
    q = _new_int8(rows, cols, rowwise, colwise, x.device)
    out, scale, out_t, scale_t, ws, nbytes = q.data, q.row_scale, q.data_t, q.col_scale, None, 0
    if colwise:
        nbytes = _quantize_int8_ws_cached(rows, cols, 1 if rowwise else 0)
        if nbytes:
            ws, nbytes = _call_workspace(nbytes, x)
    if rows and cols:
        _call("bf8_quantize_int8_bf16", idx, _lib.lib().bf8_quantize_int8_bf16, x.data_ptr(), rows, cols,
              _ptr(out), _ptr(scale), _ptr(out_t), _ptr(scale_t), _ptr(ws), nbytes)
    elif colwise:
        scale_t.fill_(2.0 ** -40 / 127)
    if rowwise and not cols:
        scale.fill_(2.0 ** -40 / 127)
    return q


def _int8_matrix(who, **tensors):
    for name, t in tensors.items():
        if t.dtype is not torch.int8:
            raise TypeError(f"{who}: {name} must be int8 codes (got {t.dtype})")
        if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
            _byte_matrix(who, **{name: t})


def _int8_scale(who, name, t, rows):
    """The scales of an operand of ``rows`` rows as the kernels read them."""
    if t.dtype is not torch.float32 or t.shape != (rows,):
        raise ValueError(f"{who}: {name} must be float32 [{rows}] (got {t.dtype} {tuple(t.shape)})")
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.contiguous().clone()


def dequant_int8(q, *, transpose=False):
    """The values of an :class:`Int8Tensor` as bf16 [rows, cols] (the fp32 product of code and scale, rounded), or with
    ``transpose`` those of its columnwise copy, [cols, rows] (a view of rows padded to 16 where rows
    is not a multiple)."""
    who = "dequant_int8"
    codes, scale = (q.data_t, q.col_scale) if transpose else (q.data, q.row_scale)
    if codes is None:
        raise ValueError(f"{who}: the tensor has no {'columnwise' if transpose else 'rowwise'} copy")
    idx = _index_of(who, codes, scale)
    _int8_matrix(who, codes=codes)
    codes = codes.contiguous()
    codes = codes if codes.data_ptr() % 8 == 0 else codes.clone()
    rows, cols = codes.shape
    scale = _int8_scale(who, "scale", scale, rows)
    out = torch.empty((rows, cols), dtype=torch.bfloat16, device=codes.device)
    if rows and cols:
        _call("bf8_dequant_int8", idx, _lib.lib().bf8_dequant_int8, codes.data_ptr(), scale.data_ptr(),
              rows, cols, out.data_ptr())
    return out[:, :q.rows] if transpose and q.rows != cols else out


def _linear_bias(who, bias, N):
    if bias.dtype is not torch.bfloat16 or bias.numel() != N:
        raise ValueError(f"{who}: bias must be bfloat16 [{N}] (got {bias.dtype} {tuple(bias.shape)})")
    bias = bias.contiguous()
    return bias if bias.data_ptr() % 8 == 0 else bias.clone()


def gemm_int8(a, a_scale, b, b_scale, *, bias=None, out_dtype=torch.bfloat16, out=None):
    """``C = a_scale[:, None] * b_scale * (A @ B.T) (+ bias)`` of int8 codes A [M, K] and B [N, K] with
    fp32 scales [M] and [N] (as :func:`quantize_int8` writes them) on the int8 MFMA; the sums are exact in
    int32. K a multiple of 16, 133120 at most (131056 for codes of -128, which no quantizer here writes), N of 8;
    C bf16 or fp32. The scales' product is formed first, in fp32: past its range C is inf, or NaN where the sum is 0."""
    who = "gemm_int8"
    idx = _index_of(who, a, a_scale, b, b_scale, bias, out)
    _int8_matrix(who, a=a, b=b)
    M, K = a.shape
    N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"{who}: inner dims differ ({K} vs {Kb})")
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise TypeError(f"{who}: out_dtype must be bfloat16 or float32")
    a_scale, b_scale = _int8_scale(who, "a_scale", a_scale, M), _int8_scale(who, "b_scale", b_scale, N)
    if out is None:
        out, ldc = torch.empty((M, N), dtype=out_dtype, device=a.device), N
    else:
        _out_matrix(who, out, (M, N), out_dtype)
        ldc = out.stride(0) if M > 1 else N
    if bias is not None:
        bias = _linear_bias(who, bias, N)
    if K == 0:  # an empty sum
        return out.zero_() if bias is None else out.copy_(bias.reshape(1, N).expand(M, N))
    L, ws = _lib.lib(), None
    ws_bytes = L.bf8_gemm_int8_workspace(M, N, K)
    if ws_bytes:
        ws, ws_bytes = _call_workspace(ws_bytes, a)
    # (a single row's stride(0) may be anything)
    _call("bf8_gemm_int8", idx, L.bf8_gemm_int8, a.data_ptr(), a.stride(0) if M > 1 else K,
          a_scale.data_ptr(), b.data_ptr(), b.stride(0) if N > 1 else K, b_scale.data_ptr(), M, N, K,
          _ptr(bias), out.data_ptr(), OUT_BF16 if out_dtype is torch.bfloat16 else OUT_F32, ldc, _ptr(ws),
          ws_bytes)
    return out


def linear_int8(x, w, w_scale, *, bias=None, out_dtype=torch.bfloat16):
    """A linear layer of int8 weights in serving: ``y = x @ W.T (+ bias)`` with bf16 x [..., K]
    quantized by token in the call and W as codes [N, K] under ``w_scale`` [N]. No gradients
    (:class:`bongard_amd.linear.Int8LinearFunction` has them)."""
    who = "linear_int8"
    idx = _index_of(who, x, w, w_scale, bias)
    _int8_matrix(who, w=w)
    shape = x.shape
    N, K = w.shape
    if shape[-1] != K:
        raise ValueError(f"{who}: inner dims differ ({shape[-1]} vs {K})")
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise TypeError(f"{who}: out_dtype must be bfloat16 or float32")
    w_scale = _int8_scale(who, "w_scale", w_scale, N)
    if bias is not None:
        bias = _linear_bias(who, bias, N)
    x = _rows_bf16(x)
    M = x.shape[0]
    out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    if K == 0:  # an empty sum
        out = out.zero_() if bias is None else out.copy_(bias.reshape(1, N).expand(M, N))
    elif M:
        L, ws = _lib.lib(), None
        ws_bytes = L.bf8_linear_int8_workspace(M, N, K)
        if ws_bytes:
            ws, ws_bytes = _call_workspace(ws_bytes, x)
        _call("bf8_linear_int8", idx, L.bf8_linear_int8, x.data_ptr(), w.data_ptr(),
              w.stride(0) if N > 1 else K, w_scale.data_ptr(), M, N, K, _ptr(bias), out.data_ptr(),
              OUT_BF16 if out_dtype is torch.bfloat16 else OUT_F32, N, _ptr(ws), ws_bytes)
    return out if len(shape) == 2 else out.view(*shape[:-1], N)


@functools.lru_cache(maxsize=4096)
def _linear_int8_forward_ws_cached(M, N, K, keep_x, keep_w):
    return int(_lib.lib().bf8_linear_int8_forward_workspace(M, N, K, keep_x, keep_w))


def linear_int8_forward(x, w, *, bias=None, keep_x=False, keep_w=False):
    """The training forward of an int8 linear in one call: ``(y, x_t, x_t_scale, w_t, w_t_scale)``, y bf16 [M, N]
    of bf16 x [M, K] and w [N, K], both quantized by row, and with ``keep_x`` (``keep_w``) the columnwise codes
    and scales that :func:`linear_int8_backward` takes (else None). The values are :func:`quantize_int8`'s and
    :func:`gemm_int8`'s. K a multiple of 16, N of 8."""
    who = "linear_int8_forward"
    idx = _index_of(who, x, w, bias)
    x, w = _rows_bf16(x), _rows_bf16(w)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"{who}: inner dims differ ({K} vs {w.shape[1]})")
    if bias is not None:
        bias = _linear_bias(who, bias, N)
    if not (M and N and K):  # nothing to launch, or an empty sum
        xq, wq = quantize_int8(x, colwise=keep_x), quantize_int8(w, colwise=keep_w)
        y = gemm_int8(xq.data, xq.row_scale, wq.data, wq.row_scale, bias=bias)
        return y, xq.data_t, xq.col_scale, wq.data_t, wq.col_scale
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    x_t = x_t_scale = w_t = w_t_scale = None
    if keep_x:
        x_t = torch.empty((K, (M + 15) // 16 * 16), dtype=torch.int8, device=x.device)
        x_t_scale = torch.empty(K, dtype=torch.float32, device=x.device)
    if keep_w:
        w_t = torch.empty((K, (N + 15) // 16 * 16), dtype=torch.int8, device=x.device)
        w_t_scale = torch.empty(K, dtype=torch.float32, device=x.device)
    ws, nbytes = _call_workspace(_linear_int8_forward_ws_cached(M, N, K, keep_x, keep_w), x)
    _call("bf8_linear_int8_forward", idx, _lib.lib().bf8_linear_int8_forward, x.data_ptr(), w.data_ptr(), M, N, K,
          _ptr(bias), y.data_ptr(), _ptr(x_t), _ptr(x_t_scale), _ptr(w_t), _ptr(w_t_scale), ws.data_ptr(), nbytes)
    return y, x_t, x_t_scale, w_t, w_t_scale


@functools.lru_cache(maxsize=4096)
def _linear_int8_backward_ws_cached(M, N, K, dx, dw):
    return int(_lib.lib().bf8_linear_int8_backward_workspace(M, N, K, dx, dw))


def linear_int8_backward(dy, w_t=None, w_t_scale=None, x_t=None, x_t_scale=None):
    """Gradients ``(dx, dw)`` of an int8 linear for bf16 ``dy`` [M, N] in one call: ``dy`` quantized by token
    for dx [M, K], the product with ``w_t`` [K, N] (W's columnwise codes, scales ``w_t_scale`` [K]), and by
    channel for dw [N, K], the product with ``x_t`` [K, M rounded up to 16] (x's, ``x_t_scale`` [K]). Without
    ``w_t`` (``x_t``) dx (dw) is None. The values are :func:`quantize_int8`'s and :func:`gemm_int8`'s. N a
    multiple of 16, K of 8; for dw M at most 133120."""
    who = "linear_int8_backward"
    idx = _index_of(who, dy, w_t, w_t_scale, x_t, x_t_scale)
    dy = _rows_bf16(dy)
    M, N = dy.shape
    if w_t is None and x_t is None:
        raise ValueError(f"{who}: nothing requested")
    K = (x_t if w_t is None else w_t).shape[0]

    def operand(name, t, scale, cols):
        if t is None:
            return None, None
        if t.dtype is not torch.int8 or t.shape != (K, cols):
            raise ValueError(f"{who}: {name} must be int8 [{K}, {cols}] (got {t.dtype} {tuple(t.shape)})")
        if scale is None:
            raise ValueError(f"{who}: {name} needs {name}_scale")
        t = t.contiguous()
        return t if t.data_ptr() % 16 == 0 else t.clone(), _int8_scale(who, f"{name}_scale", scale, K)

    w_t, w_t_scale = operand("w_t", w_t, w_t_scale, N)
    x_t, x_t_scale = operand("x_t", x_t, x_t_scale, (M + 15) // 16 * 16)
    return _linear_int8_backward(idx, dy, K, w_t, w_t_scale, x_t, x_t_scale)


def _linear_int8_backward(idx, dy, K, w_t, w_t_scale, x_t, x_t_scale):
    """:func:`linear_int8_backward` of what its checks or the forward's have seen."""
    M, N = dy.shape
    dx = None if w_t is None else torch.empty((M, K), dtype=torch.bfloat16, device=dy.device)
    dw = None if x_t is None else torch.empty((N, K), dtype=torch.bfloat16, device=dy.device)
    if not (M and N and K):  # sums of nothing
        for t in (dx, dw):
            if t is not None:
                t.zero_()
        return dx, dw
    ws, nbytes = _call_workspace(_linear_int8_backward_ws_cached(M, N, K, dx is not None, dw is not None), dy)
    _call("bf8_linear_int8_backward", idx, _lib.lib().bf8_linear_int8_backward, dy.data_ptr(), M, N, K, _ptr(w_t),
          _ptr(w_t_scale), _ptr(x_t), _ptr(x_t_scale), _ptr(dx), _ptr(dw), ws.data_ptr(), nbytes)
    return dx, dw


@dataclass
class MxInt8Tensor:
    """An 8-bit checkpoint of a bf16 tensor [rows, cols]: ``data`` int8 [rows, cols] and ``exps`` uint8
    [rows, ceil(cols / 32)], one for each block of 32 along a row; the values are
    data * 2^(exps - 133) (255: NaN), which bf16 holds exactly."""

    data: torch.Tensor
    exps: torch.Tensor


def _new_mxint8(rows, cols, device):
    return MxInt8Tensor(torch.empty((rows, cols), dtype=torch.int8, device=device),
                        torch.empty((rows, (cols + 31) // 32), dtype=torch.uint8, device=device))


def _mxint8_of(who, q, rows, cols):
    if (q.data.dtype is not torch.int8 or q.exps.dtype is not torch.uint8 or q.data.shape != (rows, cols)
            or q.exps.shape != (rows, (cols + 31) // 32)):
        raise ValueError(f"{who}: the checkpoint must be int8 [{rows}, {cols}] with uint8 exponents "
                         f"[{rows}, {(cols + 31) // 32}] (got {q.data.dtype} {tuple(q.data.shape)}, "
                         f"{q.exps.dtype} {tuple(q.exps.shape)})")
    data = q.data.contiguous()
    return data if data.data_ptr() % 8 == 0 else data.clone(), q.exps.contiguous()


def quantize_mxint8(x):
    """The 8-bit checkpoint of a bf16 tensor (flattened to [rows, cols], cols a multiple of 8) as a
    :class:`MxInt8Tensor`: of each block of 32 along a row the least power of two at which its largest
    value is within 127 steps, and the values to the nearest step (ties to even); a block that
    holds inf or NaN reads back as NaN."""
    idx = _index_of("quantize_mxint8", x)
    x = _rows_bf16(x)
    rows, cols = x.shape
    q = _new_mxint8(rows, cols, x.device)
    if rows and cols:
        _call("bf8_quantize_mxint8_bf16", idx, _lib.lib().bf8_quantize_mxint8_bf16, x.data_ptr(), rows,
              cols, q.data.data_ptr(), q.exps.data_ptr())
    return q


def dequant_mxint8(q):
    """The values of a :class:`MxInt8Tensor` as bf16 [rows, cols]."""
    who = "dequant_mxint8"
    idx = _index_of(who, q.data, q.exps)
    rows, cols = q.data.shape
    data, exps = _mxint8_of(who, q, rows, cols)
    out = torch.empty((rows, cols), dtype=torch.bfloat16, device=data.device)
    if rows and cols:
        _call("bf8_dequant_mxint8", idx, _lib.lib().bf8_dequant_mxint8, data.data_ptr(), exps.data_ptr(),
              rows, cols, out.data_ptr())
    return out


def gemm_geglu_int8(x, x_scale, w, w_scale, intermediate, *, keep_gu=False):
    """Gate/up product of int8 operands X [M, K] and W [2I, K] (gate rows then up rows) with the gated
    GELU: ``(H, checkpoint or None)``, H bf16 [M, I] = gelu_tanh(gate) * up (gate, up, the activation
    and H rounded to bf16, as :func:`geglu` does) and, with ``keep_gu``, the :class:`MxInt8Tensor` of the
    bf16 pre-activations. I must be a multiple of 128."""
    who = "gemm_geglu_int8"
    idx = _index_of(who, x, x_scale, w, w_scale)
    _int8_matrix(who, x=x, w=w)
    I = int(intermediate)
    M, K = x.shape
    N, Kw = w.shape
    if N != 2 * I or K != Kw:
        raise ValueError(f"{who}: w must have {2 * I} rows of {K} values (got {N} of {Kw})")
    if I % 128:
        raise ValueError(f"{who}: the intermediate size must be a multiple of 128 (got {I})")
    if K == 0:
        raise ValueError(f"{who}: K must not be 0")
    x_scale, w_scale = _int8_scale(who, "x_scale", x_scale, M), _int8_scale(who, "w_scale", w_scale, N)
    H = torch.empty((M, I), dtype=torch.bfloat16, device=x.device)
    gu = _new_mxint8(M, N, x.device) if keep_gu else None
    if M and I:
        _call("bf8_gemm_geglu_int8", idx, _lib.lib().bf8_gemm_geglu_int8, x.data_ptr(),
              x.stride(0) if M > 1 else K, x_scale.data_ptr(), w.data_ptr(), w.stride(0),
              w_scale.data_ptr(), M, I, K, H.data_ptr(), gu.data.data_ptr() if keep_gu else None,
              gu.exps.data_ptr() if keep_gu else None)
    return H, gu


def linear_geglu_int8(x, w, w_scale):
    """A gate/up projection of int8 weights in serving with the gated GELU: H bf16 [..., I] of bf16 x [..., K]
    quantized by token in the call and W as codes [2I, K] (gate rows then up rows) under ``w_scale`` [2I], as
    :func:`gemm_geglu_int8` computes it. I a multiple of 128. No gradients
    (:class:`bongard_amd.linear.Int8GegluMlpFunction` has them)."""
    who = "linear_geglu_int8"
    idx = _index_of(who, x, w, w_scale)
    _int8_matrix(who, w=w)
    shape = x.shape
    N, K = w.shape
    if shape[-1] != K:
        raise ValueError(f"{who}: inner dims differ ({shape[-1]} vs {K})")
    if N % 256 or K == 0:
        raise ValueError(f"{who}: the intermediate size must be a multiple of 128 and K not 0 (got {tuple(w.shape)})")
    I = N // 2
    w_scale = _int8_scale(who, "w_scale", w_scale, N)
    x = _rows_bf16(x)
    M = x.shape[0]
    out = torch.empty((M, I), dtype=torch.bfloat16, device=x.device)
    if M and I:
        L, ws = _lib.lib(), None
        ws_bytes = L.bf8_linear_geglu_int8_workspace(M, I, K)
        if ws_bytes:
            ws, ws_bytes = _call_workspace(ws_bytes, x)
        _call("bf8_linear_geglu_int8", idx, L.bf8_linear_geglu_int8, x.data_ptr(), w.data_ptr(), w.stride(0),
              w_scale.data_ptr(), M, I, K, out.data_ptr(), _ptr(ws), ws_bytes)
    return out if len(shape) == 2 else out.view(*shape[:-1], I)


def geglu_mlp_int8(x, w_gu, w_gu_scale, w_down, w_down_scale):
    """The gated MLP of int8 weights in serving: bf16 x [..., K], W_gu as codes [2I, K] (gate rows then
    up rows) and W_down [N, I], each with its scales; x and the activation are quantized by token in the
    call. No gradients (:class:`bongard_amd.linear.Int8GegluMlpFunction` has them)."""
    return linear_int8(linear_geglu_int8(x, w_gu, w_gu_scale), w_down, w_down_scale)


def geglu_mxint8(GU):
    """:func:`geglu` whose pre-activations are kept for the backward in 8 bits: ``(H bf16 [M, I], the
    MxInt8Tensor of GU [M, 2I])`` from bf16 GU in one pass. I must be a multiple of 32."""
    who = "geglu_mxint8"
    idx = _index_of(who, GU)
    if GU.dtype is not torch.bfloat16 or GU.dim() != 2 or GU.shape[1] % 64:
        raise ValueError(f"{who}: GU must be bf16 [M, 2I], I a multiple of 32 (got {GU.dtype} "
                         f"{tuple(GU.shape)})")
    GU = _rows_bf16(GU)
    M, I = GU.shape[0], GU.shape[1] // 2
    H, q = torch.empty((M, I), dtype=torch.bfloat16, device=GU.device), _new_mxint8(M, 2 * I, GU.device)
    if M and I:
        _call("bf8_geglu_mxint8", idx, _lib.lib().bf8_geglu_mxint8, GU.data_ptr(), M, I, H.data_ptr(),
              q.data.data_ptr(), q.exps.data_ptr())
    return H, q


@functools.lru_cache(maxsize=4096)
def _geglu_mlp_int8_forward_ws_cached(*args):
    return int(_lib.lib().bf8_geglu_mlp_int8_forward_workspace(*args))


def _geglu_mlp_int8_forward(x, I, gu_q, down_q, keep_gu, keep_x, keep_h):
    """The gated int8 MLP of bf16 x [M, K], M > 0, and the rowwise copies of its weights, in one call: ``(y, checkpoint
    codes, its exponents, x_t, x_t_scale, h_t, h_t_scale)``, None where not kept. The values are
    :func:`quantize_int8`'s, :func:`gemm_geglu_int8`'s and :func:`gemm_int8`'s."""
    who = "geglu_mlp_int8_forward"
    idx = _index_of(who, x, gu_q.data, gu_q.row_scale, down_q.data, down_q.row_scale)
    x = _rows_bf16(x)
    M, K = x.shape
    N = down_q.rows
    if (gu_q.rows, gu_q.cols, down_q.cols) != (2 * I, K, I):
        raise ValueError(f"{who}: weights [{gu_q.rows}, {gu_q.cols}] and [{N}, {down_q.cols}] for x [..., {K}] and the "
                         f"intermediate size {I}")
    weights = [t.contiguous() for t in (gu_q.data, gu_q.row_scale, down_q.data, down_q.row_scale)]
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    gu = _new_mxint8(M, 2 * I, x.device) if keep_gu else None
    copies = [None] * 4
    for at, keep, n in ((0, keep_x, K), (2, keep_h, I)):
        if keep:
            copies[at] = torch.empty((n, (M + 15) // 16 * 16), dtype=torch.int8, device=x.device)
            copies[at + 1] = torch.empty(n, dtype=torch.float32, device=x.device)
    ws, nbytes = _call_workspace(_geglu_mlp_int8_forward_ws_cached(M, K, I, N, keep_x, keep_h), x)
    data, exps = (gu.data, gu.exps) if keep_gu else (None, None)
    _call("bf8_geglu_mlp_int8_forward", idx, _lib.lib().bf8_geglu_mlp_int8_forward, x.data_ptr(), M, K, I, N,
          *(t.data_ptr() for t in weights), y.data_ptr(), _ptr(data), _ptr(exps), *(_ptr(t) for t in copies), ws.data_ptr(), nbytes)
    return (y, data, exps, *copies)


@functools.lru_cache(maxsize=4096)
def _geglu_mlp_int8_backward_ws_cached(*args):
    return int(_lib.lib().bf8_geglu_mlp_int8_backward_workspace(*args))


def _geglu_mlp_int8_backward(dy, K, I, needs, gu8, gu_exps, x_t, x_t_scale, h_t, h_t_scale, gu_t, gu_t_scale, down_t,
                             down_t_scale):
    """Gradients ``(dx, dW_gu, dW_down)`` (those of ``needs``, the others None) of the gated int8 MLP for bf16 dy
    [M, N], M > 0, from the columnwise codes and the checkpoint that its forward kept:
    :func:`linear_int8_backward` on H and W_down, :func:`geglu_bwd_mxint8`, the products with x and W_gu."""
    dy = _rows_bf16(dy)
    M, N = dy.shape
    dx, dgu, dd = (torch.empty(shape, dtype=torch.bfloat16, device=dy.device) if n else None
                   for n, shape in zip(needs, ((M, K), (2 * I, K), (N, I))))
    ws, nbytes = _call_workspace(_geglu_mlp_int8_backward_ws_cached(M, K, I, N, *needs), dy)
    _call("bf8_geglu_mlp_int8_backward", dy.get_device(), _lib.lib().bf8_geglu_mlp_int8_backward, dy.data_ptr(), M, K,
          I, N, _ptr(gu8), _ptr(gu_exps), _ptr(x_t), _ptr(x_t_scale), _ptr(h_t), _ptr(h_t_scale), _ptr(gu_t),
          _ptr(gu_t_scale), _ptr(down_t), _ptr(down_t_scale), _ptr(dx), _ptr(dgu), _ptr(dd), ws.data_ptr(), nbytes)
    return dx, dgu, dd


@functools.lru_cache(maxsize=4096)
def _geglu_bwd_maxima_cached(M, I):
    return int(_lib.lib().bf8_geglu_bwd_mxint8_maxima(M, I))


def _geglu_bwd_mxint8(idx, dH, data, exps):
    """:func:`geglu_bwd_mxint8` of what its checks or the forward's have seen."""
    M, I = dH.shape
    dGU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=dH.device)
    if M and I:
        _call("bf8_geglu_bwd_mxint8", idx, _lib.lib().bf8_geglu_bwd_mxint8, dH.data_ptr(),
              data.data_ptr(), exps.data_ptr(), M, I, dGU.data_ptr(), None, 0)
    return dGU


def geglu_bwd_mxint8(dH, gu, *, rowwise=False, colwise=False):
    """:func:`geglu_bwd` on the values of GU's checkpoint: dGU bf16 [M, 2I], or with ``rowwise`` or
    ``colwise`` that tensor's :func:`quantize_int8` instead (from 1024 rows on, and where its rows are too wide for
    that, by the maxima that the backward's kernel leaves: the same codes and scales)."""
    who = "geglu_bwd_mxint8"
    idx = _index_of(who, dH, gu.data, gu.exps)
    dH = _rows_bf16(dH)
    M, I = dH.shape
    if I % 32:
        raise ValueError(f"{who}: the intermediate size must be a multiple of 32 (got {I})")
    data, exps = _mxint8_of(who, gu, M, 2 * I)
    if not (rowwise or colwise):
        return _geglu_bwd_mxint8(idx, dH, data, exps)
    # both copies of dGU's codes, by the maxima and by the quantizer's own pass, us: [512, 2 x 10240] 32.5 and
    # 31.5, [1500, 2 x 2560] 27.5 and 29.9, [4096, 2 x 10240] 157 and 168
    if M < 1024 and I <= 16384 or not (M and I):
        return quantize_int8(geglu_bwd_mxint8(dH, gu), rowwise=rowwise, colwise=colwise)
    dGU = torch.empty((M, 2 * I), dtype=torch.bfloat16, device=dH.device)
    L = _lib.lib()
    ws, nbytes = _call_workspace(_geglu_bwd_maxima_cached(M, I), dH)
    _call("bf8_geglu_bwd_mxint8", idx, L.bf8_geglu_bwd_mxint8, dH.data_ptr(), data.data_ptr(),
          exps.data_ptr(), M, I, dGU.data_ptr(), ws.data_ptr(), nbytes)
    q = _new_int8(M, 2 * I, rowwise, colwise, dH.device)
    _call("bf8_quantize_int8_maxima_bf16", idx, L.bf8_quantize_int8_maxima_bf16, dGU.data_ptr(), M, 2 * I, 2,
          _ptr(q.data), _ptr(q.row_scale), _ptr(q.data_t), _ptr(q.col_scale), ws.data_ptr(), nbytes)
    return q


def column_sums(x):
    """bf16 [cols] sums over the rows of a bf16 tensor (flattened to [rows, cols], cols a multiple of 8),
    in fp32 and a fixed order: the gradient of a bias."""
    idx = _index_of("column_sums", x)
    x = _rows_bf16(x)
    rows, cols = x.shape
    if not rows:
        return x.new_zeros(cols)
    out = torch.empty(cols, dtype=torch.bfloat16, device=x.device)
    if cols:
        L = _lib.lib()
        ws, nbytes = _call_workspace(L.bf8_column_sums_workspace(rows, cols), x)
        _call("bf8_column_sums_bf16", idx, L.bf8_column_sums_bf16, x.data_ptr(), rows, cols,
              out.data_ptr(), ws.data_ptr(), nbytes)
    return out


# ---- layer norm ------------------------------------------------------------------------------
def layernorm(x, weight, bias, eps, *, want_stats=False, checkpoint=False):
    """Layer norm of the rows of a bf16 tensor [..., cols] (fp32 arithmetic): ``(y, mean, rstd,
    checkpoint)``. ``bias``: bf16 [cols] or None. ``want_stats``: the rows' fp32 mean and 1 / sqrt(var +
    eps) (else None); ``checkpoint``: the :class:`MxInt8Tensor` of x, written in the same pass (else
    None). cols: a multiple of 8, 16384 at most. No gradients
    (:func:`bongard_amd.fused_mlp.layer_norm` has them)."""
    y, stats, q = _layernorm(x, weight, bias, eps, want_stats, checkpoint)
    mean, rstd = (None, None) if stats is None else stats.unbind(0)
    return y, mean, rstd, q


def _layernorm(x, weight, bias, eps, want_stats, checkpoint):
    """:func:`layernorm` with the statistics as one tensor [2, rows]: ``(y, statistics, checkpoint)``."""
    who = "layernorm"
    idx = _index_of(who, x, weight, bias)
    shape = x.shape
    weight = _norm_weight(who, "weight", weight, shape[-1])
    bias = None if bias is None else _norm_weight(who, "bias", bias, shape[-1])
    x = _rows_bf16(x)
    rows, cols = x.shape
    y = torch.empty_like(x)
    stats = mean = rstd = q = None
    if want_stats:
        stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    if checkpoint:
        q = _new_mxint8(rows, cols, x.device)
    if rows:
        _call("bf8_layernorm_bf16", idx, _lib.lib().bf8_layernorm_bf16, x.data_ptr(), rows, cols,
              weight.data_ptr(), _ptr(bias), eps, y.data_ptr(), mean, rstd,
              q.data.data_ptr() if checkpoint else None, q.exps.data_ptr() if checkpoint else None)
    return y if len(shape) == 2 else y.view(shape), stats, q


@functools.lru_cache(maxsize=4096)
def _layernorm_ws_cached(rows, cols):
    return int(_lib.lib().bf8_layernorm_bwd_workspace(rows, cols))


def layernorm_backward(x, dy, weight, mean, rstd, *, needs=(True, True, True)):
    """Gradients ``(dx, dweight, dbias)`` of :func:`layernorm` for ``dy``, from the forward's ``mean`` and
    ``rstd`` and its input ``x`` or that input's checkpoint (an :class:`MxInt8Tensor`). ``needs``: which
    to compute (the others are None)."""
    who = "layernorm_backward"
    q = x if isinstance(x, MxInt8Tensor) else None
    idx = _index_of(who, dy, q.data if q else x, q.exps if q else None, weight, mean, rstd)
    shape = dy.shape
    weight = _norm_weight(who, "weight", weight, shape[-1])
    dy = _rows_bf16(dy)
    rows, cols = dy.shape
    if q is not None:
        data, exps = _mxint8_of(who, q, rows, cols)
    elif x.shape != shape:
        raise ValueError(f"{who}: x must be {tuple(shape)} (got {tuple(x.shape)})")
    else:
        x = _rows_bf16(x)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype is not torch.float32 or t.shape != (rows,) or not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be contiguous float32 [{rows}] (got {t.dtype} "
                             f"{tuple(t.shape)})")
    return _layernorm_backward(idx, shape, x, data if q else None, exps if q else None, dy, weight, mean.data_ptr(),
                               rstd.data_ptr(), needs)


def _layernorm_backward(idx, shape, x, data, exps, dy, weight, mean, rstd, needs):
    """:func:`layernorm_backward` of what its checks or the forward's have seen: contiguous and aligned tensors (x
    unread where ``data`` is given), the statistics' addresses."""
    rows, cols = dy.shape
    dx = torch.empty_like(dy) if needs[0] else None
    dw = torch.empty_like(weight) if needs[1] else None
    db = torch.empty_like(weight) if needs[2] else None
    if rows == 0:
        for g in (dw, db):
            if g is not None:
                g.zero_()
    elif any(needs):
        ws, nbytes = None, 0
        if needs[1] or needs[2]:
            ws, nbytes = _call_workspace(_layernorm_ws_cached(rows, cols), dy)
        _call("bf8_layernorm_bwd_bf16", idx, _lib.lib().bf8_layernorm_bwd_bf16,
              x.data_ptr() if data is None else None, _ptr(data), _ptr(exps), dy.data_ptr(), rows, cols,
              weight.data_ptr(), mean, rstd, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
    if dx is not None and len(shape) != 2:
        dx = dx.view(shape)
    return dx, dw, db
