"""RMSNorm / LayerNorm ops (``csrc/norms.cu``) with autograd and an optional fused residual add.

``rms_norm(x, w, eps)`` follows the reference definition ``x * (mean(x^2) + eps)^-1/2 * w``
(crates/brain-transformer/src/ops.rs:103-131); ``layer_norm`` uses the biased variance with eps
inside the square root (crates/brain-transformer/src/ops.rs:57-101). ``add_rms_norm(x, r, w)``
returns ``(norm(x + r), x + r)`` like ``fused_add_rmsnorm`` (crates/brain-core/src/tensor/ops_fused.rs:77-125).

If the weight carries a ``main_grad`` buffer (flat gradient storage used by the data-parallel
engine), its gradient is accumulated there by the kernel and autograd receives ``None``.
"""
from __future__ import annotations

import torch

from .. import _native
from ._common import (dtype_code, has_main_grad, launch, main_grad_beta, no_backward, ptr, rows2d, same_device,
                      stream)

_RMS, _LN = 0, 1


def _fwd(kind, x2, w, b, eps, res2=None):
    M, D = x2.shape
    y = torch.empty_like(x2)
    rstd = torch.empty(M, device=x2.device, dtype=torch.float32)
    mean = torch.empty(M, device=x2.device, dtype=torch.float32) if kind == _LN else None
    s = torch.empty_like(x2) if res2 is not None else None
    _native.call(
        "brain_norm_fwd", kind, x2.data_ptr(), x2.stride(0), ptr(res2), res2.stride(0) if res2 is not None else 0,
        w.data_ptr(), ptr(b), y.data_ptr(), y.stride(0), ptr(s), s.stride(0) if s is not None else 0,
        ptr(mean), rstd.data_ptr(), M, D, float(eps), stream(x2))
    return y, s, mean, rstd


def _bwd(kind, dy2, x2, w, b, mean, rstd, dres2=None):
    """Returns (dx, dw, db); dw/db are None when accumulated into main_grad."""
    M, D = x2.shape
    dx = torch.empty_like(x2)
    P = _native.fn("brain_norm_bwd_partials")(M)
    ws = torch.empty(2 * P * D, device=x2.device, dtype=torch.float32)
    use_main = has_main_grad(w)
    if use_main:
        dw = w.main_grad
        db = b.main_grad if (b is not None and has_main_grad(b)) else None
        dw_f32 = int(dw.dtype == torch.float32)
        bw = main_grad_beta(w)
        bb = main_grad_beta(b) if db is not None else bw
        if bw != bb:  # one accumulate flag covers both: clear the fresh one and accumulate into both
            (dw if bw == 0.0 else db).zero_()
            bw = 1.0
        acc = int(bw != 0.0)
    else:
        dw = torch.empty(D, device=x2.device, dtype=torch.float32)
        db = torch.empty(D, device=x2.device, dtype=torch.float32) if b is not None else None
        dw_f32, acc = 1, 0
    _native.call(
        "brain_norm_bwd", kind, dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), w.data_ptr(),
        ptr(mean), rstd.data_ptr(), dx.data_ptr(), dx.stride(0), ptr(dres2), dres2.stride(0) if dres2 is not None else 0,
        dw.data_ptr(), ptr(db), dw_f32, acc, ws.data_ptr(), M, D, stream(x2))
    if use_main:
        return dx, None, None
    return dx, dw.to(w.dtype), (db.to(b.dtype) if db is not None else None)


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, kind):
        x2 = rows2d(x)
        y, _, mean, rstd = _fwd(kind, x2, w, b, eps)
        ctx.save_for_backward(x2, w, b, mean, rstd)
        ctx.kind = kind
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w, b, mean, rstd = ctx.saved_tensors
        dx, dw, db = _bwd(ctx.kind, rows2d(dy), x2, w, b, mean, rstd)
        return dx.view(ctx.shape), dw, db, None, None


class _AddNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, w, b, eps, kind):
        x2, r2 = rows2d(x), rows2d(r)
        y, s, mean, rstd = _fwd(kind, x2, w, b, eps, r2)
        ctx.save_for_backward(s, w, b, mean, rstd)
        ctx.kind = kind
        ctx.shape = x.shape
        return y.view(x.shape), s.view(x.shape)

    @staticmethod
    def backward(ctx, dy, ds):
        s, w, b, mean, rstd = ctx.saved_tensors
        ds2 = rows2d(ds) if ds is not None else None
        dx, dw, db = _bwd(ctx.kind, rows2d(dy), s, w, b, mean, rstd, ds2)
        dx = dx.view(ctx.shape)
        return dx, dx, dw, db, None, None


# ------------------------------------------------------------------ CPU oracle restatements
def rms_norm_ref(x, w, eps):
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    return y.to(x.dtype)


def layer_norm_ref(x, w, b, eps):
    xf = x.float()
    mu = xf.mean(-1, keepdim=True)
    var = (xf - mu).pow(2).mean(-1, keepdim=True)
    y = (xf - mu) * torch.rsqrt(var + eps) * w.float()
    if b is not None:
        y = y + b.float()
    return y.to(x.dtype)


# ------------------------------------------------------------------ public ops
def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    if x.is_cuda:
        return _NormFn.apply(x, w, None, eps, _RMS)
    return rms_norm_ref(x, w, eps)


def layer_norm(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    if x.is_cuda:
        return _NormFn.apply(x, w, b, eps, _LN)
    return layer_norm_ref(x, w, b, eps)


def add_rms_norm(x, r, w, eps=1e-6):
    """(rms_norm(x + r), x + r) in one pass."""
    if x.is_cuda:
        return _AddNormFn.apply(x, r, w, None, eps, _RMS)
    s = x + r
    return rms_norm_ref(s, w, eps), s


def add_layer_norm(x, r, w, b=None, eps=1e-5):
    if x.is_cuda:
        return _AddNormFn.apply(x, r, w, b, eps, _LN)
    s = x + r
    return layer_norm_ref(s, w, b, eps), s


def fused_layer_norm(x, w, b=None, eps=1e-5):
    """LayerNorm with the one-pass variance of the reference's fused variant: var = max(E[x^2] - E[x]^2, 0)
    (crates/brain-core/src/tensor/ops_fused.rs:43-70). On CUDA tensors the LayerNorm kernel runs; it takes
    the two-pass variance, which equals the one-pass form in exact arithmetic and does not cancel. On the
    CPU float64 inputs are computed in float64 (the reference's precision), others in float32."""
    if x.is_cuda:
        return layer_norm(x, w, b, eps)
    ct = torch.float64 if x.dtype == torch.float64 else torch.float32
    xf = x.to(ct)
    mu = xf.mean(-1, keepdim=True)
    var = (xf.pow(2).mean(-1, keepdim=True) - mu.pow(2)).clamp_min(0.0)
    y = (xf - mu) * torch.rsqrt(var + eps) * w.to(ct)
    if b is not None:
        y = y + b.to(ct)
    return y.to(x.dtype)


# ------------------------------------------------------------------ e4m3 output (inference)
def rms_norm_fp8_ref(s, w, eps, scaling):
    y = s.float()
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    if scaling == "block":
        y = y.view(*s.shape[:-1], s.shape[-1] // 128, 128)
    amax = y.abs().amax(-1)
    scale = torch.where(amax > 0, (amax / 448.0).clamp_min(2.0 ** -126), torch.ones_like(amax))
    return (y / scale[..., None]).to(torch.float8_e4m3fn).view(s.shape), scale


def _norm_fp8(name, x, r, w, eps, scaling):
    if scaling not in ("rowwise", "block"):
        raise ValueError(f"unknown fp8 scaling {scaling!r}")
    shape = x.shape
    D = shape[-1] if shape else 0
    if not 0 < D <= 2 ** 30 or (scaling == "block" and D % 128):
        raise ValueError(f"{name}: last dimension {D} is not " +
                         ("a multiple of 128" if 0 < D <= 2 ** 30 else "one of 1 to 2^30"))
    if w.shape != (D,) or (r is not None and r.shape != shape):
        raise ValueError(f"{name}: x {tuple(x.shape)}, residual {None if r is None else tuple(r.shape)}, "
                         f"weight {tuple(w.shape)}")
    if w.dtype is not x.dtype or (r is not None and r.dtype is not x.dtype):
        raise TypeError(f"{name}: x, the residual and the weight are of one type")
    code = dtype_code(name, x)
    no_backward(name, x, r, w)
    same_device(x, r, w)
    if not x.is_cuda:
        s = x if r is None else (x.float() + r.float()).to(x.dtype)
        return *rms_norm_fp8_ref(s, w, eps, scaling), s
    w = w.contiguous()
    block = scaling == "block"
    if len(shape) == 2 and x.is_contiguous() and (r is None or r.is_contiguous()):  # as below, at less cost a call
        x2, r2, M, ldx, ldr = x, r, shape[0], D, D
        q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
        s = None if r is None else torch.empty_like(x)
    else:
        x2, r2 = rows2d(x), None if r is None else rows2d(r)
        M, ldx, ldr = x2.shape[0], x2.stride(0), 0 if r2 is None else r2.stride(0)
        q = torch.empty(shape, device=x.device, dtype=torch.float8_e4m3fn)
        s = None if r is None else torch.empty(shape, device=x.device, dtype=x.dtype)
    scale = x.new_empty((M, D // 128) if block else M, dtype=torch.float32)
    if len(shape) != 2:
        scale = scale.view(*shape[:-1], D // 128) if block else scale.view(shape[:-1])
    launch(x, "brain_norm_fp8", code, x2.data_ptr(), ldx, ptr(r2), ldr, w.data_ptr(), ptr(s), q.data_ptr(),
           scale.data_ptr(), M, D, int(block), float(eps))
    return q, scale, s


def rms_norm_fp8(x, w, eps=1e-6, scaling: str = "rowwise"):
    """``rms_norm(x, w)`` quantised to e4m3 in the same pass -> (q, scale), the operand that the fp8 GEMMs take
    (``quantization.fp8_gemm_rowwise`` / ``fp8_gemm_blockscaled``): one scale a row (``"rowwise"``, scale of
    x's leading shape) or one per 128 values (``"block"``, [..., D / 128]), amax / 448, at least 2^-126 (1 for
    zeros). The norm is quantised from float32, without a rounding to x's type in between. Inference only."""
    return _norm_fp8("rms_norm_fp8", x, None, w, eps, scaling)[:2]


def add_rms_norm_fp8(x, r, w, eps=1e-6, scaling: str = "rowwise"):
    """``add_rms_norm`` with the e4m3 output of :func:`rms_norm_fp8` -> (q, scale, x + r)."""
    return _norm_fp8("add_rms_norm_fp8", x, r, w, eps, scaling)
