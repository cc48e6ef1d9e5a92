"""Root-mean-square norm with the residual's addition, on the HIP kernels.

`rms_norm` stands beside the LayerNorm of the transformer blocks: the residual stream's sum and its
norm in one pass (`dp_rms_norm`), differentiable (`dp_rms_norm_bwd`). `rms_norm_e4m3` is the
serving form whose output feeds an 8-bit product: e4m3 values and one scale per row.

There is no CPU path: the HIP library must load (see _lib.load()).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_DT = {torch.float32: _lib.DP_F32, torch.bfloat16: _lib.DP_BF16}
_LONGEST = {torch.float32: 8192, torch.bfloat16: 16384}   # elements of a row


def _check(name, x, weight, residual, eps):
    _lib.refuse_tangents(name, x, weight, residual)
    if x.dtype not in _DT:
        raise TypeError(f"{name}: x dtype {x.dtype} (f32 / bf16)")
    if weight.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"{name}: weight dtype {weight.dtype} (f32, or x's {x.dtype})")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _LONGEST[x.dtype]:
        raise ValueError(f"{name}: x {tuple(x.shape)}: rows of 1 to {_LONGEST[x.dtype]} elements of {x.dtype}")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"{name}: weight {tuple(weight.shape)} does not match x {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{name}: residual {tuple(residual.shape)} {residual.dtype} does not match x "
                         f"{tuple(x.shape)} {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"{name}: eps {eps}")
    if not x.is_cuda:
        raise RuntimeError(f"{name}: tensors must be on the GPU (no CPU path)")
    if weight.device != x.device or (residual is not None and residual.device != x.device):
        raise RuntimeError(f"{name}: x on {x.device}, weight on {weight.device}"
                           + (f", residual on {residual.device}" if residual is not None else "")
                           + ": all must be on the same GPU")
    if x.numel() // x.shape[-1] >= 2 ** 31:
        raise ValueError(f"{name}: {x.numel() // x.shape[-1]} rows are too many")


def _rows(t, c):
    """(2-d view or copy with contiguous rows, row stride)."""
    m = t.reshape(-1, c)
    if m.stride(1) != 1 and c > 1:
        m = m.contiguous()
    return m, m.stride(0) if m.shape[0] > 1 else c


def _ptr(t):
    return None if t is None else t.data_ptr()


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        c = x.shape[-1]
        xm, ld_x = _rows(x, c)
        rows = xm.shape[0]
        w = weight.contiguous()
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        rm, ld_r, r = None, 0, None
        if residual is not None:
            rm, ld_r = _rows(residual, c)
            r = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        need = any(ctx.needs_input_grad[:3])
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if need else None
        if rows:
            with _lib.device_of(x):
                s = torch.cuda.current_stream().cuda_stream
                _lib.check(_lib.load().dp_rms_norm(y.data_ptr(), _ptr(r), _ptr(rstd), xm.data_ptr(), ld_x, _ptr(rm),
                                                   ld_r, w.data_ptr(), _DT[w.dtype], eps, rows, c, _DT[x.dtype],
                                                   C.c_void_p(s)), "dp_rms_norm")
        if need:
            ctx.save_for_backward(x if r is None else r, w, rstd)
            ctx.has_residual = r is not None
            ctx.set_materialize_grads(False)
        return y if r is None else (y, r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dres=None):
        r, w, rstd = ctx.saved_tensors
        c = r.shape[-1]
        if dy is None:   # only the sum was used
            dw = torch.zeros_like(w) if ctx.needs_input_grad[1] else None
            return dres, dw, dres if ctx.has_residual else None, None
        rm, ld_r = _rows(r, c)
        rows = rm.shape[0]
        dx = torch.empty(r.shape, device=r.device, dtype=r.dtype)
        if not rows:
            return dx, torch.zeros_like(w), dx if ctx.has_residual else None, None
        dw = torch.empty_like(w)
        dym, ld_dy = _rows(dy.to(r.dtype), c)
        drm, ld_dr = (None, 0) if dres is None else _rows(dres.to(r.dtype), c)
        lib = _lib.load()
        with _lib.device_of(r):
            n = int(lib.dp_rms_norm_bwd_ws_floats(rows, c, _DT[r.dtype]))
            ws = torch.empty(n, device=r.device, dtype=torch.float32)
            s = torch.cuda.current_stream().cuda_stream
            _lib.check(lib.dp_rms_norm_bwd(dx.data_ptr(), dw.data_ptr(), rm.data_ptr(), ld_r, rstd.data_ptr(),
                                           dym.data_ptr(), ld_dy, _ptr(drm), ld_dr, w.data_ptr(), _DT[w.dtype],
                                           ws.data_ptr(), n, rows, c, _DT[r.dtype], C.c_void_p(s)),
                       "dp_rms_norm_bwd")
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x (..., c) f32 / bf16, weight (c,) f32 or x's type -> y = r / sqrt(mean r^2 + eps) * weight with
    r = x, or, with a residual of x's shape and type, r = x + residual rounded to that type; then
    (y, r) is returned, r being the residual stream behind this addition. Sums and the norm are f32.
    Rows of up to 16384 bf16 or 8192 f32 elements. Differentiable (once, in reverse) in x, weight
    and residual."""
    _check("rms_norm", x, weight, residual, eps)
    return RMSNormFunction.apply(x, weight, residual, float(eps))


def rms_norm_e4m3(x, weight, residual=None, eps=1e-6):
    """The same norm with an 8-bit output, for serving: (y, scale, r) with y (..., c) float8_e4m3fn and
    scale (...) f32, y * scale[..., None] standing for the norm: scale = max |norm| / 448 of its row, 2^-126 at
    least (a row of zeros has scale 0). r = x + residual, or None without a residual. Has no gradient."""
    _check("rms_norm_e4m3", x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_e4m3: the 8-bit form has no gradient (use rms_norm, or torch.no_grad())")
    c = x.shape[-1]
    xm, ld_x = _rows(x, c)
    rows = xm.shape[0]
    w = weight.contiguous()
    y = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    rm, ld_r, r = None, 0, None
    if residual is not None:
        rm, ld_r = _rows(residual, c)
        r = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if rows:
        with _lib.device_of(x):
            s = torch.cuda.current_stream().cuda_stream
            _lib.check(_lib.load().dp_rms_norm_e4m3(y.data_ptr(), scale.data_ptr(), _ptr(r), xm.data_ptr(), ld_x,
                                                    _ptr(rm), ld_r, w.data_ptr(), _DT[w.dtype], eps, rows, c,
                                                    _DT[x.dtype], C.c_void_p(s)), "dp_rms_norm_e4m3")
    return y, scale, r
