"""Operators of the "gated" dynamics-parameter network, each on hand-written HIP kernels: the
gated linear recurrence over a sequence and its one-step form (csrc/gated_scan.hip), the
root-mean-square norm with the residual's addition and its 8-bit output (csrc/rms_norm.hip),
the product of 8-bit rows (csrc/linear_8bit.hip).

They take GPU tensors of float32, bfloat16 or float16 and run on the current stream of the
tensors' device; states, norms and sums are float32 whatever the element type.  The
reference's only recurrent network is torch.nn.LSTM (kvae/dynamics_parameter_network.py:18-58);
these operators have no counterpart there.
"""
import contextlib
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _capi as capi


def _device_of(*tensors):
    """The one GPU all given tensors are on; raises for CPU tensors and for a mix."""
    capi.require_gpu(*tensors)
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors on different devices: {sorted(map(str, devices))}")
    return devices.pop()


def _on(device):
    """Context in which `device` is the current one (free when it already is)."""
    if torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _rows_dense(t):
    """`t` itself when its last axis has stride 1, a contiguous copy otherwise."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _mask_bytes(mask, shape, device_tensor):
    """(T,B) or (B,) mask of any type as bytes (non-zero: the step counts), or None."""
    if mask is None:
        return None
    if tuple(mask.shape) != tuple(shape):
        raise ValueError(f"mask must have shape {tuple(shape)}, got {tuple(mask.shape)}")
    if mask.dtype not in (torch.bool, torch.uint8):
        mask = mask != 0
    return mask.view(torch.uint8)


def _scan_width(u, output_gate):
    parts = 3 if output_gate else 2
    if u.shape[-1] % parts:
        raise ValueError(f"the last axis of u holds {parts} equal parts "
                         f"({'x, forget, gate' if output_gate else 'x, forget'}), got {u.shape[-1]}")
    return u.shape[-1] // parts


def _state(h0, B, H, name):
    if h0 is None:
        return None
    if tuple(h0.shape) != (B, H):
        raise ValueError(f"{name} must have shape {(B, H)}, got {tuple(h0.shape)}")
    if h0.dtype != torch.float32:
        raise TypeError(f"{name} is float32 whatever the type of u, got {h0.dtype}")
    return h0


def _scan_struct(u, mask, H, gated):
    T, B = u.shape[:2]
    d = capi.GatedScan(T=T, B=B, H=H, dtype=capi.sequence_dtype_code(u.dtype), gated=int(gated),
                       u=u.data_ptr(), u_stride_t=u.stride(0), u_stride_b=u.stride(1))
    if mask is not None:
        d.mask, d.mask_stride_t, d.mask_stride_b = mask.data_ptr(), mask.stride(0), mask.stride(1)
    return d


def _scan_workspace(lib, d, device):
    size = lib.kvae_gated_scan_workspace_bytes(d.T, d.B, d.H, d.dtype)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _scan_forward(u, h0, mask, gated, keep):
    """(y, last, states): states, what the backward pass starts its chunks from, only if `keep`."""
    lib, (T, B) = capi.load(), u.shape[:2]
    H = u.shape[2] // (3 if gated else 2)
    with _on(u.device):
        y = torch.empty(T, B, H, dtype=u.dtype, device=u.device)
        last = torch.empty(B, H, dtype=torch.float32, device=u.device)
        states = torch.empty(-(-T // capi.SCAN_CHUNK) if keep else 0, B, H, dtype=torch.float32,
                             device=u.device)
        d = _scan_struct(u, mask, H, gated)
        d.h0, d.y, d.last = capi.ptr(h0), y.data_ptr(), last.data_ptr()
        d.states = states.data_ptr() if keep else None
        ws = _scan_workspace(lib, d, u.device)
        capi.check(lib.kvae_gated_scan_forward(C.byref(d), capi.ptr(ws), ws.numel() if ws is not None else 0,
                                               _stream(u.device)))
    return y, last, states


class GatedScanFunction(torch.autograd.Function):
    """(u, h0, mask bytes, gated) -> (y, last state)."""

    @staticmethod
    def forward(ctx, u, h0, mask, gated):
        y, last, states = _scan_forward(u, h0, mask, gated, keep=True)
        ctx.save_for_backward(u, mask, states)
        ctx.gated, ctx.has_h0 = gated, h0 is not None
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        u, mask, states = ctx.saved_tensors
        lib, (T, B) = capi.load(), u.shape[:2]
        H = u.shape[2] // (3 if ctx.gated else 2)
        with _on(u.device):
            dy = torch.zeros(T, B, H, dtype=u.dtype, device=u.device) if dy is None else _rows_dense(dy)
            dlast = dlast.contiguous() if dlast is not None else None
            du = torch.empty(u.shape, dtype=u.dtype, device=u.device)
            dh0 = torch.empty(B, H, dtype=torch.float32, device=u.device) if ctx.has_h0 else None
            d = _scan_struct(u, mask, H, ctx.gated)
            d.states, d.dy, d.dlast = states.data_ptr(), dy.data_ptr(), capi.ptr(dlast)
            d.dy_stride_t, d.dy_stride_b = dy.stride(0), dy.stride(1)
            d.du, d.dh0 = du.data_ptr(), capi.ptr(dh0)
            ws = _scan_workspace(lib, d, u.device)
            capi.check(lib.kvae_gated_scan_backward(C.byref(d), capi.ptr(ws),
                                                    ws.numel() if ws is not None else 0,
                                                    _stream(u.device)))
        return du, dh0, None, None


def gated_scan(u, h0=None, mask=None, output_gate=True):
    """Gated linear recurrence over a sequence: ``(y (T,B,H), last state (B,H) float32)``.

    ``u`` (T,B,3H) holds ``[x | forget | gate]`` along its last axis -- one projection's output,
    used in place -- or (T,B,2H) ``[x | forget]`` with ``output_gate=False``:

        f = sigmoid(forget),  c_t = f_t c_{t-1} + (1 - f_t) x_t,  y_t = c_t silu(gate_t)  (or c_t)

    from ``c_{-1} = h0`` (B,H) float32, or zeros.  ``mask`` (T,B), of any type: where it is zero the
    step is skipped (the state passes through, y is 0, no gradient, whatever u holds there), so a
    padded batch ends in each sequence's own last state, and a sequence without any step in ``h0``.
    ``u`` may have any strides over time and batch (a batch-first tensor transposed, a slice of a
    wider one) without a copy.  T = 0 returns ``h0`` as the last state.

    Differentiable (once) with respect to ``u`` and ``h0``.  The backward pass reads u and the
    gradients and a float32 state per 16 steps that the forward pass keeps; the state and every sum
    are float32, results are rounded to u's type once, and repeated calls give the same bits.
    """
    _device_of(u, h0, mask)
    if u.dim() != 3:
        raise ValueError(f"u must have shape (T, B, parts * H), got {tuple(u.shape)}")
    capi.sequence_dtype_code(u.dtype)
    T, B = u.shape[:2]
    H = _scan_width(u, output_gate)
    h0 = _state(h0, B, H, "h0")
    mask = _mask_bytes(mask, (T, B), u)
    if u.numel() == 0:
        last = h0.clone() if h0 is not None else torch.zeros(B, H, dtype=torch.float32, device=u.device)
        return u[..., :H].clone(), last       # (empty, connected to u)
    u = _rows_dense(u)
    h0 = h0.contiguous() if h0 is not None else None
    if torch.is_grad_enabled() and (u.requires_grad or (h0 is not None and h0.requires_grad)):
        return GatedScanFunction.apply(u, h0, mask, bool(output_gate))
    y, last, _ = _scan_forward(u, h0, mask, output_gate, keep=False)
    return y, last


def gated_scan_step(u, state, mask=None, output_gate=True):
    """One step of ``gated_scan`` for serving: ``u`` (B,3H or 2H) -> y (B,H); ``state`` (B,H) float32,
    contiguous, is updated in place.  ``mask`` (B): a sequence whose entry is zero keeps its state and
    gets y = 0.  One launch, one pass over u, state and y.  Records no gradient and refuses to run
    where one would be lost."""
    device = _device_of(u, state, mask)
    if u.dim() != 2:
        raise ValueError(f"u must have shape (B, parts * H), got {tuple(u.shape)}")
    code = capi.sequence_dtype_code(u.dtype)
    B, H = u.shape[0], _scan_width(u, output_gate)
    _state(state, B, H, "state")
    if not state.is_contiguous():
        raise ValueError("state is updated in place: it must be contiguous")
    if torch.is_grad_enabled() and (u.requires_grad or state.requires_grad):
        raise RuntimeError("gated_scan_step records no gradient: call it under torch.no_grad(), or "
                           "gated_scan on a sequence of one step")
    mask = _mask_bytes(mask, (B,), u)
    if u.numel() == 0:
        return u.new_zeros(B, H)
    u = _rows_dense(u)
    with _on(device):
        y = torch.empty(B, H, dtype=u.dtype, device=device)
        capi.check(capi.load().kvae_gated_scan_step(
            B, H, code, int(output_gate), u.data_ptr(), u.stride(0), capi.ptr_strided(mask),
            mask.stride(0) if mask is not None else 0, state.data_ptr(), y.data_ptr(), _stream(device)))
    return y


# -- root-mean-square norm ------------------------------------------------------------------
def _rows(t, D):
    """`t` as (rows, D) with last-axis stride 1; copies only when its leading axes do not merge."""
    if t is None:
        return None
    t = _rows_dense(t)
    try:
        return t.view(-1, D)
    except RuntimeError:
        return t.reshape(-1, D)


def _check_norm(x, weight, residual):
    device = _device_of(x, weight, residual)
    capi.sequence_dtype_code(x.dtype)
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    D = x.shape[-1]
    if tuple(weight.shape) != (D,):
        raise ValueError(f"weight must have shape {(D,)}, got {tuple(weight.shape)}")
    if weight.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"weight must be float32 or {x.dtype}, got {weight.dtype}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if residual is not None and residual.dtype != x.dtype:
        raise TypeError(f"residual must have x's type {x.dtype}, got {residual.dtype}")
    if D > capi.NORM_MAX_WIDTH:
        raise NotImplementedError(f"rows of up to {capi.NORM_MAX_WIDTH} elements, got {D}")
    return device


def _norm_struct(x2, r2, weight, eps):
    d = capi.RmsNorm(rows=x2.shape[0], D=x2.shape[1], dtype=capi.sequence_dtype_code(x2.dtype),
                     weight_dtype=capi.sequence_dtype_code(weight.dtype), x=x2.data_ptr(),
                     x_stride=x2.stride(0), weight=weight.data_ptr(), eps=eps)
    if r2 is not None:
        d.residual, d.residual_stride = r2.data_ptr(), r2.stride(0)
    return d


def _norm_forward(x, weight, residual, eps, keep):
    """(y, sum or None, rstd or None), the first two shaped like x."""
    D = x.shape[-1]
    x2, r2 = _rows(x, D), _rows(residual, D)
    with _on(x.device):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if r2 is not None else None
        rstd = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device) if keep else None
        d = _norm_struct(x2, r2, weight, eps)
        d.y, d.sum, d.rstd = y.data_ptr(), capi.ptr(total), capi.ptr(rstd)
        capi.check(capi.load().kvae_rms_norm_forward(C.byref(d), _stream(x.device)))
    return y, total, rstd


class RmsNormFunction(torch.autograd.Function):
    """(x, weight, residual or None, eps) -> y, or (y, sum) with a residual."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, total, rstd = _norm_forward(x, weight, residual, eps, keep=True)
        # The backward pass forms the unrounded sum again from x and residual where the gradient of
        # a float32 weight would show the 16-bit sum's rounding; elsewhere the stored sum serves
        # (one tensor less to keep and to read).
        again = residual is not None and x.dtype != weight.dtype
        ctx.save_for_backward(x if total is None or again else total, residual if again else None,
                              weight, rstd)
        ctx.eps, ctx.has_residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        x, residual, weight, rstd = ctx.saved_tensors
        lib, D = capi.load(), x.shape[-1]
        with _on(x.device):
            dy = torch.zeros_like(x) if dy is None else dy
            x2, r2, dy2, ds2 = _rows(x, D), _rows(residual, D), _rows(dy, D), _rows(dsum, D)
            rows = x2.shape[0]
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dweight = torch.empty(D, dtype=weight.dtype, device=x.device)
            partial = torch.empty(lib.kvae_rms_norm_backward_parts(rows), D, dtype=torch.float32,
                                  device=x.device)
            d = _norm_struct(x2, r2, weight, ctx.eps)
            d.rstd, d.dy, d.dy_stride = rstd.data_ptr(), dy2.data_ptr(), dy2.stride(0)
            if ds2 is not None:
                d.dsum, d.dsum_stride = ds2.data_ptr(), ds2.stride(0)
            d.dx, d.partial, d.dweight = dx.data_ptr(), partial.data_ptr(), dweight.data_ptr()
            capi.check(lib.kvae_rms_norm_backward(C.byref(d), _stream(x.device)))
        return dx, dweight, dx if ctx.has_residual else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """Root-mean-square norm over the last axis: ``y = r (mean r^2 + eps)^(-1/2) weight`` with
    ``r = x``; with ``residual`` (x's shape and type) ``r = x + residual`` and the result is ``(y, r)``,
    the pair a residual stack carries on, in one pass.

    ``weight`` (D) is float32 or has x's type.  The norm is taken of the unrounded sum in float32;
    y and r are rounded to x's type once.  Rows of up to 16384 elements, any row stride.
    Differentiable (once) with respect to x, residual and weight; the weight's gradient is summed
    in float32 in a fixed order."""
    _check_norm(x, weight, residual)
    if x.numel() == 0:
        r = x if residual is None else x + residual
        y = r * weight.to(x.dtype)
        return y if residual is None else (y, r)
    weight = weight.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        return RmsNormFunction.apply(x, weight, residual, float(eps))
    y, total, _ = _norm_forward(x, weight, residual, float(eps), keep=False)
    return y if residual is None else (y, total)


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} records no gradient: call it under torch.no_grad()")


def rms_norm_quantized(x, weight, residual=None, eps=1e-6):
    """``rms_norm`` with y in 8 bits for ``linear_8bit``: ``(q, scale)``, or ``(q, scale, r)`` with a
    residual.  q has x's shape in torch.float8_e4m3fn and scale x's leading shape in float32:
    ``y ~ q * scale[..., None]`` with ``scale = max(max |y| / 448, 2^-126)`` per row, to the nearest.
    A NaN stays one and does not enter the scale.  Serving only: no gradient."""
    device = _check_norm(x, weight, residual)
    _no_gradient("rms_norm_quantized", x, weight, residual)
    D = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    total = torch.empty(x.shape, dtype=x.dtype, device=device) if residual is not None else None
    if x.numel():
        x2, r2, weight = _rows(x, D), _rows(residual, D), weight.contiguous()
        with _on(device):
            d = _norm_struct(x2, r2, weight, float(eps))
            d.y, d.scale, d.sum = q.data_ptr(), scale.data_ptr(), capi.ptr(total)
            capi.check(capi.load().kvae_rms_norm_quantized(C.byref(d), _stream(device)))
    elif D == 0:
        scale.fill_(2.0 ** -126)
    return (q, scale) if residual is None else (q, scale, total)


def quantize_rows(x):
    """The last axis of x in 8 bits with one scale per row: ``(q, scale)`` as in
    ``rms_norm_quantized`` without the norm.  Lays out the weights of ``linear_8bit`` once."""
    device = _device_of(x)
    code = capi.sequence_dtype_code(x.dtype)
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    D = x.shape[-1]
    if D > capi.NORM_MAX_WIDTH:
        raise NotImplementedError(f"rows of up to {capi.NORM_MAX_WIDTH} elements, got {D}")
    _no_gradient("quantize_rows", x)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    if x.numel():
        x2 = _rows(x, D)
        with _on(device):
            capi.check(capi.load().kvae_quantize_rows(x2.shape[0], D, code, x2.data_ptr(), x2.stride(0),
                                                      q.data_ptr(), scale.data_ptr(), _stream(device)))
    elif D == 0:
        scale.fill_(2.0 ** -126)
    return q, scale


def linear_8bit(x, x_scale, weight, weight_scale, bias=None, dtype=torch.float32):
    """``y = (x * x_scale) (weight * weight_scale)^T + bias`` for 8-bit rows: x (..., K) with x_scale
    (...) as ``rms_norm_quantized`` returns them, weight (N, K) with weight_scale (N) as
    ``quantize_rows`` lays them out once; y (..., N) of ``dtype`` (float32, bfloat16 or float16).

    The sum runs over the 8-bit values on the matrix instructions in float32; scales and bias
    (float32) are applied before the one rounding to ``dtype``.  Any sizes.  Serving only: no
    gradient."""
    device = _device_of(x, x_scale, weight, weight_scale, bias)
    code = capi.sequence_dtype_code(dtype)
    for name, t in (("x", x), ("weight", weight)):
        if t.dtype != torch.float8_e4m3fn:
            raise TypeError(f"{name} must be torch.float8_e4m3fn, got {t.dtype}")
    for name, t in (("x_scale", x_scale), ("weight_scale", weight_scale), ("bias", bias)):
        if t is not None and t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x (..., K) and weight (N, K) expected, got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if x_scale.shape != x.shape[:-1] or tuple(weight_scale.shape) != (N,):
        raise ValueError(f"one scale per row expected, got {tuple(x_scale.shape)} for x {tuple(x.shape)} and "
                         f"{tuple(weight_scale.shape)} for weight {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"bias must have shape {(N,)}, got {tuple(bias.shape)}")
    _no_gradient("linear_8bit", x_scale, weight_scale, bias)
    with _on(device):
        y = torch.empty(x.shape[:-1] + (N,), dtype=dtype, device=device)
        if y.numel() == 0:
            return y
        if K == 0:
            return y.copy_(bias) if bias is not None else y.zero_()
        x, x_scale, weight, weight_scale = (t.contiguous() for t in (x, x_scale, weight, weight_scale))
        bias = bias.contiguous() if bias is not None else None
        capi.check(capi.load().kvae_linear_8bit(
            x_scale.numel(), N, K, x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(),
            weight_scale.data_ptr(), capi.ptr(bias), code, y.data_ptr(), _stream(device)))
    return y
