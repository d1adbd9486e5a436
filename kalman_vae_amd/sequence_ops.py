"""Operators of the "gated" dynamics-parameter network, each on hand-written HIP kernels: the
gated linear recurrence over a sequence and its one-step form (csrc/gated_scan.hip), the
root-mean-square norm with the residual's addition and its 8-bit output (csrc/rms_norm.hip),
the product of 8-bit rows (csrc/linear_8bit.hip).

They take GPU tensors of float32, bfloat16 or float16 and run on the current stream of the
tensors' device; states, norms and sums are float32 whatever the element type.  None has a forward-mode
derivative: tensors with a tangent (torch.autograd.forward_ad) are refused.  Only the product's
16-bit results of more than 32 rows come from sums of fewer bits (see linear_8bit).

The reference's only recurrent network is torch.nn.LSTM (kvae/dynamics_parameter_network.py:18-58);
these operators have no counterpart there.
"""
import torch

from . import _capi as capi


def _device_of(first, *others):
    """The one GPU all given tensors are on; raises for CPU tensors and for a mix."""
    device = first.device
    if not first.is_cuda:
        capi.require_gpu(first)
    for t in others:
        if t is not None and t.device != device:
            capi.require_gpu(t)
            raise ValueError(f"tensors on different devices: {device} and {t.device}")
    return device


def _mask_bytes(mask, shape):
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


def gated_scan(u, h0=None, mask=None, output_gate=True):
    """Gated linear recurrence over a sequence: ``(y (T,B,H), last state (B,H) float32)``.

    ``u`` (T,B,3H) holds ``[x | forget | gate]`` along its last axis -- one projection's output,
    used in place -- or (T,B,2H) ``[x | forget]`` with ``output_gate=False``:

        f = sigmoid(forget),  c_t = f_t c_{t-1} + (1 - f_t) x_t,  y_t = c_t silu(gate_t)  (or c_t)

    from ``c_{-1} = h0`` (B,H) float32, or zeros.  ``mask`` (T,B), of any type: where it is zero the
    step is skipped (the state passes through, y is 0, no gradient, whatever u holds there), so a
    padded batch ends in each sequence's own last state, and a sequence without any step in ``h0``.
    ``u`` may have any strides over time and batch (a batch-first tensor transposed, a slice of a
    wider one) without a copy, unless sequences that a workgroup takes together (up to 512 / H + 2)
    lie 2^31 bytes apart.  T = 0 returns ``h0`` as the last state.

    Differentiable (once) with respect to ``u`` and ``h0``.  The backward pass reads u and the
    gradients and a float32 state per 16 steps (float32; 8 steps of the 16-bit types) that the
    forward pass keeps; the state and every sum are float32, results are rounded to u's type once, and
    repeated calls give the same bits.
    """
    _device_of(u, h0, mask)
    if u.dim() != 3:
        raise ValueError(f"u must have shape (T, B, parts * H), got {tuple(u.shape)}")
    capi.sequence_dtype_code(u.dtype)
    T, B = u.shape[:2]
    H = _scan_width(u, output_gate)
    h0 = _state(h0, B, H, "h0")
    mask = _mask_bytes(mask, (T, B))
    if u.numel() == 0:
        last = h0.clone() if h0 is not None else torch.zeros(B, H, dtype=torch.float32, device=u.device)
        return u[..., :H].clone(), last       # (empty, connected to u)
    return capi.torch_entry().gated_scan(u, h0, mask, bool(output_gate))


def gated_scan_step(u, state, mask=None, output_gate=True):
    """One step of ``gated_scan`` for serving: ``u`` (B,3H or 2H) -> y (B,H); ``state`` (B,H) float32,
    contiguous, is updated in place.  ``mask`` (B): a sequence whose entry is zero keeps its state and
    gets y = 0.  One launch, one pass over u, state and y.  Records no gradient and refuses to run
    where one would be lost."""
    _device_of(u, state, mask)
    if u.dim() != 2:
        raise ValueError(f"u must have shape (B, parts * H), got {tuple(u.shape)}")
    capi.sequence_dtype_code(u.dtype)
    B, H = u.shape[0], _scan_width(u, output_gate)
    _state(state, B, H, "state")
    if not state.is_contiguous():
        raise ValueError("state is updated in place: it must be contiguous")
    if torch.is_grad_enabled() and (u.requires_grad or state.requires_grad):
        raise RuntimeError("gated_scan_step records no gradient: call it under torch.no_grad(), or "
                           "gated_scan on a sequence of one step")
    mask = _mask_bytes(mask, (B,))
    if u.numel() == 0:
        return u.new_zeros(B, H)
    return capi.torch_entry().gated_scan_step(u, state, mask, bool(output_gate))


# -- root-mean-square norm ------------------------------------------------------------------
def _check_norm(x, weight, residual):
    _device_of(x, weight, residual)
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
    y, total = capi.torch_entry().rms_norm(x, weight, residual, eps)
    return y if residual is None else (y, total)


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} records no gradient: call it under torch.no_grad()")


def rms_norm_quantized(x, weight, residual=None, eps=1e-6):
    """``rms_norm`` with y in 8 bits for ``linear_8bit``: ``(q, scale)``, or ``(q, scale, r)`` with a
    residual.  q has x's shape in torch.float8_e4m3fn and scale x's leading shape in float32:
    ``y ~ q * scale[..., None]`` with ``scale = max(max |y| / 448, 2^-126)`` per row, to the nearest.
    A NaN stays one and does not enter the scale.  Serving only: no gradient."""
    _check_norm(x, weight, residual)
    _no_gradient("rms_norm_quantized", x, weight, residual)
    if x.numel():
        q, scale, total = capi.torch_entry().rms_norm_quantized(x, weight, residual, eps)
    else:
        (q, scale), total = _empty_quantized(x), x if residual is None else x + residual
    return (q, scale) if residual is None else (q, scale, total)


def _empty_quantized(x):
    return (torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device),
            torch.full(x.shape[:-1], 2.0 ** -126, dtype=torch.float32, device=x.device))


def quantize_rows(x):
    """The last axis of x in 8 bits with one scale per row: ``(q, scale)`` as in
    ``rms_norm_quantized`` without the norm.  Lays out the weights of ``linear_8bit`` once.  Rows of up to
    16384 elements; longer ones need codes and scales of the caller's own."""
    _device_of(x)
    capi.sequence_dtype_code(x.dtype)
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    D = x.shape[-1]
    if D > capi.NORM_MAX_WIDTH:
        raise NotImplementedError(f"rows of up to {capi.NORM_MAX_WIDTH} elements, got {D}")
    _no_gradient("quantize_rows", x)
    return capi.torch_entry().quantize_rows(x) if x.numel() else _empty_quantized(x)


def linear_8bit(x, x_scale, weight, weight_scale, bias=None, dtype=torch.float32):
    """``y = (x * x_scale) (weight * weight_scale)^T + bias`` for 8-bit rows: x (..., K) with x_scale
    (...) as ``rms_norm_quantized`` returns them, weight (N, K) with weight_scale (N) as
    ``quantize_rows`` lays them out once; y (..., N) of ``dtype`` (float32, bfloat16 or float16).

    Scales and bias (float32) are applied to the sum of the products of the 8-bit values, before the one
    rounding to ``dtype``.  The sum is float32 throughout with ``dtype=torch.float32``, and with up to 32
    rows of x.  16-bit results of more rows come from the matrix instructions for 8-bit operands, at twice
    the rate: of every eight neighbouring products these cut what lies below 2^-13 of the largest
    (1e-5 of a sum of terms of like size; where larger products cancel, a small result may be lost, and
    float32 results rounded afterwards are the way to have it).  K up to 2^22, N up to 2^26, M up to 2^31
    rows, M N up to 2^40.  Serving only: no gradient."""
    _device_of(x, x_scale, weight, weight_scale, bias)
    capi.sequence_dtype_code(dtype)
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
    if x_scale.numel() == 0 or N == 0 or K == 0:
        y = torch.zeros(x.shape[:-1] + (N,), dtype=dtype, device=x.device)
        return y if bias is None else y + bias.to(dtype)
    return capi.torch_entry().linear_8bit(x, x_scale, weight, weight_scale, bias, dtype)
