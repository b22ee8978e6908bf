"""Root-mean-square norm over the last dimension, alone or with the residual's addition.

    y = RMSNormFunction.apply(x, weight, eps)
    y, s = AddRMSNormFunction.apply(x, residual, weight, eps)

    s = x + residual ,   y = s / sqrt(mean(s^2) + eps) * weight

x, residual [..., D], weight [D], all of one dtype; gradients for x, residual (the same tensor, as the gradient of a sum is)
and weight.  y is computed from s before s is rounded to the storage type; the backward pass reads s as it was written.  Rows of
any finite values are normalised, also where their squares leave fp32's range.

For an 8-bit projection behind the norm, without gradients:

    q, scale = rms_norm_e4m3(x, weight, eps)
    q, scale, s = add_rms_norm_e4m3(x, residual, weight, eps)

q is e4m3(y / scale), rounded to nearest, with one scale = max(max|y| / 448, 1e-30) per row, [..., 1] in fp32.
"""
import torch

from . import _lib

_ops = _lib.load_ops()


def _check(x, residual, weight, eps):
    assert x.dim() >= 1 and weight.shape == x.shape[-1:], "weight must be [D] for x [..., D]"
    assert residual is None or residual.shape == x.shape, "residual must have x's shape"
    assert weight.dtype == x.dtype and (residual is None or residual.dtype == x.dtype)
    assert eps >= 0


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        _check(x, None, weight, eps)
        x, weight = x.contiguous(), weight.contiguous()
        y, = torch.ops.rms.forward(x, None, weight, float(eps))
        ctx.save_for_backward(x, weight)
        ctx.eps = float(eps)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        x, weight = saved = ctx.saved_tensors
        grads = torch.ops.rms.backward(grad_y.contiguous(), None, x, weight, ctx.eps)
        return (*_ops.no_second_derivative(grads, (grad_y, *saved)), None)


class AddRMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        """Returns (y, s)."""
        _check(x, residual, weight, eps)
        x, residual, weight = x.contiguous(), residual.contiguous(), weight.contiguous()
        y, s = torch.ops.rms.forward(x, residual, weight, float(eps))
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(s, weight)
        ctx.eps = float(eps)
        return y, s

    @staticmethod
    def backward(ctx, grad_y, grad_s):
        s, weight = saved = ctx.saved_tensors
        gy = torch.zeros_like(s) if grad_y is None else grad_y.contiguous()
        grads = torch.ops.rms.backward(gy, None if grad_s is None else grad_s.contiguous(), s, weight, ctx.eps)
        d_s, d_w = _ops.no_second_derivative(grads, [t for t in (grad_y, grad_s, *saved) if t is not None])
        return d_s, d_s, d_w, None


_lib.bind_apply(RMSNormFunction, _lib.RMS, _ops.rms_apply)
_lib.bind_apply(AddRMSNormFunction, _lib.ADD_RMS, _ops.add_rms_apply)


def _e4m3(x, residual, weight, eps):
    out = _ops.rms_e4m3(x, residual, weight, eps)
    if out is not NotImplemented:
        return out
    _check(x, residual, weight, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError("the 8-bit norm has no gradients: call it under torch.no_grad()")
    residual = None if residual is None else residual.contiguous()
    return tuple(torch.ops.rms.e4m3(x.contiguous(), residual, weight.contiguous(), float(eps)))


def rms_norm_e4m3(x, weight, eps):
    """(q [..., D] float8_e4m3fn, scale [..., 1] float32)"""
    return _e4m3(x, None, weight, eps)


def add_rms_norm_e4m3(x, residual, weight, eps):
    """(q [..., D] float8_e4m3fn, scale [..., 1] float32, s [..., D])"""
    assert residual is not None
    return _e4m3(x, residual, weight, eps)
