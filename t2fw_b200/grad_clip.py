"""Global gradient norm over many tensors, and clipping by it.

    total = global_norm(tensors)                        # sqrt of the sum of all squares, a device scalar
    total = clip_grad_norm_(parameters, max_norm)       # scales the parameters' .grad in place
    clipped, total = clip_grads(grads, max_norm)        # leaves its inputs as they are

Every tensor is multiplied by min(1, max_norm / (total + 1e-6)), the factor of torch.nn.utils.clip_grad_norm_, whose arguments
the in-place form takes in the same places (the 2-norm is the only one); where the factor is 1 it writes nothing.  Two kernel launches for up to 512 tensors, no synchronisation with the host, sums in
fp64 over vectors of 16 bytes; total is fp32 (fp64 if a tensor is).  A total that is infinite or NaN goes into the factor as it is.  Tensors may be
of different dtypes; they are dense CUDA tensors of one device, and those that are scaled in place do not share memory.
"""
import torch

from . import _lib

_ops = _lib.load_ops()


def global_norm(tensors):
    """sqrt of the sum of the squares of all elements (0 for no tensors)."""
    tensors = list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    with torch.no_grad():
        return torch.ops.gradclip.norm(tensors)


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative or NaN")
    return max_norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clips the gradients of `parameters` (a tensor or an iterable of tensors; those without a gradient are passed over) in
    place and returns their norm before.  Any norm_type but 2 is refused.  error_if_nonfinite waits for the norm on the host
    and raises before anything is written."""
    max_norm = _max_norm(max_norm)
    if isinstance(norm_type, bool) or float(norm_type) != 2.0:
        raise ValueError("norm_type must be 2")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters]
    grads = [g for g in grads if g is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite and not torch.isfinite(global_norm(grads)):
        raise RuntimeError("the norm of the gradients is not finite, so they cannot be clipped")
    total = _ops.grad_clip(grads, max_norm, True)
    if total is NotImplemented:
        with torch.no_grad():
            total = torch.ops.gradclip.clip_(grads, max_norm)
    return total


def clip_grads(grads, max_norm):
    """(list of clipped gradients, norm before).  The results lie in one allocation, which lives as long as one of them does and
    is what torch.save writes for any of them: clone a result that is kept or saved by itself.
    Not differentiable: a derivative through the result raises."""
    max_norm = _max_norm(max_norm)
    grads = list(grads)
    if not grads:
        return [], torch.tensor(0.0)
    r = _ops.grad_clip(grads, max_norm, False)
    if r is not NotImplemented:
        return r[1], r[0]
    with torch.no_grad():
        total, *clipped = torch.ops.gradclip.clip(grads, max_norm)
    total, *clipped = _ops.no_second_derivative([total, *clipped], grads)
    return clipped, total
