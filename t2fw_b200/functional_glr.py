"""The gated linear recurrence: a state of one number per channel, with a scan over the sequence.

    outputs, next_state = GLRFunction.apply(value, forget, state)

    h_t = forget_t * h_{t-1} + value_t ,   outputs_t = h_t ,   next_state = h_T = outputs[:, -1], bit for bit

value, forget, outputs [B, T, D]; state, next_state [B, D]; gradients for all three inputs.  It is what the decay rule
(`LFWFunction`) becomes with a key and a query of one element, and like there the gates are taken as given.

    outputs, next_state = GLRFusedFunction.apply(vg, state)

is the layer core around it on a projection output vg [B, T, 2*D] = value | gate pre-activation, read in place:
a = sigmoid(gate), h_t = a_t h_{t-1} + (1 - a_t) value_t.  The state is carried in fp32 (fp64 for fp64 tensors) and rounded
where it is written; the gradients of the gates use the outputs as they were written.

Both are additions: the reference has the matrix-state recurrences only.
"""
import torch

from . import _lib

_ops = _lib.load_ops()


def _contiguous(t):
    return None if t is None else t.contiguous()


class GLRFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, value, forget, state):
        """Returns (outputs [B,T,D], next_state [B,D])."""
        assert value.shape == forget.shape
        for other in (forget, state):
            assert other.dtype == value.dtype

        outputs, next_state = torch.ops.glr.forward(value, forget, state)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(forget, outputs, state)
        return outputs, next_state

    @staticmethod
    def backward(ctx, grad_output, grad_state):
        forget, outputs, state = saved = ctx.saved_tensors
        go = torch.zeros_like(outputs) if grad_output is None else grad_output.contiguous()
        grads = torch.ops.glr.backward(go, _contiguous(grad_state), forget, outputs, state)
        return _ops.no_second_derivative(grads, [t for t in (grad_output, grad_state, *saved) if t is not None])


class GLRFusedFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, vg, state):
        """Returns (outputs [B,T,D], next_state [B,D])."""
        assert vg.dim() == 3 and state.dim() == 2 and vg.shape[2] == 2 * state.shape[1], "vg must be [B, T, 2*D]"
        assert state.shape[0] == vg.shape[0], "state must be [B, D]"
        assert vg.dtype == state.dtype
        vg = vg.contiguous()
        state = state.contiguous()
        outputs, next_state = torch.ops.glr.fused_forward(vg, state)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(vg, outputs, state)
        return outputs, next_state

    @staticmethod
    def backward(ctx, grad_output, grad_state):
        vg, outputs, state = saved = ctx.saved_tensors
        go = torch.zeros_like(outputs) if grad_output is None else grad_output.contiguous()
        grads = torch.ops.glr.fused_backward(go, _contiguous(grad_state), vg, outputs, state)
        return _ops.no_second_derivative(grads, [t for t in (grad_output, grad_state, *saved) if t is not None])


_lib.bind_apply(GLRFunction, _lib.GLR, _ops.glr_apply)
_lib.bind_apply(GLRFusedFunction, _lib.GLR_FUSED, _ops.glr_fused_apply)
