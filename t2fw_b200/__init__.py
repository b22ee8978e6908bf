"""t2fw_b200: the fast-weight recurrences of T2FW (decay rule "LFW", delta rule "DFW") as
hand-written sm_100a CUDA behind the reference's Python API.

    from t2fw_b200.functional_lfw import LFWFunction
    from t2fw_b200.functional_dfw import DFWFunction

and, beside them, a gated linear recurrence with a state of one number per channel, a root-mean-square norm that adds the
residual, and gradient clipping:

    from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads, global_norm

The native libraries are built ahead of time (python -m t2fw_b200.build) and loaded on first
use; there is no CPU or PyTorch fallback: if the libraries are missing the import fails.
"""
__version__ = "0.1.0"
