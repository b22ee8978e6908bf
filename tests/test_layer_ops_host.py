"""What the operators around the recurrences refuse, without a GPU: the classes' assertions, tensors that are not on a GPU, and
the C ABI's argument checks, which come before any CUDA call."""
import ctypes

import pytest
import torch

from t2fw_b200 import _lib
from t2fw_b200.decode import glr_decode_step
from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction
from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction, add_rms_norm_e4m3, rms_norm_e4m3
from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads, global_norm

ONE = 16      # any non-null pointer: nothing is dereferenced where a check fails


def _fails(rc, code, text):
    assert rc == code and text in _lib.load_core().t2fw_last_error().decode()


def test_shapes_and_types_assert():
    x, f, s = torch.randn(2, 5, 4), torch.rand(2, 5, 4), torch.zeros(2, 4)
    for a in ((x, f[:, :4], s), (x, f.double(), s), (x, f, s.half())):
        with pytest.raises(AssertionError):
            GLRFunction.apply(*a)
    for a in ((x, s), (torch.randn(2, 5, 8), s[:1]), (torch.randn(2, 5, 8).half(), s), (torch.randn(5, 8), s)):
        with pytest.raises(AssertionError):
            GLRFusedFunction.apply(*a)
    w = torch.ones(4)
    for a in ((x, w[:3], 1e-5), (x, w.half(), 1e-5), (x, w, -1.0), (x, w, float("nan"))):
        with pytest.raises(AssertionError):
            RMSNormFunction.apply(*a)
        with pytest.raises(AssertionError):
            rms_norm_e4m3(*a)
    for fn in (AddRMSNormFunction.apply, add_rms_norm_e4m3):
        with pytest.raises(AssertionError):
            fn(x, x[:1], w, 1e-5)


def test_cpu_tensors_are_a_runtime_error():
    x, f, s, w = torch.randn(2, 1, 4), torch.rand(2, 1, 4), torch.zeros(2, 4), torch.ones(4)
    for call in (lambda: GLRFunction.apply(x, f, s), lambda: GLRFusedFunction.apply(torch.randn(2, 1, 8), s),
                 lambda: glr_decode_step(x, f, s, s.clone(), torch.empty_like(x)), lambda: RMSNormFunction.apply(x, w, 1e-5),
                 lambda: AddRMSNormFunction.apply(x, x, w, 1e-5), lambda: rms_norm_e4m3(x, w, 1e-5),
                 lambda: global_norm([x]), lambda: clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        clip_grad_norm_(p, 1.0)
    assert torch.equal(p.grad, torch.ones(3))


def test_clipping_refuses_impossible_limits_and_passes_over_nothing():
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip_grads([torch.ones(2)], bad)
        with pytest.raises(ValueError):
            clip_grad_norm_([], bad)
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0
    assert clip_grads([], 1.0)[0] == [] and float(global_norm(iter([]))) == 0


def test_c_entries_check_first():
    lib = _lib.load_core()
    _fails(lib.t2fw_glr_forward(None, ONE, ONE, ONE, ONE, 1, 1, 1, 0, None), 1, "null")
    _fails(lib.t2fw_glr_forward(ONE, ONE, ONE, ONE, ONE, 1, 0, 1, 0, None), 1, "positive")
    _fails(lib.t2fw_glr_forward(ONE, ONE, ONE, ONE, ONE, 1, 1, 1, 7, None), 1, "dtype")
    for B, T, D in ((1 << 41, 1, 1), (1 << 20, 1 << 20, 2), (1 << 62, 1 << 62, 1 << 62), (3, 1 << 39, 1)):
        _fails(lib.t2fw_glr_forward(ONE, ONE, ONE, ONE, ONE, B, T, D, 0, None), 1, "range")
    _fails(lib.t2fw_glr_backward(ONE, None, ONE, ONE, ONE, ONE, None, ONE, 1, 1, 1, 0, None), 1, "null")
    _fails(lib.t2fw_glr_fused_forward(ONE, ONE, ONE, None, 1, 1, 1, 0, None), 1, "null")
    _fails(lib.t2fw_glr_fused_backward(ONE, None, None, ONE, ONE, ONE, ONE, 1, 1, 1, 0, None), 1, "null")
    _fails(lib.t2fw_rms_norm_forward(ONE, ONE, ONE, ONE, None, 1, 1, 0.0, 0, None), 1, "together")
    _fails(lib.t2fw_rms_norm_forward(ONE, None, ONE, ONE, None, 0, 1, 0.0, 0, None), 1, "positive")
    _fails(lib.t2fw_rms_norm_forward(ONE, None, ONE, ONE, None, 1 << 31, 1, 0.0, 0, None), 1, "range")
    _fails(lib.t2fw_rms_norm_forward(ONE, None, ONE, ONE, None, 1, 1, -1.0, 0, None), 1, "eps")
    _fails(lib.t2fw_rms_norm_e4m3(ONE, None, ONE, ONE, ONE, None, 1, 1, 0.0, 3, None), 2, "8-bit")
    _fails(lib.t2fw_rms_norm_backward(ONE, None, ONE, ONE, ONE, ONE, 4, 8, 0.0, 0, None, 0, None), 3, "scratch")
    assert lib.t2fw_rms_norm_backward_scratch_bytes(0, 8, 0) == 0
    assert lib.t2fw_rms_norm_backward_scratch_bytes(4, 8, 0) > 0


def test_c_clipping_checks_its_lists():
    lib = _lib.load_core()

    def call(ptrs=(16, 32), outs=(48, 64), numel=(1, 1), dtypes=(0, 2), n=2, max_norm=1.0, total=ONE, tdt=2, scratch=ONE, size=None):
        size = lib.t2fw_grad_clip_scratch_bytes(2) if size is None else size
        arr = lambda t, v: (t * len(v))(*v)  # noqa: E731
        return lib.t2fw_grad_clip(arr(ctypes.c_void_p, ptrs), arr(ctypes.c_void_p, outs), arr(ctypes.c_int64, numel),
                                  arr(ctypes.c_int, dtypes), n, max_norm, total, tdt, scratch, size, None)

    _fails(call(n=0), 1, "number of tensors")
    _fails(call(ptrs=(16, None)), 1, "tensor 1: null")
    _fails(call(outs=(16, 64)), 1, "in place or none")
    _fails(call(outs=(48, None)), 1, "output 1: null")
    _fails(call(numel=(0, 1)), 1, "tensor 0: size")
    _fails(call(numel=(1 << 43, (1 << 43) + 1)), 1, "tensor 1: size")
    _fails(call(dtypes=(0, 9)), 1, "tensor 1: unknown dtype")
    _fails(call(max_norm=-1.0), 1, "max_norm")
    _fails(call(max_norm=float("nan")), 1, "max_norm")
    _fails(call(total=None), 1, "null")
    _fails(call(tdt=0), 1, "norm is float32")
    _fails(call(size=8), 3, "scratch")
    assert lib.t2fw_grad_clip_scratch_bytes(0) == 0


def test_model_options_that_do_not_exist():
    from t2fw_b200.gpt2_fw import GPT2FW, GPT2FWConfig, Linear8

    def _config(rule="glr", norm="rms"):
        return GPT2FWConfig(vocab_size=200, n_positions=128, d_model=64, n_head=1, n_layer=2, rule=rule, norm=norm)

    for cfg in (_config("dfw"), _config("glr", "layer")):
        with pytest.raises(RuntimeError, match="8-bit"):
            GPT2FW(cfg).eight_bit_()
    with pytest.raises(RuntimeError, match="8-bit"):
        GPT2FW(_config()).eight_bit_()      # fp32
    with pytest.raises(RuntimeError, match="8-bit"):
        Linear8(torch.nn.Linear(4, 4, bias=False).half())
    with pytest.raises(ValueError, match="norm"):
        GPT2FW(_config(norm="batch"))
    with pytest.raises(RuntimeError, match="multiples of 16"):
        Linear8(torch.nn.Linear(16, 24).half())
    with pytest.raises(ValueError, match="rule"):
        GPT2FW(_config(rule="rnn"))


def test_clipping_takes_the_places_of_torchs_arguments():
    """The third argument is the norm's type, of which there is one, and the fourth asks for an error."""
    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (1.0, float("inf"), float("nan"), 0, -2.0, True, False, "inf"):
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_([p], 1.0, bad)
    for good in (2, 2.0, "2"):
        assert float(clip_grad_norm_([p], 1.0, good)) == 0 and float(clip_grad_norm_([p], 1.0, good, True)) == 0
    assert float(clip_grad_norm_([p], 1.0, norm_type=2.0, error_if_nonfinite=True)) == 0


def test_schemas_name_what_is_written():
    """An operator that returns nothing and is said to write nothing may be dropped or moved by what reads schemas."""
    for op, written in ((torch.ops.glr.decode_step, {"state_out", "outputs"}), (torch.ops.gradclip.clip_, {"tensors"}),
                        (torch.ops.lfw.decode_step, {"state_out", "outputs"})):
        schema = op.default._schema
        assert schema.is_mutable
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written
    for op in (torch.ops.glr.forward, torch.ops.glr.fused_backward, torch.ops.rms.backward, torch.ops.rms.e4m3, torch.ops.gradclip.norm,
               torch.ops.gradclip.clip):
        assert not op.default._schema.is_mutable


def test_c_norm_refuses_outputs_over_inputs():
    """A row may be read again after a first write.  (Sizes that no call here gets to work on: the check comes before any CUDA call.)"""
    lib = _lib.load_core()
    x, r, w, y, s = (k << 20 for k in range(1, 6))
    text = "shares memory"
    for bad in ((x, r, w, x, s), (x, r, w, y, r), (x, r, w, y, x), (x, r, w, x + 62, s), (x, r, w, y, r - 62), (x, r, w, w, s)):
        _fails(lib.t2fw_rms_norm_forward(*bad, 4, 8, 0.0, 0, None), 1, text)
    _fails(lib.t2fw_rms_norm_forward(x, None, w, x, None, 4, 8, 0.0, 0, None), 1, text)
    _fails(lib.t2fw_rms_norm_e4m3(x, r, w, r + 63, y, s, 4, 8, 0.0, 0, None), 1, text)
    _fails(lib.t2fw_rms_norm_e4m3(x, r, w, y, w, s, 4, 8, 0.0, 0, None), 1, text)
    size = lib.t2fw_rms_norm_backward_scratch_bytes(4, 8, 0)
    for d_s, d_w, scratch in ((x, y, s), (r, y, s), (y, w, s), (y, s, x - size + 16)):
        _fails(lib.t2fw_rms_norm_backward(x, r, 7 << 20, w, d_s, d_w, 4, 8, 0.0, 0, scratch, size, None), 1, text)
