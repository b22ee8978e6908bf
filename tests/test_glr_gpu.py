"""The gated linear recurrence (GLRFunction, GLRFusedFunction, glr_decode_step) against its definition in 64 bits."""
import pytest
import torch

from layer_ref import assert_within, glr, glr_fused, rounded, unit

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]
# relative error of sigmoid(g) and 1 - sigmoid(g) for |g| < 16 in units of u: the exponential's argument and result (a fast
# one is documented as 2 + 1.16 |g| steps of 2u), a sum, a reciprocal of 2 steps, a product; then the product with the value
GATE_ERR = 2 * (2 + 1.16 * 16) + 8
# one token, around the lengths of a part, several parts with a ragged end; widths around a vector and a tile
SHAPES = [(1, 1, 1), (3, 1, 72), (2, 2, 8), (1, 3, 7), (5, 31, 64), (2, 33, 100), (3, 64, 65), (1, 127, 128), (2, 128, 40),
          (2, 129, 96), (1, 255, 24), (4, 257, 56), (3, 333, 77), (2, 513, 264), (1, 1025, 129), (2, 2050, 72), (40, 19, 200)]


def _inputs(B, T, D, dtype, dev, gates, seed, offset=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def make(t):
        if not offset:
            return t.to(dtype)
        flat = torch.empty(t.numel() + offset, dtype=dtype, device=dev)[offset:]
        return flat.copy_(t.reshape(-1)).view(t.shape)

    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    gate = rnd(B, T, D) + (4.0 if gates == "open" else 0.0)
    x, go, s, gs = rnd(B, T, D), rnd(B, T, D), rnd(B, D), rnd(B, D)
    f = {"open": torch.sigmoid(gate), "sigmoid": torch.sigmoid(gate), "signed": torch.tanh(gate),
         "reset": torch.sigmoid(gate) * (rnd(B, T, D) > -1), "ones": torch.ones_like(gate)}[gates]
    return [make(t) for t in (x, f, s, go, gs)] + [make(torch.cat([x, gate], -1))]


def _check_plain(B, T, D, dtype, dev, gates, seed, offset=0):
    from t2fw_b200.functional_glr import GLRFunction

    x, f, s, go, gs, _ = _inputs(B, T, D, dtype, dev, gates, seed, offset)
    leaves = [t.requires_grad_(True) for t in (x, f, s)]
    out, nxt = GLRFunction.apply(*leaves)
    grads = torch.autograd.grad([out, nxt], leaves, [go, gs])
    ref, _ = glr(x, f, s, go, gs, dtype)
    for name, got in zip(("outputs", "next_state", "d_value", "d_forget", "d_state"), (out, nxt, *grads)):
        assert got.dtype == dtype
        assert_within(got, *ref[name], name)
    with torch.no_grad():
        again = GLRFunction.apply(*leaves)
    assert torch.equal(again[0], out) and torch.equal(again[1], nxt)


def _check_fused(B, T, D, dtype, dev, gates, seed, offset=0):
    from t2fw_b200.functional_glr import GLRFusedFunction

    _, _, s, go, gs, vg = _inputs(B, T, D, dtype, dev, gates, seed, offset)
    leaves = [vg.requires_grad_(True), s.requires_grad_(True)]
    out, nxt = GLRFusedFunction.apply(*leaves)
    grads = torch.autograd.grad([out, nxt], leaves, [go, gs])
    ref = glr_fused(vg, s, go, gs, dtype, GATE_ERR)
    for name, got in zip(("outputs", "next_state", "d_vg", "d_state"), (out, nxt, *grads)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_definition(cuda, shape, dtype):
    _check_plain(*shape, dtype, cuda, "open", sum(shape))
    _check_fused(*shape, dtype, cuda, "open", sum(shape) + 1)


@pytest.mark.parametrize("gates", ["sigmoid", "signed", "reset", "ones"])
def test_gate_distributions(cuda, gates):
    _check_plain(2, 700, 136, torch.float32, cuda, gates, 3)
    _check_plain(2, 700, 136, torch.bfloat16, cuda, gates, 4)
    if gates == "sigmoid":
        _check_fused(2, 700, 136, torch.float16, cuda, gates, 5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_unaligned_tensors(cuda, dtype, offset):
    _check_plain(2, 300, 64, dtype, cuda, "open", 6, offset)
    _check_fused(2, 300, 64, dtype, cuda, "open", 7, offset)


@pytest.mark.parametrize("B,T,D", [(1, 12000, 64), (1, 9001, 136), (700, 40, 64), (96, 300, 768), (2, 3000, 2048),
                                   (40, 400, 501), (30, 100, 1002)])
def test_larger_grids(cuda, B, T, D):
    _check_plain(B, T, D, torch.bfloat16, cuda, "open", 8)
    _check_fused(B, T, D, torch.bfloat16, cuda, "open", 9)


def test_gradients_against_differences(cuda):
    from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction

    x, f, s, _, _, vg = _inputs(2, 37, 5, torch.float64, cuda, "signed", 10)
    assert torch.autograd.gradcheck(GLRFunction.apply, [t.requires_grad_(True) for t in (x, f, s)])
    assert torch.autograd.gradcheck(GLRFusedFunction.apply, [vg.requires_grad_(True), s])


def test_an_output_that_nothing_used(cuda):
    from t2fw_b200.functional_glr import GLRFunction

    x, f, s, go, gs, _ = _inputs(2, 150, 48, torch.float32, cuda, "open", 11)
    leaves = [t.requires_grad_(True) for t in (x, f, s)]
    zero = torch.zeros_like
    for up in ((go, None), (None, gs)):
        outs = GLRFunction.apply(*leaves)
        used = [(o, u) for o, u in zip(outs, up) if u is not None]
        got = torch.autograd.grad([o for o, _ in used], leaves, [u for _, u in used])
        full = [u if u is not None else zero(o) for o, u in zip(outs, up)]
        want = torch.autograd.grad(GLRFunction.apply(*leaves), leaves, full)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [5, 700])
def test_nan_and_infinity_stay_where_the_recurrence_has_them(cuda, T):
    """A step that is no finite number makes its channel's later ones so, and no other.  Which kind of number it is agrees too,
    but for the channel of an infinite gate: the steps of a run are composed into h -> P h + L there, with P and L both
    infinite, and infinity minus infinity is NaN where the steps one by one may stay at an infinity."""
    from t2fw_b200.functional_glr import GLRFunction

    x, f, s, go, gs, _ = _inputs(2, T, 40, torch.float32, cuda, "open", 12)
    x[0, T // 2, 3] = float("nan")
    f[1, T // 2, 9] = float("inf")
    f[1, T // 3, 10] = float("nan")
    s[0, 20] = float("inf")
    f[0, T // 2, 20] = 0.0            # infinity times zero
    x[1, 0, 30] = float("-inf")
    ref, _ = glr(x, f, s, go, gs, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, f, s)]
    out, nxt = GLRFunction.apply(*leaves)
    grads = torch.autograd.grad([out, nxt], leaves, [go, gs])
    for name, got in zip(("outputs", "next_state", "d_value", "d_forget", "d_state"), (out, nxt, *grads)):
        want = ref[name][0]
        assert bool((torch.isfinite(got) == torch.isfinite(want)).all()), name
        kind = torch.ones(2, 40, dtype=torch.bool, device=cuda)
        kind[1, 9] = False
        kind = (kind if want.dim() == 2 else kind[:, None]).expand_as(want)
        assert bool((torch.isnan(got) == torch.isnan(want))[kind].all()), name
        inf = kind & torch.isinf(want)
        assert bool((got[inf].double() == want[inf]).all()), name
        fine = torch.isfinite(want)
        assert_within(got[fine], want[fine], ref[name][1][fine], name)


def test_zero_states_meet_gates_whose_product_overflows(cuda):
    """Gates of 2 over hundreds of steps in front of the first value: the state is zero, not infinity times zero.  And a gate of
    zero ends what was before, also where the gates behind it overflow."""
    from t2fw_b200.functional_glr import GLRFunction

    f = torch.full((1, 1200, 16), 2.0, device=cuda)
    x, s = torch.zeros_like(f), torch.zeros(1, 16, device=cuda)
    x[:, 1190] = 1.0
    out, nxt = GLRFunction.apply(x, f, s)
    assert not out[:, :1190].any() and torch.equal(out[0, 1190:, 0], 2.0 ** torch.arange(10, device=cuda))
    s += 1.0
    f[:, 0] = 0.0
    out, nxt = GLRFunction.apply(x, f, s)
    assert not out[:, :1190].any() and torch.equal(nxt, torch.full_like(nxt, 512.0))


def test_no_wrong_finite_numbers_where_products_overflow(cuda):
    """A tiny state in front of gates whose product leaves the range: what the recurrence gives, or no finite number."""
    from t2fw_b200.functional_glr import GLRFunction

    for D in (16, 17):
        f = torch.full((1, 1200, D), 2.0, device=cuda)
        x, s = torch.zeros_like(f), torch.full((1, D), 2.0 ** -100, device=cuda)
        out, nxt = GLRFunction.apply(x, f, s)
        want = torch.tensor([2.0 ** (t - 100) if t < 1000 else float("inf") for t in range(1, 1201)], device=cuda, dtype=torch.float64)
        assert torch.equal(out[0, :127, 0].double(), want[:127])
        same = out[0].double() == want[:, None]
        assert bool((same | ~torch.isfinite(out[0])).all()) and not torch.isfinite(nxt).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D", [(1, 1), (3, 77), (256, 768), (1000, 129), (512, 1024), (513, 1023)])
def test_decode_steps(cuda, B, D, dtype):
    """Steps into own buffers, the state in place or in turn, against the definition on the state as it was rounded."""
    from t2fw_b200.decode import glr_decode_step
    from t2fw_b200.functional_glr import GLRFunction

    g = torch.Generator(device=cuda).manual_seed(B + D)
    s = torch.randn(B, D, generator=g, device=cuda).to(dtype)
    one, two, out = s.clone(), s.clone(), torch.empty(B, 1, D, dtype=dtype, device=cuda)
    other = torch.empty_like(two)
    for _ in range(3):
        x = torch.randn(B, 1, D, generator=g, device=cuda).to(dtype)
        f = torch.sigmoid(torch.randn(B, 1, D, generator=g, device=cuda)).to(dtype)
        ref = f[:, 0].double() * one.double() + x[:, 0].double()
        tol = rounded(ref, 2 * unit(dtype) * ((f[:, 0].double() * one.double()).abs() + x[:, 0].double().abs()), dtype)
        o, n = GLRFunction.apply(x, f, one)
        assert glr_decode_step(x, f, one, one, out)[1] is one
        assert_within(out[:, 0], ref, tol, "outputs")
        assert torch.equal(out[:, 0], one) and torch.equal(o, out) and torch.equal(n, one)
        glr_decode_step(x, f, two, other, out)
        assert torch.equal(other, one)
        two, other = other, two


def test_split_sequence_continues(cuda):
    """A prompt in two calls, the second from the first one's state, and single steps behind it."""
    from t2fw_b200.functional_glr import GLRFunction

    x, f, s, go, gs, _ = _inputs(2, 400, 72, torch.float32, cuda, "open", 13)
    ref, _ = glr(x, f, s, go, gs, torch.float32)
    state, parts = s, []
    for a, b in ((0, 150), (150, 398), (398, 399), (399, 400)):
        o, state = GLRFunction.apply(x[:, a:b].contiguous(), f[:, a:b].contiguous(), state)
        parts.append(o)
    assert_within(torch.cat(parts, 1), ref["outputs"][0], 2 * ref["outputs"][1], "outputs")


def test_other_streams_and_two_calls_at_once(cuda):
    from t2fw_b200.functional_glr import GLRFunction

    data = [_inputs(2, 900, 128, torch.float16, cuda, "open", 20 + i)[:3] for i in range(2)]
    want = [GLRFunction.apply(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(GLRFunction.apply(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, n in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(n, want[i][1])


def test_captured_training_step_replays(cuda):
    """Forward and backward in one graph; replays follow the inputs."""
    from t2fw_b200.functional_glr import GLRFunction

    x, f, s, go, gs, _ = _inputs(2, 600, 96, torch.float16, cuda, "open", 30)
    leaves = [t.requires_grad_(True) for t in (x, f, s)]

    def step():
        out, nxt = GLRFunction.apply(*leaves)
        return (out, nxt, *torch.autograd.grad([out, nxt], leaves, [go, gs]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for k in range(2):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        want = step()
        for a, b in zip(res, want):
            assert torch.equal(a, b)


def test_a_changed_output_is_noticed(cuda):
    from t2fw_b200.functional_glr import GLRFunction

    x, f, s, go, gs, _ = _inputs(1, 20, 8, torch.float32, cuda, "open", 31)
    out, nxt = GLRFunction.apply(x.requires_grad_(True), f.requires_grad_(True), s)
    with torch.no_grad():
        out.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, x, go)


def test_second_derivative_and_forward_mode_are_refused(cuda):
    import torch.autograd.forward_ad as fw

    from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction

    x, f, s, go, gs, vg = _inputs(1, 20, 8, torch.float32, cuda, "open", 32)
    for fn, ins in ((GLRFunction, (x, f, s)), (GLRFusedFunction, (vg, s))):
        for cls in (fn, type("Sub", (fn,), {})):
            leaves = [t.clone().requires_grad_(True) for t in ins]
            first = torch.autograd.grad(cls.apply(*leaves), leaves, [go, gs])
            again = torch.autograd.grad(cls.apply(*leaves), leaves, [go, gs], create_graph=True)
            for a, b in zip(first, again):
                assert torch.equal(a, b)
            with pytest.raises(RuntimeError, match="not implemented"):
                torch.autograd.grad(again[0].sum(), leaves[0])
        with fw.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
            fn.apply(fw.make_dual(ins[0], torch.ones_like(ins[0])), *ins[1:])


def test_refusals(cuda):
    from t2fw_b200.decode import glr_decode_step
    from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction

    x, f, s, _, _, vg = _inputs(2, 6, 8, torch.float16, cuda, "open", 33)
    with pytest.raises(AssertionError):
        GLRFunction.apply(x, f[:, :5], s)
    with pytest.raises(AssertionError):
        GLRFunction.apply(x, f.float(), s)
    with pytest.raises(RuntimeError, match="contiguous"):
        GLRFunction.apply(x.transpose(0, 1).contiguous().transpose(0, 1), f, s)
    with pytest.raises(RuntimeError, match="state must be"):
        GLRFunction.apply(x, f, s[:1])
    with pytest.raises(RuntimeError, match="empty"):
        GLRFunction.apply(x[:, :0], f[:, :0], s)
    with pytest.raises(RuntimeError, match="CUDA"):
        GLRFunction.apply(x, f, s.cpu())
    with pytest.raises(AssertionError):
        GLRFusedFunction.apply(vg[..., :15], s)
    with pytest.raises(RuntimeError, match="dtype"):
        GLRFunction.apply(*(t.int() for t in (x, f, s)))
    one, out = x[:, :1].contiguous(), torch.empty(2, 1, 8, dtype=torch.float16, device=cuda)
    gate = f[:, :1].contiguous()
    with pytest.raises(RuntimeError, match="share memory"):
        glr_decode_step(one, gate, s, s, one)
    both = torch.zeros(3, 8, dtype=torch.float16, device=cuda)
    with pytest.raises(RuntimeError, match="state_out"):
        glr_decode_step(one, gate, both[:2], both[1:], out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES + [(8, 1024, 768), (700, 40, 64), (1, 9001, 136), (40, 400, 501)])
def test_the_final_state_is_the_last_output(cuda, shape, dtype):
    """Bit for bit, and so is the state's gradient f_1 r_1 where d_value holds r_1 unrounded: who goes on from the state goes on
    from what was reported."""
    from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction

    x, f, s, go, gs, vg = _inputs(*shape, dtype, cuda, "open", 40 + sum(shape))
    leaves = [t.requires_grad_(True) for t in (x, f, s)]
    out, nxt = GLRFunction.apply(*leaves)
    assert torch.equal(nxt, out[:, -1])
    dx, _, ds = torch.autograd.grad([out, nxt], leaves, [go, gs])
    if dtype in (torch.float32, torch.float64):
        assert torch.equal(ds, f[:, 0] * dx[:, 0])
    out, nxt = GLRFusedFunction.apply(vg, s)
    assert torch.equal(nxt, out[:, -1])


@pytest.mark.parametrize("D", [16, 17])
def test_a_finite_last_output_is_a_finite_state(cuda, D):
    """128 gates of 1, then 128 of 2: the product of a part is 2^128, beyond fp32, but no state is."""
    from t2fw_b200.functional_glr import GLRFunction

    f = torch.ones(1, 256, D, device=cuda)
    f[:, 128:] = 2.0
    x, s = torch.zeros_like(f), torch.full((1, D), 2.0 ** -100, device=cuda)
    out, nxt = GLRFunction.apply(x, f, s)
    assert torch.equal(nxt, out[:, -1]) and bool((nxt == 2.0 ** 28).all())
    leaves = [t.requires_grad_(True) for t in (x, f.flip(1).contiguous(), torch.zeros_like(s))]
    dx, _, ds = torch.autograd.grad(GLRFunction.apply(*leaves)[1], leaves, s)
    assert bool((dx[:, 0] == 2.0 ** 27).all()) and bool((ds == 2.0 ** 28).all())


@pytest.mark.parametrize("native", [True, False])
def test_a_decode_step_marks_what_it_writes(cuda, native):
    """A backward pass that saved the state or the outputs' buffer raises instead of reading what a step left there."""
    from t2fw_b200.decode import glr_decode_step
    from t2fw_b200.functional_glr import GLRFunction

    step = glr_decode_step if native else torch.ops.glr.decode_step
    x, f, s, go, _, _ = _inputs(2, 1, 8, torch.float32, cuda, "open", 50)
    for written in ("state", "outputs"):
        gate = f.clone().requires_grad_(True)
        state, out = s.clone(), torch.zeros_like(x)
        if written == "state":
            y, _ = GLRFunction.apply(x, gate, state)       # saves the state
        else:
            y = gate * out
        step(x, f, state, state, out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, gate, go)
    state, other, out = s.clone(), s.clone(), torch.zeros_like(x)
    step(x, f, state, other, out)
    assert (x._version, f._version, state._version, other._version, out._version) == (0, 0, 0, 1, 1)
    with pytest.raises(RuntimeError, match="share memory"):
        step(x, f, state, other, x)
    assert x._version == 0 and other._version == 1
    with torch.inference_mode():
        state, other, out = s.clone(), s.clone(), torch.zeros_like(x)
    step(x, f, state, other, out)
    step(x, f, state, state, out)
    assert torch.equal(state, out[:, 0]) and torch.equal(other, state)
