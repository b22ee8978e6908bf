"""The root-mean-square norm (RMSNormFunction, AddRMSNormFunction and the 8-bit forms) against its definition in 64 bits."""
import pytest
import torch

from layer_ref import TINY, assert_within, rms_norm, unit

pytestmark = pytest.mark.gpu

EPS = 1e-5
DTYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]
# (leading sizes, D): single values, around a vector, a warp's row, a block's row, rows beyond what registers hold
SHAPES = [((1,), 1), ((3,), 7), ((2, 3), 8), ((5,), 100), ((1,), 256), ((300,), 264), ((300,), 330), ((5,), 1002), ((3,), 6002), ((7,), 768), ((2, 33), 1001), ((1100,), 128),
          ((9,), 2048), ((3,), 5000), ((2,), 16384), ((3,), 20001), ((1,), 70000), ((2500,), 24)]


def _inputs(lead, D, dtype, dev, seed, offset=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def make(*shape):
        t = torch.randn(*shape, generator=g, device=dev)
        if not offset:
            return t.to(dtype)
        return torch.empty(t.numel() + offset, dtype=dtype, device=dev)[offset:].copy_(t.reshape(-1)).view(t.shape)

    return make(*lead, D), make(*lead, D), make(D), make(*lead, D), make(*lead, D)


def _check(lead, D, dtype, dev, seed, offset=0):
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction

    x, res, w, gy, gs = _inputs(lead, D, dtype, dev, seed, offset)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    y, s = AddRMSNormFunction.apply(*leaves, EPS)
    dx, dr, dw = torch.autograd.grad([y, s], leaves, [gy, gs])
    ref = rms_norm(x, res, w, EPS, gy, gs, dtype)
    for name, got in (("y", y), ("sum", s), ("d_s", dx), ("d_s", dr), ("d_weight", dw)):
        assert got.dtype == dtype
        assert_within(got, *ref[name], "add " + name)
    y = RMSNormFunction.apply(x, w, EPS)
    dx, dw = torch.autograd.grad(y, [x, w], gy)
    ref = rms_norm(x, None, w, EPS, gy, None, dtype)
    for name, got in (("y", y), ("d_s", dx), ("d_weight", dw)):
        assert_within(got, *ref[name], name)
    again = torch.autograd.grad(RMSNormFunction.apply(x, w, EPS), [x, w], gy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,D", SHAPES)
def test_matches_definition(cuda, lead, D, dtype):
    _check(lead, D, dtype, cuda, D)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_unaligned_tensors(cuda, dtype, offset):
    _check((40,), 128, dtype, cuda, 5, offset)
    _check((3,), 2048, dtype, cuda, 6, offset)


def test_many_rows(cuda):
    _check((20000,), 64, torch.bfloat16, cuda, 7)
    _check((8192,), 768, torch.float16, cuda, 8)


def _check_e4m3(x, res, w, out, dtype):
    s = x.double() + (0 if res is None else res.double())
    D = x.shape[-1]
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * w.double()
    scale = (y.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-30)
    k = (D / 32 + 26) * unit(dtype)
    q, sc = out[:2]
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    assert sc.dtype == torch.float32 and sc.shape == x.shape[:-1] + (1,)
    assert_within(sc, scale, k * scale, "scale")
    # a value between two neighbours of the grid goes to the nearer one: half a step is 2^-4 of the value, 2^-10 below the
    # smallest normal 2^-6; computed, it is off by k before that
    v = y / sc.double()
    assert_within(q.double(), v, 2.0 ** -4 * v.abs().clamp_min(2.0 ** -6) + 2 * k * v.abs(), "q")
    assert (q.double().abs().amax(-1) == 448).logical_or(s.abs().amax(-1) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES[:3])
@pytest.mark.parametrize("lead,D", SHAPES)
def test_eight_bit_forms(cuda, lead, D, dtype):
    from t2fw_b200.functional_norm import AddRMSNormFunction, add_rms_norm_e4m3, rms_norm_e4m3

    x, res, w, _, _ = _inputs(lead, D, dtype, cuda, D + 1)
    _check_e4m3(x, None, w, rms_norm_e4m3(x, w, EPS), dtype)
    out = add_rms_norm_e4m3(x, res, w, EPS)
    _check_e4m3(x, res, w, out, dtype)
    assert torch.equal(out[2], AddRMSNormFunction.apply(x, res, w, EPS)[1])


def test_eight_bit_rounding_is_the_nearest(cuda):
    """Against torch's own conversion where y / scale is exact: weights that are powers of two over rows of equal magnitude."""
    from t2fw_b200.functional_norm import rms_norm_e4m3

    D = 256
    w = torch.linspace(-448, 448, D, device=cuda)
    w[0] = 448.0
    x = torch.ones(1, D, device=cuda)
    q, scale = rms_norm_e4m3(x, w, 0.0)      # rstd = 1, y = w, scale = 1
    assert float(scale) == 1.0
    assert torch.equal(q.float()[0], w.to(torch.float8_e4m3fn).float())


def test_rows_of_zeros(cuda):
    from t2fw_b200.functional_norm import RMSNormFunction, rms_norm_e4m3

    x = torch.zeros(3, 96, dtype=torch.float16, device=cuda, requires_grad=True)
    w = torch.ones(96, dtype=torch.float16, device=cuda)
    y = RMSNormFunction.apply(x, w, EPS)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert not y.any()
    assert_within(dx, torch.full((3, 96), EPS ** -0.5, device=cuda, dtype=torch.float64),
                  torch.full((3, 96), EPS ** -0.5 * (2.0 ** -11 + 2.0 ** -20), device=cuda, dtype=torch.float64))
    with torch.no_grad():
        q, scale = rms_norm_e4m3(x, w, EPS)
    assert not q.float().any() and torch.equal(scale, torch.full_like(scale, 1e-30))


def test_nan_and_infinity_stay_in_their_row(cuda):
    from t2fw_b200.functional_norm import AddRMSNormFunction, rms_norm_e4m3

    for D in (64, 1001):
        x, res, w, _, _ = _inputs((5,), D, torch.float32, cuda, 9)
        x[1, 3], x[3, 7] = float("nan"), float("inf")
        y, s = AddRMSNormFunction.apply(x, res, w, EPS)
        q, scale = rms_norm_e4m3(x, w, EPS)
        assert y[1].isnan().all() and q[1].float().isnan().all() and scale[1].isnan().all()
        assert y[3, 7].isnan() and not y[3, :7].any() and q[3].float().isnan().all()
        for i in (0, 2, 4):
            assert torch.isfinite(y[i]).all() and torch.isfinite(q[i].float()).all()
        x[1, 3], x[3, 7] = 1.0, 1.0
        w[5] = float("nan")
        q, scale = rms_norm_e4m3(x, w, EPS)
        assert scale.isnan().all()


def test_gradients_against_differences(cuda):
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction

    x, res, w, _, _ = (t.requires_grad_(True) for t in _inputs((3,), 13, torch.float64, cuda, 10))
    assert torch.autograd.gradcheck(lambda a, b: RMSNormFunction.apply(a, b, 0.1), [x, w])
    assert torch.autograd.gradcheck(lambda a, b, c: AddRMSNormFunction.apply(a, b, c, 0.1), [x, res, w])


def test_an_output_that_nothing_used(cuda):
    from t2fw_b200.functional_norm import AddRMSNormFunction

    x, res, w, gy, gs = _inputs((6,), 96, torch.float32, cuda, 11)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    for k in range(2):
        got = torch.autograd.grad(AddRMSNormFunction.apply(*leaves, EPS)[k], leaves, (gy, gs)[k])
        want = torch.autograd.grad(AddRMSNormFunction.apply(*leaves, EPS), leaves,
                                   [gy if k == 0 else torch.zeros_like(gy), gs if k == 1 else torch.zeros_like(gs)])
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_captured_training_step_replays_beside_another(cuda):
    """Two captured steps with a workspace each, replayed in turn and at once."""
    from t2fw_b200.functional_norm import AddRMSNormFunction

    steps = []
    for seed in (12, 13):
        x, res, w, gy, gs = _inputs((500,), 200, torch.bfloat16, cuda, seed)
        leaves = [t.requires_grad_(True) for t in (x, res, w)]

        def step(leaves=leaves, up=(gy, gs)):
            outs = AddRMSNormFunction.apply(*leaves, EPS)
            return (*outs, *torch.autograd.grad(outs, leaves, up))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res_ = step()
        steps.append((step, graph, res_, torch.cuda.Stream()))
    for _ in range(3):
        for _, graph, _, st in steps:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for step, _, res_, _ in steps:
            for a, b in zip(res_, step()):
                assert torch.equal(a, b)


def test_strided_and_mixed_arguments(cuda):
    """Other strides are copied; what the native entry point does not take goes through the class with the same result."""
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction, add_rms_norm_e4m3

    x, res, w, gy, gs = _inputs((6, 5), 64, torch.float16, cuda, 14)
    want = AddRMSNormFunction.apply(x, res, w, EPS)
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    for got in (AddRMSNormFunction.apply(xt, res, w, EPS), type("Sub", (AddRMSNormFunction,), {}).apply(x, res, w, EPS)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(RMSNormFunction.apply(x, w, 0), RMSNormFunction.apply(x, w, 0.0))
    a, b = add_rms_norm_e4m3(xt, res, w, EPS), add_rms_norm_e4m3(x, res, w, EPS)
    assert all(torch.equal(p.float(), q.float()) for p, q in zip(a, b))
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    y, s = AddRMSNormFunction.apply(*leaves, EPS)
    got = torch.autograd.grad([y, s], leaves, [gy.transpose(0, 1).contiguous().transpose(0, 1), gs])
    for p, q in zip(got, torch.autograd.grad(AddRMSNormFunction.apply(*leaves, EPS), leaves, [gy, gs])):
        assert torch.equal(p, q)


def test_refusals(cuda):
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction, add_rms_norm_e4m3, rms_norm_e4m3

    x, res, w, gy, _ = _inputs((4,), 16, torch.float16, cuda, 15)
    with pytest.raises(AssertionError):
        RMSNormFunction.apply(x, w[:8], EPS)
    with pytest.raises(AssertionError):
        AddRMSNormFunction.apply(x, res[:2], w, EPS)
    with pytest.raises(AssertionError):
        RMSNormFunction.apply(x, w.float(), EPS)
    with pytest.raises(AssertionError):
        RMSNormFunction.apply(x, w, -1.0)
    with pytest.raises(RuntimeError, match="empty"):
        RMSNormFunction.apply(x[:0], w, EPS)
    with pytest.raises(RuntimeError, match="CUDA"):
        RMSNormFunction.apply(x.cpu(), w.cpu(), EPS)
    with pytest.raises(RuntimeError, match="8-bit"):
        rms_norm_e4m3(x.double(), w.double(), EPS)
    with pytest.raises(RuntimeError, match="no gradients"):
        add_rms_norm_e4m3(x, res, w.requires_grad_(True), EPS)
    with torch.no_grad():
        add_rms_norm_e4m3(x, res, w, EPS)
    for cls in (RMSNormFunction, type("Sub", (RMSNormFunction,), {})):
        g, = torch.autograd.grad(cls.apply(x, w, EPS), w, gy, create_graph=True)
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(g.float().sum(), w)


@pytest.mark.parametrize("dtype", DTYPES[:3])
@pytest.mark.parametrize("D", [8, 96, 1001, 1002, 2048, 70000])
def test_eight_bit_rows_of_zeros_with_a_tiny_eps(cuda, D, dtype):
    """y is 0, so q is, however large 1 / sqrt(eps) / scale would be."""
    from t2fw_b200.functional_norm import add_rms_norm_e4m3, rms_norm_e4m3

    x, w = torch.zeros(3, D, dtype=dtype, device=cuda), torch.ones(D, dtype=dtype, device=cuda)
    x[1, D // 2] = 1.0
    for eps in (1e-17, 8e-18, 1e-20, 1e-36):
        for q, scale in (rms_norm_e4m3(x, w, eps), add_rms_norm_e4m3(x, torch.zeros_like(x), w, eps)[:2]):
            assert not q[::2].float().any() and torch.equal(scale[::2], torch.full_like(scale[::2], 1e-30))
            assert float(q[1, D // 2].float()) == 448.0 and int((q[1].float() != 0).sum()) == 1


@pytest.mark.parametrize("D", [64, 33, 40000])
def test_eight_bit_rows_below_the_smallest_scale(cuda, D):
    """x = 1e-12, w = 1e-30: y is 0.995e-30 and the scale 1e-30; e4m3 holds 0.9375 and 1 there."""
    from t2fw_b200.functional_norm import rms_norm_e4m3

    x = torch.full((2, D), 1e-12, device=cuda)
    q, scale = rms_norm_e4m3(x, torch.full((D,), 1e-30, device=cuda), 1e-26)
    assert torch.equal(scale, torch.full_like(scale, 1e-30)) and bool((q.float() == 1.0).all())


# powers of two that take the squares, and their sums, out of fp32's range (fp64's) but not the values themselves
FAR = {torch.bfloat16: [63, 64, 100, 118, -50, -56, -64, -100], torch.float32: [63, 64, 100, 118, -50, -56, -64, -100],
       torch.float64: [511, 512, 700, -440, -460, -512]}


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("lead,D", [((5,), 8), ((3,), 7), ((9,), 24), ((5,), 100), ((5,), 264), ((4,), 330), ((3,), 768), ((5,), 1001), ((5,), 1002),
                                    ((3,), 2048), ((3,), 6002), ((2,), 8192), ((2,), 16384), ((3,), 20001), ((2,), 70000)])
def test_squares_that_leave_the_range(cuda, lead, D, dtype):
    """With eps = 0 the norm does not depend on a row's size, and a power of two changes no rounding: y and d_weight are those of
    the rows at size 1, and d_s is smaller by the power.  Rows of every size lie beside one another.  At 2^118 a d_s of less than
    2^-8 lies below the smallest normal number, 2^-126: its two last roundings (the product with 1 / rms and the sum with gs or the
    storage type) are then off by half of the smallest subnormal each, 2^118 times as much at size 1."""
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction

    x, res, w, gy, gs = _inputs(lead, D, dtype, cuda, D + 20)
    powers = FAR[dtype]
    big = lambda t, f: (t.detach().double() * f).to(dtype)  # noqa: E731
    for shift in range(len(powers)):
        far = [0 if i % 3 == 1 else powers[(i + shift) % len(powers)] for i in range(lead[0])]
        up = torch.tensor([[2.0 ** k] for k in far], device=cuda, dtype=torch.float64)      # the host's powers are exact, pow() here is not
        down = 1.0 / up
        leaves = [t.requires_grad_(True) for t in (big(x, up), big(res, up), w.detach().clone())]
        assert torch.equal(leaves[0].double(), x.double() * up)
        y, s = AddRMSNormFunction.apply(*leaves, 0.0)
        dx, dr, dw = torch.autograd.grad([y, s], leaves, [gy, big(gs, down)])
        ref = rms_norm(x, res, w, 0.0, gy, gs, dtype)
        ref["d_s"] = (ref["d_s"][0], ref["d_s"][1] + 2 * TINY[dtype] * up)
        for name, got in (("y", y), ("sum", s.double() * down), ("d_s", dx.double() * up), ("d_s", dr.double() * up), ("d_weight", dw)):
            assert_within(got, *ref[name], "add " + name)
        y = RMSNormFunction.apply(leaves[0], leaves[2], 0.0)
        dx, dw = torch.autograd.grad(y, [leaves[0], leaves[2]], gy)
        ref = rms_norm(x, None, w, 0.0, gy, None, dtype)
        ref["d_s"] = (ref["d_s"][0], ref["d_s"][1] + 2 * TINY[dtype] * up)
        for name, got in (("y", y), ("d_s", dx.double() * up), ("d_weight", dw)):
            assert_within(got, *ref[name], name)
        for i in range(lead[0]):      # a row is what it is alone, whatever lies beside it
            assert torch.equal(RMSNormFunction.apply(leaves[0][i:i + 1], leaves[2], 0.0)[0], y[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead,D", [((5,), 8), ((5,), 100), ((5,), 264), ((3,), 768), ((5,), 1001), ((3,), 2048), ((2,), 16384), ((3,), 20001)])
def test_eight_bit_rows_of_any_size(cuda, lead, D, dtype):
    """The same for the 8-bit form; and weights that take the products s w, which y never is, out of the range."""
    from t2fw_b200.functional_norm import add_rms_norm_e4m3

    x, res, w, _, _ = _inputs(lead, D, dtype, cuda, D + 21)
    s = x.double() + res.double()
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True)) * w.double()
    k = (D / 32 + 26) * unit(dtype)
    for kx, kw in ((0, 0), (64, 0), (118, 0), (-56, 0), (-100, 0), (30, 100), (118, 100), (-50, -90), (-100, -60)):
        q, scale, _ = add_rms_norm_e4m3((x.double() * 2.0 ** kx).to(dtype), (res.double() * 2.0 ** kx).to(dtype),
                                        (w.double() * 2.0 ** kw).to(dtype), 0.0)
        want = (y.abs().amax(-1, keepdim=True) / 448 * 2.0 ** kw).clamp_min(1e-30)
        assert_within(scale, want, k * want, "scale %d %d" % (kx, kw))
        v = y * 2.0 ** kw / scale.double()
        assert_within(q.double(), v, 2.0 ** -4 * v.abs().clamp_min(2.0 ** -6) + 2 * k * v.abs(), "q %d %d" % (kx, kw))


def test_the_smallest_eps_is_not_zero(cuda):
    from t2fw_b200.functional_norm import RMSNormFunction, rms_norm_e4m3

    for dtype in DTYPES[:3]:
        for D in (64, 1001, 70000):
            x, w = torch.zeros(2, D, dtype=dtype, device=cuda), torch.ones(D, dtype=dtype, device=cuda)
            assert not RMSNormFunction.apply(x, w, 1e-60).any() and not rms_norm_e4m3(x, w, 1e-60)[0].float().any()
