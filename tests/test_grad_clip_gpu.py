"""Global gradient norm and clipping (t2fw_b200/grad_clip.py) against 64-bit arithmetic."""
import pytest
import torch

from layer_ref import assert_within, clip, rounded, unit

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]
SHAPES = [(1,), (7,), (3, 5), (1000,), (64, 64), (8192,), (8193,), (257, 129), (100000,), (2, 3, 5, 7)]


def _grads(dtypes, dev, seed, shapes=SHAPES, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(std * torch.randn(s, generator=g, device=dev)).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def _check_total(total, ref, any64):
    """fp64 sums, rounded to the result's type: fp32's half step is 2^-24."""
    assert total.dim() == 0 and total.dtype == (torch.float64 if any64 else torch.float32)
    assert abs(float(total) - float(ref)) <= float(ref) * (2.0 ** -40 if any64 else 2.0 ** -24 + 2.0 ** -40)


def _check_scaled(got, grads, c):
    for a, g in zip(got, grads):
        assert a.dtype == g.dtype and a.shape == g.shape
        ref = g.double() * c
        # the factor is off by the norm's rounding, its own sum's and division's, and the product is rounded
        u = unit(g.dtype)
        assert_within(a, ref, rounded(ref, 5 * 2.0 ** -24 * ref.abs() + u * ref.abs(), g.dtype), str(g.dtype))


@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES[:3], DTYPES])
@pytest.mark.parametrize("factor", [0.01, 0.7, 3.0, 0.0])
def test_norm_and_clipping(cuda, dtypes, factor):
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads, global_norm

    grads = _grads(dtypes, cuda, 1)
    ref, _ = clip(grads, 1.0)
    max_norm = factor * float(ref)
    _, c = clip(grads, max_norm)
    any64 = torch.float64 in dtypes
    _check_total(global_norm(grads), ref, any64)
    out, total = clip_grads(grads, max_norm)
    _check_total(total, ref, any64)
    _check_scaled(out, grads, c)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    total = clip_grad_norm_(params, max_norm)
    _check_total(total, ref, any64)
    for p, a in zip(params, out):
        assert torch.equal(p.grad, a)


def test_same_as_torch(cuda):
    from t2fw_b200.grad_clip import clip_grad_norm_

    params = [torch.nn.Parameter(torch.zeros(s, device=cuda)) for s in SHAPES]
    for p, g in zip(params, _grads([torch.float32], cuda, 2)):
        p.grad = g
    copy = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(copy, params):
        p.grad = q.grad.clone()
    copy.append(torch.nn.Parameter(torch.zeros(3, device=cuda)))      # without a gradient
    want = torch.nn.utils.clip_grad_norm_(copy, 5.0)
    got = clip_grad_norm_(iter(params + [copy[-1]]), 5.0)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
    for p, q in zip(params, copy):
        assert_within(p.grad, q.grad.double(), 1e-5 * q.grad.double().abs() + 1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_into_a_bucket(cuda, dtype):
    """Gradients one behind the other in one buffer, at any offset; what lies between and around them is left alone."""
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads

    sizes = [1, 3, 17, 8192, 5, 8191, 40001, 2]
    flat = torch.randn(sum(sizes) + 3 * len(sizes) + 3, device=cuda).to(dtype)
    before, at, views = flat.clone(), 3, []
    for n in sizes:
        views.append((at, n))
        at += n + 3
    params = []
    for a, n in views:
        p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda))
        p.grad = flat[a:a + n]
        params.append(p)
    grads = [before[a:a + n] for a, n in views]
    ref, c = clip(grads, 2.0)
    out, total = clip_grads([p.grad for p in params], 2.0)
    _check_scaled(out, grads, c)
    assert torch.equal(flat, before)
    _check_total(clip_grad_norm_(params, 2.0), ref, dtype == torch.float64)
    mask = torch.ones_like(flat, dtype=torch.bool)
    for (a, n), o in zip(views, out):
        assert torch.equal(flat[a:a + n], o)
        mask[a:a + n] = False
    assert torch.equal(flat[mask], before[mask])


def test_many_tensors(cuda):
    """More than one table of addresses."""
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads

    grads = _grads([torch.float32, torch.bfloat16], cuda, 3, [(i % 37 + 1,) for i in range(1300)])
    ref, c = clip(grads, 1.0)
    out, total = clip_grads(grads, 1.0)
    _check_total(total, ref, False)
    _check_scaled(out, grads, c)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    clip_grad_norm_(params, 1.0)
    assert all(torch.equal(p.grad, o) for p, o in zip(params, out))


def test_strides_that_cover_their_memory(cuda):
    from t2fw_b200.grad_clip import clip_grads

    g = torch.randn(30, 50, device=cuda).t()
    ref, c = clip([g], 1.0)
    (o,), total = clip_grads([g], 1.0)
    assert o.stride() == g.stride()
    _check_total(total, ref, False)
    _check_scaled([o], [g], c)


def test_results_are_tensors_of_their_own(cuda):
    """They share an allocation and nothing else: a change of one, also by autograd's books, is none of the others."""
    from t2fw_b200.grad_clip import clip_grads

    grads = _grads(DTYPES, cuda, 8)
    out, _ = clip_grads(grads, 1.0)
    spans = sorted((o.data_ptr(), o.data_ptr() + o.nbytes) for o in out)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and all(o.data_ptr() % 512 == 0 for o in out)
    kept = [o.clone() for o in out]
    w = torch.ones_like(out[4]).requires_grad_(True)
    y = (w * out[4]).sum()      # saves a result
    for i, o in enumerate(out):
        if i != 4:
            assert not o._is_view() and o.is_contiguous() and not o.requires_grad
            o.add_(1.0)
    y.backward()
    assert torch.equal(w.grad, kept[4]) and torch.equal(out[4], kept[4])
    assert torch.equal(out[0], kept[0] + 1.0)
    del out[1:], y
    assert torch.equal(torch.clone(out[0]), kept[0] + 1.0) and out[0].to("cpu").shape == grads[0].shape


def test_large_tensor(cuda):
    from t2fw_b200.grad_clip import clip_grads, global_norm

    g = torch.randn(50_000_001, device=cuda).to(torch.bfloat16)
    ref, c = clip([g], 100.0)
    (o,), total = clip_grads([g], 100.0)
    _check_total(total, ref, False)
    _check_scaled([o], [g], c)
    assert torch.equal(global_norm([g]), total) and torch.equal(clip_grads([g], 100.0)[0][0], o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_values_whose_squares_leave_the_range(cuda, dtype, size):
    from t2fw_b200.grad_clip import clip_grads

    grads = [(size * torch.randn(5000, device=cuda)).to(dtype), torch.zeros(9, dtype=dtype, device=cuda)]
    ref, c = clip(grads, size)
    out, total = clip_grads(grads, size)
    _check_total(total, ref, False)
    _check_scaled(out, grads, c)


def test_nonfinite_norms(cuda):
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads

    for bad in (float("inf"), float("nan")):
        grads = _grads([torch.float32], cuda, 4)
        grads[4][3, 3] = bad
        out, total = clip_grads(grads, 1.0)
        assert torch.equal(total.isnan(), torch.tensor(bad != bad, device=cuda)) and not torch.isfinite(total)
        for o, g in zip(out, grads):      # what multiplication by 0 or by NaN gives
            want = g * (1.0 / torch.tensor(bad, device=cuda))
            assert torch.equal(o.isnan(), want.isnan()) and torch.equal(o[~o.isnan()], want[~want.isnan()])
        p = torch.nn.Parameter(torch.zeros_like(grads[4]))
        p.grad = grads[4].clone()
        with pytest.raises(RuntimeError, match="not finite"):
            clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert torch.equal(p.grad.nan_to_num(), grads[4].nan_to_num())
        clip_grad_norm_(p, float("inf"))      # inf / inf and inf / nan
        assert p.grad.isnan().all()
    g = torch.randn(10, device=cuda)
    assert torch.equal(clip_grads([g], float("inf"))[0][0], g)


def test_empty_and_zero(cuda):
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads, global_norm

    assert float(clip_grad_norm_([], 1.0)) == 0 and clip_grads([], 1.0)[0] == [] and float(global_norm([])) == 0
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(2, device=cuda))], 1.0)) == 0
    e, z = torch.empty(0, 3, device=cuda), torch.zeros(5, device=cuda)
    out, total = clip_grads([e, z, e], 1.0)
    assert float(total) == 0 and out[0].shape == (0, 3) and not out[1].any()
    out, total = clip_grads([e], 0.0)
    assert float(total) == 0 and total.is_cuda
    out, _ = clip_grads([z, z], 0.0)       # the same tensor twice, into two results
    assert not out[0].any() and out[0].data_ptr() != out[1].data_ptr()


def test_gradients_made_with_a_graph(cuda):
    from t2fw_b200.grad_clip import clip_grads

    w = torch.randn(20, device=cuda, requires_grad=True)
    g, = torch.autograd.grad(w.pow(3).sum(), w, create_graph=True)
    (o,), total = clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(o.sum(), w)
    with torch.no_grad():
        (o,), _ = clip_grads([g], 1.0)
    assert not o.requires_grad


def test_change_in_place_is_noticed(cuda):
    from t2fw_b200.grad_clip import clip_grad_norm_

    w = torch.randn(20, device=cuda, requires_grad=True)
    p = torch.nn.Parameter(torch.zeros(20, device=cuda))
    p.grad = torch.randn(20, device=cuda)
    y = (w * p.grad).sum()      # saves the gradient
    clip_grad_norm_(p, 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_streams_and_graphs(cuda):
    """Two captured calls with a workspace each, replayed at once on two streams."""
    from t2fw_b200.grad_clip import clip_grads

    runs = []
    for seed in (5, 6):
        grads = _grads([torch.float16], cuda, seed, std=0.1 * seed)
        clip_grads(grads, 1.0)
        graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            res = clip_grads(grads, 1.0)
        runs.append((grads, graph, st, res))
    for k in range(4):
        for grads, graph, st, _ in runs:
            for g in grads:
                g.mul_(1.5 if k % 2 else 0.5)
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for grads, _, _, (out, total) in runs:
            want, t = clip_grads(grads, 1.0)
            assert torch.equal(total, t) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda):
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads, global_norm

    g = torch.randn(40, device=cuda)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip_grads([g], bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        global_norm([g, g.cpu()])
    with pytest.raises(RuntimeError, match="dense"):
        clip_grads([g[::2]], 1.0)
    with pytest.raises(RuntimeError, match="dense"):
        global_norm([g[:1].expand(5)])
    with pytest.raises(RuntimeError, match="dtype"):
        global_norm([g.int()])
    with pytest.raises(RuntimeError, match="dense"):
        global_norm([g.to_sparse()])
    before = g.clone()
    params = [torch.nn.Parameter(torch.zeros(30, device=cuda)) for _ in range(2)]
    for grads in ((g[:30], g[10:]), (g[:30], g[:30])):
        for p, t in zip(params, grads):
            p.grad = t
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grad_norm_(params, 1.0)
    assert torch.equal(g, before)


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("place", range(8))
def test_one_large_value_in_eight(cuda, dtype, place):
    """The squares of eight neighbours are added in fp32, in three levels: 3 * 2^-24 of their sum, half of that of the norm, which
    is then rounded (2^-24).  Small values whose squares lie just below half a step of the large one's are where that is reached."""
    from t2fw_b200.grad_clip import global_norm

    for small in (2.0 ** -12, 2.43e-4, 3.4e-4, 2.0 ** -11, 1e-3):
        v = torch.full((8,), small, device=cuda)
        v[place] = 1.0
        g = v.repeat(4096).to(dtype)
        ref = g.double().square().sum().sqrt()
        assert abs(float(global_norm([g])) - float(ref)) <= (2.5 * 2.0 ** -24 + 2.0 ** -40) * float(ref)
