"""The operators around the recurrences on more than 2^31 elements, whose last ones lie beyond 32-bit offsets, and as the first
call of a process inside a capture."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("B,T,D", [(1, 1050000, 2056), (141000, 16, 1000), (3, 1450001, 503)])
def test_recurrence(cuda, B, T, D):
    """f = 1/2 and x = 1 everywhere: h is 2 after a few steps (2 - 2^-t rounds to it) and r is 2 but near the end; all of them
    are numbers that bf16 holds exactly."""
    from t2fw_b200.functional_glr import GLRFunction

    assert B * T * D > 2 ** 31
    x = torch.ones(B, T, D, dtype=torch.bfloat16, device=cuda)
    f = torch.full_like(x, 0.5)
    s = torch.full((B, D), 2.0, dtype=torch.bfloat16, device=cuda)
    for b, t, d in ((0, 0, 1), (B - 1, T - 2, D - 1), (B - 1, T - 5, 0)):
        x[b, t, d] = 9.0
    leaves = [t.requires_grad_(True) for t in (x, f, s)]
    out, nxt = GLRFunction.apply(*leaves)
    dx, df, ds = torch.autograd.grad(out, leaves, x.detach())      # the gradient of each output is x
    for b, want in ((0, {}), (B - 1, {})):
        n = min(T, 12)
        xs, h = x[b].detach().double(), s[b].detach().double()
        first = []
        for t in range(n):
            h = 0.5 * h + xs[t]
            first.append(h)
        assert torch.equal(out[b, :n].double(), torch.stack(first).bfloat16().double())
        h, r = torch.full((D,), 2.0, device=cuda, dtype=torch.float64), torch.zeros(D, device=cuda, dtype=torch.float64)
        last, back = [], []
        for t in range(T - n, T):
            h = 0.5 * h + xs[t]
            last.append(h)
        if T > 40:      # the start has died away
            assert torch.equal(out[b, T - n:].double(), torch.stack(last).bfloat16().double())
        for t in range(T - 1, T - 1 - n, -1):
            r = xs[t] + 0.5 * r
            back.append(r)
        assert torch.equal(dx[b, T - n:].double(), torch.stack(back[::-1]).bfloat16().double())
        rest = (dx[b, T - n:].double() * out[b, T - n - 1:T - 1].double()) if T > n else None
        if rest is not None:
            assert bool(((df[b, T - n:].double() - rest).abs() <= 2.0 ** -7 * rest.abs()).all())
    assert torch.equal(nxt, out[:, -1]) and bool((ds[:, 2:] == 1.0).all())


def test_norm(cuda):
    from t2fw_b200.functional_norm import AddRMSNormFunction, rms_norm_e4m3

    rows, D = 1050000, 2056
    x = torch.ones(rows, D, dtype=torch.bfloat16, device=cuda)
    x[rows - 1, ::2] = -3.0
    w = torch.ones(D, dtype=torch.bfloat16, device=cuda)
    with torch.no_grad():
        q, scale = rms_norm_e4m3(x, w, 0.0)
        y, s = AddRMSNormFunction.apply(x, x, w, 0.0)
    assert bool((q[:-1].view(torch.uint8) == q[0, 0].view(torch.uint8)).all()) and float(q[0, 0].float()) == 448.0
    assert float(q[-1, 0].float()) == -448.0 and float(q[-1, 1].float()) == 144.0      # 448 / 3, to the nearest of 144 and 160
    assert torch.equal(s[-1], 2 * x[-1]) and torch.equal(s[0], 2 * x[0])
    assert bool((y[:-1] == 1.0).all()) and abs(float(y[-1, 0]) + 3 / 5 ** 0.5) < 2.0 ** -7
    del q, scale, y, s
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    from t2fw_b200.functional_norm import RMSNormFunction

    dx, dw = torch.autograd.grad(RMSNormFunction.apply(*leaves, 0.0), leaves, x.detach())
    # a row of equal values: the gradient along it is none, but for some six roundings of terms of size 1
    assert bool((dx[:-1].abs() <= 8 * 2.0 ** -24).all())
    # rows - 1 ones and the last row's 9 / sqrt(5) or 1 / sqrt(5); a sum of a million in fp32, rounded to bf16's half step
    assert bool(((dw.double() - rows).abs() <= rows * 2.0 ** -8).all())


def test_clipping(cuda):
    from t2fw_b200.grad_clip import clip_grad_norm_

    n = 2 ** 31 + 20001
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device=cuda))
    p.grad = torch.full((n,), 2.0, dtype=torch.bfloat16, device=cuda)
    total = clip_grad_norm_(p, 1e9)
    assert abs(float(total) - 2.0 * n ** 0.5) <= 1e-6 * float(total) and bool((p.grad == 2.0).all())
    clip_grad_norm_(p, float(total) / 4)
    assert bool((p.grad == 0.5).all())


FIRST = """
import torch
from t2fw_b200.functional_glr import GLRFusedFunction
from t2fw_b200.functional_norm import AddRMSNormFunction
from t2fw_b200.grad_clip import clip_grads
x = torch.randn(2, 300, 128, device="cuda")
vg = torch.randn(2, 300, 256, device="cuda")
s, w = torch.zeros(2, 128, device="cuda"), torch.ones(128, device="cuda")
torch.cuda.synchronize()
def step():
    out, _ = GLRFusedFunction.apply(vg, s)
    y, r = AddRMSNormFunction.apply(out, x, w, 1e-5)
    return (*clip_grads([y, r], 1.0)[0],)
g = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(g):
    got = step()
g.replay()
with torch.no_grad():
    want = step()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("equal")
"""


@pytest.mark.parametrize("env", [{}, {"T2FW_DISABLE_PDL": "1"}])
def test_first_calls_of_a_process_inside_a_capture(cuda, env):
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, env=dict(os.environ, **env), capture_output=True, text=True,
                       timeout=240)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("B,T,D", [(1, 1050000, 2056), (3, 1450001, 503)])
def test_fused_recurrence(cuda, B, T, D):
    """Gates of sigmoid(0) = 1/2 and values of 2 everywhere, rows of 2 D: the numbers of test_recurrence again."""
    from t2fw_b200.functional_glr import GLRFusedFunction

    assert B * T * D > 2 ** 31
    vg = torch.zeros(B, T, 2 * D, dtype=torch.bfloat16, device=cuda)
    vg[..., :D] = 2.0
    s = torch.full((B, D), 2.0, dtype=torch.bfloat16, device=cuda)
    for b, t, d in ((0, 0, 1), (B - 1, T - 2, D - 1), (B - 1, T - 5, 0)):
        vg[b, t, d] = 18.0
    leaves = [vg.requires_grad_(True), s.requires_grad_(True)]
    out, nxt = GLRFusedFunction.apply(*leaves)
    assert torch.equal(nxt, out[:, -1])
    dvg, ds = torch.autograd.grad(out, leaves, torch.ones_like(out))
    n = 12
    for b in {0, B - 1}:
        xs, h, first, last = 0.5 * vg[b, :, :D].detach(), s[b].detach().double(), [], []
        for t in range(n):
            h = 0.5 * h + xs[t].double()
            first.append(h)
        assert torch.equal(out[b, :n].double(), torch.stack(first).bfloat16().double())
        h = torch.full((D,), 2.0, device=cuda, dtype=torch.float64)
        for t in range(T - n, T):
            h = 0.5 * h + xs[t].double()
            last.append(h)
        assert torch.equal(out[b, T - n:].double(), torch.stack(last).bfloat16().double())
        for t in (*range(n), *range(T - n, T)):
            r = 2.0 - 2.0 ** (t - T + 1) if t >= T - 60 else 2.0
            before = (out[b, t - 1] if t else s[b]).double()
            want = torch.cat([torch.full_like(before, 0.5 * r), 0.25 * r * (before - vg[b, t, :D].double())])
            assert bool(((dvg[b, t].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20).all())
        del xs
    assert bool((ds.double() - 1.0).abs().max() <= 2.0 ** -8)
