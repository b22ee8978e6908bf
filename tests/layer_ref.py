"""Plain 64-bit implementations of the gated linear recurrence, the root-mean-square norm and gradient clipping, each with a
bound on how far a computation in the storage type may be from it.

Counted in the bounds: a rounding to a type is off by at most half a step, eps/2 of the value, plus half of the type's
smallest subnormal; u = 2^-24 is that of fp32, in which everything is carried (2^-53 for fp64 storage)."""
import torch

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150, torch.float64: 0.0}


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(ref, err, dtype):
    """Bound for a value `ref` that is known up to `err` and then rounded to dtype once."""
    return err + half_step(dtype) * (ref.abs() + err) + TINY[dtype]


def assert_within(got, ref, tol, what=""):
    got = got.detach().double().to(ref.device)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = int(((got - ref).abs() / tol).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError("%s: %d of %d off, worst at %d: %r instead of %r, %r allowed" % (
            what, int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]), float(ref.reshape(-1)[i]), float(tol.reshape(-1)[i])))


# ---- gated linear recurrence ---------------------------------------------------------------------

def recurrence(x, f, start, roundings, u, reverse=False):
    """h_t = f_t h_{t-1} + x_t along dim 1 in the inputs' type, and the bound E_t on a computation in which every step costs
    `roundings` of relative size u: E_t = |f_t| E_{t-1} + roundings u M_t with M the recurrence of the absolute values.  A
    computation in parts multiplies gates first and states later; a term still goes through one multiplication by a gate and
    one rounding of it per step, and through one addition per step at most."""
    T = x.shape[1]
    h, E = torch.empty_like(x), torch.empty_like(x)
    s, m, e = start, start.abs(), torch.zeros_like(start)
    for t in (range(T - 1, -1, -1) if reverse else range(T)):
        s = f[:, t] * s + x[:, t]
        m = f[:, t].abs() * m + x[:, t].abs()
        e = f[:, t].abs() * e + roundings * u * m
        h[:, t], E[:, t] = s, e
    return h, E


def glr(x, f, state, go, gs, dtype, gate_err=0.0):
    """{name: (reference, bound)} for outputs, next_state and the three gradients; gate_err: relative error, in units of u, of
    gates and values that were computed from something else."""
    u, c = unit(dtype), 4.0 + gate_err
    x, f, state, go, gs = (t.detach().double() for t in (x, f, state, go, gs))
    h, E = recurrence(x, f, state, c, u)
    out_err = rounded(h, E, dtype)
    # r_t = go_t + f_{t+1} r_{t+1}; behind the last step stands gs with a gate of 1
    ahead = torch.cat([f[:, 1:], torch.ones_like(f[:, :1])], dim=1)
    r, Er = recurrence(go, ahead, gs, c, u, reverse=True)
    before = torch.cat([state[:, None], h[:, :-1]], dim=1)
    before_err = torch.cat([torch.zeros_like(state[:, None]), out_err[:, :-1]], dim=1)      # read as it was written
    df = r * before
    df_err = r.abs() * before_err + Er * (before.abs() + before_err) + 2 * u * df.abs()
    ds = f[:, 0] * r[:, 0]
    ds_err = f[:, 0].abs() * Er[:, 0] + c * u * ds.abs()
    return {"outputs": (h, out_err), "next_state": (h[:, -1], rounded(h[:, -1], E[:, -1], dtype)),
            "d_value": (r, rounded(r, Er, dtype)), "d_forget": (df, rounded(df, df_err, dtype)),
            "d_state": (ds, rounded(ds, ds_err, dtype))}, (r, Er, before, before_err)


def glr_fused(vg, state, go, gs, dtype, gate_err):
    v, g = vg.detach().double().chunk(2, dim=-1)
    a, rest, u = torch.sigmoid(g), torch.sigmoid(-g), unit(dtype)
    ref, (r, Er, before, before_err) = glr(rest * v, a, state, go, gs, dtype, gate_err)
    dv, dg = rest * r, a * rest * r * (before - v)
    dv_err = rest * Er + (gate_err + 2) * u * dv.abs()
    k = a * rest
    dg_err = k * (Er * (before - v).abs() + (r.abs() + Er) * (before_err + 2 * u * (before.abs() + v.abs()))) + \
        (2 * gate_err + 4) * u * dg.abs()
    ref["d_vg"] = (torch.cat([dv, dg], -1), torch.cat([rounded(dv, dv_err, dtype), rounded(dg, dg_err, dtype)], -1))
    del ref["d_value"], ref["d_forget"]
    return ref


# ---- root-mean-square norm -------------------------------------------------------------------------

def rms_norm(x, residual, weight, eps, gy, gs, dtype):
    """{name: (reference, bound)}: y, sum, d_s, d_weight.  A sum over a row is formed from at least 32 partial sums and then
    in a tree: D/32 + 16 roundings at most."""
    u, D = unit(dtype), x.shape[-1]
    exact_s = residual is None
    s = x.detach().double() + (0 if exact_s else residual.detach().double())
    w, gy = weight.detach().double(), gy.double()
    k = (D / 32 + 16) * u
    rstd = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    y = s * rstd * w
    ref = {"y": (y, rounded(y, (k + 6 * u) * y.abs() + (0 if exact_s else u) * y.abs(), dtype)),
           "sum": (s, rounded(s, u * s.abs(), dtype))}
    g = w * gy
    mean_gs, mean_abs = (g * s).mean(-1, keepdim=True), (g * s).abs().mean(-1, keepdim=True)
    ds = rstd * (g - s * rstd.square() * mean_gs)
    scale = rstd * (g.abs() + s.abs() * rstd.square() * mean_abs)
    # the gradients read s as it was written: off by half a step in each of the four places where it stands
    read = 0.0 if exact_s else half_step(dtype) + 2 * u
    ds_err = (4 * read + 2 * k + 10 * u) * scale + TINY[dtype] * rstd * 4 * (1 + scale)
    if gs is not None:
        ds = ds + gs.double()
        ds_err = ds_err + 2 * u * ds.abs()
    ref["d_s"] = (ds, rounded(ds, ds_err, dtype))
    flat = lambda t: t.reshape(-1, D)  # noqa: E731
    dw = flat(gy * s * rstd).sum(0)
    rows = flat(s).shape[0]
    dw_err = ((rows + 8) * u + k + 2 * read) * flat(gy * s * rstd).abs().sum(0) + TINY[dtype] * flat(gy.abs() * rstd).sum(0)
    ref["d_weight"] = (dw, rounded(dw, dw_err, dtype))
    return ref


# ---- clipping --------------------------------------------------------------------------------------

def clip(tensors, max_norm):
    """(norm, factor) in 64 bits"""
    total = torch.sqrt(sum(t.detach().double().square().sum() for t in tensors))
    return total, (max_norm / (total + 1e-6)).clamp_max(1.0)
