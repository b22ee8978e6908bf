"""Performance cases of the operators of a gated-linear-recurrence language model's training and serving step.

A case names the operator (`op`), the pass, sizes and storage type:

  glr    the gated linear recurrence h_t = f_t h_{t-1} + x_t over [B, T, D]; `fused`: value and gate pre-activation in one
         projection output [B, T, 2*D], f = sigmoid(gate), x = (1 - f) value
         pass "fwd" (prefill), "train" (forward, gradients of every input), "step" (one token into caller-owned buffers)
  norm   root-mean-square norm over rows of D, with the residual's addition (`add`) or without
         pass "train" (forward, gradients), "e4m3" (inference: 8-bit output with one scale per row)
  clip   global norm of a model's gradients and clipping by it; the gradients have the shapes of the repository's language
         model with d_model D, `layers` layers and `vocab` rows in its table
         pass "inplace" (`.grad` of parameters, in one flat buffer as a data-parallel bucket holds them), "new" (a list of
         gradients to a list of clipped ones)

`own` chooses between the framework's kernels and the operators written with elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
E4M3_MAX, MIN_SCALE = 448.0, 1e-30


def _glr(name, kind, B, T, D, dtype, gates, fused=False):
    return {"name": name, "op": "glr", "pass": kind, "fused": fused, "B": B, "T": T, "D": D, "dtype": dtype, "gates": gates}


def _norm(name, kind, rows, D, dtype, add):
    return {"name": name, "op": "norm", "pass": kind, "rows": rows, "D": D, "dtype": dtype, "add": add}


def _clip(name, kind, D, layers, vocab, dtype, max_norm):
    return {"name": name, "op": "clip", "pass": kind, "D": D, "layers": layers, "vocab": vocab, "dtype": dtype,
            "max_norm": max_norm}


def listed():
    return [
        # serving: one token of 256 sequences, the state advanced into a second buffer (latency of a small call)
        _glr("glr_step_b256", "step", 256, 1, 768, "fp16", "open"),
        # prefill of three prompts of ragged length, a width that is no multiple of a tile
        _glr("glr_prefill_b3", "fwd", 3, 777, 1016, "bf16", "open"),
        # training at the benchmark's shape: batch 8, sequence 1024, d_model 768
        _glr("glr_train_b8", "train", 8, 1024, 768, "fp16", "sigmoid"),
        # one long sequence, through the layer form that reads the projection output in place
        _glr("glr_fused_train_long", "train", 1, 65536, 1024, "bf16", "open", fused=True),
        # full precision at odd sizes
        _glr("glr_train_fp32", "train", 3, 333, 77, "fp32", "sigmoid"),
        # serving: one token of 32 sequences into an 8-bit projection
        _norm("norm_e4m3_b32", "e4m3", 32, 768, "fp16", True),
        # training at the benchmark's shape; odd sizes without a residual
        _norm("norm_train_b8", "train", 8192, 768, "fp16", True),
        _norm("norm_train_odd", "train", 2051, 1001, "bf16", False),
        # prefill of 16384 tokens of a wider model into an 8-bit projection
        _norm("norm_e4m3_prefill", "e4m3", 16384, 2048, "bf16", True),
        # every gradient of the small model (124 M values), an ordinary step whose norm stays below the limit
        _clip("clip_inplace_l12", "inplace", 768, 12, 50304, "fp16", 1024.0),
        # a tiny model (28 tensors): launches for little work; four layers, clipped
        _clip("clip_new_tiny", "new", 128, 2, 512, "fp32", 0.25),
        _clip("clip_new_l4", "new", 768, 4, 50304, "bf16", 1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    D = _log(rng, 24, hi)
    return rng.choice([D, (D + 7) // 8 * 8, (D + 63) // 64 * 64])


def draw(rng):
    kind = rng.choice(["step", "glr", "glr", "glr", "norm", "norm", "clip"])
    dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    gates = rng.choice(["sigmoid", "open"])
    if kind == "step":
        c = _glr("", "step", _log(rng, 1, 4096), 1, _width(rng, 2048), dtype, gates)
    elif kind == "glr":
        T, D = _log(rng, 2, 65536), _width(rng, 2048)
        B = _log(rng, 1, max(1, min(256, (1 << 25) // (T * D))))
        T = min(T, max(2, (1 << 25) // (B * D)))
        c = _glr("", rng.choice(["train", "train", "fwd"]), B, T, D, dtype, gates, fused=rng.random() < 0.5)
    elif kind == "norm":
        D = _width(rng, 8192)
        c = _norm("", rng.choice(["train", "e4m3"]), _log(rng, 1, max(1, min(65536, (1 << 25) // D))), D, dtype,
                  rng.random() < 0.7)
    else:
        D = 64 * _log(rng, 1, 12)
        c = _clip("", rng.choice(["inplace", "new"]), D, rng.randint(1, 4), 64 * _log(rng, 4, 700), dtype,
                  rng.choice([0.25, 1.0, 4.0]))
        if c["pass"] == "inplace":
            c["max_norm"] = 1024.0      # clipped gradients would be others in the next pass over the same state
    c.pop("name", None)
    return c


def _shapes(case):
    """Parameter shapes of the language model with one projection to query, key, value and gate."""
    D = case["D"]
    block = [(D,), (D,), (4 * D, D), (4 * D,), (D, D), (D,), (D,), (D,), (4 * D, D), (4 * D,), (D, 4 * D), (D,)]
    return [(case["vocab"], D), (1024, D)] + block * case["layers"] + [(D,), (D,)]


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    st = {"case": case}
    train = case["pass"] == "train"
    if case["op"] == "glr":
        B, T, D = case["B"], case["T"], case["D"]
        gate = rnd(B, T, D) + (4.0 if case["gates"] == "open" else 0.0)
        if case["fused"]:
            ins = [torch.cat([rnd(B, T, D), gate], dim=-1), rnd(B, D)]
        else:
            ins = [rnd(B, T, D), torch.sigmoid(gate), rnd(B, D)]
        st["in"] = [t.to(dtype).requires_grad_(train) for t in ins]
        if train:
            st["up"] = [rnd(B, T, D).to(dtype), rnd(B, D).to(dtype)]
        if case["pass"] == "step":
            st["next"] = torch.empty(B, D, dtype=dtype, device=dev)
            st["out"] = torch.empty(B, 1, D, dtype=dtype, device=dev)
    elif case["op"] == "norm":
        rows, D = case["rows"], case["D"]
        ins = [rnd(rows, D), 4.0 * rnd(rows, D), 1.0 + 0.1 * rnd(D)] if case["add"] else [rnd(rows, D), 1.0 + 0.1 * rnd(D)]
        st["in"] = [t.to(dtype).requires_grad_(train) for t in ins]
        if train:
            st["up"] = [rnd(rows, D).to(dtype) for _ in range(2 if case["add"] else 1)]
    else:
        shapes = _shapes(case)
        sizes = [math.prod(s) for s in shapes]
        flat = (1e-3 * rnd(sum(sizes))).to(dtype)
        grads = [t.view(s) for t, s in zip(flat.split(sizes), shapes)]
        if case["pass"] == "inplace":
            st["flat"] = flat
            st["params"] = [torch.nn.Parameter(torch.zeros_like(t)) for t in grads]
            for p, t in zip(st["params"], grads):
                p.grad = t
        else:
            st["grads"] = [t.clone() for t in grads]
    return st


# ---- plain forms --------------------------------------------------------------------------------

def _scan(x, f):
    """All h_t of h_t = f_t h_{t-1} + x_t from zero, along dim 1, by doubling the reach of every step."""
    reach = 1
    while reach < x.shape[1]:
        x = torch.cat([x[:, :reach], x[:, reach:] + f[:, reach:] * x[:, :-reach]], dim=1)
        f = torch.cat([f[:, :reach], f[:, reach:] * f[:, :-reach]], dim=1)
        reach *= 2
    return x


def _from(x, f, start):
    """The same from a state: it enters through the first step."""
    return _scan(torch.cat([x[:, :1] + f[:, :1] * start[:, None], x[:, 1:]], dim=1), f)


def _gates(case, ins):
    if not case["fused"]:
        return ins[0].float(), ins[1].float(), None
    v, g = ins[0].float().chunk(2, dim=-1)
    return torch.sigmoid(-g) * v, torch.sigmoid(g), (v, torch.sigmoid(-g))


def _plain_glr(st):
    case, dtype = st["case"], DTYPES[st["case"]["dtype"]]
    ins = [t.detach() for t in st["in"]]
    x, f, parts = _gates(case, ins)
    s = ins[-1].float()
    h = _from(x, f, s)
    if case["pass"] == "step":
        st["out"].copy_(h)
        st["next"].copy_(h[:, -1])
        return st["out"], st["next"]
    out = (h.to(dtype), h[:, -1].to(dtype))
    if case["pass"] == "fwd":
        return out
    go, gs = (t.float() for t in st["up"])
    # r_t = go_t + f_{t+1} r_{t+1}: the same scan from the last step to the first, with the gates one step on
    go = torch.cat([go[:, :-1], go[:, -1:] + gs[:, None]], dim=1)
    ahead = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], dim=1)
    r = _scan(go.flip(1), ahead.flip(1)).flip(1)
    before = torch.cat([s[:, None], h[:, :-1]], dim=1)
    d_s = (f[:, 0] * r[:, 0]).to(dtype)
    if case["fused"]:
        v, rest = parts
        return (*out, torch.cat([rest * r, f * rest * r * (before - v)], dim=-1).to(dtype), d_s)
    return (*out, r.to(dtype), (r * before).to(dtype), d_s)


def _plain_norm(st):
    case, dtype = st["case"], DTYPES[st["case"]["dtype"]]
    ins = [t.detach().float() for t in st["in"]]
    s, w = (ins[0] + ins[1] if case["add"] else ins[0]), ins[-1]
    rstd = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
    y = s * rstd * w
    if case["pass"] == "e4m3":
        scale = (y.abs().amax(-1, keepdim=True) / E4M3_MAX).clamp_min(MIN_SCALE)
        q = (y / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return (q, scale, s.to(dtype)) if case["add"] else (q, scale)
    up = [t.float() for t in st["up"]]
    g = w * up[0]
    d_s = rstd * (g - s * rstd * rstd * (g * s).mean(-1, keepdim=True))
    d_w = (up[0] * s * rstd).sum(0).to(dtype)
    if case["add"]:
        d_s = (d_s + up[1]).to(dtype)
        return y.to(dtype), s.to(dtype), d_s, d_s, d_w
    return y.to(dtype), d_s.to(dtype), d_w


def _plain_clip(st):
    case = st["case"]
    grads = [p.grad for p in st["params"]] if case["pass"] == "inplace" else st["grads"]
    total = torch.sqrt(torch.stack([t.double().square().sum() for t in grads]).sum()).float()
    c = (case["max_norm"] / (total + 1e-6)).clamp_max(1.0)
    if case["pass"] == "inplace":
        [t.copy_(t.float() * c) for t in grads]
        return total, st["flat"]
    return total, [(t.float() * c).to(t.dtype) for t in grads]


# ---- the framework's operators --------------------------------------------------------------------

def _own_glr(st):
    from t2fw_b200.decode import glr_decode_step
    from t2fw_b200.functional_glr import GLRFunction, GLRFusedFunction

    case = st["case"]
    if case["pass"] == "step":
        return glr_decode_step(*st["in"], st["next"], st["out"])
    fn = GLRFusedFunction if case["fused"] else GLRFunction
    if case["pass"] == "fwd":
        with torch.no_grad():
            return fn.apply(*st["in"])
    out, nxt = fn.apply(*st["in"])
    return (out.detach(), nxt.detach(), *torch.autograd.grad([out, nxt], st["in"], st["up"]))


def _own_norm(st):
    from t2fw_b200.functional_norm import AddRMSNormFunction, RMSNormFunction, add_rms_norm_e4m3, rms_norm_e4m3

    case = st["case"]
    if case["pass"] == "e4m3":
        return (add_rms_norm_e4m3 if case["add"] else rms_norm_e4m3)(*st["in"], EPS)
    if case["add"]:
        y, s = AddRMSNormFunction.apply(*st["in"], EPS)
        return (y.detach(), s.detach(), *torch.autograd.grad([y, s], st["in"], st["up"]))
    y = RMSNormFunction.apply(*st["in"], EPS)
    return (y.detach(), *torch.autograd.grad([y], st["in"], st["up"]))


def _own_clip(st):
    from t2fw_b200.grad_clip import clip_grad_norm_, clip_grads

    case = st["case"]
    if case["pass"] == "inplace":
        return clip_grad_norm_(st["params"], case["max_norm"]), st["flat"]
    clipped, total = clip_grads(st["grads"], case["max_norm"])
    return total, clipped


def run(state):
    op = state["case"]["op"]
    if own:
        return {"glr": _own_glr, "norm": _own_norm, "clip": _own_clip}[op](state)
    with torch.no_grad():
        return {"glr": _plain_glr, "norm": _plain_norm, "clip": _plain_clip}[op](state)


def work(case):
    """Inputs once, outputs once; operations of the formulas as written, a special function as one."""
    e = 4 if case["dtype"] == "fp32" else 2
    train = case["pass"] == "train"
    if case["op"] == "glr":
        n, rows = case["B"] * case["T"] * case["D"], case["B"] * case["D"]
        elems = 3 * n + 2 * rows                             # value, gate, outputs; state in and out
        if train:
            elems += 3 * n + 2 * rows                        # upstream gradients, gradients of value, gate and state
        flops = ((6 if case["fused"] else 2) + ((8 if case["fused"] else 4) if train else 0)) * n
        return {"bytes": e * elems, "flops": flops}
    if case["op"] == "norm":
        n, D = case["rows"] * case["D"], case["D"]
        if case["pass"] == "e4m3":
            return {"bytes": e * ((3 if case["add"] else 1) * n + D) + n + 4 * case["rows"], "flops": (7 if case["add"] else 6) * n}
        # x, y, dy, dx; with a residual it, the sum, the sum's gradient too (one gradient serves x and the residual)
        return {"bytes": e * ((7 if case["add"] else 4) * n + 2 * D), "flops": (16 if case["add"] else 14) * n}
    n = sum(math.prod(s) for s in _shapes(case))
    clipped = 1e-3 * math.sqrt(n) > case["max_norm"]
    new = case["pass"] == "new"
    return {"bytes": e * n * (2 if new or clipped else 1) + 4, "flops": 3 * n}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _exact_glr(case, st):
    ins = [t.detach().double() for t in st["in"]]
    state, T = ins[-1], case["T"]
    if case["fused"]:
        D = case["D"]
        v, a = ins[0][..., :D], 1.0 / (1.0 + torch.exp(-ins[0][..., D:]))
        x, f = (1.0 - a) * v, a
    else:
        x, f = ins[0], ins[1]
    h = torch.empty_like(x)
    last = state
    for t in range(T):
        last = torch.addcmul(x[:, t], f[:, t], last)
        h[:, t] = last
    if case["pass"] != "train":
        return h, last
    go, carry = st["up"][0].double(), st["up"][1].double()
    r = torch.empty_like(x)
    for t in range(T - 1, -1, -1):
        r[:, t] = go[:, t] + carry
        carry = f[:, t] * r[:, t]
    d_f = r * torch.cat([state.unsqueeze(1), h[:, :-1]], dim=1)
    if not case["fused"]:
        return h, last, r, d_f, carry
    # x = (1 - a) v:  d_a = d_f - r v,  d_g = a (1 - a) d_a
    return h, last, torch.cat([(1.0 - a) * r, a * (1.0 - a) * (d_f - r * v)], dim=-1), carry


def _exact_norm(case, st):
    ins = [t.detach().double().requires_grad_(True) for t in st["in"]]
    s = ins[0] + ins[1] if case["add"] else ins[0]
    y = s * torch.rsqrt(s.square().sum(-1, keepdim=True) / case["D"] + EPS) * ins[-1]
    if case["pass"] == "e4m3":
        scale = torch.clamp(y.abs().max(dim=-1, keepdim=True).values / E4M3_MAX, min=MIN_SCALE)
        return (y / scale, scale, s) if case["add"] else (y / scale, scale)
    outs = [y, s] if case["add"] else [y]
    return (*outs, *torch.autograd.grad(outs, ins, [t.double() for t in st["up"]]))


def _exact_clip(case, st):
    flat = st["flat"].double() if case["pass"] == "inplace" else torch.cat([t.double().reshape(-1) for t in st["grads"]])
    total = torch.sqrt(torch.dot(flat, flat))
    c = min(1.0, case["max_norm"] / (float(total) + 1e-6))
    if case["pass"] == "inplace":
        return total, flat * c
    return total, [t.double() * c for t in st["grads"]]


def exact(case, seed):
    st = prepare(case, seed)
    with torch.set_grad_enabled(case["op"] == "norm"):
        got = {"glr": _exact_glr, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](case, st)
    detach = lambda v: [detach(t) for t in v] if isinstance(v, (list, tuple)) else v.detach()  # noqa: E731
    return detach(got)
