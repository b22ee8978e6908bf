"""The gated linear recurrence, the root-mean-square norm and gradient clipping as the language model uses them together."""
import copy

import pytest
import torch
import torch.nn.functional as F

from layer_ref import assert_within, clip

pytestmark = pytest.mark.gpu


def _config(rule="glr", norm="rms", **kw):
    from t2fw_b200.gpt2_fw import GPT2FWConfig

    return GPT2FWConfig(**{**dict(vocab_size=200, n_positions=128, d_model=64, n_head=1, n_layer=2, rule=rule, norm=norm), **kw})


def _norm(m, x):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + m.eps) * m.weight


def reference_loss(model, ids, targets):
    """The model with rule="glr" and norm="rms" from its definition, in the type of its parameters, on the CPU."""
    x = model.wte(ids) + model.wpe(torch.arange(ids.shape[1]))
    for blk in model.blocks:
        v, g = blk.attn.qkv(_norm(blk.ln1, x)).chunk(2, dim=-1)
        a, h, hs = torch.sigmoid(g), torch.zeros_like(v[:, 0]), []
        for t in range(v.shape[1]):
            h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
            hs.append(h)
        x = x + blk.attn.proj(torch.stack(hs, 1))
        x = x + blk.out(F.gelu(blk.fc(_norm(blk.ln2, x)), approximate="tanh"))
    logits = F.linear(_norm(model.ln_f, x), model.wte.weight)
    return F.cross_entropy(logits.flatten(0, 1), targets.flatten())


def test_training_step_matches_the_definition(cuda):
    """fp32 model against the same model in 64 bits on the CPU: loss, every gradient, the clipped gradients and their norm."""
    from t2fw_b200.gpt2_fw import GPT2FW
    from t2fw_b200.grad_clip import clip_grad_norm_

    torch.backends.cuda.matmul.allow_tf32 = False
    torch.manual_seed(3)
    model = GPT2FW(_config())
    for p in model.parameters():      # norms and biases away from 1 and 0
        p.data.add_(0.05 * torch.randn_like(p))
    exact = copy.deepcopy(model).double()
    model = model.to(cuda)
    ids = torch.randint(0, 200, (3, 101))
    want = reference_loss(exact, ids[:, :-1], ids[:, 1:])
    want.backward()
    got = model(ids[:, :-1].to(cuda), targets=ids[:, 1:].to(cuda))
    got.backward()
    # Nothing here is rounded below fp32 (2^-24).  A value passes some 20 layers of operations, each a sum of up to 256 products,
    # so a relative error of 20 * 256 * 2^-24 = 3e-4 of the largest entry of a tensor is more than the roundings can make.
    tol = 20 * 256 * 2.0 ** -24
    assert abs(float(got.detach()) - float(want.detach())) <= tol * float(want.detach())
    for (name, p), q in zip(model.named_parameters(), exact.parameters()):
        assert_within(p.grad.cpu(), q.grad, torch.full_like(q.grad, tol * float(q.grad.abs().max())), name)
    total, c = clip([q.grad for q in exact.parameters()], 0.5)
    before = [p.grad.clone() for p in model.parameters()]
    norm = clip_grad_norm_(model.parameters(), 0.5)
    assert c < 1 and abs(float(norm) - float(total)) <= tol * float(total)
    for p, b in zip(model.parameters(), before):
        assert_within(p.grad, b.double() * (0.5 / (float(norm) + 1e-6)), 2.0 ** -21 * b.double().abs() + 2.0 ** -149)


@pytest.mark.parametrize("rule", ["dfw", "lfw", "glr"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_all_pairs_of_rule_and_norm_train(cuda, rule, norm):
    from t2fw_b200.gpt2_fw import GPT2FW
    from t2fw_b200.grad_clip import clip_grad_norm_

    torch.manual_seed(4)
    model = GPT2FW(_config(rule, norm)).half().to(cuda)
    ids = torch.randint(0, 200, (2, 71), device=cuda)
    for _ in range(2):
        model.zero_grad()
        loss = model(ids[:, :-1], targets=ids[:, 1:])
        loss.backward()
        clip_grad_norm_(model.parameters(), 1.0, error_if_nonfinite=True)
        assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in model.parameters())
        assert all(bool(p.grad.any()) for p in model.parameters())


def test_model_without_blocks(cuda):
    from t2fw_b200.gpt2_fw import GPT2FW

    model = GPT2FW(_config(n_layer=0)).to(cuda)
    ids = torch.randint(0, 200, (2, 9), device=cuda)
    want = F.linear(_norm(model.ln_f, model.wte(ids) + model.wpe(torch.arange(9, device=cuda))), model.wte.weight)
    got = model(ids)
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_eight_bit_linear(cuda, dtype):
    """Norm and projection in 8 bits against 64-bit products of the same 8-bit values."""
    from t2fw_b200.functional_norm import rms_norm_e4m3
    from t2fw_b200.gpt2_fw import Linear8

    torch.manual_seed(5)
    lin = torch.nn.Linear(64, 96).to(cuda, dtype)
    lin8 = Linear8(lin)
    # half a step of e4m3 is 2^-4 of a value, 2^-10 of the scale below the smallest normal
    w = lin.weight.double()
    back = lin8.weight.double() * lin8.scale.double().t()
    assert_within(back, w, 2.0 ** -4 * w.abs() + 2.0 ** -10 * lin8.scale.double().t() + 2.0 ** -20 * w.abs())
    for rows in ((7,), (1,), (2, 33)):
        x = torch.randn(*rows, 64, device=cuda).to(dtype)
        with torch.no_grad():
            q, s = rms_norm_e4m3(x, torch.ones(64, device=cuda, dtype=dtype), 1e-5)
            y = lin8((q, s))
        ref = q.double() * s.double() @ back.t() + lin.bias.double()
        # products of two 4-bit significands are exact, their fp32 sum, the two scales and the bias are not: 64 + 4 roundings
        mag = (q.double() * s.double()).abs() @ back.t().abs() + lin.bias.double().abs()
        assert y.dtype == dtype and y.shape == (*rows, 96)
        assert_within(y, ref, torch.finfo(dtype).eps / 2 * ref.abs() + 70 * 2.0 ** -24 * mag + 2.0 ** -24)


@pytest.mark.parametrize("rule", ["glr", "lfw"])
def test_eight_bit_model_runs(cuda, rule):
    from t2fw_b200.gpt2_fw import GPT2FW

    torch.manual_seed(6)
    model = GPT2FW(_config(rule)).bfloat16().to(cuda)
    ids = torch.randint(0, 200, (2, 50), device=cuda)
    with torch.no_grad():
        got = copy.deepcopy(model).eight_bit_()(ids)
    assert got.shape == (2, 50, 256) and torch.isfinite(got).all()
    with pytest.raises(RuntimeError, match="no gradients"):
        copy.deepcopy(model).eight_bit_()(ids)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 32, 1000, 8192])
def test_eight_bit_linear_at_the_models_sizes(cuda, rows, dtype):
    """d_model to the widths behind the norms: value | gate, and query | key | value | gate or the feed-forward layer's first."""
    from t2fw_b200.functional_norm import rms_norm_e4m3
    from t2fw_b200.gpt2_fw import GPT2FWConfig, Linear8

    d = GPT2FWConfig().d_model
    torch.manual_seed(7)
    x = torch.randn(rows, d, device=cuda).to(dtype)
    with torch.no_grad():
        q, s = rms_norm_e4m3(x, 1 + 0.1 * torch.randn(d, device=cuda).to(dtype), 1e-5)
    for out in (2 * d, 4 * d):
        lin8 = Linear8(torch.nn.Linear(d, out).to(cuda, dtype))
        with torch.no_grad():
            y = lin8((q, s))
        assert y.dtype == dtype and y.shape == (rows, out)
        _check_product(y, q, s, lin8)


def _check_product(y, q, s, lin8):
    """y against 64-bit products of the same 8-bit values: those of two 4-bit significands are exact, their fp32 sum, the two
    scales and the bias are not, d + 4 roundings."""
    w = lin8.weight.double() * lin8.scale.double().t()
    a = q.double().flatten(0, -2) * s.double().flatten(0, -2)
    ref = a @ w.t() + lin8.bias.double()
    mag = a.abs() @ w.abs().t() + lin8.bias.double().abs()
    tol = torch.finfo(y.dtype).eps / 2 * ref.abs() + (q.shape[-1] + 6) * 2.0 ** -24 * mag + 2.0 ** -24
    assert_within(y.flatten(0, -2), ref, tol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rule", ["glr", "lfw"])
def test_eight_bit_model_at_full_width(cuda, rule, dtype):
    """Every 8-bit norm and projection inside the model, on what it was given there: the norm against its definition, the product
    against 64 bits.  And a model that is cast behind eight_bit_() raises."""
    from t2fw_b200.gpt2_fw import GPT2FW, GPT2FWConfig

    torch.manual_seed(8)
    model = GPT2FW(GPT2FWConfig(vocab_size=500, n_positions=256, n_layer=2, rule=rule, norm="rms")).to(cuda, dtype)
    for p in model.parameters():
        p.data.add_(0.02 * torch.randn_like(p))
    model.eight_bit_()
    seen = []

    def norm_hook(m, args, out):
        x, residual = args[0], args[1] if len(args) > 1 else None
        (q, scale), s = (out[0], out[1]) if residual is not None else (out, None)
        total = x.double() + (0 if residual is None else residual.double())
        if s is not None:
            assert_within(s, total, (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * total.abs() + 2.0 ** -25)
        y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + m.eps) * m.weight.double()
        k = (x.shape[-1] / 32 + 26) * 2.0 ** -24
        want = (y.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-30)
        assert_within(scale, want, k * want)
        v = y / scale.double()
        assert_within(q.double(), v, 2.0 ** -4 * v.abs().clamp_min(2.0 ** -6) + 2 * k * v.abs())
        seen.append("norm")

    def product_hook(m, args, out):
        _check_product(out, *args[0], m)
        seen.append("product")

    for blk in model.blocks:
        for m, hook in ((blk.ln1, norm_hook), (blk.ln2, norm_hook), (blk.attn.qkv, product_hook), (blk.fc, product_hook)):
            m.register_forward_hook(hook)
    ids = torch.randint(0, 500, (2, 130), device=cuda)
    with torch.no_grad():
        logits = model(ids)
    assert torch.isfinite(logits).all() and sorted(seen) == ["norm"] * 4 + ["product"] * 4
    other = torch.bfloat16 if dtype == torch.float16 else torch.float16
    with torch.no_grad(), pytest.raises(RuntimeError):
        model.to(other)(ids)
