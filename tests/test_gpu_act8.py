"""Linear8, LayerNorm8 and hooks that capture in 8 bits: gradients against the formulas on
the rounded rows, factors against the folds of those rows, and a run of all of them.

A sum of K fp32 terms is off by at most K 2^-23 times the sum of their magnitudes; a
bf16 product of the library's rounds its result by 2^-8."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

BF, F4 = torch.bfloat16, torch.float32
U2 = 2.0 ** -23


def mods():
    from ifkfac_b200 import activation_hooks, checkpoint8, engine
    return activation_hooks, checkpoint8, engine


def randn(*shape, seed=0, dtype=F4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rounded(x):
    _, c8, _ = mods()
    return c8.dequantize_rows(c8.quantize_rows(x.reshape(-1, x.shape[-1])), F4).double()


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_linear8_forward_is_linear_and_gradients_are_the_formulas(bias, autocast):
    _, c8, _ = mods()
    torch.manual_seed(0)
    ref = nn.Linear(200, 72, bias=bias).cuda()
    m = c8.Linear8.from_linear(ref)
    x = randn(3, 50, 200).requires_grad_()
    with torch.autocast("cuda", dtype=BF, enabled=autocast):
        y, want = m(x), ref(x)
    assert y.dtype == want.dtype and torch.equal(y, want)
    dy = randn(3, 50, 72, seed=1, dtype=y.dtype)
    gx, = torch.autograd.grad(want, x, dy, retain_graph=True)
    y.backward(dy)
    assert torch.equal(x.grad, gx)                           # the input gradient is nn.Linear's
    d, X = dy.reshape(-1, 72).double(), rounded(x.detach())
    assert m.weight.grad.dtype == F4
    assert ((m.weight.grad.double() - d.t() @ X).abs() <= 151 * U2 * (d.abs().t() @ X.abs())).all()
    if bias:
        assert ((m.bias.grad.double() - d.sum(0)).abs() <= 151 * U2 * d.abs().sum(0)).all()
    # against differences: the loss is linear in W and b, up to X's rounding (at most a / 64 a group)
    V = randn(72, 200, seed=2)
    num = (F.linear(x.detach().reshape(-1, 200).double(), V.double()) * d).sum()
    a = x.detach().reshape(-1, 200).abs()
    a = F.pad(a, (0, 24)).view(150, 7, 32).amax(-1, keepdim=True).expand(150, 7, 32).reshape(150, 224)[:, :200]
    slack = (d.abs() @ V.double().abs() * a.double() / 64).sum()
    assert abs(float((m.weight.grad.double() * V.double()).sum() - num)) <= float(slack)


def test_linear8_frozen_and_inference():
    _, c8, _ = mods()
    m = c8.Linear8(64, 32).cuda()
    x = randn(5, 64)
    with torch.no_grad():
        assert torch.equal(m(x), F.linear(x, m.weight, m.bias))
    assert m._last_rows is None
    m.weight.requires_grad_(False)
    xg = x.clone().requires_grad_()
    m(xg).sum().backward()
    assert m.weight.grad is None and torch.allclose(m.bias.grad, torch.full((32,), 5.0, device="cuda"))
    assert torch.allclose(xg.grad, m.weight.sum(0).expand(5, 64), rtol=1e-5, atol=1e-5)
    m = c8.Linear8(64, 32).cuda().to(BF)
    m(x.to(BF)).sum().backward()
    assert m.weight.grad.dtype == BF and m.bias.grad.dtype == BF
    with pytest.raises(TypeError):
        m(x)                                                 # fp32 rows, bf16 weight
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(TypeError):
        m(x)
    empty = c8.Linear8(64, 32).cuda()
    empty(x[:0]).sum().backward()
    assert (empty.weight.grad == 0).all() and (empty.bias.grad == 0).all()


@pytest.mark.parametrize("affine,bias", [(True, True), (True, False), (False, False)])
def test_layernorm8_is_the_functional_pair(affine, bias):
    _, c8, _ = mods()
    ref = nn.LayerNorm(96, elementwise_affine=affine, bias=bias).cuda()
    if affine:
        ref.weight.data += 0.1 * randn(96, seed=3)
    m = c8.LayerNorm8.from_layer_norm(ref)
    x = randn(4, 7, 96).requires_grad_()
    dy = randn(4, 7, 96, seed=1)
    y = m(x)
    yy, saved = c8.layer_norm_forward(x.detach().reshape(-1, 96), ref.weight, ref.bias, save=True, checkpoint=True)
    assert torch.equal(y.reshape(-1, 96), yy) and torch.allclose(y, ref(x), rtol=1e-5, atol=1e-5)
    y.backward(dy)
    dx, dw, db = c8.layer_norm_backward(dy.reshape(-1, 96), saved, ref.weight)
    assert torch.equal(x.grad.reshape(-1, 96), dx)
    if affine:
        assert torch.equal(m.weight.grad, dw)
    if bias:
        assert torch.equal(m.bias.grad, db)
    with torch.autocast("cuda", dtype=BF):
        assert m(x).dtype == BF
    with torch.no_grad():
        assert torch.equal(m(x), y)
    with pytest.raises(ValueError):
        m(x[..., :95])


def _capture(mode, precision, subsample, model, x, **kw):
    AH, _, _ = mods()
    hooks = AH.RawActivationHooks(model, damping=1e-2, augment_bias=True, max_seq_rows=subsample,
                                  batched=mode == "batched", deferred=mode == "deferred", precision=precision, **kw)
    hooks.enable()
    for k in range(3):
        torch.manual_seed(100 + k)  # the subsamples' randperm
        model(x[k]).square().sum().backward()
    return hooks


@pytest.mark.parametrize("mode", ["batched", "deferred"])
@pytest.mark.parametrize("precision", [0, 1, 2])
@pytest.mark.parametrize("subsample", [0, 64])
@pytest.mark.parametrize("conv", [False, True])
def test_hooks_fold_the_rounded_rows(mode, precision, subsample, conv, monkeypatch):
    """Factors captured in 8 bits are, bit for bit, those of folding the rounded rows
    (values exact in both types), with nn.Linear and with Linear8, whose rows are shared."""
    AH, c8, engine = mods()
    torch.manual_seed(0)
    base = nn.Sequential(nn.Linear(40, 24), nn.GELU(), nn.Linear(24, 16)).cuda()
    x = [randn(2, 100, 40, seed=k) for k in range(3)]
    model = base
    if conv:
        model = c8.convert(nn.Sequential(*base))
        assert type(model[0]) is c8.Linear8
    packed = []
    pack = engine.quantize_rows
    monkeypatch.setattr(engine, "quantize_rows", lambda *a, **k: packed.append(1) or pack(*a, **k))
    hooks = _capture(mode, precision, subsample, model, x, capture_8bit=True)
    # 3 passes x 2 layers, X and delta; a Linear8 layer's X is packed already
    assert len(packed) == (6 if conv else 12)
    pend = hooks._pending_X if mode == "batched" else hooks._raw_X
    rows = [c for m in hooks.linear_layers for c in pend[m]]
    assert rows and all(isinstance(c, engine.PackedRows) and c.ones for c in rows)
    keep = [(t, m, list(p[m])) for t, p in
            ((0, pend), (1, hooks._pending_G if mode == "batched" else hooks._raw_G)) for m in hooks.linear_layers]
    want = []
    for t, m, chunks in keep:
        f = engine.Factor(chunks[0].cols, "cuda", precision)
        engine.fold_segments([f], [[c.unpack() for c in chunks]], None)
        want.append(f)
    monkeypatch.setattr(type(hooks), "_UNPACK_BYTES", 20000)  # several fold calls
    if mode == "batched":
        hooks.flush()
    factors = hooks.get_factors()
    for (t, m, _), f in zip(keep, want):
        got = (hooks._R_X if t == 0 else hooks._R_G)[m]
        assert torch.equal(got, f.R[: f.rows_R]), (t, m)
        assert f.rows_seen == (hooks._n_rows_X if t == 0 else hooks._n_rows_G)[m] == 3 * (subsample or 200)
    assert len(factors) == 2
    hooks.clear()
    assert not any(pend[m] for m in hooks.linear_layers)
    hooks.remove()
    if conv:
        model(x[0]).sum().backward()
        assert model[0]._last_rows is None and not model[0]._share_rows   # nothing kept once the hooks are gone


def test_paused_hooks_keep_no_rows():
    AH, c8, _ = mods()
    model = c8.convert(nn.Sequential(nn.Linear(40, 24))).cuda()
    hooks = AH.RawActivationHooks(model, batched=True, capture_8bit=True)
    hooks.enable()
    hooks.pause()
    model(randn(5, 40)).sum().backward()
    assert model[0]._last_rows is None and not hooks._pending_X[model[0]]
    hooks.resume()
    with torch.no_grad():                                     # no backward pass: the hooks pack X themselves
        model(randn(5, 40))
    assert hooks._pending_X[model[0]][0].rows == 5
    hooks.remove()


def test_rows_that_no_hook_took_are_not_the_next_passs():
    """forward() called past the hooks leaves its rows; a pass without gradients has none of its own."""
    hooks_mod, c8, engine = mods()
    model = nn.Sequential(c8.Linear8(64, 32, device="cuda"))
    hooks = hooks_mod.RawActivationHooks(model, batched=True, capture_8bit=True)
    hooks.enable()
    first, second = randn(40, 64, seed=1), randn(24, 64, seed=2)
    model[0].forward(first)
    with torch.no_grad():
        model(second)
    kept, = hooks._pending_X[model[0]]
    assert torch.equal(kept.unpack(F4).x.double(), rounded(second))
    hooks.remove()


def test_conv_inputs_stay_images():
    AH, _, engine = mods()
    model = nn.Sequential(nn.Conv2d(3, 8, 3, padding=1), nn.Flatten(), nn.Linear(8 * 36, 5)).cuda()
    hooks = AH.RawActivationHooks(model, damping=1e-2, max_conv_rows=0, batched=True, capture_8bit=True)
    hooks.enable()
    for k in range(8):
        model(randn(40, 3, 6, 6, seed=k)).square().sum().backward()
    conv, lin = hooks.linear_layers
    assert hooks._pending_X[conv][0].geo is not None
    assert isinstance(hooks._pending_G[conv][0], engine.PackedRows) and hooks._pending_G[conv][0].rows == 40 * 36
    hooks.flush()
    assert hooks.get_factors().keys() == {conv, lin}
    hooks.remove()


def test_a_run_of_all_of_them():
    """A small decoder block as bench.py's workloads have it: LayerNorm8 into Linear8 under
    autocast, captured in 8 bits by IFKFAC, three steps over one refresh interval.  Its
    gradients are those of the same model with the layers' own rules done by hand."""
    from ifkfac_b200 import IFKFAC
    _, c8, _ = mods()

    class Block(nn.Module):
        def __init__(self, d=64):
            super().__init__()
            self.ln, self.fc, self.fc2 = nn.LayerNorm(d), nn.Linear(d, 4 * d), nn.Linear(4 * d, d)

        def forward(self, x):
            return x + self.fc2(F.gelu(self.fc(self.ln(x))))

    torch.manual_seed(0)
    model = c8.convert(nn.Sequential(Block(), Block())).cuda()
    opt = IFKFAC(model, lr=1e-2, damping=1e-2, factor_update_freq=2, momentum=0.9, use_true_bf16=True,
                 max_seq_rows=0, batched_qr=True, capture_8bit=True)
    x, t = randn(6, 80, 64), randn(6, 80, 64, seed=1)
    seen = {}

    def keep(m, inp, out):
        seen[m] = (inp[0].detach(), out)
        out.retain_grad()

    hs = [m.register_forward_hook(keep) for m in model.modules() if isinstance(m, (c8.Linear8, c8.LayerNorm8))]
    w0 = [p.detach().clone() for p in model.parameters()]
    for step in range(3):
        model.zero_grad()  # the layer norms' parameters are not the optimizer's
        with torch.autocast("cuda", dtype=BF):
            loss = (model(x) - t).square().mean()
        loss.backward()
        for m, (inp, out) in seen.items():
            d = out.grad.reshape(-1, out.shape[-1])
            if isinstance(m, c8.Linear8):
                D, X = d.double(), rounded(inp)
                assert ((m.weight.grad.double() - D.t() @ X).abs() <= 481 * U2 * (D.abs().t() @ X.abs())).all()
            else:
                x2 = inp.reshape(-1, 64)
                _, s = c8.layer_norm_forward(x2, m.weight, m.bias, m.eps, out.dtype, save=True, checkpoint=True)
                _, dw, db = c8.layer_norm_backward(d, s, m.weight)
                assert torch.equal(m.weight.grad, dw) and torch.equal(m.bias.grad, db)
        opt.step()
        assert torch.isfinite(loss)
    assert len(opt._factors) == 4 and all(torch.isfinite(f).all() for p in opt._factors.values() for f in p)
    for m in opt.hooks.linear_layers:
        assert torch.isfinite(m.weight).all()
    moved = [not torch.equal(p, q) for p, q in zip(model.parameters(), w0)]
    assert sum(moved) >= 8                                    # the weights and biases of the four Linear8 layers
    for h in hs:
        h.remove()
    opt.cleanup()
