"""Linear8, LayerNorm8 and hooks that capture in 8 bits in the places of the layers they
replace: dtypes under autocast, several sets of hooks, threads, captured training steps."""
import threading

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

BF, F4 = torch.bfloat16, torch.float32


def mods():
    from ifkfac_b200 import activation_hooks, checkpoint8, engine
    return activation_hooks, checkpoint8, engine


def randn(*shape, seed=0, dtype=F4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("dtype", [F4, BF])
def test_converted_norms_have_the_dtype_of_those_they_replace(dtype, autocast):
    """nn.LayerNorm gives fp32 under autocast, and so does a converted one unless it is asked not to:
    in a post-norm block its output is the residual stream."""
    _, c8, _ = mods()
    ref = nn.LayerNorm(96, device="cuda", dtype=F4 if autocast else dtype)
    x = randn(5, 7, 96, dtype=dtype)
    with torch.autocast("cuda", dtype=BF, enabled=autocast):
        want = ref(x)
        y = c8.convert(nn.Sequential(ref))[0](x)
        narrow = c8.convert(nn.Sequential(ref), autocast_norms=True)[0](x)
        direct = c8.LayerNorm8(96, device="cuda", autocast_output=False)(x)
    assert y.dtype == want.dtype == (F4 if autocast else dtype)
    assert narrow.dtype == (BF if autocast else dtype) and direct.dtype == want.dtype
    # both are fp32 statistics and one rounding: 2^-8 of the value in bf16; in fp32 sums of 96 terms and a few products
    tol = 2.0 ** -8 if y.dtype == BF else 104 * 2.0 ** -23
    assert ((y.double() - want.double()).abs() <= 2 * tol * (1 + want.double().abs())).all()


def test_a_converted_post_norm_block_keeps_its_residual_stream():
    _, c8, _ = mods()

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.fc, self.norm = nn.Linear(64, 64), nn.LayerNorm(64)

        def forward(self, x):
            return self.norm(x + self.fc(x))

    torch.manual_seed(0)
    model = nn.Sequential(Block(), Block()).cuda()
    x = randn(3, 64)
    with torch.autocast("cuda", dtype=BF):
        want = model(x)
        got = c8.convert(model)(x)
    assert want.dtype == got.dtype == F4
    got.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


def counted(monkeypatch, engine):
    packed, pack = [], engine.quantize_rows
    monkeypatch.setattr(engine, "quantize_rows", lambda *a, **k: packed.append(1) or pack(*a, **k))
    return packed


def rounded(x):
    _, c8, _ = mods()
    return c8.dequantize_rows(c8.quantize_rows(x.reshape(-1, x.shape[-1])), F4)


def test_several_sets_of_hooks_share_a_layers_rows(monkeypatch):
    """Hooks that do not capture in 8 bits leave the rows to those that do, two sets that do both get
    them, and one that goes takes nothing from the other."""
    AH, c8, engine = mods()
    model = nn.Sequential(c8.Linear8(40, 24, device="cuda"))
    plain = AH.RawActivationHooks(model, batched=True)
    one, two = (AH.RawActivationHooks(model, batched=True, capture_8bit=True) for _ in range(2))
    for h in (plain, one, two):
        h.enable()
    packed = counted(monkeypatch, engine)
    x = randn(50, 40)
    with torch.no_grad():
        model(x)                                             # no rows of the layer's own
    assert len(packed) == 2
    for h in (one, two):
        h.clear()
    del packed[:]
    y = model(x)
    assert not packed and model[0]._last_rows is None
    a, b = one._pending_X[model[0]][0], two._pending_X[model[0]][0]
    assert a.q is b.q and torch.equal(a.unpack(F4).x, rounded(x))
    assert isinstance(plain._pending_X[model[0]][0], engine.Rows)
    y.sum().backward()
    del packed[:]
    one.remove()
    model(x)
    assert not packed and torch.equal(two._pending_X[model[0]][1].unpack(F4).x, rounded(x))
    two.remove()
    plain.remove()


def test_rows_of_a_pass_within_another_ones_hooks():
    """A forward pass of the layer, of as many rows, between a pass and its hooks."""
    AH, c8, engine = mods()
    model = nn.Sequential(c8.Linear8(40, 24, device="cuda"))
    first, second = randn(50, 40, seed=1), randn(50, 40, seed=2)
    handle = model[0].register_forward_hook(lambda m, i, o: [m.forward(second), None][1])
    hooks = AH.RawActivationHooks(model, batched=True, capture_8bit=True)
    hooks.enable()
    model(first)
    kept, = hooks._pending_X[model[0]]
    assert torch.equal(kept.unpack(F4).x, rounded(first))
    hooks.remove()
    handle.remove()


def test_threads_in_one_layer_keep_their_own_rows():
    AH, c8, engine = mods()
    model = nn.Sequential(c8.Linear8(64, 16, device="cuda"))
    hooks = AH.RawActivationHooks(model, batched=True, capture_8bit=True)
    got = {}
    accumulate = hooks._accumulate
    hooks._accumulate = lambda m, c, *a: (got.setdefault(threading.get_ident(), []).append(c), accumulate(m, c, *a))
    hooks.enable()
    xs = [randn(32, 64, seed=k) for k in range(4)]
    ids, start = {}, threading.Barrier(4)

    def work(k):
        ids[k] = threading.get_ident()
        start.wait()
        for _ in range(25):
            model(xs[k])
        start.wait()                                         # no thread's identity is used again

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(4):
        want = rounded(xs[k])
        assert len(got[ids[k]]) == 25
        for c in got[ids[k]]:
            c = c if isinstance(c, engine.PackedRows) else engine.PackedRows.pack(c)
            assert torch.equal(c.unpack(F4).x, want)
    hooks.remove()


def test_a_captured_training_step():
    """Forward and backward of LayerNorm8 and Linear8 captured in a graph and replayed on new inputs: the
    bits of the eager step."""
    _, c8, _ = mods()
    torch.manual_seed(0)
    model = c8.convert(nn.Sequential(nn.LayerNorm(96), nn.Linear(96, 72), nn.GELU(), nn.Linear(72, 40))).cuda()
    params = list(model.parameters())
    x = randn(130, 96)

    def step():
        with torch.autocast("cuda", dtype=BF, cache_enabled=False):
            loss = model(x).float().square().mean()
        return torch.autograd.grad(loss, params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6):
        x.copy_(randn(130, 96, seed=seed))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_recomputed_and_offloaded_activations():
    """The same gradients, bit for bit, with the block recomputed in its backward pass and with the saved
    rows kept on the host meanwhile."""
    from torch.utils.checkpoint import checkpoint
    _, c8, _ = mods()
    torch.manual_seed(0)
    model = c8.convert(nn.Sequential(nn.LayerNorm(64), nn.Linear(64, 128), nn.GELU(), nn.Linear(128, 64))).cuda()
    x = randn(6, 30, 64).requires_grad_()

    def grads(run):
        with torch.autocast("cuda", dtype=BF):
            loss = run(x).float().square().mean()
        return torch.autograd.grad(loss, [x, *model.parameters()])

    want = grads(model)
    assert all(torch.equal(p, q) for p, q in zip(grads(lambda t: checkpoint(model, t, use_reentrant=False)), want))
    with torch.autograd.graph.save_on_cpu():
        got = grads(model)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
