"""8-bit rows and layer norm on the host: the format, the checks of arguments, the
conversion of a model.  Nothing here runs on a GPU."""
import ctypes

import numpy as np
import pytest
import torch
import torch.nn as nn

from ifkfac_b200 import _lib
from ifkfac_b200 import checkpoint8 as c8
from tests import q8_reference as ref

FAKE = ctypes.c_void_p(4096)


def test_format_bounds():
    """The oracle's format keeps what include/ifk.h promises: |x - value| <= 2^e <= a / 64."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((64, 100)) * np.exp(rng.uniform(-40, 40, (64, 1)))
    x[3] = 0
    codes, scales = ref.quantize(x)
    v = ref.values(codes, scales, 100)
    step = np.repeat(np.exp2(scales.astype(float) - 127), 32, axis=1)[:, :100]
    assert (np.abs(x - v) <= step).all()
    a = np.abs(np.pad(x, ((0, 0), (0, 28)))).reshape(64, 4, 32).max(-1)
    assert (np.exp2(scales.astype(float) - 127)[a > 0] <= a[a > 0] / 64).all()
    assert codes.shape == (64, 128) and (codes[:, 100:] == 0).all()


@pytest.mark.parametrize("n,pitch", [(1, 32), (31, 32), (32, 32), (33, 64), (4096, 4096), (4097, 4128)])
def test_pitch(n, pitch):
    assert _lib.lib().ifk_q8_pitch(n) == pitch
    assert _lib.lib().ifk_q8_pitch(0) == 0


def test_q8_argument_errors_before_any_gpu_work():
    L = _lib.lib()

    def quant(x=FAKE, ld=64, dt=_lib.BF16, idx=None, src=8, rows=8, n=64, codes=FAKE, ldc=64, scales=FAKE, lds=2):
        return L.ifk_q8_quantize(x, ld, dt, idx, src, rows, n, codes, ldc, scales, lds, None, None)

    assert quant(rows=-1) == _lib.ERR_SHAPE
    assert quant(n=0) == _lib.ERR_SHAPE
    assert quant(ld=63) == _lib.ERR_SHAPE
    assert quant(dt=2) == _lib.ERR_DTYPE
    assert quant(x=None) == _lib.ERR_ARG
    assert quant(codes=None) == _lib.ERR_ARG
    assert quant(codes=ctypes.c_void_p(4100)) == _lib.ERR_ARG       # codes are 16-byte aligned
    assert quant(n=65, ld=80) == _lib.ERR_SHAPE                     # the pitch of 65 columns is 96
    assert quant(ldc=72) == _lib.ERR_SHAPE                          # not a multiple of 16
    assert quant(lds=1) == _lib.ERR_SHAPE
    assert quant(idx=FAKE, src=0) == _lib.ERR_SHAPE
    assert quant(rows=0, x=None, codes=None) == _lib.OK             # nothing to do

    def deq(codes=FAKE, ldc=64, scales=FAKE, lds=2, idx=None, src=8, rows=8, n=64, out=FAKE, ld=64, dt=_lib.F32):
        return L.ifk_q8_dequantize(codes, ldc, scales, lds, idx, src, rows, n, out, ld, dt, None, None)

    assert deq(out=None) == _lib.ERR_ARG
    assert deq(scales=None) == _lib.ERR_ARG
    assert deq(ld=63) == _lib.ERR_SHAPE
    assert deq(ldc=32) == _lib.ERR_SHAPE
    assert deq(dt=3) == _lib.ERR_DTYPE
    assert deq(idx=FAKE, src=-1) == _lib.ERR_SHAPE
    assert deq(rows=0, out=None) == _lib.OK


def test_wgrad_argument_errors_before_any_gpu_work():
    L = _lib.lib()
    need = L.ifk_q8_wgrad_workspace(8, 16, 64, _lib.BF16)
    assert need > 0
    assert L.ifk_q8_wgrad_workspace(8, 0, 64, _lib.BF16) == 0
    assert L.ifk_q8_wgrad_workspace(-1, 16, 64, _lib.BF16) == 0
    assert L.ifk_q8_wgrad_workspace(8, 16, 64, 7) == 0

    def wgrad(delta=FAKE, ld=16, dt=_lib.BF16, codes=FAKE, ldc=64, scales=FAKE, lds=2, rows=8, n_out=16, n_in=64,
              dW=FAKE, ldw=64, ws=FAKE, wsb=need):
        return L.ifk_q8_wgrad(delta, ld, dt, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, None, 0, None, ws,
                              wsb, None)

    assert wgrad(dW=None) == _lib.ERR_ARG
    assert wgrad(delta=None) == _lib.ERR_ARG
    assert wgrad(codes=None) == _lib.ERR_ARG
    assert wgrad(dt=5) == _lib.ERR_DTYPE
    assert wgrad(rows=-1) == _lib.ERR_SHAPE
    assert wgrad(n_out=0) == _lib.ERR_SHAPE
    assert wgrad(n_in=0) == _lib.ERR_SHAPE
    assert wgrad(ld=15) == _lib.ERR_SHAPE
    assert wgrad(ldw=63) == _lib.ERR_SHAPE
    assert wgrad(ldc=48) == _lib.ERR_SHAPE
    assert wgrad(ws=None) == _lib.ERR_WORKSPACE
    assert wgrad(ws=ctypes.c_void_p(4097)) == _lib.ERR_WORKSPACE
    assert wgrad(wsb=need - 1) == _lib.ERR_WORKSPACE


def test_layernorm_argument_errors_before_any_gpu_work():
    L = _lib.lib()

    def fwd(x=FAKE, ldx=64, xd=_lib.F32, w=FAKE, b=FAKE, wd=_lib.F32, rows=4, n=64, eps=1e-5, y=FAKE, ldy=64,
            yd=_lib.BF16, codes=None, ldc=64, scales=None, lds=2):
        return L.ifk_layernorm(x, ldx, xd, w, b, wd, rows, n, eps, y, ldy, yd, None, None, codes, ldc, scales, lds,
                               None)

    assert fwd(x=None) == _lib.ERR_ARG
    assert fwd(y=None) == _lib.ERR_ARG
    assert fwd(codes=FAKE) == _lib.ERR_ARG                  # codes without scales
    assert fwd(codes=FAKE, scales=FAKE, ldc=32) == _lib.ERR_SHAPE
    assert fwd(n=0) == _lib.ERR_SHAPE
    assert fwd(rows=-1) == _lib.ERR_SHAPE
    assert fwd(ldx=63) == _lib.ERR_SHAPE
    assert fwd(ldy=63) == _lib.ERR_SHAPE
    assert fwd(xd=2) == _lib.ERR_DTYPE
    assert fwd(wd=2) == _lib.ERR_DTYPE
    assert fwd(eps=-1e-5) == _lib.ERR_ARG
    assert fwd(eps=float("nan")) == _lib.ERR_ARG
    assert fwd(rows=0, x=None, y=None) == _lib.OK

    need = L.ifk_layernorm_backward_workspace(4, 64)
    assert need > 0 and L.ifk_layernorm_backward_workspace(4, 0) == 0

    def bwd(dy=FAKE, ldy=64, yd=_lib.F32, x=FAKE, ldx=64, xd=_lib.F32, codes=None, scales=None, mean=FAKE, w=FAKE,
            wd=_lib.F32, dx=FAKE, lddx=64, dw=FAKE, ws=FAKE, wsb=need):
        return L.ifk_layernorm_backward(dy, ldy, yd, x, ldx, xd, codes, 64, scales, 2, mean, FAKE, w, wd, 4, 64, dx,
                                        lddx, dw, None, None, ws, wsb, None)

    assert bwd(dy=None) == _lib.ERR_ARG
    assert bwd(mean=None) == _lib.ERR_ARG
    assert bwd(dx=None) == _lib.ERR_ARG
    assert bwd(x=None) == _lib.ERR_ARG                      # neither the rows nor their 8-bit form
    assert bwd(codes=FAKE, scales=FAKE) == _lib.ERR_ARG     # both
    assert bwd(x=None, codes=FAKE) == _lib.ERR_ARG          # codes without scales
    assert bwd(ldy=63) == _lib.ERR_SHAPE
    assert bwd(ldx=63) == _lib.ERR_SHAPE
    assert bwd(lddx=63) == _lib.ERR_SHAPE
    assert bwd(xd=9) == _lib.ERR_DTYPE
    assert bwd(ws=None) == _lib.ERR_WORKSPACE
    assert bwd(wsb=need - 1) == _lib.ERR_WORKSPACE


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    q = c8.Q8Rows(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 2, dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="CUDA"):
        c8.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        c8.dequantize_rows(q)
    with pytest.raises(ValueError, match="CUDA"):
        c8.weight_grad(x, q)
    with pytest.raises(ValueError, match="CUDA"):
        c8.layer_norm_forward(x)
    with pytest.raises(ValueError, match="CUDA"):
        c8.LayerNorm8(64)(x)
    with pytest.raises(ValueError, match="CUDA"):
        c8.Linear8(64, 8)(x)


def test_q8rows_checks_its_layout():
    z = lambda *s: torch.zeros(*s, dtype=torch.int8)
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    q = c8.Q8Rows(z(6, 96), u(6, 3), 70)
    assert (q.rows, q.cols, q.nbytes) == (6, 70, 6 * 99)
    assert q[2:5].rows == 3 and q[2:5].codes.data_ptr() == q.codes[2].data_ptr()
    with pytest.raises(TypeError):
        q[::2]
    for codes, scales, cols in ((z(6, 70), u(6, 3), 70), (z(6, 96), u(6, 2), 70), (z(6, 96), u(5, 3), 70),
                                (z(6, 96), u(6, 3), 64), (z(6, 96), u(6, 3), 0),
                                (z(96, 6).t(), u(6, 3), 70)):
        with pytest.raises(ValueError):
            c8.Q8Rows(codes, scales, cols)
    with pytest.raises(TypeError):
        c8.Q8Rows(u(6, 96), u(6, 3), 70)


def test_convert_keeps_parameters_and_structure():
    lin = nn.Linear(8, 8)
    model = nn.Sequential(nn.LayerNorm(8), lin, nn.GELU(), lin, nn.Linear(8, 3, bias=False),
                          nn.LayerNorm((4, 8)), nn.LayerNorm(3, elementwise_affine=False))
    names = dict(model.named_parameters())
    out = c8.convert(model)
    assert out is model and dict(model.named_parameters()) == names
    assert type(model[0]) is c8.LayerNorm8 and type(model[1]) is c8.Linear8 and type(model[4]) is c8.Linear8
    assert model[1] is model[3]                              # a shared layer stays shared
    assert type(model[5]) is nn.LayerNorm                    # two normalised dimensions: left alone
    assert type(model[6]) is c8.LayerNorm8 and model[6].weight is None
    assert model[1].weight is lin.weight and model[4].bias is None and model[0].eps == 1e-5
    hooked = nn.Sequential(nn.Linear(4, 4))
    hooked[0].register_forward_hook(lambda *a: None)
    assert type(c8.convert(hooked)[0]) is nn.Linear          # its hooks would be lost
    only = c8.convert(nn.Sequential(nn.Linear(4, 4), nn.LayerNorm(4)), linear=False)
    assert type(only[0]) is nn.Linear and type(only[1]) is c8.LayerNorm8
    assert type(c8.convert(nn.Linear(4, 4))) is c8.Linear8
    with pytest.raises(ValueError):
        c8.LayerNorm8((4, 8))


def test_capture_8bit_needs_a_mode_that_keeps_rows():
    from ifkfac_b200.activation_hooks import RawActivationHooks
    model = nn.Sequential(nn.Linear(4, 4))
    with pytest.raises(ValueError, match="batched or deferred"):
        RawActivationHooks(model, capture_8bit=True)
    RawActivationHooks(model, capture_8bit=True, deferred=True)
    hooks = RawActivationHooks(model, capture_8bit=True, batched=True)
    hooks.enable()
    with pytest.raises(ValueError, match="CUDA"):
        model(torch.randn(3, 4))
    hooks.remove()


def test_modules_take_their_input_by_name():
    """nn.Linear and nn.LayerNorm call it `input`; here the call gets as far as the check of the device."""
    for m in (c8.Linear8(8, 4), c8.LayerNorm8(8)):
        with pytest.raises(ValueError, match="CUDA"):
            m(input=torch.randn(2, 8))


@pytest.mark.parametrize("make", [lambda: nn.Linear(8, 8), lambda: nn.LayerNorm(8)])
def test_convert_keeps_what_a_layer_carries(make):
    plain = make()
    plain.tag, plain.info = "q", {"k": 1}
    plain.register_buffer("mask", torch.ones(8))
    plain.register_buffer("scratch", torch.ones(2), persistent=False)
    plain.extra = nn.Parameter(torch.zeros(3))
    plain.weight.requires_grad_(False)
    plain.eval()
    keys = list(nn.Sequential(plain).state_dict())
    model = c8.convert(nn.Sequential(plain))
    new = model[0]
    assert type(new) in (c8.Linear8, c8.LayerNorm8) and type(plain) in (nn.Linear, nn.LayerNorm)
    assert new.tag == "q" and new.info is plain.info and new.mask is plain.mask and new.extra is plain.extra
    assert list(model.state_dict()) == keys and "scratch" in dict(new.named_buffers())
    assert new.weight is plain.weight and not new.weight.requires_grad and not new.training
    new.register_buffer("later", torch.ones(1))              # containers of its own
    assert "later" not in plain._buffers
    assert repr(new).startswith(type(new).__name__)


@pytest.mark.parametrize("hook", [
    lambda m: m.register_state_dict_pre_hook(lambda *a: None), lambda m: m._register_state_dict_hook(lambda *a: None),
    lambda m: m.register_load_state_dict_post_hook(lambda *a: None),
    lambda m: m._register_load_state_dict_pre_hook(lambda *a: None),
    lambda m: m.register_forward_pre_hook(lambda *a: None), lambda m: m.register_full_backward_hook(lambda *a: None),
    lambda m: setattr(m, "forward", lambda x: x)])
def test_convert_leaves_layers_with_hooks_or_a_forward_of_their_own(hook):
    for make, cls in ((lambda: nn.Linear(8, 8), nn.Linear), (lambda: nn.LayerNorm(8), nn.LayerNorm)):
        m = make()
        hook(m)
        assert c8.convert(nn.Sequential(m))[0] is m and type(m) is cls


def _rows(n=4):
    return c8.Q8Rows(torch.zeros(n, 32, dtype=torch.int8), torch.ones(n, 1, dtype=torch.uint8), 20)


def test_a_passs_rows_go_to_the_hooks_of_that_pass():
    m, q, out, other = c8.Linear8(20, 4), _rows(), torch.zeros(2), torch.zeros(2)
    m.share_rows()
    m.share_rows()
    m._pass = c8._PassRows(q, out, m._share_rows)
    assert m.take_rows(other) is None and m._last_rows is q  # another pass's output
    assert m.take_rows(out) is q and m._last_rows is q       # two sets of hooks each take them
    assert m.take_rows(out) is q and m._last_rows is None
    assert m.take_rows(out) is None
    m.unshare_rows()
    assert m._share_rows == 1
    m.unshare_rows()
    m.unshare_rows()
    assert m._share_rows == 0


def test_copies_and_pickles_of_a_layer_hold_no_rows():
    import copy
    import io
    m, out = c8.Linear8(20, 4), torch.zeros(2)
    m._pass = c8._PassRows(_rows(), out, 1)
    assert copy.deepcopy(m)._last_rows is None
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    back = torch.load(f, weights_only=False)
    assert back._last_rows is None and torch.equal(back.weight, m.weight)
    assert m._last_rows is not None


def test_hooks_leave_the_layers_as_they_found_them():
    from ifkfac_b200.activation_hooks import RawActivationHooks
    model = c8.convert(nn.Sequential(nn.Linear(4, 4)))
    sets = [RawActivationHooks(model, capture_8bit=True, batched=True) for _ in range(2)]
    plain = RawActivationHooks(model, batched=True)
    for h in (*sets, plain):
        h.enable()
    assert model[0]._share_rows == 2
    plain.remove()
    sets[0].remove()
    sets[0].remove()
    assert model[0]._share_rows == 1                         # the other set still gets its rows
    sets[1].remove()
    assert model[0]._share_rows == 0


@pytest.mark.parametrize("precision,size", [(_lib.PREC_AUTO, 4), (_lib.PREC_BF16, 2), (_lib.PREC_FP32, 2)])
def test_rows_are_unpacked_a_share_at_a_time(precision, size):
    """One layer's chunks too: every fold call but one of a single chunk stays under the limit, and each
    table's chunks stay in their order."""
    from ifkfac_b200.activation_hooks import RawActivationHooks
    from ifkfac_b200.engine import PackedRows, Rows
    hooks = RawActivationHooks(nn.Sequential(nn.Linear(20, 4)), capture_8bit=True, batched=True, precision=precision)
    calls = []
    hooks._fold_batch = lambda entries: calls.append(entries)
    hooks._UNPACK_BYTES = 10 * 20 * size
    chunks = [PackedRows(_rows(n), torch.float32, ones=True) for n in (3, 4, 2, 2, 50, 1, 9, 9, 1)]
    plain = Rows(torch.zeros(1000, 20))                      # not unpacked: counts for nothing
    entries = [("X", "a", chunks[:4]), ("G", "a", [plain] + chunks[4:6]), ("X", "b", chunks[6:])]
    hooks._fold_entries(entries)
    for e in calls:
        assert len({(t, m) for t, m, _ in e}) == len(e) and all(cs for _, _, cs in e)
        packed = [c for _, _, cs in e for c in cs if isinstance(c, PackedRows)]
        assert len(packed) == 1 or sum(c.rows * 20 * size for c in packed) <= hooks._UNPACK_BYTES
    for table, module, want in entries:
        got = [c for e in calls for t, m, cs in e if (t, m) == (table, module) for c in cs]
        assert got == want
    assert len(calls) == 5                                   # 3 4 2 | 2 | 50 | 1 9 | 9 1
    calls.clear()
    hooks._fold_entries([("X", "a", [plain] * 3), ("G", "a", [plain])])
    assert calls == [[("X", "a", [plain] * 3), ("G", "a", [plain])]]


def test_a_delta_read_in_place_needs_no_room_for_a_copy():
    L = _lib.lib()
    at, rows, n_out, n_in = _lib.BF16 | _lib.DELTA_IN_PLACE, 16384, 4096, 4096
    full, less = (L.ifk_q8_wgrad_workspace(rows, n_out, n_in, d) for d in (_lib.BF16, at))
    assert full - less == 2 * rows * n_out and 0 < less < 1 << 26
    assert L.ifk_q8_wgrad_workspace(rows, n_out, n_in, _lib.F32 | _lib.DELTA_IN_PLACE) == 0
    need = L.ifk_q8_wgrad_workspace(8, 16, 64, at)

    def wgrad(delta=FAKE, ld=16, dt=at, wsb=need):
        return L.ifk_q8_wgrad(delta, ld, dt, FAKE, 64, FAKE, 2, 8, 16, 64, FAKE, 64, None, 0, None, FAKE, wsb, None)

    assert wgrad(delta=ctypes.c_void_p(4104)) == _lib.ERR_ARG
    assert wgrad(ld=20) == _lib.ERR_ARG
    assert wgrad(ld=15) == _lib.ERR_SHAPE
    assert wgrad(dt=_lib.F32 | _lib.DELTA_IN_PLACE) == _lib.ERR_DTYPE
    assert wgrad(wsb=need - 1) == _lib.ERR_WORKSPACE
    assert wgrad(dt=_lib.BF16, wsb=need) == _lib.ERR_WORKSPACE  # any alignment: room for the copy


def test_a_layer_made_of_a_hooked_one_starts_without_hooks():
    m = nn.Linear(20, 4)
    m.register_full_backward_hook(lambda *a: None)
    new = c8.Linear8.from_linear(m)
    assert new.weight is m.weight and not new._backward_hooks and new._is_full_backward_hook is None
    new._pass = c8._PassRows(_rows(), torch.zeros(2), 1)
    assert new.take_rows().rows == 4 and new.take_rows() is None   # without an output: the last pass's
    bare = nn.Linear(20, 4)
    bare.register_full_backward_hook(lambda *a: None).remove()
    assert type(c8.convert(nn.Sequential(bare))[0]) is c8.Linear8  # its hooks are gone: nothing to lose
