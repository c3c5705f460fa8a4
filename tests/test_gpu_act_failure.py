"""Bounded device-side waits of the layer norm's backward pass and of the weight gradient.

A barrier that lacks an arrival (DEBUG_WITHHOLD, or-ed to the gradient's element type) makes
the waits on it run out after two seconds.  The call returns, leaves IFK_ERR_TIMEOUT in its
status word and NaN where its result is not valid, so that a training step that looks at no
status word does not go on with a gradient that only looks like one; the next call is right."""
import pytest
import torch

from ifkfac_b200 import _lib

F4, BF = torch.float32, torch.bfloat16
CODE = {F4: _lib.F32, BF: _lib.BF16}


def c8():
    from ifkfac_b200 import checkpoint8
    return checkpoint8


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("rows,n,xd", [(4800, 96, F4), (2600, 768, BF), (310, 8192, F4), (40, 768, F4)])
def test_layer_norm_backward_without_a_row(rows, n, xd, checkpoint):
    L = _lib.lib()
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, n, generator=g, device="cuda").to(xd)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(xd)
    w = 1 + 0.1 * torch.randn(n, generator=g, device="cuda")
    _, saved = c8().layer_norm_forward(x, w, save=True, checkpoint=checkpoint)
    want = c8().layer_norm_backward(dy, saved, w)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dx, dw, db = torch.zeros_like(dy), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    nbytes = L.ifk_layernorm_backward_workspace(rows, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    q = saved.q8.args() if checkpoint else (None, 0, None, 0)
    rc = L.ifk_layernorm_backward(dy.data_ptr(), n, CODE[xd] | _lib.DEBUG_WITHHOLD, None if checkpoint else x.data_ptr(), n,
                                  CODE[xd], *q, saved.mean.data_ptr(), saved.rstd.data_ptr(), w.data_ptr(), _lib.F32, rows,
                                  n, dx.data_ptr(), n, dw.data_ptr(), db.data_ptr(), status.data_ptr(), ws.data_ptr(),
                                  nbytes, stream())
    assert rc == _lib.OK
    torch.cuda.synchronize()
    assert status.item() == _lib.ERR_TIMEOUT
    assert torch.isnan(dx[0]).all() and torch.isnan(dw).all() and torch.isnan(db).all()
    good = ~torch.isnan(dx).any(1)                 # the other blocks' rows: whole, and right
    assert torch.equal(dx[good], want[0][good]) and torch.isnan(dx[~good]).all()
    if rows > 148 * 16:
        assert int(good.sum()) > rows * 9 // 10
    status.zero_()
    again = c8().layer_norm_backward(dy, saved, w, status=status)
    assert all(torch.equal(p, t) for p, t in zip(again, want)) and status.item() == 0


@pytest.mark.gpu
def test_layer_norm_backward_that_waits_for_nothing():
    """Rows read without copies (an odd pitch) have no such wait: the flag changes nothing."""
    L = _lib.lib()
    x = torch.randn(7, 41, device="cuda")[:, :40]
    dy = torch.randn(7, 40, device="cuda")
    _, saved = c8().layer_norm_forward(x, save=True)
    want = c8().layer_norm_backward(dy, saved)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dx = torch.zeros_like(dy)
    rc = L.ifk_layernorm_backward(dy.data_ptr(), 40, _lib.F32 | _lib.DEBUG_WITHHOLD, saved.x.data_ptr(), 41, _lib.F32, None,
                                  0, None, 0, saved.mean.data_ptr(), saved.rstd.data_ptr(), None, _lib.F32, 7, 40,
                                  dx.data_ptr(), 40, None, None, status.data_ptr(), None, 0, stream())
    assert rc == _lib.OK and torch.equal(dx, want[0]) and status.item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n_in,n_out,dtype", [
    (300, 200, 130, BF),          # one tile, one pair
    (1024, 768, 2304, BF),        # tiles cut into shares
    (700, 300, 520, F4),
    (2100, 2049, 2570, BF),       # a wave of tiles, and more than one accumulator
    (2100, 2049, 2570, F4)])
def test_weight_grad_without_codes(rows, n_in, n_out, dtype):
    L = _lib.lib()
    g = torch.Generator(device="cuda").manual_seed(1)
    q = c8().quantize_rows(torch.randn(rows, n_in, generator=g, device="cuda"))
    delta = torch.randn(rows, n_out, generator=g, device="cuda").to(dtype)
    want = c8().weight_grad(delta, q, bias=True)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dW, db = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    nbytes = L.ifk_q8_wgrad_workspace(rows, n_out, n_in, CODE[dtype])
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    rc = L.ifk_q8_wgrad(delta.data_ptr(), n_out, CODE[dtype] | _lib.DEBUG_WITHHOLD, *q.args(), rows, n_out, n_in,
                        dW.data_ptr(), n_in, db.data_ptr(), 0, status.data_ptr(), ws.data_ptr(), nbytes, stream())
    assert rc == _lib.OK
    torch.cuda.synchronize()
    assert status.item() == _lib.ERR_TIMEOUT
    # the first pair's first tile; a share of it that another pair has is right
    assert torch.isnan(dW[0, : min(n_in, 256)]).all()
    assert torch.equal(db, want[1])                    # its sums do not go through the pair
    far = dW[:, -1]                                    # and tiles of other pairs are whole
    if n_in > 256 * 3:
        assert torch.equal(far, want[0][:, -1])
    status.zero_()
    again = c8().weight_grad(delta, q, bias=True, status=status)
    assert all(torch.equal(p, t) for p, t in zip(again, want)) and status.item() == 0


def test_the_flag_does_not_hide_other_errors():
    import ctypes
    L, fake, flag = _lib.lib(), ctypes.c_void_p(4096), _lib.DEBUG_WITHHOLD
    bwd = lambda dt, dy=fake: L.ifk_layernorm_backward(dy, 64, dt, fake, 64, _lib.F32, None, 0, None, 0, fake, fake, None,
                                                       _lib.F32, 4, 64, fake, 64, None, None, None, None, 0, None)
    assert bwd(_lib.F32 | flag, None) == _lib.ERR_ARG and bwd(9 | flag) == _lib.ERR_DTYPE and bwd(512) == _lib.ERR_DTYPE
    wgrad = lambda dt, ws=fake: L.ifk_q8_wgrad(fake, 16, dt, fake, 64, fake, 2, 8, 16, 64, fake, 64, None, 0, None, ws,
                                               1 << 30, None)
    assert wgrad(_lib.BF16 | flag, None) == _lib.ERR_WORKSPACE and wgrad(5 | flag) == _lib.ERR_DTYPE
    # it belongs to these two calls: an element type with it is none elsewhere
    assert L.ifk_q8_quantize(fake, 64, _lib.F32 | flag, None, 8, 8, 64, fake, 64, fake, 2, None, None) == _lib.ERR_DTYPE
