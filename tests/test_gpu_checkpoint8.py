"""8-bit rows, the weight gradient from them and layer norm against 64-bit oracles.

Tolerances.  u = 2^-24 is half a step of fp32; h is half a step of the output's
type.  A sum of K fp32 terms, in any order and with rounding or truncation, is off
by at most K 2u times the sum of the terms' magnitudes (S below)."""
import numpy as np
import pytest
import torch

from tests import q8_reference as ref

pytestmark = pytest.mark.gpu

BF, F4 = torch.bfloat16, torch.float32
U2 = 2.0 ** -23
HALF = {BF: 2.0 ** -8, F4: 2.0 ** -24}


def c8():
    from ifkfac_b200 import checkpoint8
    return checkpoint8


def buffer(rows, n, dtype, pad=0, seed=0, spread=100.0, scale=1.0):
    """rows x n values, a view into a buffer whose pitch is n + pad."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, n + pad, generator=g, device="cuda") * scale
    x *= torch.exp(torch.rand(n + pad, generator=g, device="cuda") * np.log(spread))
    return x.to(dtype)[:, :n]


# ---- rows to 8 bits and back ----

@pytest.mark.parametrize("dtype", [BF, F4])
@pytest.mark.parametrize("rows,n,pad", [(1, 1, 0), (1, 768, 0), (3, 31, 0), (5, 32, 0), (7, 33, 0), (300, 1025, 3),
                                        (2, 70001, 0), (1000, 64, 8), (129, 257, 7), (3000, 1, 0), (700, 3, 1),
                                        (2500, 4, 4), (900, 8, 0), (600, 9, 7), (5000, 17, 0)])
def test_quantize_matches_the_format_bit_for_bit(rows, n, pad, dtype):
    x = buffer(rows, n, dtype, pad, seed=n)
    if rows > 2:
        x[1] = 0
    q = c8().quantize_rows(x)
    codes, scales = ref.quantize(x.double().cpu().numpy())
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    want = ref.values(codes, scales, n)
    for out in (BF, F4):
        v = c8().dequantize_rows(q, out)
        assert v.dtype == out and np.array_equal(v.double().cpu().numpy(), want)


def test_quantize_extremes():
    """Ties, the clip at 127, powers of two, denormals, the largest numbers, signs of zero,
    and groups with a NaN or an infinity, which read back as NaN without touching others."""
    x = torch.zeros(6, 96)
    x[0, :8] = torch.tensor([64.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -63.5])   # e = 0: ties to even
    x[0, 32:36] = torch.tensor([127.9, -127.9, 127.5, 126.5])                 # clipped at +-127
    x[1, :3] = torch.tensor([2.0 ** -126, 2.0 ** -140, -(2.0 ** -149)])       # denormal steps
    x[1, 32:34] = torch.tensor([3.4e38, -3.4028234663852886e38])
    x[1, 64:66] = torch.tensor([-0.0, 0.0])
    x[2, 5] = float("nan")
    x[3, 40] = float("inf")
    x[3, 41] = 1.0
    x[4, 95] = -float("inf")
    x[5] = torch.linspace(-1, 1, 96)
    q = c8().quantize_rows(x.cuda())
    codes, scales = ref.quantize(x.double().numpy())
    assert np.array_equal(q.codes.cpu().numpy(), codes) and np.array_equal(q.scales.cpu().numpy(), scales)
    v = c8().dequantize_rows(q, F4).cpu().numpy()
    nan = np.zeros((6, 96), bool)
    nan[2, :32] = nan[3, 32:64] = nan[4, 64:] = True
    assert np.array_equal(np.isnan(v), nan)
    assert np.array_equal(v[~nan].astype(np.float64), ref.values(codes, scales, 96)[~nan])


@pytest.mark.parametrize("dtype", [BF, F4])
def test_gather_of_rows(dtype):
    x = buffer(500, 200, dtype, pad=4)
    idx = torch.randint(0, 500, (77,), device="cuda")
    idx[3] = idx[4]                                        # the same row twice
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = c8().quantize_rows(x, index=idx, status=status)
    whole = c8().quantize_rows(x)
    assert torch.equal(q.codes, whole.codes[idx]) and torch.equal(q.scales, whole.scales[idx])
    assert torch.equal(c8().dequantize_rows(whole, dtype, index=idx, status=status), c8().dequantize_rows(q, dtype))
    assert status.item() == 0
    idx[10], idx[11] = -1, 500                             # refused on the device: zero rows and a status
    q = c8().quantize_rows(x, index=idx, status=status)
    assert status.item() == 8 and (q.codes[10:12] == 0).all() and (q.codes[12] != 0).any()
    status.zero_()
    v = c8().dequantize_rows(whole, dtype, index=idx, status=status)
    assert status.item() == 8 and (v[10:12] == 0).all() and (v[12] != 0).any()


def test_empty_rows_and_slices():
    x = buffer(0, 40, BF)
    q = c8().quantize_rows(x)
    assert q.rows == 0 and c8().dequantize_rows(q).shape == (0, 40)
    full = c8().quantize_rows(buffer(9, 40, BF))
    assert torch.equal(c8().dequantize_rows(full[2:7]), c8().dequantize_rows(full)[2:7])
    # a transposed view and rows of stride 0 are read as the values they stand for
    t = buffer(40, 9, F4).t()
    assert torch.equal(c8().quantize_rows(t).codes, c8().quantize_rows(t.contiguous()).codes)
    e = buffer(1, 40, F4).expand(5, 40)
    assert torch.equal(c8().quantize_rows(e).codes, c8().quantize_rows(e.contiguous()).codes)


def test_rows_far_into_a_large_buffer():
    """Offsets past 2^31 elements: the last rows of a 2.2 G element buffer."""
    rows, n = 34000, 65536
    x = torch.zeros(rows, n, dtype=BF, device="cuda")
    x[-3:] = buffer(3, n, BF, seed=5)
    q = c8().quantize_rows(x)
    tail = c8().quantize_rows(x[-3:].clone())
    assert torch.equal(q.codes[-3:], tail.codes) and torch.equal(q.scales[-3:], tail.scales)
    idx = torch.tensor([rows - 1, 0, rows - 2], device="cuda")
    v = c8().dequantize_rows(q, BF, index=idx)
    assert torch.equal(v[0], c8().dequantize_rows(tail, BF)[2]) and (v[1] == 0).all()


# ---- weight gradient ----

def wgrad_oracle(delta, q):
    x = c8().dequantize_rows(q, F4).double()
    d = delta.double()
    return d.t() @ x, d.sum(0), d.abs().t() @ x.abs(), d.abs().sum(0)


def check_wgrad(dW, db, delta, q, extra=1):
    W, b, SW, Sb = wgrad_oracle(delta, q)
    k = delta.shape[0] + extra
    assert ((dW.double() - W).abs() <= k * U2 * SW).all(), float(((dW.double() - W).abs() / (SW + 1e-300)).max() / U2)
    assert ((db.double() - b).abs() <= k * U2 * Sb).all()


@pytest.mark.parametrize("dtype", [BF, F4])
@pytest.mark.parametrize("rows,n_in,n_out,pad", [
    (1, 1, 1, 0), (1, 256, 512, 0), (2, 33, 65, 1), (63, 128, 256, 0), (64, 128, 256, 8), (65, 129, 257, 0),
    (200, 1000, 40, 0), (777, 96, 1030, 5), (1024, 768, 2304, 0), (4097, 160, 300, 4), (9000, 72, 24, 0)])
def test_weight_grad(rows, n_in, n_out, pad, dtype):
    q = c8().quantize_rows(buffer(rows, n_in, BF, seed=rows))
    delta = buffer(rows, n_out, dtype, pad, seed=rows + 1, spread=10.0, scale=1e-3)
    dW, db = c8().weight_grad(delta, q, bias=True)
    check_wgrad(dW, db, delta, q)
    again, db2 = c8().weight_grad(delta, q, bias=True)
    assert torch.equal(dW, again) and torch.equal(db, db2)     # the order of the sums is fixed
    only, none = c8().weight_grad(delta, q)
    assert none is None and torch.equal(only, dW)


@pytest.mark.parametrize("dtype", [BF, F4])
def test_weight_grad_into_views_and_accumulated(dtype):
    """out inside a wider buffer: what lies around it stays; accumulate adds."""
    rows, n_in, n_out = 300, 200, 130
    q = c8().quantize_rows(buffer(rows, n_in, BF))
    delta = buffer(rows, n_out, dtype, seed=2, scale=1e-3)
    W = torch.full((n_out + 2, n_in + 3), 7.0, device="cuda")
    b = torch.full((n_out + 2,), 7.0, device="cuda")
    c8().weight_grad(delta, q, out=W[1:-1, 1:-2], out_bias=b[1:-1])
    check_wgrad(W[1:-1, 1:-2], b[1:-1], delta, q)
    assert (W[0] == 7).all() and (W[-1] == 7).all() and (W[:, 0] == 7).all() and (W[:, -2:] == 7).all()
    assert b[0] == 7 and b[-1] == 7
    first, fb = W[1:-1, 1:-2].clone(), b[1:-1].clone()
    c8().weight_grad(delta, q, out=W[1:-1, 1:-2], out_bias=b[1:-1], accumulate=True)
    # one more rounded addition of the same values: exactly twice them
    assert torch.equal(W[1:-1, 1:-2], 2 * first) and torch.equal(b[1:-1], 2 * fb)
    assert (W[0] == 7).all() and (W[:, -2:] == 7).all() and b[-1] == 7


def test_weight_grad_of_no_rows():
    q = c8().quantize_rows(buffer(0, 40, BF))
    out = torch.full((5, 40), 3.0, device="cuda")
    ob = torch.full((5,), 3.0, device="cuda")
    d = torch.empty(0, 5, dtype=BF, device="cuda")
    c8().weight_grad(d, q, out=out, out_bias=ob, accumulate=True)
    assert (out == 3).all() and (ob == 3).all()
    c8().weight_grad(d, q, out=out, out_bias=ob)
    assert (out == 0).all() and (ob == 0).all()


def test_weight_grad_nonfinite_rows():
    """A NaN group poisons its own 32 columns; an infinite delta its own output row."""
    rows, n_in, n_out = 130, 100, 70
    x = buffer(rows, n_in, F4)
    x[100, 40] = float("nan")
    q = c8().quantize_rows(x)
    for dtype in (BF, F4):
        delta = buffer(rows, n_out, dtype, seed=3)
        dW, _ = c8().weight_grad(delta, q)
        bad = torch.zeros(n_out, n_in, dtype=torch.bool, device="cuda")
        bad[:, 32:64] = True
        assert torch.equal(torch.isnan(dW), bad)
        delta[5, 7] = float("inf")
        dW, db = c8().weight_grad(delta, q, bias=True)
        want = torch.isfinite(wgrad_oracle(delta, q)[0])
        assert torch.equal(torch.isfinite(dW), want)
        assert torch.isinf(db[7]) and torch.isfinite(db[:7]).all() and torch.isfinite(db[8:]).all()


def test_weight_grad_of_wide_range_delta():
    """fp32 deltas over the whole exponent range: the three-term split loses nothing that fp32 keeps."""
    rows = 96
    q = c8().quantize_rows(buffer(rows, 64, BF))
    g = torch.Generator(device="cuda").manual_seed(1)
    delta = torch.randn(rows, 48, generator=g, device="cuda") * torch.exp2(
        torch.randint(-100, 90, (48,), generator=g, device="cuda").float())
    dW, db = c8().weight_grad(delta, q, bias=True)
    check_wgrad(dW, db, delta, q)


# ---- layer norm ----

def ln_tolerance(x, z, rstd, mean, n):
    """Error of the normalised rows: the two sums of the statistics run over at most
    min(n, 96) terms in a row with the differences from a first mean as terms, so z is
    off by at most (96 + 8) 2u (1 + |z|), and the stored mean's rounding adds |mean| u rstd."""
    return (min(n, 96) + 8) * U2 * (1 + z.abs()) + U2 * mean.abs() * rstd


LN_SIZES = [(1, 1, 0), (1, 2048, 0), (3, 2, 0), (5, 31, 0), (17, 64, 0), (33, 256, 8), (40, 257, 0), (9, 512, 1),
            (300, 768, 0), (12, 1000, 4), (50, 1024, 0), (21, 1537, 7), (11, 2056, 0), (6, 4096, 0), (3, 8191, 3),
            (4, 8192, 0), (2, 16384, 0), (2, 20001, 0), (1300, 40, 0), (700, 1280, 0),
            # rows enough to be walked through rings in shared memory
            (4800, 96, 0), (2501, 1280, 0), (2600, 768, 8), (1300, 4096, 0), (310, 8192, 0), (605, 6000, 16),
            (300, 16384, 0)]


@pytest.mark.parametrize("xd,yd", [(F4, F4), (F4, BF), (BF, BF), (BF, F4)])
@pytest.mark.parametrize("rows,n,pad", LN_SIZES)
def test_layer_norm(rows, n, pad, xd, yd):
    x = buffer(rows, n, xd, pad, seed=n, spread=8.0) + (0.5 if pad == 0 else 0.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = 1 + 0.1 * torch.randn(n, generator=g, device="cuda")
    b = 0.1 * torch.randn(n, generator=g, device="cuda")
    dy = torch.randn(rows, n + pad, generator=g, device="cuda").to(yd)[:, :n]
    eps = 1e-5
    Y, Z, R, M = ref.layer_norm(x, w, b, eps)
    tz = ln_tolerance(x.double(), Z, R, M, n)
    for checkpoint in (False, True):
        y, saved = c8().layer_norm_forward(x, w, b, eps, yd, save=True, checkpoint=checkpoint)
        assert y.dtype == yd
        assert ((y.double() - Y).abs() <= HALF[yd] * Y.abs() + tz * w.abs() + 2 * U2 * (Y.abs() + b.abs())).all()
        assert torch.equal(y, c8().layer_norm_forward(x, w, b, eps, yd)[0])
        z, tzq = Z, tz
        if checkpoint:
            assert saved.x is None
            q = c8().quantize_rows(x)
            assert torch.equal(q.codes, saved.q8.codes) and torch.equal(q.scales, saved.q8.scales)
            z = (c8().dequantize_rows(q, F4).double() - M) * R
            tzq = ln_tolerance(x.double(), z, R, M, n)
        dx, dw, db = c8().layer_norm_backward(dy, saved, w, status=status)
        assert status.item() == 0
        DX, DW, DB = ref.layer_norm_backward(dy, z, R, w)
        gw = (dy.double() * w.double()).abs()
        k = (min(n, 96) + 8) * U2
        mg, mz = gw.mean(1, keepdim=True), (gw * z.abs()).mean(1, keepdim=True)
        tdx = R * (k * (gw + mg + z.abs() * mz) + tzq * mz + z.abs() * (gw * tzq).mean(1, keepdim=True)) \
            + k * DX.abs()
        assert dx.dtype == xd and ((dx.double() - DX).abs() <= HALF[xd] * DX.abs() + tdx).all()
        ady = dy.double().abs()
        assert ((dw.double() - DW).abs() <= (rows + 4) * U2 * (ady * z.abs()).sum(0) + (ady * tzq).sum(0)).all()
        assert ((db.double() - DB).abs() <= (rows + 4) * U2 * ady.sum(0)).all()
        again = c8().layer_norm_backward(dy, saved, w)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
        dx1, none, none1 = c8().layer_norm_backward(dy, saved, w, weight_grads=False)
        assert none is None and none1 is None and torch.equal(dx1, dx)


@pytest.mark.parametrize("n", [48, 1500, 9000])
def test_layer_norm_without_weight_or_bias_and_bf16_weights(n):
    x = buffer(10, n, F4, spread=4.0)
    dy = buffer(10, n, F4, seed=1, spread=1.0)
    one, zero = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    y, s = c8().layer_norm_forward(x, save=True)
    yy, ss = c8().layer_norm_forward(x, one, zero, save=True)
    assert torch.equal(y, yy)
    assert torch.equal(c8().layer_norm_forward(x, one)[0], y) and torch.equal(c8().layer_norm_forward(x, None, zero)[0], y)
    for p, q in zip(c8().layer_norm_backward(dy, s), c8().layer_norm_backward(dy, ss, one)):
        assert torch.equal(p, q)
    wb = (one + 0.1 * buffer(1, n, F4, seed=4, spread=1.0)[0]).to(BF)
    bb = (0.1 * buffer(1, n, F4, seed=5, spread=1.0)[0]).to(BF)
    assert torch.equal(c8().layer_norm_forward(x, wb, bb)[0], c8().layer_norm_forward(x, wb.float(), bb.float())[0])
    for p, q in zip(c8().layer_norm_backward(dy, s, wb), c8().layer_norm_backward(dy, s, wb.float())):
        assert torch.equal(p, q)


@pytest.mark.parametrize("n", [96, 1500, 20000])
def test_layer_norm_odd_rows(n):
    """Constant rows (variance 0: y = b), rows far from zero, and non-finite rows, which
    stay in their own row of y and dx."""
    x = buffer(8, n, F4, spread=2.0)
    x[1] = 3.0
    x[2] += 10000.0
    x[4, n // 2] = float("nan")
    x[6, 0] = float("inf")
    w, b = torch.full((n,), 2.0, device="cuda"), torch.full((n,), 0.25, device="cuda")
    y, s = c8().layer_norm_forward(x, w, b, save=True)
    Y, Z, R, M = ref.layer_norm(x, w, b, 1e-5)
    assert torch.equal(y[1], b)
    ok = torch.tensor([0, 1, 2, 3, 5, 7], device="cuda")
    tol = ln_tolerance(x.double(), Z, R, M, n)[ok] * 2 + 2 * U2 * (Y[ok].abs() + 0.25)
    assert ((y.double() - Y)[ok].abs() <= tol).all()
    assert torch.isnan(y[[4, 6]]).all() and torch.isfinite(y[ok]).all()
    dx, dw, db = c8().layer_norm_backward(torch.ones_like(y), s, w)
    assert torch.isnan(dx[[4, 6]]).all() and torch.isfinite(dx[ok]).all()
    assert torch.isnan(dw).all() and torch.equal(db, torch.full_like(db, 8.0))


@pytest.mark.parametrize("n", [65, 1100])
def test_layer_norm_no_rows(n):
    x = torch.empty(0, n, device="cuda")
    y, s = c8().layer_norm_forward(x, save=True, checkpoint=True)
    dx, dw, db = c8().layer_norm_backward(torch.empty(0, n, device="cuda"), s)
    assert y.shape == dx.shape == (0, n) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("rows,n", [(7, 40), (3, 1300), (2, 9000)])
def test_layer_norm_gradient_against_differences(rows, n):
    """Central differences of the forward kernel along a random direction.  The
    truncation is estimated from a second step of twice the length (their difference is
    three times it); fp32 outputs off by tol_y move a difference by sum |dy| tol_y / h."""
    x = buffer(rows, n, F4, spread=3.0)
    w = 1 + 0.1 * buffer(1, n, F4, seed=3, spread=1.0)[0]
    b = buffer(1, n, F4, seed=4, spread=1.0)[0]
    dy = buffer(rows, n, F4, seed=5, spread=1.0)
    v = buffer(rows, n, F4, seed=6, spread=1.0)
    _, s = c8().layer_norm_forward(x, w, b, save=True)
    dx, dw, db = c8().layer_norm_backward(dy, s, w)

    def loss(dir_x=0.0, dir_w=0.0, dir_b=0.0):
        # powers of two times v: the step itself is exact up to the sum's rounding
        xx = x + dir_x * v
        y, _ = c8().layer_norm_forward(xx, w + dir_w * v[0], b + dir_b * v[0])
        return float((y.double() * dy.double()).sum()), xx

    Y, Z, R, M = ref.layer_norm(x, w, b, 1e-5)
    tol_y = (ln_tolerance(x.double(), Z, R, M, n) * w.abs() + 2 * U2 * (Y.abs() + b.abs())) * 2
    h = 2.0 ** -6
    noise = float((dy.double().abs() * tol_y).sum()) / h
    step_noise = float((dx.double().abs() * U2 * x.abs().double()).sum()) / h
    for key, grad in (("dir_x", (dx.double() * v.double()).sum()), ("dir_w", (dw.double() * v[0].double()).sum()),
                      ("dir_b", (db.double() * v[0].double()).sum())):
        d1 = (loss(**{key: h})[0] - loss(**{key: -h})[0]) / (2 * h)
        d2 = (loss(**{key: 2 * h})[0] - loss(**{key: -2 * h})[0]) / (4 * h)
        assert abs(float(grad) - d1) <= abs(d2 - d1) + noise + step_noise, key


# ---- streams, graphs ----

def test_graph_replays_on_new_values_and_other_streams():
    """Captured once, replayed on new inputs; two graphs replayed in turn; a side stream."""
    rows, n, m = 260, 192, 136
    x, dy, delta = buffer(rows, n, F4), buffer(rows, n, BF, seed=1), buffer(rows, m, F4, seed=2)
    w = torch.ones(n, device="cuda")

    def step():
        y, s = c8().layer_norm_forward(x, w, None, out_dtype=BF, save=True, checkpoint=True)
        q = c8().quantize_rows(y)
        return (y, *c8().layer_norm_backward(dy, s, w), *c8().weight_grad(delta, q, bias=True))

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in (10, 11):
        x.copy_(buffer(rows, n, F4, seed=seed))
        delta.copy_(buffer(rows, m, F4, seed=seed + 50))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            g.replay()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_weight_gradients_queued_behind_one_another():
    """A call's kernels overlap their launches: calls in a row without a wait, the inputs overwritten right behind
    them, and the same in a graph, have the bits of calls one at a time."""
    jobs = []
    for k, (rows, n_in, n_out, dt, pad) in enumerate(((1, 96, 2304, BF, 0), (65, 521, 72, F4, 3), (700, 768, 1030, BF, 0),
                                                      (3000, 48, 513, BF, 3), (64, 2048, 520, BF, 0),
                                                      (1000, 300, 264, F4, 0))):
        jobs.append((buffer(rows, n_out, dt, pad, seed=k), c8().quantize_rows(buffer(rows, n_in, F4, seed=k + 50))))
    want = []
    for delta, q in jobs:
        want.append(c8().weight_grad(delta, q, bias=True))
        torch.cuda.synchronize()

    def same(got):
        return all(torch.equal(p, t) for a, b in zip(got, want) for p, t in zip(a, b))

    for _ in range(3):
        got = [c8().weight_grad(delta, q, bias=True) for delta, q in jobs]
        assert same([(w.clone(), b.clone()) for w, b in got])
    got = []
    for delta, q in jobs:
        d = delta.clone()
        r = c8().Q8Rows(q.codes.clone(), q.scales.clone(), q.cols)
        got.append(c8().weight_grad(d, r, bias=True))
        d.fill_(3.0)
        r.codes.zero_()
        r.scales.fill_(1)
    assert same(got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [c8().weight_grad(delta, q, bias=True) for delta, q in jobs]
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert same(got)


def test_python_refusals():
    x = buffer(6, 64, BF)
    q = c8().quantize_rows(x)
    with pytest.raises(TypeError):
        c8().quantize_rows(x.half())
    with pytest.raises(ValueError):
        c8().quantize_rows(x[0])
    with pytest.raises(ValueError):
        c8().quantize_rows(x[:, :0])
    with pytest.raises(ValueError):
        c8().quantize_rows(x, index=torch.zeros(2, 2, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        c8().dequantize_rows(q, torch.float16)
    with pytest.raises(ValueError):
        c8().weight_grad(x[:5], q)                       # rows differ
    with pytest.raises(ValueError):
        c8().weight_grad(x, q, accumulate=True)
    with pytest.raises(ValueError):
        c8().weight_grad(x, q, out=torch.empty(64, 63, device="cuda"))
    with pytest.raises(ValueError):
        c8().weight_grad(x, q, out=torch.empty(64, 64, dtype=BF, device="cuda"))
    with pytest.raises(ValueError):
        c8().weight_grad(x.cpu(), q)
    with pytest.raises(ValueError):
        c8().layer_norm_forward(x, torch.ones(63, device="cuda"))
    with pytest.raises(TypeError):
        c8().layer_norm_forward(x, torch.ones(64, device="cuda"), torch.ones(64, device="cuda", dtype=BF))
    _, s = c8().layer_norm_forward(x, save=True)
    with pytest.raises(ValueError):
        c8().layer_norm_backward(x[:5], s)
    for bad in (torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")):
        with pytest.raises(TypeError):
            c8().quantize_rows(x, status=bad)
    with pytest.raises(RuntimeError):
        c8().quantize_rows(x[:0], index=torch.zeros(3, dtype=torch.int64, device="cuda"))  # rows of nothing


def test_calls_on_two_streams_at_once():
    """Calls that overlap on the GPU share nothing: each has its own workspace."""
    rows, n, m = 2600, 512, 384
    xs = [buffer(rows, n, BF, seed=k) for k in range(2)]
    ds = [buffer(rows, m, BF, seed=10 + k) for k in range(2)]
    w = torch.ones(n, device="cuda")

    def work(k):
        y, s = c8().layer_norm_forward(xs[k], w, None, save=True, checkpoint=True)
        q = c8().quantize_rows(y)
        return (y, *c8().layer_norm_backward(xs[1 - k], s, w), *c8().weight_grad(ds[k], q, bias=True))

    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(work(k))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


@pytest.mark.parametrize("xd", [BF, F4])
@pytest.mark.parametrize("rows,n,pad", [(40, 768, 0), (1300, 1000, 0), (33, 1001, 0), (9, 4096, 1), (700, 96, 3),
                                        (3, 9000, 0), (2, 17000, 0)])
def test_layer_norm_of_a_bf16_model(rows, n, pad, xd):
    """bf16 weights and a missing bias, on rows of either type, aligned or not: the bits of the same
    weights in fp32, forward (with and without 8-bit rows) and backward."""
    x = buffer(rows, n, xd, pad, spread=4.0)
    dy = buffer(rows, n, xd, pad, seed=1, spread=1.0)
    wb = (1 + 0.1 * buffer(1, n, F4, seed=4, spread=1.0)[0]).to(BF)
    bb = (0.1 * buffer(1, n, F4, seed=5, spread=1.0)[0]).to(BF)
    for w, b in ((wb, bb), (wb, None), (None, bb)):
        f = [None if t is None else t.float() for t in (w, b)]
        for checkpoint in (False, True):
            y, s = c8().layer_norm_forward(x, w, b, save=True, checkpoint=checkpoint)
            yy, ss = c8().layer_norm_forward(x, *f, save=True, checkpoint=checkpoint)
            assert torch.equal(y, yy) and torch.equal(s.mean, ss.mean) and torch.equal(s.rstd, ss.rstd)
            if checkpoint:
                assert torch.equal(s.q8.codes, ss.q8.codes) and torch.equal(s.q8.scales, ss.q8.scales)
            for p, q in zip(c8().layer_norm_backward(dy, s, w), c8().layer_norm_backward(dy, ss, f[0])):
                assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [BF, F4])
def test_weight_grad_of_a_slice_of_rows(dtype):
    """Rows from the middle of a batch: codes and scales that start anywhere, and are not copied."""
    q = c8().quantize_rows(buffer(400, 40, BF))
    delta = buffer(400, 72, dtype, seed=2, scale=1e-3)
    for lo, hi in ((0, 400), (3, 130), (129, 130), (255, 400), (7, 7)):
        part = q[lo:hi]
        dW, db = c8().weight_grad(delta[lo:hi], part, bias=True)
        check_wgrad(dW, db, delta[lo:hi], part)
        own = c8().Q8Rows(part.codes.clone(), part.scales.clone(), 40)
        assert torch.equal(dW, c8().weight_grad(delta[lo:hi].clone(), own)[0])
