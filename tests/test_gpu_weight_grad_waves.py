"""The weight gradient from 8-bit rows where a pair of CTAs has more than one tile or more
than one accumulator's worth of rows: whole waves of tiles, tiles cut behind them, and
accumulators added to the result (and to what was there before).

Tolerance.  A tile is one of 256 x 256 and a wave has 74 of them; an accumulator sums at
most 120 products of 16 rows (1920 rows, or 640 in the three terms of an fp32 delta)
before it is added to the result with rounding.  Each of the 120 additions is off by at
most one fp32 step 2u = 2^-23 of what has been summed so far, each addition of an
accumulator, of a tile's shares or to the previous content by u.  With S the sum of the
terms' magnitudes an element is off by at most (120 2u + (accumulators + 3) u) S."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F4 = torch.bfloat16, torch.float32
U = 2.0 ** -24
ADDS = 120


def c8():
    from ifkfac_b200 import checkpoint8
    return checkpoint8


def accumulators(rows, dtype):
    return -(-rows // (640 if dtype == F4 else 1920))


def inputs(rows, n_in, n_out, dtype, pad=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = c8().quantize_rows(torch.randn(rows, n_in, generator=g, device="cuda"))
    delta = (torch.randn(rows, n_out + pad, generator=g, device="cuda") * 1e-3).to(dtype)[:, :n_out]
    return delta, q


def oracle(delta, q):
    x, d = c8().dequantize_rows(q, F4).double(), delta.double()
    return d.t() @ x, d.sum(0), d.abs().t() @ x.abs(), d.abs().sum(0)


SIZES = [
    (2100, 2049, 2570, 0),      # 99 tiles: a wave, 25 tiles cut, the last of them ragged on both sides
    (2100, 2049, 2570, 5),      # delta's rows not aligned
    (2000, 512, 9472, 0),       # 74 tiles: a wave and nothing left
    (4097, 4096, 4096, 0),      # 256 tiles: three waves, 34 tiles cut, more than two accumulators a tile
    (700, 260, 256 * 75, 8),    # 150 tiles: two waves, two tiles shared by all pairs
]


@pytest.mark.parametrize("dtype", [BF, F4])
@pytest.mark.parametrize("rows,n_in,n_out,pad", SIZES)
def test_waves_of_tiles(rows, n_in, n_out, pad, dtype):
    delta, q = inputs(rows, n_in, n_out, dtype, pad)
    W, b, SW, Sb = oracle(delta, q)
    tol = (2 * ADDS + accumulators(rows, dtype) + 3) * U
    dW, db = c8().weight_grad(delta, q, bias=True)
    assert ((dW.double() - W).abs() <= tol * SW).all(), float(((dW.double() - W).abs() / (SW + 1e-300)).max() / U)
    assert ((db.double() - b).abs() <= rows * 2 * U * Sb).all()
    again, db2 = c8().weight_grad(delta, q, bias=True)
    assert torch.equal(again, dW) and torch.equal(db2, db)
    # into a view of a wider buffer, and added to what it holds
    buf = torch.full((n_out + 2, n_in + 3), 7.0, device="cuda")
    into, into_b = buf[1:-1, 1:-2], torch.empty(n_out, device="cuda")
    c8().weight_grad(delta, q, out=into, out_bias=into_b)
    assert torch.equal(into, dW) and torch.equal(into_b, db)
    before = torch.randn(n_out, n_in, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda") * 1e-2
    into.copy_(before)
    into_b.fill_(0.5)
    c8().weight_grad(delta, q, out=into, out_bias=into_b, accumulate=True)
    assert ((into.double() - (W + before)).abs() <= tol * (SW + before.abs())).all()
    assert ((into_b.double() - (b + 0.5)).abs() <= rows * 2 * U * (Sb + 0.5)).all()
    for edge in (buf[0], buf[-1], buf[:, 0], buf[:, -2:]):
        assert (edge == 7).all()


@pytest.mark.parametrize("dtype", [BF, F4])
def test_long_sums_do_not_drift(dtype):
    """65536 rows of positive codes and deltas, 74 tiles: 35 accumulators a tile (103 in three
    terms).  Of a sum that grows evenly the average partial sum is half of it, so the bound above
    halves; rows of 1/2 to 1 and 1 to 2 keep every partial sum within 5% of even growth.
    The mean loss is the truncations' alone, as the additions between accumulators round to
    nearest: it stays under 2e-6.  (Measured: 1.1e-6 in bf16, 4e-8 in three terms; with one
    accumulator over all rows 3.5e-4 in either type.)"""
    rows, n_in, n_out = 65536, 512, 9472
    g = torch.Generator(device="cuda").manual_seed(3)
    q = c8().quantize_rows(torch.rand(rows, n_in, generator=g, device="cuda") + 1)
    delta = ((torch.rand(rows, n_out, generator=g, device="cuda") + 1) / 2).to(dtype)
    dW, _ = c8().weight_grad(delta, q)
    some = torch.cat([torch.arange(64), torch.arange(4700, 4764), torch.arange(n_out - 64, n_out)]).cuda()
    x = c8().dequantize_rows(q, F4).double()
    W = delta[:, some].double().t() @ x
    err = (dW[some].double() - W) / W
    bound = 1.05 * (ADDS + accumulators(rows, dtype) / 2 + 1) * U
    assert float(err.abs().max()) <= bound
    assert abs(float(err.mean())) <= 2e-6


def test_transient_memory_of_an_aligned_delta():
    """16384 rows of bf16, 2048 to 2048: outputs and the shares of cut tiles, and no copy of delta (67 MB)."""
    delta, q = inputs(16384, 2048, 2048, BF)
    c8().weight_grad(delta, q, bias=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    dW, db = c8().weight_grad(delta, q, bias=True)
    peak = torch.cuda.max_memory_allocated() - before
    parts = 2 * 74 * 256 * 256 * 4
    assert peak <= dW.nbytes + db.nbytes + parts + 592 * 2048 * 4 + (1 << 21)
    odd = torch.empty(16384, 2049, dtype=BF, device="cuda")[:, :2048]
    odd.copy_(delta)
    other, _ = c8().weight_grad(odd, q)
    assert torch.equal(other, dW)
