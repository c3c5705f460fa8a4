"""The operators of 8-bit activation checkpoints and of layer norm: cases, plain forms and calls.

A case is one pass through one operator at one size:

* ``roundtrip``  rows quantised to the 8-bit checkpoint and read back;
* ``wgrad``      a Linear layer's weight and bias gradient from its 8-bit input rows;
* ``ln_forward`` layer norm without a backward pass;
* ``ln_train``   layer norm forward and backward, from the saved input or from its 8-bit checkpoint.

The checkpoint format: groups of 32 consecutive columns of a row share a power-of-two scale 2^e with
e = floor(log2(max |x|)) - 6 (at least -126, at most 121), stored as the byte e + 127; a value is
code * 2^e with an integer code in [-127, 127], rounded to the nearest (ties to even) and clipped.
Rows of codes are padded to a multiple of 32 columns.
"""
import math

import torch

own = False  # True: run() calls the framework's operators instead of the plain forms

GROUP = 32
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token's activations: the smallest call, all latency
        {"name": "roundtrip_token", "op": "roundtrip", "rows": 1, "n": 768, "dtype": "bf16", "pick": 0, "pad": 0},
        # a training step's captured rows of a 4096-wide layer
        {"name": "roundtrip_step", "op": "roundtrip", "rows": 16384, "n": 4096, "dtype": "bf16", "pick": 0, "pad": 0},
        # the hooks' random subsample of 2048 rows, an odd width inside a wider fp32 buffer
        {"name": "roundtrip_sample", "op": "roundtrip", "rows": 8191, "n": 1025, "dtype": "fp32", "pick": 2048,
         "pad": 3},
        # weight gradient of one token: an outer product, bound by writing the gradient
        {"name": "wgrad_token", "op": "wgrad", "rows": 1, "n_in": 2048, "n_out": 8192, "dtype": "bf16", "pad": 0},
        # a narrow decoder block's fused projection: few tiles, so the rows are split
        {"name": "wgrad_block", "op": "wgrad", "rows": 8192, "n_in": 768, "n_out": 2304, "dtype": "bf16", "pad": 0},
        # odd sizes, an fp32 gradient that is a slice of a wider buffer
        {"name": "wgrad_odd", "op": "wgrad", "rows": 1001, "n_in": 521, "n_out": 1030, "dtype": "fp32", "pad": 5},
        # the largest: one 4096 x 4096 layer over 16384 rows
        {"name": "wgrad_step", "op": "wgrad", "rows": 16384, "n_in": 4096, "n_out": 4096, "dtype": "bf16", "pad": 0},
        # one token through a layer norm
        {"name": "ln_token", "op": "ln_forward", "rows": 1, "n": 2048, "dtype": "bf16", "out": "bf16", "pad": 0},
        # evaluation of a batch of sequences: fp32 residual stream, bf16 into the next layer
        {"name": "ln_eval", "op": "ln_forward", "rows": 4096, "n": 1280, "dtype": "fp32", "out": "bf16", "pad": 0},
        # a narrow decoder's layer norm over 8 x 1024 tokens, checkpointed in 8 bits
        {"name": "ln_train_q8", "op": "ln_train", "rows": 8192, "n": 768, "dtype": "fp32", "out": "bf16", "pad": 0,
         "q8": True},
        # odd sizes and pitch, checkpointed in 8 bits
        {"name": "ln_train_odd", "op": "ln_train", "rows": 333, "n": 1537, "dtype": "fp32", "out": "fp32", "pad": 7,
         "q8": True},
        # a wide layer norm over a training step's rows, from its saved input
        {"name": "ln_train_wide", "op": "ln_train", "rows": 16384, "n": 4096, "dtype": "bf16", "out": "bf16",
         "pad": 0, "q8": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _width(rng, lo, hi):
    """A width: round ones (multiples of 64) and odd ones."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(("roundtrip", "wgrad", "wgrad", "ln_forward", "ln_train"))
    dtype = rng.choice(("bf16", "fp32"))
    pad = rng.choice((0, 0, 8, rng.randint(1, 40)))
    if op == "wgrad":
        n_in, n_out = _width(rng, 16, 8192), _width(rng, 16, 8192)
        most = (1 << 38) // (n_in * n_out) // (3 if dtype == "fp32" else 1)
        return {"op": op, "rows": _log(rng, 1, min(16384, most)), "n_in": n_in, "n_out": n_out, "dtype": dtype,
                "pad": pad}
    n = _width(rng, 1 if op == "roundtrip" else 16, 16384)
    rows = _log(rng, 1, min(16384, (1 << 25) // n))
    if op == "roundtrip":
        pick = rng.randint(1, rows) if rng.random() < 0.4 else 0
        return {"op": op, "rows": rows, "n": n, "dtype": dtype, "pick": pick, "pad": pad}
    case = {"op": op, "rows": rows, "n": n, "dtype": dtype, "out": rng.choice(("bf16", dtype)), "pad": pad}
    if op == "ln_train":
        case["q8"] = rng.random() < 0.6
    return case


def _rows(g, rows, n, dtype, pad, column_scale):
    """rows x n values, a view of a buffer whose pitch is n + pad."""
    x = torch.randn(rows, n + pad, generator=g, device="cuda")
    x *= torch.exp(torch.rand(n + pad, generator=g, device="cuda") * math.log(column_scale))
    return x.to(DTYPES[dtype])[:, :n]


def _codes(x):
    """(codes int8, scales uint8) of x in the checkpoint format, by elementary operations."""
    rows, n = x.shape
    ld = -(-n // GROUP) * GROUP
    v = torch.zeros(rows, ld, device=x.device)
    v[:, :n] = x.float()
    v = v.view(rows, ld // GROUP, GROUP)
    top = v.abs().amax(dim=2, keepdim=True)
    # floor(log2(top)) from the exponent field of the fp32 value (zero and denormals fall below the clamp)
    e = ((top.view(torch.int32) >> 23) - 127 - 6).clamp(-126, 121)
    inv = ((127 - e) << 23).view(torch.float32)
    codes = torch.round(v * inv).clamp(-127, 127).to(torch.int8).view(rows, ld)
    return codes, (e + 127).to(torch.uint8).view(rows, ld // GROUP)


def _values(codes, scales, n):
    """fp32 values of a checkpoint."""
    rows, ld = codes.shape
    scale = (scales.to(torch.int32) << 23).view(torch.float32)
    return (codes.float().view(rows, ld // GROUP, GROUP) * scale[:, :, None]).view(rows, ld)[:, :n]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, pad = case["rows"], case["pad"]
    if case["op"] == "wgrad":
        x = _rows(g, rows, case["n_in"], "bf16", 0, 100.0)
        if rows >= 16:
            x[torch.arange(0, rows, 16, device="cuda")] = 0  # padding tokens
        codes, scales = _codes(x)
        delta = torch.randn(rows, case["n_out"] + pad, generator=g, device="cuda") * 1e-3
        delta = delta.to(DTYPES[case["dtype"]])[:, : case["n_out"]]
        return {"case": case, "codes": codes, "scales": scales, "delta": delta}
    n = case["n"]
    x = _rows(g, rows, n, case["dtype"], pad, 100.0 if case["op"] == "roundtrip" else 8.0)
    state = {"case": case, "x": x, "index": None}
    if case["op"] == "roundtrip":
        if rows >= 16:
            x[torch.arange(0, rows, 16, device="cuda")] = 0
        if case["pick"]:
            state["index"] = torch.randperm(rows, generator=g, device="cuda")[: case["pick"]]
        return state
    state["weight"] = 1.0 + 0.1 * torch.randn(n, generator=g, device="cuda")
    state["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda")
    if case["op"] == "ln_train":
        state["dy"] = (torch.randn(rows, n, generator=g, device="cuda") * 1e-2).to(DTYPES[case["out"]])
    return state


def _plain(s):
    c = s["case"]
    if c["op"] == "roundtrip":
        x = s["x"] if s["index"] is None else s["x"][s["index"]]
        codes, scales = _codes(x)
        return _values(codes, scales, c["n"]).to(x.dtype)
    if c["op"] == "wgrad":
        d = s["delta"].float()
        return d.t() @ _values(s["codes"], s["scales"], c["n_in"]), d.sum(0)
    x, w = s["x"].float(), s["weight"]
    mean = x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + EPS)
    y = ((x - mean) * rstd * w + s["bias"]).to(DTYPES[c["out"]])
    if c["op"] == "ln_forward":
        return y
    if c["q8"]:
        x = _values(*_codes(s["x"]), c["n"])
    xh = (x - mean) * rstd
    dy = s["dy"].float()
    gw = dy * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xh).sum(0), dy.sum(0)


def _calls(s):
    from ifkfac_b200 import checkpoint8 as c8
    c = s["case"]
    if c["op"] == "roundtrip":
        return c8.dequantize_rows(c8.quantize_rows(s["x"], index=s["index"]), dtype=s["x"].dtype)
    if c["op"] == "wgrad":
        return c8.weight_grad(s["delta"], c8.Q8Rows(s["codes"], s["scales"], c["n_in"]), bias=True)
    out = DTYPES[c["out"]]
    if c["op"] == "ln_forward":
        return c8.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=out)[0]
    y, saved = c8.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=out, save=True,
                                     checkpoint=c["q8"])
    return (y, *c8.layer_norm_backward(s["dy"], saved, s["weight"]))


def run(state):
    return _calls(state) if own else _plain(state)


def work(case):
    size = {"bf16": 2, "fp32": 4}
    rows, e = case["rows"], size[case["dtype"]]
    if case["op"] == "wgrad":
        i, o = case["n_in"], case["n_out"]
        groups = -(-i // GROUP)
        return {"bytes": rows * (o * e + i + groups) + 4 * o * (i + 1), "flops": 2.0 * rows * o * i + rows * o}
    n = case["n"]
    groups = -(-n // GROUP)
    if case["op"] == "roundtrip":
        rows = case["pick"] or rows
        return {"bytes": rows * (2 * n * e + n + groups) + (8 * rows if case["pick"] else 0), "flops": 4.0 * rows * n}
    o = size[case["out"]]
    if case["op"] == "ln_forward":
        return {"bytes": rows * n * (e + o) + 8 * n, "flops": 8.0 * rows * n}
    # forward reads x and writes y; backward reads dy and the saved rows and writes dx; a checkpoint is written too
    saved = 2 * (rows * (n + groups)) if case["q8"] else rows * n * e
    return {"bytes": rows * n * (2 * e + 2 * o) + saved + 16 * rows + 20 * n, "flops": 20.0 * rows * n}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]

    def held(x):
        """The values of x in the checkpoint format, in 64 bits: frexp gives max = m 2^k with m in [1/2, 1)."""
        n = x.shape[1]
        v = torch.nn.functional.pad(x.double(), (0, -n % GROUP)).unflatten(1, (-1, GROUP))
        k = torch.frexp(v.abs().amax(-1, keepdim=True)).exponent.double()
        step = torch.exp2((k - 7).clamp(-126, 121))
        step = torch.where(v.abs().amax(-1, keepdim=True) > 0, step, torch.full_like(step, 2.0 ** -126))
        return ((v / step).round().clamp(-127, 127) * step).flatten(1)[:, :n]

    if c["op"] == "roundtrip":
        return held(s["x"] if s["index"] is None else s["x"][s["index"]])
    if c["op"] == "wgrad":
        exps = s["scales"].double().repeat_interleave(GROUP, dim=1) - 127
        x = (s["codes"].double() * torch.exp2(exps))[:, : c["n_in"]]
        d = s["delta"].double()
        return torch.mm(d.t(), x), torch.einsum("ro->o", d)
    x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = (var + EPS).sqrt()
    y = (x - mean) / sd * w + b
    if c["op"] == "ln_forward":
        return y
    z = ((held(s["x"]) if c["q8"] else x) - mean) / sd
    dy = s["dy"].double()
    # the gradient of y = z w + b with z normalised: g less its components along 1 and z
    g = dy * w / sd
    dx = g - g.sum(1, keepdim=True) / c["n"] - z * ((g * z).sum(1, keepdim=True) / c["n"])
    return y, dx, torch.einsum("rn,rn->n", dy, z), torch.einsum("rn->n", dy)
