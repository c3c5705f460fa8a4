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
