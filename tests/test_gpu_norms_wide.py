"""GPU: rows beyond the ones that stay in registers (16384 elements), against fp64."""
import numpy as np
import pytest
import torch

from oracle import norm_oracle as orc
from transformer_vae_amd import functional as F

pytestmark = pytest.mark.gpu

H = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def n64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("value", [0.7, -3.3, 1.0])
@pytest.mark.parametrize("d", [16392, 40000, 2000000])
def test_equal_values_add_up(d, value):
    """Sums of equal terms: what a long row's additions lose is the same each time, so nothing averages out."""
    x, w = torch.full((2, d), value, device=dev()), torch.full((d,), 0.3, device=dev())
    y = F.rms_norm(x, w, 0.0)
    want = orc.norm_forward(n64(x), n64(w), None, 0.0, True)[0]
    # a square, seven additions in fp32, the division, the root, two products, within 16 h
    assert (np.abs(n64(y) - want) <= 16 * H * np.abs(want)).all()


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("d", [16392, 40000, 2000000])
def test_equal_gradients_add_up(d, rms):
    """g = dy w the same everywhere: mean g is g, and of dv nothing but -xh mean(g xh) is left."""
    gen = torch.Generator(device=dev()).manual_seed(d)
    x = torch.randn(2, d, generator=gen, device=dev()) + (0.5 if rms else 0.0)
    x.requires_grad_(True)
    dy = torch.full((2, d), 0.7, device=dev())
    (dx,) = torch.autograd.grad(F.rms_norm(x, None, 1e-6) if rms else F.layer_norm(x, None, None, 1e-6), x, dy)
    _, xh, rstd = orc.norm_forward(n64(x), None, None, 1e-6, rms)
    want = orc.norm_backward(n64(dy), xh, rstd, None, rms)[0]
    # each of g, mean g and xh mean(g xh) costs at most 16 h of itself; xh (off by 8 h) of the mean's terms: 24 h of |g| mean |xh|
    bound = H * rstd * (32 * 0.7 + 24 * 0.7 * np.abs(xh) * np.abs(xh).mean(1, keepdims=True) + 16 * np.abs(xh) * np.abs((0.7 * xh).mean(1, keepdims=True)))
    off = np.abs(n64(dx) - want)
    assert (off <= bound).all(), (off.max(), (off / bound).max())


@pytest.mark.parametrize("unlike", [64, 1])
@pytest.mark.parametrize("parts", [32, 64, 7])
@pytest.mark.parametrize("d", [20000, 200000, 2000000])
def test_rows_of_segments_that_start_unlike_their_rest(d, parts, unlike):
    """Concatenated blocks with a header: whatever places the first guess of the mean comes from, it must not decide the result."""
    g = torch.Generator(device=dev()).manual_seed(d + parts)
    x = torch.randn(3, d, generator=g, device=dev())
    for k in range(parts):
        at = (k * ((d + 7) // 8) // parts) * 8                # where a segment of whole groups of eight starts
        x[:, at:at + unlike] += 1000.0
    y = F.layer_norm(x, eps=1e-6)
    v = n64(x)
    want, _, rstd = orc.norm_forward(v, None, None, 1e-6, False)
    # a difference to the mean costs 2 h of itself (mean and remainder), the statistics and the products 16 h of the value; the mean
    # is off by 2 h of the first guess's remaining distance, a standard deviation at most, and of itself
    bound = H * (20 * np.abs(want) + 4 + 2 * rstd * np.abs(v.mean(1, keepdims=True)))
    off = np.abs(n64(y) - want)
    assert (off <= bound).all(), (off.max(), (off / bound).max())
