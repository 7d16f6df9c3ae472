"""GPU: input gradients of the norms with frozen weights."""
import pytest
import torch

from transformer_vae_amd import functional as F

pytestmark = pytest.mark.gpu

H = 2.0 ** -24


@pytest.mark.parametrize("shape", [(5, 96), (33, 301), (512, 2048), (513, 2048), (40, 2049)])
@pytest.mark.parametrize("rms", [False, True])
def test_frozen_weights_keep_the_input_gradient(shape, rms):
    """dx alone against dx beside dw and db, in fp32: the same bits from one kernel (beyond 512 rows of 2048), else two orders of
    the sums of a row."""
    gen = torch.Generator(device="cuda").manual_seed(shape[1])
    x, dy = (torch.randn(shape, generator=gen, device="cuda") for _ in range(2))
    w = 1 + 0.2 * torch.randn(shape[1], generator=gen, device="cuda")
    x.requires_grad_(True)
    got = []
    for need in (True, False):
        wt = w.clone().requires_grad_(need)
        y = F.rms_norm(x, wt) if rms else F.layer_norm(x, wt, torch.zeros_like(w))
        got.append([torch.autograd.grad(y, (x, wt) if need else (x,), dy, retain_graph=True)[0] for _ in range(2)])
    assert torch.equal(*got[0]) and torch.equal(*got[1])
    a, b = got[0][0], got[1][0]
    if shape[0] > 512 or shape[1] > 2048:
        assert torch.equal(a, b)
    # either order of n terms is off by at most (n / 64 + 32) h of the sum of their magnitudes; both sums enter dx with rstd and
    # xh, whose products and the subtraction cost 8 h more of what they subtract
    v = x.detach().double()
    c = v if rms else v - v.mean(1, keepdim=True)
    rstd = (c.square().mean(1, keepdim=True)).rsqrt()
    xh, g = c * rstd, (dy * w).double().abs()
    n = 2 * (shape[1] / 64 + 40) * H
    bound = n * rstd * (g + g.mean(1, keepdim=True) + xh.abs() * (g * xh.abs()).mean(1, keepdim=True))
    assert ((a - b).double().abs() <= bound).all()
