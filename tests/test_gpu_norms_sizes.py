"""GPU: norm and dropout calls near the limits of their sizes."""
import pytest
import torch

from oracle import norm_oracle as orc
from transformer_vae_amd import functional as F

pytestmark = pytest.mark.gpu


def test_dropout_over_more_threads_than_a_launch_has():
    # 2^31 - 1 rows of two groups of eight: 2^32 threads, one for each; the input is one row, read with a stride of 0
    rows, d, p, rng = 2 ** 31 - 1, 9, 0.5, (3, 4)
    x = torch.arange(1.0, d + 1, device="cuda")
    out = F.dropout(x.expand(rows, d), p, rng)
    edge = 2 ** 23 * 256 // 2                    # the first row of the second launch, were it 2^23 workgroups of 256 threads
    for at in (0, edge - 32, rows // 2, rows - 64):
        keep = torch.from_numpy(orc.keep(64, d, p, *rng, first_row=at)).cuda()
        assert torch.equal(out[at:at + 64], torch.where(keep, x * orc.scale(p), 0.0)), at


def test_weight_gradients_of_rows_beyond_a_launch():
    # the last sums take 1024 threads for 64 columns: 2^32 threads at 2^28 of them
    d = 2 ** 28 + 200
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(1, d, generator=gen, device="cuda").bfloat16() for _ in range(2))
    w, b = (torch.ones(d, device="cuda", dtype=torch.bfloat16).requires_grad_(True) for _ in range(2))
    dw, db = torch.autograd.grad(F.layer_norm(x, w, b, 1e-5), (w, b), dy)
    assert torch.equal(db, dy[0])
    mean, var = x.double().mean(), x.double().var(unbiased=False)
    h, u = 2.0 ** -24, 2.0 ** -8
    for at in range(0, d, 2 ** 26):
        v = x[0, at:at + 2 ** 26].double()
        g = dy[0, at:at + 2 ** 26].double()
        want = g * (v - mean) * (var + 1e-5).rsqrt()
        # the mean is off by 2 h of itself and of the first guess's distance, the rest are products
        off = (dw[at:at + 2 ** 26].double() - want).abs()
        assert (off <= (u + 16 * h) * want.abs() + 16 * h * g.abs() + 2.0 ** -126).all(), at
