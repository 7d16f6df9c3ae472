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
