"""GPU: norm and dropout calls of 32 MiB and more, whose accesses go past the caches, against the oracle.  Tolerances and the derivation
of each are test_gpu_norms's."""
import pytest

import test_gpu_norms as base

pytestmark = pytest.mark.gpu

LIMIT = 32 << 20


@pytest.mark.parametrize("shape,x,w,r,rms,p,return_sum", [
    # x alone
    ((24001, 768), "bf16", "f32", "", False, 0.0, False), ((17001, 1024), "f16", "f16", "", True, 0.0, False),
    ((9001, 1024), "f32", "f32", "", False, 0.0, False), ((1100, 16384), "bf16", "f32", "", False, 0.0, False),
    # residual, dropout and the returned sum, in one type and beside an fp32 residual
    ((24001, 768), "bf16", "bf16", "bf16", False, 0.1, False), ((17001, 1024), "bf16", "f32", "f32", True, 0.1, True),
    ((9001, 1024), "f32", "f32", "f32", False, 0.1, True), ((17001, 1024), "f16", "f32", "f16", True, 0.25, True),
    ((1100, 16384), "bf16", "bf16", "bf16", False, 0.1, True), ((11001, 1536), "bf16", "f32", "f32", False, 0.0, True),
    ((350001, 48), "f16", "f16", "f16", False, 0.5, False),
], ids=str)
def test_norms(shape, x, w, r, rms, p, return_sum):
    assert shape[0] * shape[1] * base.TYPES[x].itemsize >= LIMIT
    base.check(shape, x, w, r, rms, p, return_sum, seed=shape[1])


@pytest.mark.parametrize("x,r", [("f32", ""), ("bf16", ""), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("d", [77, 1000])              # 77: a workgroup's groups lie in up to a hundred rows
def test_dropout(d, x, r):
    rows = LIMIT // (d * base.TYPES[x].itemsize) + 3
    base.test_dropout((rows, d), x, r)
