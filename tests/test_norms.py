"""CPU: the norm and dropout oracle against published vectors and differences, and what the operators refuse."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import transformer_vae_amd as amd
from oracle import norm_oracle as orc
from transformer_vae_amd import _lib
from transformer_vae_amd import functional as F


def test_philox_known_answers():
    # the known-answer vectors published with the generator: all-zero, all-one and the digits of pi
    def run(ctr, key):
        return [int(v) for v in orc.philox4x32([np.array(c) for c in ctr], key)]
    assert run([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert run([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert run([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_keep_decisions_are_independent_draws(p):
    # 2^20 decisions: the kept share is within five standard deviations, neighbours and the next offset are uncorrelated
    k = orc.keep(1024, 1024, p, 7, 3).astype(np.float64)
    q = 1.0 - orc.threshold(p) / 65536.0
    sd = np.sqrt(q * (1 - q) / k.size)
    assert abs(k.mean() - q) < 5 * sd
    for other in (np.roll(k, 1, 1), np.roll(k, 1, 0), orc.keep(1024, 1024, p, 7, 4), orc.keep(1024, 1024, p, 8, 3)):
        cov = ((k - q) * (other - q)).mean() / (q * (1 - q))
        assert abs(cov) < 5 / np.sqrt(k.size)


@pytest.mark.parametrize("rms", [False, True])
def test_oracle_gradients_against_differences(rms):
    rng = np.random.default_rng(1)
    v, w, b, dy = rng.normal(size=(5, 13)), rng.normal(size=13), rng.normal(size=13), rng.normal(size=(5, 13))
    y, xh, rstd = orc.norm_forward(v, w, None if rms else b, 1e-6, rms)
    dv, dw, db = orc.norm_backward(dy, xh, rstd, w, rms)

    def loss(v, w, b):
        return (orc.norm_forward(v, w, None if rms else b, 1e-6, rms)[0] * dy).sum()

    h = 1e-5
    for k in range(8):
        u = rng.normal(size=v.shape)
        num = (loss(v + h * u, w, b) - loss(v - h * u, w, b)) / (2 * h)
        assert num == pytest.approx((dv * u).sum(), rel=1e-7, abs=1e-7)
        u = rng.normal(size=13)
        assert (loss(v, w + h * u, b) - loss(v, w - h * u, b)) / (2 * h) == pytest.approx((dw * u).sum(), rel=1e-7, abs=1e-7)
        if not rms:
            assert (loss(v, w, b + h * u) - loss(v, w, b - h * u)) / (2 * h) == pytest.approx((db * u).sum(), rel=1e-7, abs=1e-7)


def test_operators_refuse_cpu_tensors():
    x, w = torch.randn(4, 16), torch.ones(16)
    for call in (lambda: F.layer_norm(x, w, w), lambda: F.rms_norm(x, w), lambda: F.dropout(x, 0.1), lambda: F.dropout_add(x, x, 0.1),
                 lambda: F.dropout_add_layer_norm(x, x, w, w), lambda: F.dropout_add_rms_norm(x, x, w),
                 lambda: amd.LayerNorm(16)(x), lambda: amd.RMSNorm(16)(x), lambda: amd.Dropout(0.1)(x),
                 lambda: amd.DropoutAddLayerNorm(16, 0.1)(x, x), lambda: amd.DropoutAddRMSNorm(16, 0.1)(x, x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_modules_check_their_arguments_and_keep_parameter_names():
    with pytest.raises(ValueError, match="last axis"):
        amd.LayerNorm((4, 16))
    for cls in (amd.DropoutAddLayerNorm, amd.DropoutAddRMSNorm, amd.Dropout):
        with pytest.raises(ValueError):
            cls(16, 1.5) if cls is not amd.Dropout else cls(-0.1)
    with pytest.raises(ValueError, match="16 features"):
        amd.LayerNorm(16)(torch.randn(2, 8))
    assert set(amd.LayerNorm(8).state_dict()) == set(torch.nn.LayerNorm(8).state_dict()) == set(amd.DropoutAddLayerNorm(8).state_dict())
    assert set(amd.RMSNorm(8).state_dict()) == {"weight"} == set(amd.DropoutAddRMSNorm(8).state_dict())
    x = torch.randn(2, 8)
    assert amd.Dropout(0.5).eval()(x) is x


def test_decoder_options():
    cfg = SimpleNamespace(t5=SimpleNamespace(d_model=32), funnel=SimpleNamespace(d_model=32, layer_norm_eps=1e-9), latent_size=11, n_latent_tokens=3)
    for key in ("", "no_norm"):
        dec = amd.VAE_DECODER_MODELS[key](cfg)
        assert dec.dropout_rate == 0.0
        assert amd.VAE_DECODER_MODELS[key](cfg, dropout_rate=0.2).dropout_rate == 0.2
        with pytest.raises(ValueError, match="dropout_rate"):
            amd.VAE_DECODER_MODELS[key](cfg, dropout_rate=1.2)
    cfg.latent_decoder_dropout = 0.1
    dec = amd.VAE_DECODER_MODELS[""](cfg)
    assert dec.dropout_rate == 0.1 and dec._active_dropout() == 0.1 and dec.eval()._active_dropout() == 0.0


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


# Each call stands for one refusal; none reaches the GPU.  Pointers are never followed.
P = ctypes.c_void_p(4096)
FWD = dict(kind=0, x=P, xo=8, xi=0, res=None, ro=0, ri=0, grp=1, w=None, b=None, eps=1e-5, p=0.0, rng=None, seed=0, off=0, y=P, sum=None,
           mean=None, rstd=None, rows=4, d=8, t=0, wt=0, rt=0, stream=None)
BWD = dict(kind=0, dy=P, yo=8, yi=0, ds=None, so=0, si=0, x=P, xo=8, xi=0, res=None, ro=0, ri=0, grp=1, w=None, mean=P, rstd=P, p=0.0, rng=None,
           seed=0, off=0, dx=None, dr=None, dw=None, db=None, rows=4, d=8, t=0, wt=0, rt=0, ws=None, nb=0, stream=None)
DROP = dict(x=P, xo=8, xi=0, res=None, ro=0, ri=0, grp=1, out=P, rows=4, d=8, p=0.1, rng=None, seed=0, off=0, t=0, ot=0, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(kind=2), "unknown norm"), (dict(t=2), "unknown dtype"), (dict(t=1, wt=3), "weights"), (dict(t=3, wt=3, rt=1), "residual"),
    (dict(x=None), "null pointer"), (dict(y=None), "null pointer"), (dict(rows=0), "bad shape"), (dict(d=0), "bad shape"),
    (dict(rows=1 << 31), "bad shape"), (dict(d=1 << 31), "bad shape"), (dict(grp=3), "groups"), (dict(grp=0), "groups"),
    (dict(p=-0.1), "probability"), (dict(p=float("nan")), "probability"), (dict(p=1.1), "probability"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(mean=P), "mean and rstd"), (dict(rstd=P), "mean and rstd"),
    (dict(kind=1, b=P), "no bias"), (dict(kind=1, mean=P, rstd=P), "mean and rstd"),
])
def test_norm_fwd_refusals(lib, change, words):
    assert lib.tvae_norm_fwd(*{**FWD, **change}.values()) == 1
    assert words in lib.tvae_last_error().decode()


@pytest.mark.parametrize("change,words", [
    (dict(dy=None), "null pointer"), (dict(rstd=None), "null pointer"), (dict(mean=None), "needs mean"), (dict(kind=1), "neither"),
    (dict(dw=P, rows=4000), "workspace"), (dict(dw=P, ws=P, nb=16, rows=4000), "workspace"), (dict(x=None), "null pointer"), (dict(t=1, rt=3), "residual"),
    (dict(p=2.0), "probability"), (dict(rows=6, grp=4), "groups"),
])
def test_norm_bwd_refusals(lib, change, words):
    assert lib.tvae_norm_bwd(*{**BWD, **change}.values()) == 1
    assert words in lib.tvae_last_error().decode()


@pytest.mark.parametrize("change,words", [
    (dict(t=2), "unknown dtype"), (dict(ot=7), "unknown dtype"), (dict(t=1, ot=3), "one type"), (dict(x=None), "null pointer"),
    (dict(out=None), "null pointer"), (dict(rows=0), "bad shape"), (dict(d=-1), "bad shape"), (dict(grp=3), "groups"),
    (dict(p=1.0000001), "probability"), (dict(p=float("nan")), "probability"),
])
def test_dropout_refusals(lib, change, words):
    assert lib.tvae_dropout(*{**DROP, **change}.values()) == 1
    assert words in lib.tvae_last_error().decode()


def test_backward_workspace_query(lib):
    q = lib.tvae_norm_bwd_workspace_bytes
    assert q(0, 8) == q(8, 0) == q(1 << 31, 8) == q(8, 1 << 31) == -1
    assert q(1, 1) == q(512, 2048) == 0 and q(513, 1) >= 8 and q(1, 2049) >= 2 * 4 * 2049
    # the partial sums stay small next to the rows themselves
    assert q(245760, 1024) <= 245760 * 1024 * 2 // 16


def test_missing_extension_is_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(_lib, "HOST_PATH", str(tmp_path / "_host.so"))
    with pytest.raises(RuntimeError, match="has not been built"):
        F.layer_norm(torch.randn(2, 8))
