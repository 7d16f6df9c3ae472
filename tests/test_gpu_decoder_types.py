"""GPU: the decoders' dropout and native norm where latents and parameters are of different types, against the stock paths."""
from types import SimpleNamespace

import pytest
import torch

import transformer_vae_amd as amd

pytestmark = pytest.mark.gpu

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64


def dev():
    return torch.device("cuda:0")


def u_of(t):
    return torch.finfo(t).eps / 2


def t5_cfg(L):
    from transformers import T5Config
    return SimpleNamespace(t5=T5Config(d_model=64, d_ff=160, num_layers=1, num_heads=2, vocab_size=8), latent_size=L, n_latent_tokens=3)


@pytest.mark.parametrize("L", [24, 64])              # 64: the latents are the hidden states
@pytest.mark.parametrize("z_type,p_type,autocast", [(F32, F32, None), (BF16, F32, None), (F16, F32, None), (F32, BF16, None), (F32, F16, None),
                                                    (BF16, BF16, None), (F16, BF16, None), (BF16, F16, None), (F32, F32, BF16), (BF16, F32, BF16),
                                                    (F32, F32, F16)])
def test_t5_decoder_of_mixed_types(z_type, p_type, autocast, L):
    """Types as the stock block's, values too.  With u the wider rounding of the types that take part: the norms' outputs differ by
    at most three roundings, each product's result by two more; a 160 x 64 product of random weights stretches an error by up to
    1 + (64/160)^1/2 = 1.6 against its result, the way through the relu by 2^1/2, the 64 x 160 one by 2.6: ((3 * 1.6 + 2) 1.4 * 2.6 + 2) u
    < 32 u of the branch, in the 2-norm.  Backward the same chain once more: 64 u of a gradient's norm."""
    torch.manual_seed(4)
    stock = amd.VAE_DECODER_MODELS["t5_norm"](t5_cfg(L)).to(dev(), p_type)
    own = amd.VAE_DECODER_MODELS["t5_norm"](t5_cfg(L), native_norm=True).to(dev(), p_type)
    own.load_state_dict(stock.state_dict())
    z = torch.randn(4, 3, L, device=dev()).to(z_type).requires_grad_(True)
    outs, grads = [], []
    for dec in (stock, own):
        with torch.autocast("cuda", dtype=autocast or BF16, enabled=autocast is not None):
            out = dec(z)
        outs.append(out)
        grads.append(torch.autograd.grad(out.float().square().sum(), [z, *dec.parameters()]))
    assert outs[0].dtype == outs[1].dtype and outs[0].shape == outs[1].shape
    u = max(u_of(t) for t in (z_type, p_type, autocast or F32)) + 2 * u_of(F32)
    a, c = (t.detach().double() for t in outs)
    assert (a - c).norm() <= 32 * u * a.norm()
    for p, q in zip(*grads):
        assert p.dtype == q.dtype
        assert (p.double() - q.double()).norm() <= 64 * u * p.double().norm()


@pytest.mark.parametrize("z_type,p_type", [(BF16, F32), (F32, BF16), (F16, F32)])
def test_t5_decoder_of_mixed_types_with_a_dropout_rate(z_type, p_type):
    """A dropout rate brings the native norm along, in evaluation too."""
    torch.manual_seed(4)
    stock = amd.VAE_DECODER_MODELS["t5_norm"](t5_cfg(24)).to(dev(), p_type)
    drop = amd.VAE_DECODER_MODELS["t5_norm"](t5_cfg(24), dropout_rate=0.5).to(dev(), p_type)
    drop.load_state_dict(stock.state_dict())
    z = torch.randn(4, 3, 24, device=dev()).to(z_type)
    a, c = stock(z), drop.eval()(z)
    assert a.dtype == c.dtype and (a.double() - c.double()).norm() <= 32 * max(u_of(z_type), u_of(p_type)) * a.double().norm()
    out = drop.train()(z)
    assert out.dtype == a.dtype and torch.isfinite(out).all()


@pytest.mark.parametrize("key", ["", "no_norm", "t5_norm"])
@pytest.mark.parametrize("L", [24, 64])
def test_double_latents_with_a_dropout_rate(key, L):
    """The latent decoders compute float64 in fp32 and return float64; a dropout rate changes nothing about that."""
    cfg = t5_cfg(L)
    cfg.funnel = SimpleNamespace(d_model=64, layer_norm_eps=1e-9)
    torch.manual_seed(4)
    dec = amd.VAE_DECODER_MODELS[key](cfg, dropout_rate=0.25).to(dev(), F64)
    z = torch.randn(4, 3, L, device=dev(), dtype=F64, requires_grad=True)
    dec.train()
    torch.manual_seed(9)
    out = dec(z)
    assert out.dtype == F64
    grads = torch.autograd.grad(out.square().sum(), [z, *dec.parameters()])
    assert all(g.dtype == F64 and torch.isfinite(g).all() for g in grads)
    single = amd.VAE_DECODER_MODELS[key](cfg, dropout_rate=0.25).to(dev())
    single.load_state_dict(dec.state_dict())
    single.train()
    torch.manual_seed(9)
    want = single(z.detach().float())
    # the same keep decisions; the stock products of t5_norm run in fp64 there and in fp32 here: 64 and 160 terms, twice 1.6 * 2.6
    # of their rounding and a rounding a step, within 64 of fp32's in the 2-norm
    assert (out.detach() - want.detach().double()).norm() <= 64 * u_of(F32) * out.detach().norm()
    assert dec.eval()(z).dtype == F64


def test_norm_parameters_of_two_types_with_a_dropout_rate():
    """The default decoder takes them without a rate, and so it does with one."""
    cfg = t5_cfg(24)
    cfg.funnel = SimpleNamespace(d_model=64, layer_norm_eps=1e-9)
    torch.manual_seed(4)
    dec = amd.VAE_DECODER_MODELS[""](cfg, dropout_rate=0.25).to(dev(), BF16)
    dec.norm.bias.data = torch.randn(64, device=dev())
    z = torch.randn(4, 3, 24, device=dev()).to(BF16).requires_grad_(True)
    assert dec.eval()(z).dtype == BF16
    out = dec.train()(z)
    grads = torch.autograd.grad(out.float().square().sum(), [z, *dec.parameters()])
    assert out.dtype == BF16 and all(torch.isfinite(g).all() for g in grads)
    assert [g.dtype for g in grads] == [t.dtype for t in (z, *dec.parameters())]
