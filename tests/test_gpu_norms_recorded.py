"""GPU: recorded programs of the norm and dropout operators give what the eager calls give, on inputs they were not recorded with."""
import io

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import transformer_vae_amd as amd
from transformer_vae_amd import functional as F

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


def inputs(rows, d, seed, dtype=torch.float32):
    g = torch.Generator(device=dev()).manual_seed(seed)
    x, r, dy = (torch.randn(rows, d, generator=g, device=dev()).to(dtype) for _ in range(3))
    w, b = torch.randn(d, generator=g, device=dev()), torch.randn(d, generator=g, device=dev())
    return x, r, w, b, dy, torch.randint(0, 1 << 60, (2,), generator=g, device=dev())


CALLS = {
    "layer_norm": lambda x, r, w, b, dy, rng: F.layer_norm(x, w, b),
    "rms_norm": lambda x, r, w, b, dy, rng: F.rms_norm(x, w),
    "dropout": lambda x, r, w, b, dy, rng: F.dropout(x, 0.25, rng),
    "dropout_add": lambda x, r, w, b, dy, rng: F.dropout_add(x, r, 0.25, rng),
    "post_norm": lambda x, r, w, b, dy, rng: F.dropout_add_layer_norm(x, r, w, b, 1e-5, 0.25, rng),
    "pre_norm": lambda x, r, w, b, dy, rng: F.dropout_add_rms_norm(x, r, w, 1e-5, 0.25, rng, True),
}


def same(got, want):
    got, want = ((t,) if torch.is_tensor(t) else tuple(t) for t in (got, want))
    return len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("name", CALLS)
def test_traced_calls(name):
    call, dtype = CALLS[name], torch.bfloat16 if name == "pre_norm" else torch.float32
    traced = torch.jit.trace(call, inputs(5, 64, 1, dtype))
    for rows, seed in ((5, 2), (700, 3)):
        new = inputs(rows, 64, seed, dtype)
        assert same(traced(*new), call(*new))
    # and through a file, and with gradients
    file = io.BytesIO()
    torch.jit.save(traced, file)
    file.seek(0)
    loaded, new = torch.jit.load(file), inputs(33, 64, 4, dtype)
    leaves = [t.requires_grad_(True) for t in new[:4]]
    for _ in range(3):                       # the first runs of a traced module profile it, later ones are optimised
        grads = []
        for f in (loaded, call):
            out = f(*new)
            out = out[0] if isinstance(out, tuple) else out
            grads.append([g for g in torch.autograd.grad(out, leaves, new[4], allow_unused=True) if g is not None])
        assert grads[0] and same(*grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_recorded_training_step(dtype):
    def step(x, r, w, b, dy, rng):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w, b)]
        n, s = F.dropout_add_layer_norm(*leaves, 1e-5, 0.1, rng, True)
        z = F.dropout_add(n, s, 0.2, rng)
        return (z.detach(), *torch.autograd.grad(z, leaves, dy))

    graph = make_fx(step)(*inputs(40, 96, 1, dtype))
    assert sum("tvae." in str(n.target) for n in graph.graph.nodes) == 4       # two forward, two backward
    for seed in (2, 3):
        new = inputs(40, 96, seed, dtype)
        assert same(graph(*new), step(*new))


def test_traced_dropout_draws_anew():
    x = torch.ones(64, 64, device=dev())
    traced = torch.jit.trace(lambda t: F.dropout(t, 0.5), x, check_trace=False)
    a, b = traced(x), traced(x)
    assert not torch.equal(a, b) and all(set(t.unique().tolist()) == {0.0, 2.0} for t in (a, b))


def test_traced_decoder():
    """The t5_norm decoder on its own norm, recorded for inference at one batch size and used at another."""
    from types import SimpleNamespace
    from transformers import T5Config
    cfg = SimpleNamespace(t5=T5Config(d_model=64, d_ff=160, num_layers=1, num_heads=2, vocab_size=8), latent_size=64, n_latent_tokens=3)
    dec = amd.VAE_DECODER_MODELS["t5_norm"](cfg, native_norm=True).to(dev()).eval()
    g = torch.Generator(device=dev()).manual_seed(1)
    with torch.no_grad():
        traced = torch.jit.trace(dec, torch.randn(2, 3, 64, generator=g, device=dev()))
        for batch in (2, 9):
            z = torch.randn(batch, 3, 64, generator=g, device=dev())
            assert torch.equal(traced(z), dec(z))


@pytest.mark.parametrize("name", CALLS)
def test_a_program_recorded_below_autograd_keeps_its_gradients(name):
    """Recorded with inputs that require gradients, the graph holds the calls that stand below autograd; run as it is, it must not
    give results without a history."""
    call, dtype = CALLS[name], torch.bfloat16 if name == "pre_norm" else torch.float32

    def leaves(seed):
        new = inputs(40, 96, seed, dtype)
        return [t.requires_grad_(True) for t in new[:4]] + list(new[4:])

    graph = make_fx(lambda *t: call(*t))(*leaves(1))
    new, grads = leaves(2), []
    for f in (graph, call):
        out = f(*new)
        outs = out if isinstance(out, tuple) else (out,)
        assert all(t.requires_grad for t in outs)
        grads.append([g for g in torch.autograd.grad(outs, new[:4], [new[4]] * len(outs), allow_unused=True) if g is not None])
    assert grads[0] and same(*grads)


def test_a_recorded_backward_pass_is_not_differentiated():
    def step(x, w, dy):
        y = F.rms_norm(x, w)
        return torch.autograd.grad(y, (x, w), dy)

    x, r, w, b, dy, rng = inputs(40, 96, 1)
    x.requires_grad_(True), w.requires_grad_(True)
    graph = make_fx(step)(x, w, dy)
    got = graph(x, w, dy)
    assert same([t.detach() for t in got], step(x, w, dy))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got[0].sum().backward()
