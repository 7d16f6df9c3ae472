"""CPU: the norm and dropout operators under what records or transforms a program.  Fake tensors of the GPU stand for the inputs:
shapes and types without storage, so no kernel runs."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import transformer_vae_amd as amd
from transformer_vae_amd import _lib
from transformer_vae_amd import functional as F


@pytest.fixture(scope="module", autouse=True)
def operators():
    _lib.host()


CALLS = [
    (lambda x, w: F.layer_norm(x, w, w), "norm", 1),
    (lambda x, w: F.rms_norm(x, w), "norm", 1),
    (lambda x, w: F.dropout(x, 0.1, (1, 2)), "dropout", 1),
    (lambda x, w: F.dropout(x, 0.1), "dropout", 1),
    (lambda x, w: F.dropout_add(x, x, 0.1, (1, 2)), "dropout", 1),
    (lambda x, w: F.dropout_add_layer_norm(x, x, w, w, 1e-5, 0.1, None, True), "norm", 2),
    (lambda x, w: F.dropout_add_rms_norm(x, x, w, 1e-5, 0.1, (1, 2)), "norm", 1),
]


@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("call,name,outputs", CALLS)
def test_a_recorded_program_holds_the_operator(call, name, outputs, needs_grad):
    """Not the allocation of its output alone, which a replay would return as it is."""
    with FakeTensorMode():
        x, w = torch.empty(4, 6, 16, device="cuda"), torch.empty(16, device="cuda")
        want = call(x, w)
        want = want if isinstance(want, tuple) else (want,)
        assert len(want) == outputs and all(t.shape == x.shape and t.dtype == x.dtype for t in want)
        nodes = [n for n in make_fx(call)(x, w).graph.nodes if n.op == "call_function"]
        assert [str(n.target) for n in nodes].count(f"tvae.{name}.default") == 1
        if needs_grad:
            w.requires_grad_(True)
            x.requires_grad_(True)
        traced = torch.jit.trace(call, (x, w), check_trace=False)
        assert [n.kind() for n in traced.graph.nodes()].count(f"tvae::{name}") == 1


def test_a_recorded_program_draws_its_own_state():
    with FakeTensorMode():
        x = torch.empty(4, 16, device="cuda")
        targets = [str(n.target) for n in make_fx(lambda x: F.dropout(x, 0.5))(x).graph.nodes]
    assert any("random_" in t for t in targets)


@pytest.mark.parametrize("key", ["", "no_norm"])
def test_a_recorded_decoder_holds_the_operator(key):
    from types import SimpleNamespace
    cfg = SimpleNamespace(t5=SimpleNamespace(d_model=16), funnel=SimpleNamespace(d_model=16, layer_norm_eps=1e-9), latent_size=16,
                          n_latent_tokens=3, latent_decoder_dropout=0.1)
    with FakeTensorMode(), torch.device("cuda"):
        dec = amd.VAE_DECODER_MODELS[key](cfg)       # as wide as the model: its linear is the identity
        graph = make_fx(lambda z: dec(z))(torch.empty(2, 3, 16, device="cuda")).graph
    assert any(str(n.target).startswith("tvae.") for n in graph.nodes)


def test_recorded_operators_check_their_arguments():
    """A recorded graph calls the operators directly, with whatever it is given."""
    ops = torch.ops.tvae
    with FakeTensorMode():
        x, w = torch.empty(4, 16, device="cuda"), torch.empty(16, device="cuda")
        rstd, rng = torch.empty(4, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda")
        norm = lambda x=x, r=None, w=w, b=None, eps=1e-5, p=0.0, rng=None: ops.norm(x, r, w, b, 0, eps, p, rng, 0, 0, False)
        back = lambda dy=x, ds=None, x=x, r=None, w=w, mean=rstd, rstd=rstd, p=0.0, rng=None, t=torch.float32: ops.norm_backward(
            dy, ds, x, r, w, mean, rstd, 0, p, rng, 0, 0, t, [True, False, True, False])
        assert [tuple(t.shape) for t in norm()] == [(4, 16)] and [tuple(t.shape) for t in back()] == [(4, 16), (16,)]
        for call, error, words in [
                (lambda: norm(w=w[:8]), ValueError, "weight must be"), (lambda: norm(r=x[:2]), ValueError, "residual must be"),
                (lambda: norm(b=w.half(), w=w.half()), TypeError, "weight must be"), (lambda: norm(eps=-1.0), ValueError, "eps"),
                (lambda: norm(p=1.5), ValueError, "between 0 and 1"), (lambda: norm(p=0.5, rng=rng[:1]), ValueError, "rng"),
                (lambda: norm(x=x.double()), TypeError, "float64"), (lambda: norm(x=torch.empty((), device="cuda")), ValueError, "without axes"),
                (lambda: norm(x=x[:, :0], w=w[:0]), ValueError, "empty"),
                (lambda: ops.dropout(x, x[:2], 0.1, None, 0, 0), ValueError, "residual must be"),
                (lambda: ops.dropout(x, None, 0.1, rng.int(), 0, 0), ValueError, "rng"),
                (lambda: back(x=x[:2]), ValueError, "x must be"), (lambda: back(rstd=rstd[:2]), ValueError, "rstd"),
                (lambda: back(mean=rstd.half()), ValueError, "mean"), (lambda: back(w=w[:8]), ValueError, "weight must be"),
                (lambda: back(t=torch.bfloat16), TypeError, "types"), (lambda: back(ds=x, r=x, x=x.bfloat16()), TypeError, "x must be")]:
            with pytest.raises(error, match=words):
                call()
    with pytest.raises(NotImplementedError):        # no kernel for tensors of the CPU
        ops.dropout(torch.empty(4, 16), None, 0.1, None, 0, 0)


@pytest.mark.parametrize("place", range(4))
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_derivatives_are_refused(place, needs_grad):
    """A tangent on any input, in any grad mode: never a result without one."""
    import torch.autograd.forward_ad as fw
    with FakeTensorMode(), fw.dual_level():
        t = [torch.empty(s, device="cuda", requires_grad=needs_grad) for s in ((4, 16), (4, 16), (16,), (16,))]
        t[place] = fw.make_dual(t[place], torch.empty_like(t[place]))
        x, r, w, b = t
        calls = [lambda: F.dropout_add_layer_norm(x, r, w, b, 1e-5, 0.1, (1, 2), True)]
        if place != 1:
            calls.append(lambda: F.layer_norm(x, w, b))
        if place != 3:
            calls.append(lambda: F.dropout_add_rms_norm(x, r, w))
        if place < 2:
            calls.append(lambda: F.dropout_add(x, r, 0.1, (1, 2)))
        if place == 0:
            calls += [lambda: F.dropout(x, 0.1), lambda: F.rms_norm(x)]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_what_stands_for_a_dropout_state():
    """A tensor, or two integers in any sequence; another thing is a TypeError, another number of them a ValueError."""
    import numpy as np
    with FakeTensorMode():
        x = torch.empty(4, 16, device="cuda")
        for rng in ((1, 2), [1, 2], np.array([1, 2]), (np.int64(1), True), (-1, 2 ** 64 - 1)):
            assert F.dropout(x, 0.5, rng).shape == x.shape
        for rng, error in ((7, TypeError), ("12", TypeError), (torch.Generator(), TypeError), ((1, 2.5), TypeError), (("1", "2"), TypeError), ({1, 2}, TypeError),
                           ((1,), ValueError), ([1, 2, 3], ValueError), ((), ValueError)):
            for call in (lambda: F.dropout(x, 0.5, rng), lambda: F.dropout_add_rms_norm(x, x, p=0.5, rng=rng)):
                with pytest.raises(error, match="rng must be a tensor or two ints"):
                    call()
