"""GPU: norm and dropout operators against the fp64 oracle, at the sizes, types and layouts where they can go wrong.

Tolerances are element-wise bounds counted in roundings.  With u = eps/2 of a type (the most a rounding to it is off,
relative to the value) and h = 2^-24 that of fp32:
  * an output costs u of its own type;
  * v = residual + scale x costs h (|scale x| + |v|);
  * a sum over n terms costs at most CHAIN(n) h of the sum of their magnitudes, CHAIN(n) = n / 64 + 32: no sum here runs
    serially over more than 8 in 512 of a row's elements before a tree of at most 32 steps;
  * rstd costs half of its argument's relative error and 4 h of its own (square root, reciprocal, division);
  * dw and db add rows serially for at most min(rows, 512) steps, then in a tree.
Dropout alone is one product and one rounding, the same in fp32 here and in the kernel: equality."""
import numpy as np
import pytest
import torch

import transformer_vae_amd as amd
from oracle import norm_oracle as orc
from transformer_vae_amd import _lib
from transformer_vae_amd import functional as F

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
H = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def u_of(t):
    return torch.finfo(t).eps / 2


def n64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def chain(n):
    return n / 64 + 32


def tiny(t):
    """Half of the smallest subnormal: what an underflowing store may lose."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


class Expect:
    """fp64 values of one call and the bounds on a kernel's distance from them."""

    def __init__(self, x, r, w, b, eps, rms, p, rng, dy=None, ds=None, types=None):
        d = x.shape[-1]
        x2 = None if x is None else n64(x).reshape(-1, d)
        r2 = None if r is None else n64(r).reshape(-1, d)
        w, b = n64(w), n64(b)
        rows = x2.shape[0]
        kept, sc = (np.ones((rows, d), bool), 1.0) if p == 0 else (orc.keep(rows, d, p, *rng), orc.scale(p))
        xs = np.where(kept, x2 * sc, 0.0)
        v = xs if r is None else xs + r2
        y, xh, rstd = orc.norm_forward(v, w, b, eps, rms)
        one = np.ones(d) if w is None else w
        c = chain(d)
        mean_abs = np.abs(v).mean(1, keepdims=True)
        # the deviation v - mean and, relative to it, the statistics
        e_v = H * (2 * np.abs(xs) + 3 * np.abs(v) + (0 if rms else (c + 2) * mean_abs))
        e_xh = e_v * rstd + H * (c + 8) * np.abs(xh) + rstd * (e_v * np.abs(xh)).mean(1, keepdims=True) * np.abs(xh)
        self.y, self.s = y, v
        self.e_y = u_of(types["y"]) * np.abs(y) + np.abs(one) * e_xh + 4 * H * (np.abs(xh * one) + np.abs(y)) + tiny(types["y"])
        self.e_s = u_of(types["s"]) * np.abs(v) + H * (2 * np.abs(xs) + np.abs(v)) + tiny(types["s"])
        if dy is None:
            return
        dy2 = n64(dy).reshape(-1, d)
        dv, self.dw, self.db = orc.norm_backward(dy2, xh, rstd, w, rms)
        g = np.abs(dy2 * one)
        s2 = (dy2 * one * xh).mean(1, keepdims=True)
        # the backward pass takes the mean in fp32 from the forward pass: h of it once more
        e_xh = e_xh + H * rstd * np.abs(v.mean(1, keepdims=True)) * (0 if rms else 2)
        e_s2 = (g * e_xh).mean(1, keepdims=True) + H * (c + 4) * (g * np.abs(xh)).mean(1, keepdims=True)
        e_s1 = 0 if rms else H * (c + 4) * g.mean(1, keepdims=True)
        inner = np.abs(dv) / rstd
        e_dv = rstd * (4 * H * (g + np.abs(xh * s2)) + e_s1 + np.abs(xh) * e_s2 + e_xh * np.abs(s2) + 4 * H * inner) + H * (c + 8) * np.abs(dv)
        if ds is not None:
            ds2 = n64(ds).reshape(-1, d)
            dv = dv + ds2
            e_dv = e_dv + 2 * H * (np.abs(ds2) + np.abs(dv))
        self.dr, self.e_dr = dv, e_dv + u_of(types["s"]) * np.abs(dv) + tiny(types["s"])
        self.dx = np.where(kept, dv * sc, 0.0)
        self.e_dx = np.where(kept, e_dv * sc + (u_of(types["y"]) + H) * np.abs(self.dx) + tiny(types["y"]), 0.0)
        steps = min(rows, 512) + 32
        self.e_dw = u_of(types["w"]) * np.abs(self.dw) + H * steps * np.abs(dy2 * xh).sum(0) + (np.abs(dy2) * e_xh).sum(0) + tiny(types["w"])
        self.e_db = u_of(types["w"]) * np.abs(self.db) + H * steps * np.abs(dy2).sum(0) + tiny(types["w"])


def close(got, want, bound, what):
    got = n64(got).reshape(want.shape)
    assert np.isfinite(got).all(), what
    off = np.abs(got - want)
    worst = (off - bound).argmax()
    assert (off <= bound).all(), f"{what}: {off.flat[worst]:.3g} off at {worst}, {bound.flat[worst]:.3g} allowed, value {want.flat[worst]:.6g}"


def make(shape, x, w, r, seed, seq=None, bias=True, train=True, spread=1.0):
    g = torch.Generator(device=dev()).manual_seed(seed)
    d = shape[-1]

    def normal(*s):
        return torch.randn(s, generator=g, device=dev())

    if seq:
        xt = (normal(shape[0], seq, d) * spread + 0.5 * normal(d)).to(TYPES[x])[:, :shape[1]]
    else:
        xt = (normal(*shape) * spread + 0.5 * normal(d)).to(TYPES[x])
    rt = None if not r else (2 * normal(*shape)).to(TYPES[r])
    wt = None if not w else (1 + 0.2 * normal(d)).to(TYPES[w])
    bt = None if not w or not bias else (0.2 * normal(d)).to(TYPES[w])
    dy = normal(*shape).to(TYPES[x])
    ds = normal(*shape).to(TYPES[r or x])
    if train:
        xt, rt, wt, bt = (None if t is None else t.detach().requires_grad_(True) for t in (xt, rt, wt, bt))
    return xt, rt, wt, bt, dy, ds


def check(shape, x, w, r="", rms=False, p=0.0, return_sum=False, seq=None, eps=1e-6, seed=1, spread=1.0):
    """A forward and backward pass through the public entry points against the oracle."""
    xt, rt, wt, bt, dy, ds = make(shape, x, w, r, seed, seq, not rms, spread=spread)
    rng = (0x123456789ABCDEF0 + seed, 3)
    if rms:
        out = F.rms_norm(xt, wt, eps) if not r and not p and not return_sum else F.dropout_add_rms_norm(xt, rt, wt, eps, p, rng, return_sum)
    else:
        out = F.layer_norm(xt, wt, bt, eps) if not r and not p and not return_sum else F.dropout_add_layer_norm(xt, rt, wt, bt, eps, p, rng, return_sum)
    y, s = out if return_sum else (out, None)
    types = {"y": TYPES[x], "s": TYPES[r or x], "w": TYPES[w or x]}
    want = Expect(xt, rt, wt, bt, eps, rms, p, rng, dy, ds if return_sum else None, types)
    assert y.dtype == types["y"] and y.shape == xt.shape
    close(y, want.y, want.e_y, "y")
    leaves = {k: t for k, t in (("dx", xt), ("dr", rt), ("dw", wt), ("db", bt)) if t is not None}
    outs, cots = ([y, s], [dy, ds]) if return_sum else ([y], [dy])
    if return_sum:
        assert s.dtype == types["s"]
        close(s, want.s, want.e_s, "s")
    for k, g in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), cots)):
        assert g.dtype == leaves[k].dtype and g.shape == leaves[k].shape
        close(g, getattr(want, k), getattr(want, "e_" + k), k)
    # inference runs the same arithmetic: the same bits
    with torch.no_grad():
        if r or p or return_sum:
            f = F.dropout_add_rms_norm(xt, rt, wt, eps, p, rng) if rms else F.dropout_add_layer_norm(xt, rt, wt, bt, eps, p, rng)
        else:
            f = F.rms_norm(xt, wt, eps) if rms else F.layer_norm(xt, wt, bt, eps)
    assert torch.equal(f, y)


# lengths: one element, below / at / above a group of eight, the widths that models have, odd ones, and each side of the
# places where another kernel or another number of lanes takes over
LENGTHS = [1, 2, 7, 8, 9, 63, 64, 65, 77, 127, 128, 129, 136, 255, 256, 264, 511, 512, 513, 520, 768, 769, 776, 1000, 1023, 1024, 1025, 1280, 1536, 1537, 1544, 2047, 2048,
           2049, 2056, 4095, 4096, 4104, 5000, 6143, 6144, 6145, 6152, 8191, 8192, 8193, 8200, 16001, 16384, 16385, 16392, 32768, 32776, 40000]


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("d", LENGTHS)
def test_row_lengths(d, rms):
    rows = 3 if d > 4096 else 37
    for x, w in (("f32", "f32"), ("bf16", "f32")):
        check((rows, d), x, w, rms=rms, seed=d)


@pytest.mark.parametrize("rms", [False, True], ids=["layer", "rms"])
@pytest.mark.parametrize("d", [5, 77, 512, 768, 1030, 1280, 1533, 4096, 5120, 6141, 9000, 33000])
@pytest.mark.parametrize("x,w,r", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("bf16", "f32", "f32"), ("f16", "f16", "f16"),
                                   ("f16", "f32", "f16"), ("bf16", "bf16", "f32"), ("f16", "", "f32"), ("bf16", "f32", "")])
def test_fused_types(d, x, w, r, rms):
    for p, return_sum in ((0.1, False), (0.25, True), (0.0, True)):
        check((4 if d > 4096 else 21, d), x, w, r, rms, p, return_sum, seed=d + len(x))


@pytest.mark.parametrize("x,w,r", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f32")])
@pytest.mark.parametrize("d", [*range(1, 26), 517, 518, 519, 521, 1029, 1030, 1031, 1033, 16379, 16381, 16382, 16383])
def test_cut_packs(d, x, w, r):
    # every remainder of a pack of eight and of four, in the first pack and in later ones
    check((3, d), x, w, r, d % 2 == 0, 0.1, True, seed=d)
    check((3, d), x, w, "", d % 2 == 1, seed=d)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 31, 32, 33, 64, 65, 255, 257, 511, 512, 513, 1025, 4099, 20011])
def test_row_counts(rows):
    for d in (3, 40, 77, 768, 2048, 2049) if rows <= 513 else (40, 768):
        check((rows, d), "f32", "f32", seed=rows)
        check((rows, d), "bf16", "f32", "bf16", rms=True, p=0.1, seed=rows)


def test_many_rows_reach_every_loop():
    check((300007, 24), "f32", "f32", seed=5)
    check((70001, 136), "bf16", "f32", "bf16", p=0.1, seed=6)


@pytest.mark.parametrize("d", [8, 77, 768, 2050])
def test_first_tokens_of_longer_sequences(d):
    for rms in (False, True):
        check((6, 5, d), "f32", "f32", "", rms, seq=11, seed=d)
        check((6, 5, d), "bf16", "f32", "bf16", rms, 0.1, True, seq=7, seed=d)


@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_layouts_give_the_same_bits(x):
    g = torch.Generator(device=dev()).manual_seed(3)
    t = TYPES[x]
    for d in (7, 77, 512):
        base = torch.randn(4, 6, 2 * d, generator=g, device=dev()).to(t)
        w, b = torch.randn(d, generator=g, device=dev()), torch.randn(d, generator=g, device=dev())
        layouts = [base[..., :d], base[..., 1:d + 1], base.transpose(0, 1)[..., :d], base[::2, 1:5, d:], base[:, :1, :d].expand(4, 9, d),
                   torch.randn(d, 24, generator=g, device=dev()).to(t).t(), base.reshape(2, 2, 6, 2 * d)[:, :, 1:, :d], base[0, 0, :d]]
        for x in layouts:
            dy = torch.randn(x.shape, generator=g, device=dev()).to(t)
            got = []
            for v in (x, x.contiguous()):
                v = v.detach().requires_grad_(True)
                y = F.dropout_add_layer_norm(v, dy, w, b, 1e-5, 0.1, (5, 6))
                got.append((y, *torch.autograd.grad(y, v, dy), F.dropout(v, 0.3, (1, 2)), F.rms_norm(v, w)))
            assert all(torch.equal(p, q) for p, q in zip(*got)), (d, x.shape, x.stride())
        # cotangents of other layouts: a slice, an expanded scalar, a transposed one
        x = torch.randn(6, 4, d, generator=g, device=dev()).to(t).requires_grad_(True)
        wg = w.clone().requires_grad_(True)
        for dy in (base.transpose(0, 1)[..., :d], torch.ones((), device=dev(), dtype=t).expand(6, 4, d), base[..., ::2].transpose(0, 1)):
            y = F.rms_norm(x, wg)
            a = torch.autograd.grad(y, (x, wg), dy, retain_graph=True)
            c = torch.autograd.grad(y, (x, wg), dy.contiguous())
            assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_expanded_input_sums_its_gradient():
    x = torch.randn(1, 5, 64, device=dev(), requires_grad=True)
    w = torch.randn(64, device=dev())
    dy = torch.randn(7, 5, 64, device=dev())
    (a,) = torch.autograd.grad(F.layer_norm(x.expand(7, 5, 64), w), x, dy)
    xd = x.detach().expand(7, 5, 64).contiguous().requires_grad_(True)
    (c,) = torch.autograd.grad(F.layer_norm(xd, w), xd, dy)
    assert torch.equal(a, c.sum(0, keepdim=True))


# ---- dropout alone -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("x,r", [("f32", ""), ("bf16", ""), ("f16", ""), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("shape", [(1,), (5,), (8,), (1, 1), (3, 7), (70, 9), (33, 64), (5, 6, 77), (2, 3, 4, 24), (4, 20011), (1, 300007), (70001, 3)])
def test_dropout(shape, x, r):
    g = torch.Generator(device=dev()).manual_seed(shape[-1])
    xt = torch.randn(shape, generator=g, device=dev()).to(TYPES[x]).requires_grad_(True)
    rt = torch.randn(shape, generator=g, device=dev()).to(TYPES[r]).requires_grad_(True) if r else None
    dy = torch.randn(shape, generator=g, device=dev()).to(TYPES[r or x])
    for p, rng in ((0.1, (2 ** 63 + 11, 2 ** 40 + 1)), (0.5, (-3, -4))):
        rows = xt.numel() // shape[-1]
        keep = torch.from_numpy(orc.keep(rows, shape[-1], p, *rng).reshape(shape)).to(dev())
        sc = orc.scale(p)
        y = F.dropout(xt, p, rng) if rt is None else F.dropout_add(xt, rt, p, rng)
        want = torch.where(keep, xt.detach().float() * sc, 0.0)
        if rt is not None:
            want = want + rt.detach().float()
        assert torch.equal(y.detach(), want.to(TYPES[r or x]))
        grads = torch.autograd.grad(y, [xt] if rt is None else [xt, rt], dy)
        assert torch.equal(grads[0], torch.where(keep, dy.float() * sc, 0.0).to(TYPES[x]))
        if rt is not None:
            assert torch.equal(grads[1], dy)


def test_dropout_probabilities():
    x = torch.randn(50, 333, device=dev(), requires_grad=True)
    for p in (0.0, 2.0 ** -18):                   # the nearest multiple of 2^-16 is 0
        assert torch.equal(F.dropout(x, p, (1, 2)), x)
    y = F.dropout(x, 1.0, (1, 2))
    assert not y.any()
    assert not torch.autograd.grad(y, x, torch.ones_like(x))[0].any()
    for p in (2.0 ** -16, 0.999999, 1 - 2.0 ** -16, 1.5 / 65536, 2.5 / 65536):
        keep = torch.from_numpy(orc.keep(50, 333, p, 1, 2)).to(dev())
        assert torch.equal(F.dropout(x, p, (1, 2)), torch.where(keep, x.detach() * orc.scale(p), 0.0)), p
    x1 = torch.ones(4096, 512, device=dev())
    m = F.dropout(x1, 0.1).mean().item()           # unbiased: within five standard deviations of 1
    assert abs(m - 1) < 5 * (0.1 / 0.9 / x1.numel()) ** 0.5


def test_dropped_infinities_and_nans_are_zero():
    keep = orc.keep(64, 80, 0.5, 9, 9)
    x = torch.randn(64, 80, device=dev())
    x[torch.from_numpy(~keep).to(dev())] = float("nan")
    x[0, ~torch.from_numpy(keep[0]).to(dev())] = float("inf")
    r, w = torch.randn(64, 80, device=dev()), torch.randn(80, device=dev())
    clean = torch.where(torch.from_numpy(keep).to(dev()), x, 0.0)
    assert torch.equal(F.dropout(x, 0.5, (9, 9)), F.dropout(clean, 0.5, (9, 9)))
    assert torch.equal(F.dropout_add_layer_norm(x, r, w, None, p=0.5, rng=(9, 9)), F.dropout_add_layer_norm(clean, r, w, None, p=0.5, rng=(9, 9)))
    # and the cotangent's
    a = torch.randn(64, 80, device=dev(), requires_grad=True)
    dy = torch.randn(64, 80, device=dev())
    dy[torch.from_numpy(~keep).to(dev())] = float("nan")
    (g,) = torch.autograd.grad(F.dropout(a, 0.5, (9, 9)), a, dy)
    assert torch.isfinite(g).all() and not g[torch.from_numpy(~keep).to(dev())].any()


def test_infinities_and_nans_stay_in_their_rows():
    for rms in (False, True):
        for d in (77, 768, 5000, 40000):
            x = torch.randn(5, d, device=dev())
            clean = x.clone()
            x[1, 3], x[3, d - 1] = float("nan"), float("inf")
            w = torch.ones(d, device=dev())
            f = (lambda t: F.rms_norm(t, w)) if rms else (lambda t: F.layer_norm(t, w, w))
            y, z = f(x), f(clean)
            assert torch.equal(y[[0, 2, 4]], z[[0, 2, 4]])
            assert y[1].isnan().all() and y[3].isnan().any()


def test_rows_of_equal_values():
    for d in (1, 77, 1000, 1024, 3000, 20000, 40000):
        for value in (0.0, 0.1, -1234.567):
            x = torch.full((3, d), value, device=dev(), requires_grad=True)
            w = torch.full((d,), 2.0, device=dev(), requires_grad=True)
            b = torch.full((d,), 0.25, device=dev())
            y = F.layer_norm(x, w, b, 1e-9)
            # what the deviations can be off is a rounding of the value; the eps of the latent decoder's norm multiplies it by 3e4
            assert (y - 0.25).abs().max().item() <= 2 * 31623 * abs(value) * H, (d, value)
            gx, gw = torch.autograd.grad(y, (x, w), torch.randn(3, d, device=dev()))
            assert torch.isfinite(gx).all() and torch.isfinite(gw).all()
        z = F.rms_norm(torch.zeros(3, d, device=dev()), torch.ones(d, device=dev()))
        assert not z.any()


def test_large_offsets_keep_their_digits():
    # rows at 1000 with unit spread: the second pass over the deviations keeps them
    for d in (77, 1024, 6000, 36000):
        g = torch.Generator(device=dev()).manual_seed(d)
        x = torch.randn(9, d, generator=g, device=dev()) + 1000.0
        y = F.layer_norm(x, eps=1e-6)
        want = orc.norm_forward(n64(x), None, None, 1e-6, False)[0]
        # inputs are exact: a deviation costs a rounding of itself after one of the mean's remainder
        bound = H * ((chain(d) + 8) * np.abs(want) + 16 * 4)
        close(y, want, bound, d)


@pytest.mark.parametrize("start", [0, 1000])
@pytest.mark.parametrize("d", [20000, 2000000])
def test_long_rows_that_start_unlike_their_rest(d, start):
    # the deviations are summed about a guess of the mean that the row's unlike part must not decide
    g = torch.Generator(device=dev()).manual_seed(d)
    x = torch.randn(3, d, generator=g, device=dev())
    x[:, start:start + 2048] += 1000.0
    y = F.layer_norm(x, eps=1e-6)
    v = n64(x)
    want, _, rstd = orc.norm_forward(v, None, None, 1e-6, False)
    # a thread adds d / 256 terms; six standard deviations of that many roundings, on the value and on the mean
    bound = H * (6 * np.sqrt(d / 256) + 8) * (np.abs(want) + rstd * np.abs(v - v.mean(1, keepdims=True)).mean(1, keepdims=True))
    close(y, want, bound, d)


def test_gradient_against_differences():
    g = torch.Generator(device=dev()).manual_seed(8)
    x, r = (torch.randn(12, 200, generator=g, device=dev()).requires_grad_(True) for _ in range(2))
    w, b = ((1 + 0.2 * torch.randn(200, generator=g, device=dev())).requires_grad_(True) for _ in range(2))
    cy, cs = torch.randn(12, 200, generator=g, device=dev()), torch.randn(12, 200, generator=g, device=dev())

    def loss(*t):
        y, s = F.dropout_add_layer_norm(*t, 1e-5, 0.25, (4, 2), True)
        return (y.double() * cy).sum() + (s.double() * cs).sum()

    grads = torch.autograd.grad(loss(x, r, w, b), (x, r, w, b))
    for k in range(4):
        u = torch.randn((x, r, w, b)[k].shape, generator=g, device=dev())
        u /= u.norm()
        h = 2.0 ** -4
        with torch.no_grad():
            at = [[t.detach() + (sgn * h * u if j == k else 0) for j, t in enumerate((x, r, w, b))] for sgn in (1, -1)]
            num = ((loss(*at[0]) - loss(*at[1])) / (2 * h)).item()
        # each of the 2400 outputs of the two losses is off by up to ~4 roundings of values up to 8: 2400 * 8 * 4 * 2^-24 / h at
        # worst, a fiftieth of that in the mean; the difference quotient itself is off by h^2/6 times the third derivative
        assert abs(num - (grads[k] * u).sum().item()) <= 2400 * 8 * 4 * H / h / 50 + h * h, k


def test_no_rows_and_refusals():
    x = torch.empty(0, 16, device=dev(), requires_grad=True)
    w = torch.ones(16, device=dev(), requires_grad=True)
    y, s = F.dropout_add_layer_norm(x, x, w, None, p=0.1, return_sum=True)
    assert y.shape == s.shape == (0, 16)
    gx, gw = torch.autograd.grad(y.sum() + s.sum(), (x, w))
    assert gx.shape == (0, 16) and not gw.any()
    assert F.dropout(torch.empty(3, 0, device=dev()), 0.5).shape == (3, 0)
    assert F.rms_norm(torch.empty(2, 0, 16, device=dev()), w).shape == (2, 0, 16)
    x, w = torch.randn(4, 16, device=dev()), torch.ones(16, device=dev())
    rng = torch.tensor([1, 2], device=dev())
    for call, error, words in [
            (lambda: F.layer_norm(x, w[:8]), ValueError, "weight must be"),
            (lambda: F.layer_norm(x, w, w.half()), TypeError, "float32"),
            (lambda: F.layer_norm(x.bfloat16(), w, w.bfloat16()), TypeError, "one type"),
            (lambda: F.layer_norm(x.double(), None), TypeError, "float64"),
            (lambda: F.rms_norm(x.int()), TypeError, "int32"),
            (lambda: F.layer_norm(x, w.cpu()), ValueError, "is on cpu"),
            (lambda: F.layer_norm(x, w, w, -1e-6), ValueError, "eps"),
            (lambda: F.layer_norm(x, w, w, float("nan")), ValueError, "eps"),
            (lambda: F.layer_norm(torch.empty(3, 0, device=dev())), ValueError, "empty"),
            (lambda: F.layer_norm(torch.tensor(1.0, device=dev())), ValueError, "without axes"),
            (lambda: F.dropout(x, 1.5), ValueError, "between 0 and 1"),
            (lambda: F.dropout(x, float("nan")), ValueError, "between 0 and 1"),
            (lambda: F.dropout(x, 0.1, rng.int()), ValueError, "rng"),
            (lambda: F.dropout(x, 0.1, rng.cpu()), ValueError, "rng"),
            (lambda: F.dropout(x, 0.1, torch.zeros(3, dtype=torch.int64, device=dev())), ValueError, "rng"),
            (lambda: F.dropout(x, 0.1, rng.repeat_interleave(2)[::2]), ValueError, "rng"),
            (lambda: F.dropout_add(x, None, 0.1), ValueError, "missing"),
            (lambda: F.dropout_add(x, x[:1], 0.1), ValueError, "residual must be"),
            (lambda: F.dropout_add(x, x.bfloat16(), 0.1), TypeError, "residual"),
            (lambda: F.dropout_add_rms_norm(x.half(), x.bfloat16(), w), TypeError, "residual"),
            (lambda: F.dropout_add_layer_norm(x, x[:, :8], w), ValueError, "residual must be")]:
        with pytest.raises(error, match=words):
            call()


def test_second_derivatives_are_refused():
    x = torch.randn(4, 16, device=dev(), requires_grad=True)
    for y in (F.layer_norm(x), F.dropout(x, 0.5)):
        (g,) = torch.autograd.grad(y.sum() + (y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


@pytest.mark.parametrize("shape", [(5, 96), (33, 301), (1000, 300), (3, 5000), (3, 20000)])
def test_partial_gradients(shape):
    """Only the gradients that are asked for; each equals the one from asking for all."""
    for return_sum in (False, True):
        xt, rt, wt, bt, dy, ds = make(shape, "bf16", "f32", "bf16", 4)
        def run(need):
            ts = [t.detach().requires_grad_(k in need) for k, t in zip("xrwb", (xt, rt, wt, bt))]
            out = F.dropout_add_layer_norm(*ts, 1e-5, 0.1, (8, 8), return_sum)
            outs, cots = (list(out), [dy, ds]) if return_sum else ([out], [dy])
            return dict(zip(need, torch.autograd.grad(outs, [t for t in ts if t.requires_grad], cots)))
        full = run("xrwb")
        for need in ("x", "r", "w", "b", "xr", "wb", "xw"):
            part = run(need)
            assert all(torch.equal(part[k], full[k]) for k in need), (need, return_sum)
    # the sum alone is used: the norm has no part
    y, s = F.dropout_add_layer_norm(xt, rt, wt, bt, 1e-5, 0.1, (8, 8), True)
    gx, gr, gw = torch.autograd.grad(s, (xt, rt, wt), ds, allow_unused=True)
    assert gw is None and torch.equal(gr, ds)
    (want,) = torch.autograd.grad(F.dropout(xt, 0.1, (8, 8)), xt, ds)
    assert torch.equal(gx, want)


def test_shared_gradient_without_dropout():
    # one tensor for both inputs' gradients: accumulating into one must not change the other
    x = torch.randn(8, 64, device=dev(), requires_grad=True)
    r = torch.randn(8, 64, device=dev(), requires_grad=True)
    dy = torch.randn(8, 64, device=dev())
    for _ in range(2):
        F.dropout_add_rms_norm(x, r).backward(dy)
    (g,) = torch.autograd.grad(F.dropout_add_rms_norm(x, r), x, dy)
    assert torch.equal(x.grad, 2 * g) and torch.equal(r.grad, 2 * g)
    x.grad.mul_(3)
    assert torch.equal(r.grad, 2 * g)
    # the same tensor as both inputs
    a = torch.randn(8, 64, device=dev(), requires_grad=True)
    (ga,) = torch.autograd.grad(F.dropout_add_layer_norm(a, a), a, dy)
    (gb,) = torch.autograd.grad(F.layer_norm(2 * a), a, dy)
    assert torch.allclose(ga, gb, rtol=0, atol=8 * H * 16)


# ---- state: rng, streams, graphs, determinism, surroundings ------------------------------------------------------------------

def test_rng_forms_agree_and_follow_the_seed():
    x = torch.randn(40, 100, device=dev())
    for seed, off in ((5, 6), (-1, 2 ** 62), (2 ** 63 + 5, 1)):
        wrap = lambda v: v - 2 ** 64 if v >= 2 ** 63 else v
        t = torch.tensor([wrap(seed), wrap(off)], device=dev())
        assert torch.equal(F.dropout(x, 0.3, (seed, off)), F.dropout(x, 0.3, t))
    torch.manual_seed(11)
    a, b = F.dropout(x, 0.3), F.dropout(x, 0.3)
    torch.manual_seed(11)
    assert torch.equal(a, F.dropout(x, 0.3)) and not torch.equal(a, b)
    # a state that changes before the backward pass is an error, not a wrong gradient
    t = F.dropout_rng(dev())
    xg = x.clone().requires_grad_(True)
    for f in (lambda: F.dropout(xg, 0.3, t), lambda: F.dropout_add_rms_norm(xg, None, p=0.3, rng=t)):
        y = f()
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_results_repeat_bit_for_bit():
    xt, rt, wt, bt, dy, _ = make((5003, 768), "bf16", "f32", "bf16", 2)
    runs = []
    for _ in range(3):
        y = F.dropout_add_layer_norm(xt, rt, wt, bt, 1e-5, 0.1, (1, 1))
        runs.append((y, *torch.autograd.grad(y, (xt, rt, wt, bt), dy)))
    assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(runs[0], r))


def test_fused_and_single_operators_drop_the_same_elements():
    for d in (77, 640):
        x, r = torch.randn(90, d, device=dev()), torch.randn(90, d, device=dev())
        w, b = torch.randn(d, device=dev()), torch.randn(d, device=dev())
        s0 = F.dropout_add(x, r, 0.2, (3, 4))
        y, s = F.dropout_add_layer_norm(x, r, w, b, 1e-5, 0.2, (3, 4), True)
        assert torch.equal(s, s0) and torch.equal(y, F.layer_norm(s0, w, b, 1e-5))
        y, s = F.dropout_add_rms_norm(x, r, w, 1e-5, 0.2, (3, 4), True)
        assert torch.equal(s, s0) and torch.equal(y, F.rms_norm(s0, w, 1e-5))


def test_two_streams_at_once():
    # two backward passes in flight share nothing
    a, b = make((4096, 768), "bf16", "f32", "bf16", 5), make((4096, 768), "bf16", "f32", "bf16", 6)

    def go(t):
        leaves = [q.detach().requires_grad_(True) for q in t[:4]]
        y = F.dropout_add_layer_norm(*leaves, 1e-5, 0.1, (1, 2))
        return (y.detach(), *torch.autograd.grad(y, leaves, t[4]))

    want = go(a), go(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(4):
        for i, (s, t) in enumerate(((s1, a), (s2, b))):
            with torch.cuda.stream(s):
                got[i].append(go(t))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(r, want[i]))


def test_captured_steps_replay():
    """Forward and backward in a graph, replayed with new inputs and new states among eager work; two graphs side by side."""
    w = (1 + 0.1 * torch.randn(96, device=dev())).requires_grad_(True)
    b = torch.randn(96, device=dev()).requires_grad_(True)

    def step(x, r, dy, rng):
        xg, rg = x.detach().requires_grad_(True), r.detach().requires_grad_(True)
        y, s = F.dropout_add_layer_norm(xg, rg, w, b, 1e-5, 0.2, rng, True)
        z = F.dropout_add(y, s, 0.1, rng)
        return (z.detach(), *torch.autograd.grad(z, (xg, rg, w, b), dy))

    g = torch.Generator(device=dev()).manual_seed(1)

    def inputs():
        return [torch.randn(700, 96, generator=g, device=dev()) for _ in range(3)] + [torch.randint(0, 1 << 60, (2,), generator=g, device=dev())]

    graphs = [amd.GraphedStep(step, inputs()) for _ in range(2)]
    for k in range(4):
        for gr in graphs:
            new = inputs()
            got = [t.clone() for t in gr(*new)]
            want = step(*new)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want)), k


@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
@pytest.mark.parametrize("op", ["norm", "dropout"])
def test_capture_beside_a_living_eager_graph_is_refused(op):
    """The leaf's accumulation node is the eager graph's, on the default stream: refused in the capture, not outside it."""
    w = torch.randn(96, device=dev(), requires_grad=True)
    x = torch.randn(40, 96, device=dev(), requires_grad=True)

    def step(dy):
        y = F.rms_norm(x, w) if op == "norm" else F.dropout(x, 0.25, (3, 4))
        return torch.autograd.grad(y, (x, w) if op == "norm" else x, dy)

    dy = torch.randn(40, 96, device=dev())
    want = step(dy)
    alive = (x * w).sum()
    with pytest.raises(RuntimeError, match="keep a graph of the same leaves alive"):
        amd.GraphedStep(step, [dy])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                # another stream alone is no reason
        got = step(dy)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del alive
    graphed = amd.GraphedStep(step, [dy])
    for _ in range(3):
        got = [t.clone() for t in graphed(dy)]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_recomputed_forward_draws_the_same():
    # activation checkpointing runs the forward pass again under the generator state that it saved
    from torch.utils.checkpoint import checkpoint
    w = torch.randn(64, device=dev(), requires_grad=True)
    x = torch.randn(30, 64, device=dev(), requires_grad=True)

    def block(t):
        return F.dropout_add_rms_norm(t, t, w, p=0.3) + F.dropout(t, 0.5)

    grads = []
    for f in (block, lambda t: checkpoint(block, t, use_reentrant=False)):
        torch.manual_seed(6)
        y = f(x)
        grads.append((y.detach(), *torch.autograd.grad(y.square().sum(), (x, w))))
    assert all(torch.equal(p, q) for p, q in zip(*grads))


def test_captured_dropout_draws_anew():
    x = torch.ones(64, 64, device=dev())
    gr = amd.GraphedStep(lambda t: F.dropout(t, 0.5), [x])
    seen = [gr(x).clone() for _ in range(3)]
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    assert all(set(t.unique().tolist()) == {0.0, 2.0} for t in seen)


@pytest.mark.parametrize("d", [5, 77, 768, 5000, 40000])
def test_surroundings_stay_as_they_are(d):
    """Outputs with a margin on both sides through the C interface: nothing but the rows is written."""
    lib, rows, pad = _lib.lib(), 7, 64
    stream = torch.cuda.current_stream().cuda_stream
    for dt, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        x, dy = (torch.randn(rows, d, device=dev()).to(dt) for _ in range(2))
        w = torch.ones(d, device=dev(), dtype=dt)
        nb = lib.tvae_norm_bwd_workspace_bytes(rows, d)

        def room(n, t):
            return torch.full((n + 2 * pad,), float("nan"), dtype=t, device=dev())

        outs = {k: room(rows * d, dt) for k in ("y", "s", "dx", "dr", "drop")}
        outs.update({k: room(d, dt) for k in ("dw", "db")})
        outs.update(mean=room(rows, torch.float32), rstd=room(rows, torch.float32), ws=room(max(nb // 4, 1), torch.float32))
        ptr = {k: t.data_ptr() + pad * t.element_size() for k, t in outs.items()}
        xp, rp = x.data_ptr(), dy.data_ptr()
        assert lib.tvae_norm_fwd(0, xp, d, 0, rp, d, 0, 1, w.data_ptr(), w.data_ptr(), 1e-5, 0.1, None, 1, 2, ptr["y"], ptr["s"], ptr["mean"],
                                 ptr["rstd"], rows, d, code, code, code, stream) == 0
        assert lib.tvae_norm_bwd(0, rp, d, 0, None, 0, 0, xp, d, 0, rp, d, 0, 1, w.data_ptr(), ptr["mean"], ptr["rstd"], 0.1, None, 1, 2, ptr["dx"],
                                 ptr["dr"], ptr["dw"], ptr["db"], rows, d, code, code, code, ptr["ws"], nb, stream) == 0
        assert lib.tvae_dropout(xp, d, 0, None, 0, 0, 1, ptr["drop"], rows, d, 0.1, None, 1, 2, code, code, stream) == 0
        torch.cuda.synchronize()
        for k, t in outs.items():
            assert t[:pad].isnan().all() and t[-pad:].isnan().all(), k
            if k != "ws":
                assert not t[pad:-pad].isnan().any(), k


def test_offsets_beyond_32_bits():
    # 2.2e9 elements: the last rows lie past 2^31 elements, in the input, the output and the gradients
    rows, d = 1100003, 2000
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=dev())
    tail, head = torch.randn(64, d, device=dev()).to(x.dtype), torch.randn(64, d, device=dev()).to(x.dtype)
    x.zero_()
    x[:64], x[-64:] = head, tail
    w = torch.randn(d, device=dev())
    x.requires_grad_(True)
    wg = w.clone().requires_grad_(True)
    y = F.layer_norm(x, wg, None, 1e-5)
    assert torch.equal(y[-64:], F.layer_norm(tail, w, None, 1e-5)) and torch.equal(y[:64], F.layer_norm(head, w, None, 1e-5))
    gx, gw = torch.autograd.grad(y, (x, wg), y.detach())
    del y
    t2 = tail.clone().requires_grad_(True)
    yt = F.layer_norm(t2, w, None, 1e-5)
    assert torch.equal(gx[-64:], torch.autograd.grad(yt, t2, yt.detach())[0])
    assert torch.isfinite(gw).all()
    del gx
    z = F.dropout(x.detach(), 0.5, (1, 2))
    keep = torch.from_numpy(orc.keep(64, d, 0.5, 1, 2, rows - 64)).to(dev())
    assert torch.equal(z[-64:], torch.where(keep, tail.float() * 2, 0.0).to(z.dtype))


# ---- used together and in the framework's own paths ----------------------------------------------------------------------

@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_sub_layers_in_sequence(x):
    """A pre-norm block and a post-norm block as a model chains them: module by module against one fp64 evaluation."""
    torch.manual_seed(5)
    d, p = 96, 0.2
    t = TYPES[x]
    lin1, lin2 = (torch.nn.Linear(d, d, device=dev(), dtype=t) for _ in range(2))
    pre, post, first = (amd.DropoutAddRMSNorm(d, p, device=dev(), dtype=t), amd.DropoutAddLayerNorm(d, p, device=dev(), dtype=t),
                        amd.RMSNorm(d, device=dev(), dtype=t))
    h = torch.randn(5, 7, d, device=dev()).to(t).requires_grad_(True)
    n = first(h)
    n, s = pre(lin1(n), h, rng=(1, 1), return_sum=True)
    out = post(lin2(n), s, rng=(1, 2))
    dy = torch.randn_like(out)
    params = [h, first.weight, pre.weight, post.weight, post.bias, lin1.weight, lin2.weight]
    grads = torch.autograd.grad(out, params, dy)

    L = [q.detach().double().cpu().requires_grad_(True) for q in params]
    b1, b2 = lin1.bias.detach().double().cpu(), lin2.bias.detach().double().cpu()
    rms = lambda v, w: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w

    def drop(v, rng):
        k = torch.from_numpy(orc.keep(35, d, p, *rng).reshape(5, 7, d))
        return torch.where(k, v * orc.scale(p), 0.0)

    n64_ = rms(L[0], L[1])
    s64 = L[0] + drop(n64_ @ L[5].T + b1, (1, 1))
    v = s64 + drop(rms(s64, L[2]) @ L[6].T + b2, (1, 2))
    o64 = (v - v.mean(-1, keepdim=True)) * torch.rsqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5) * L[3] + L[4]
    want = torch.autograd.grad(o64, L, dy.double().cpu())
    # five roundings to the type lie one after another forward and five backward, each u of values of unit size; products
    # over 96 add their own in fp32: 40 u in the 2-norm is four times their sum
    for a, c in zip([out, *grads], [o64.detach(), *want]):
        assert (a.detach().double().cpu() - c).norm() <= 40 * u_of(t) * c.norm()


def _cfg(d, L, **more):
    from types import SimpleNamespace
    return SimpleNamespace(t5=SimpleNamespace(d_model=d), funnel=SimpleNamespace(d_model=d, layer_norm_eps=1e-9), latent_size=L, n_latent_tokens=3, **more)


@pytest.mark.parametrize("L", [24, 64])
def test_decoders_with_dropout(L):
    for key in ("", "no_norm"):
        torch.manual_seed(3)
        plain = amd.VAE_DECODER_MODELS[key](_cfg(64, L)).to(dev())
        dec = amd.VAE_DECODER_MODELS[key](_cfg(64, L, latent_decoder_dropout=0.25)).to(dev())
        dec.load_state_dict(plain.state_dict())
        z = torch.randn(4, 3, L, device=dev(), requires_grad=True)
        assert torch.equal(dec.eval()(z), plain(z))                       # no dropout outside training
        dec.train()
        torch.manual_seed(9)
        out = dec(z)
        torch.manual_seed(9)
        rng = F.dropout_rng(dev())
        w, b = dec._linear_params()
        r = z if w is None else F.latent_decode(z, w, b)
        want = F.dropout(r, 0.25, rng) if key else F.dropout_add_layer_norm(r, None, dec.norm.weight, dec.norm.bias, 1e-9, 0.25, rng)
        assert torch.equal(out, want)
        vae = amd.EncoderDecoderVAE(amd.VAE_ENCODER_MODELS[""](_cfg(64, L)).to(dev()), dec)
        h = torch.randn(4, 6, 64, device=dev(), requires_grad=True)
        o = vae(input_encoding=h)
        (o.reg_loss + o.reconstructed_encoding.square().sum()).backward()
        assert all(torch.isfinite(q.grad).all() for q in [h, *vae.parameters()])


def test_t5_decoder_on_native_norm():
    from transformers import T5Config
    cfg = _cfg(64, 24)
    cfg.t5 = T5Config(d_model=64, d_ff=160, num_layers=1, num_heads=2, vocab_size=8)
    torch.manual_seed(4)
    stock = amd.VAE_DECODER_MODELS["t5_norm"](cfg).to(dev())
    own = amd.VAE_DECODER_MODELS["t5_norm"](cfg, native_norm=True).to(dev())
    own.load_state_dict(stock.state_dict())
    z = torch.randn(4, 3, 24, device=dev(), requires_grad=True)
    dy = torch.randn(4, 3, 64, device=dev())
    a, c = stock(z), own(z)
    # the two differ by the order of fp32 sums over 64 and 160 elements: 64 roundings of the result's size is an upper bound
    assert (a - c).norm() <= 64 * H * a.norm()
    for p, q in zip(torch.autograd.grad(a, [z, *stock.parameters()], dy), torch.autograd.grad(c, [z, *own.parameters()], dy)):
        assert (p - q).norm() <= 64 * H * 4 * p.norm()
    drop = amd.VAE_DECODER_MODELS["t5_norm"](cfg, dropout_rate=0.5).to(dev())
    drop.load_state_dict(stock.state_dict())
    assert torch.equal(drop.eval()(z), c)
    torch.manual_seed(1)
    out = drop.train()(z)
    torch.manual_seed(1)
    rng = F.dropout_rng(dev())
    h = F.latent_decode(z, *own._linear_params())
    branch = own.norm.DenseReluDense(F.rms_norm(h, own.norm.layer_norm.weight, own.norm.layer_norm.variance_epsilon))
    assert torch.equal(out, F.dropout_add(branch, h, 0.5, rng))


def test_modules_follow_training_mode():
    x, r = torch.randn(6, 64, device=dev()), torch.randn(6, 64, device=dev())
    m = amd.DropoutAddLayerNorm(64, 0.5).to(dev())
    drop = amd.Dropout(0.5)
    assert torch.equal(m.eval()(x, r), F.layer_norm(x + r, m.weight, m.bias))
    assert torch.equal(m.train()(x, r, rng=(1, 2)), F.dropout_add_layer_norm(x, r, m.weight, m.bias, 1e-5, 0.5, (1, 2)))
    assert torch.equal(drop(x, rng=(1, 2)), F.dropout(x, 0.5, (1, 2))) and torch.equal(drop(x, r, (1, 2)), F.dropout_add(x, r, 0.5, (1, 2)))
    assert torch.equal(drop.eval()(x, r), x + r)
    stock = torch.nn.LayerNorm(64).to(dev())
    assert (amd.LayerNorm(64).to(dev())(x) - stock(x)).abs().max() <= 64 * H * 4
