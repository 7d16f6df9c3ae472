"""Cases of the norm and dropout operators: plain forms in elementary torch operations, and the framework's own calls.

``layer_norm``, ``rms_norm``, ``dropout`` (alone and added to a residual) and ``dropout_add_norm`` (residual + dropout,
then one of the norms), over rows of ``d`` features.  ``own`` chooses between the plain form and the framework.

Dropout's keep decision is a pure function of (seed, offset, row, column): Philox4x32 with ten rounds (Salmon, Moraes, Dror
and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011), key = seed, counter = (column // 8, row, offset low,
offset high); the four words give sixteen bits to each of eight neighbouring columns, low half first.  An element is
dropped where its sixteen bits are below T = round(65536 p), and kept elements are scaled by 65536 / (65536 - T)."""
from functools import reduce

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------------------------
# cases: op, batch x tokens rows of d features (x is the first `tokens` of `seq` tokens of every sequence), the types of
# x, weights (w) and residual (r, "" = none), p, whether the backward pass runs, whether the sum is returned too
# ------------------------------------------------------------------------------------------------------------------

def _case(name, op, batch, tokens, d, x, w="", r="", norm="", p=0.0, train=True, seq=0, keep_sum=False):
    c = {"op": op, "batch": batch, "tokens": tokens, "seq": max(seq, tokens), "d": d, "x": x, "w": w, "r": r, "norm": norm,
         "p": p, "train": train, "sum": keep_sum}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token of the width-1024 model: latency alone
        _case("layer norm, one token", "layer_norm", 1, 1, 1024, "bf16", "bf16", train=False),
        # latent codes of the default width 77, 1023 x 5 of them, in fp32: odd rows of odd length
        _case("layer norm, latents of 77", "layer_norm", 1023, 5, 77, "f32", "f32"),
        # the decoded latents of a global batch of 8192 x 30 tokens of width 1024
        _case("layer norm, 8192 x 30 x 1024", "layer_norm", 8192, 30, 1024, "bf16", "bf16"),
        # a generation step of a batch of 8 at width 512
        _case("rms norm, 8 tokens", "rms_norm", 8, 1, 512, "f32", "f32", train=False),
        # a wide, odd feature axis in fp16 with fp32 weights (mixed precision), few rows
        _case("rms norm, rows of 16001", "rms_norm", 61, 13, 16001, "f16", "f32"),
        # the first 60 tokens of longer hidden states, mixed precision
        _case("rms norm, 1024 x 60 of 237 x 768", "rms_norm", 1024, 60, 768, "bf16", "f32", seq=237),
        # the smallest training batch: 8 x 5 latent tokens of width 512
        _case("dropout, 8 x 5 x 512", "dropout", 8, 5, 512, "f32", p=0.1),
        # latents of width 77 added to a residual of the same kind, 1023 x 30
        _case("dropout + residual, rows of 77", "dropout", 1023, 30, 77, "f16", r="f16", p=0.25),
        # the decoded latents of a global batch of 8192 x 30
        _case("dropout, 8192 x 30 x 1024", "dropout", 8192, 30, 1024, "bf16", p=0.1),
        # a post-norm sub-layer at a batch of 70 x 5 tokens
        _case("post-norm sub-layer, 70 x 5 x 768", "dropout_add_norm", 70, 5, 768, "f32", "f32", "f32", "layer", p=0.1),
        # a post-norm sub-layer over the hidden states of 1024 sequences of 237 tokens
        _case("post-norm sub-layer, 1024 x 237 x 768", "dropout_add_norm", 1024, 237, 768, "bf16", "bf16", "bf16", "layer", p=0.1),
        # a pre-norm sub-layer with the residual stream in fp32, mixed precision
        _case("pre-norm sub-layer, 512 x 60 x 1024", "dropout_add_norm", 512, 60, 1024, "bf16", "f32", "f32", "rms", p=0.1, keep_sum=True),
    ]


def draw(rng):
    op = rng.choice(["layer_norm", "rms_norm", "dropout", "dropout_add_norm"])
    x = rng.choice(["f32", "bf16", "bf16", "f16"])
    near = rng.choice([x, "f32"])                        # a narrow type throughout, or fp32 weights and residual beside it
    train = rng.random() < 0.75
    d = int(round(2.0 ** rng.uniform(3.0, 14.3)))
    if rng.random() < 0.6:
        d = max(8, d // 64 * 64 if d >= 64 else d // 8 * 8)
    most = 1 << 26                                       # elements: a quarter of the largest listed case's
    rows = int(round(2.0 ** rng.uniform(0.0, min(18.0, 26.0 - max(3.0, d.bit_length())))))
    tokens = rng.choice([1, 5, 30, 60, 237])
    tokens = min(tokens, rows)
    batch = max(1, min(rows // tokens, most // (tokens * d)))
    seq = tokens + rng.choice([0, 0, 1, 37])
    norm = rng.choice(["layer", "rms"])
    p = rng.choice([0.05, 0.1, 0.1, 0.25, 0.5])
    if op in ("layer_norm", "rms_norm"):
        return _case("", op, batch, tokens, d, x, near, seq=seq, train=train)
    if op == "dropout":
        return _case("", op, batch, tokens, d, x, r=rng.choice(["", near]), p=p, train=train, seq=seq)
    return _case("", op, batch, tokens, d, x, near, near, norm, p=p if train else 0.0, train=train, seq=seq, keep_sum=rng.random() < 0.5)


def work(case):
    e = case["batch"] * case["tokens"] * case["d"]
    bx, br = BYTES[case["x"]], BYTES.get(case["r"], 0)
    bw = BYTES.get(case["w"], 0) * case["d"]
    biased = case["op"] == "layer_norm" or case["norm"] == "layer"
    out = br if case["op"] == "dropout" and br else bx
    total = e * (bx + br + out) + bw * (2 if biased else 1)             # x, residual, weights -> result
    if case["sum"]:
        total += e * br
    if case["train"]:
        total += e * (out + bx + br) + bw * (2 if biased else 1)        # its gradient -> gradients of x, residual, weights
        if case["sum"]:
            total += e * br
    per = {"layer_norm": 8, "rms_norm": 5, "dropout": 2, "dropout_add_norm": 10}[case["op"]]
    return {"bytes": total, "flops": e * per * (3 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(seed)
    b, n, s, d = case["batch"], case["tokens"], case["seq"], case["d"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    def leaf(t, kind):
        return t.to(TYPES[kind]).requires_grad_(case["train"])

    out = case["r"] if case["op"] == "dropout" and case["r"] else case["x"]
    st = {"case": case, "x": None, "r": None, "w": None, "b": None, "dy": None, "ds": None, "rng": None}
    # hidden states: unit spread around feature offsets, which is what a trained layer hands on
    st["x"] = (normal(b, s, d) + 0.5 * normal(d)).to(TYPES[case["x"]])[:, :n].detach().requires_grad_(case["train"])
    if case["r"]:
        st["r"] = leaf(2.0 * normal(b, n, d), case["r"])
    if case["w"]:
        st["w"] = leaf(1.0 + 0.2 * normal(d), case["w"])
        if case["op"] == "layer_norm" or case["norm"] == "layer":
            st["b"] = leaf(0.2 * normal(d), case["w"])
    if case["train"]:
        st["dy"] = normal(b, n, d).to(TYPES[out])
        if case["sum"]:
            st["ds"] = normal(b, n, d).to(TYPES[case["r"]])
    st["rng"] = torch.randint(0, 1 << 62, (2,), generator=gen, device=dev)
    return st


EPS = {"layer_norm": 1e-9, "layer": 1e-9, "rms_norm": 1e-6, "rms": 1e-6}


# ------------------------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------------------------

def _philox_round(state, k):
    c0, c1, c2, c3, k0, k1 = state
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57              # exact modulo 2^64, which holds all of a 32 x 32 bit product
    return ((b >> 32 & MASK32) ^ c1 ^ k0, b & MASK32, (a >> 32 & MASK32) ^ c3 ^ k1, a & MASK32,
            (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32)


def _keep(rng, rows, d, threshold):
    groups = (d + 7) // 8
    dev = rng.device
    g = torch.arange(groups, device=dev).repeat(rows, 1)
    r = torch.arange(rows, device=dev)[:, None].expand(rows, groups)
    seed, offset = rng[0], rng[1]
    first = (g, r, offset & MASK32, offset >> 32 & MASK32, seed & MASK32, seed >> 32 & MASK32)
    words = torch.stack(reduce(_philox_round, range(10), first)[:4], dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1)
    return halves.reshape(rows, groups * 8)[:, :d] >= threshold


def _plain(st):
    case = st["case"]
    x = st["x"].detach()
    shape, d = x.shape, x.shape[-1]
    rows = x.numel() // d
    v = x.float()
    keep = None
    if case["p"] > 0:
        t = round(65536 * case["p"])
        scale = 65536.0 / (65536 - t)
        keep = _keep(st["rng"], rows, d, t).view(shape)
        v = torch.where(keep, v * scale, 0.0)
    if case["r"]:
        v = v + st["r"].detach().float()
    norm = case["norm"] or case["op"]
    res, out = {}, TYPES[case["r"] if case["op"] == "dropout" and case["r"] else case["x"]]
    if case["op"] == "dropout":
        res["y"] = v.to(out)
        if case["train"]:
            dv = st["dy"].float()
    else:
        w = st["w"].detach().float()
        c = v - v.mean(-1, keepdim=True) if norm.startswith("layer") else v
        rs = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS[norm])
        xh = c * rs
        y = xh * w
        res["y"] = (y if st["b"] is None else y + st["b"].detach().float()).to(out)
        if case["train"]:
            dy = st["dy"].float()
            gw = dy * w
            dv = gw - xh * (gw * xh).mean(-1, keepdim=True)
            if norm.startswith("layer"):
                dv = dv - gw.mean(-1, keepdim=True)
            dv = dv * rs
            if case["sum"]:
                dv = dv + st["ds"].float()
            res["dw"] = (dy * xh).sum((0, 1)).to(st["w"].dtype)
            if st["b"] is not None:
                res["db"] = dy.sum((0, 1)).to(st["b"].dtype)
    if case["sum"]:
        res["s"] = v.to(TYPES[case["r"]])
    if case["train"]:
        res["dx"] = (dv if keep is None else torch.where(keep, dv * scale, 0.0)).to(x.dtype)
        if case["r"]:
            res["dr"] = dv.to(TYPES[case["r"]])
    return res


# ------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------

def _own(st):
    from transformer_vae_amd import functional as F
    case, x, r, w, b = st["case"], st["x"], st["r"], st["w"], st["b"]
    op, s = case["op"], None
    if op == "layer_norm":
        y = F.layer_norm(x, w, b, EPS["layer"])
    elif op == "rms_norm":
        y = F.rms_norm(x, w, EPS["rms"])
    elif op == "dropout":
        y = F.dropout(x, case["p"], st["rng"]) if r is None else F.dropout_add(x, r, case["p"], st["rng"])
    elif case["norm"] == "layer":
        y = F.dropout_add_layer_norm(x, r, w, b, EPS["layer"], case["p"], st["rng"], return_sum=case["sum"])
    else:
        y = F.dropout_add_rms_norm(x, r, w, EPS["rms"], case["p"], st["rng"], return_sum=case["sum"])
    if case["sum"]:
        y, s = y
    res = {"y": y}
    if s is not None:
        res["s"] = s
    if case["train"]:
        leaves = {k: t for k, t in (("dx", x), ("dr", r), ("dw", w), ("db", b)) if t is not None}
        outs, cots = ([y], [st["dy"]]) if s is None else ([y, s], [st["dy"], st["ds"]])
        res.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), cots)))
    return res


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------------
# 64-bit values: the definition differentiated by autograd in float64, a block of rows at a time; the keep decisions from
# products of 16-bit halves, so that nothing here relies on wrapping
# ------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    d = case["d"]
    flat = {k: None if st[k] is None else st[k].detach().reshape(-1, d) for k in ("x", "r", "dy", "ds")}
    rows, dev = flat["x"].shape[0], flat["x"].device
    norm = case["norm"] or case["op"]
    t = round(65536 * case["p"])
    seed64, off64 = (int(v) for v in st["rng"].tolist())

    def times(word, m):
        """(high, low) 32 bits of word * m."""
        w0, w1, m0, m1 = word % 65536, word // 65536, m % 65536, m // 65536
        mid = w0 * m0 // 65536 + w1 * m0 % 65536 + w0 * m1 % 65536
        return w1 * m1 + w1 * m0 // 65536 + w0 * m1 // 65536 + mid // 65536, mid % 65536 * 65536 + w0 * m0 % 65536

    def kept(first, count):
        zero = torch.zeros((count, -(-d // 8)), dtype=torch.int64, device=dev)
        ctr = [zero + torch.arange(zero.shape[1], device=dev), zero + torch.arange(first, first + count, device=dev).unsqueeze(1),
               zero + off64 % 2 ** 32, zero + off64 // 2 ** 32]
        for i in range(10):
            (ah, al), (bh, bl) = times(ctr[0], 0xD2511F53), times(ctr[2], 0xCD9E8D57)
            k0, k1 = (seed64 + i * 0x9E3779B9) % 2 ** 32, (seed64 // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32
            ctr = [bh ^ ctr[1] ^ k0, bl, ah ^ ctr[3] ^ k1, al]
        draws = [part for word in ctr for part in (word % 65536, word // 65536)]
        return torch.stack(draws, 2).flatten(1)[:, :d] >= t

    parts = {}
    sums = {}
    step = max(1, (1 << 24) // d)
    for r0 in range(0, rows, step):
        sl = slice(r0, min(rows, r0 + step))
        leaves = {"dx": flat["x"][sl].double()}
        if case["r"]:
            leaves["dr"] = flat["r"][sl].double()
        if case["w"]:
            leaves["dw"] = st["w"].detach().double()
            if st["b"] is not None:
                leaves["db"] = st["b"].detach().double()
        leaves = {k: v.clone().requires_grad_(case["train"]) for k, v in leaves.items()}
        v = leaves["dx"]
        if case["p"] > 0:
            v = torch.where(kept(r0, sl.stop - r0), v, torch.zeros_like(v)) * (65536 / (65536 - t))
        if case["r"]:
            v = v + leaves["dr"]
        y = v
        if case["op"] != "dropout":
            if norm.startswith("layer"):
                y = (v - v.mean(1, True)) / (v.var(1, unbiased=False, keepdim=True) + EPS[norm]).sqrt()
            else:
                y = v / ((v ** 2).mean(1, True) + EPS[norm]).sqrt()
            y = y * leaves["dw"]
            if "db" in leaves:
                y = y + leaves["db"]
        got = {"y": y.detach()}
        if case["sum"]:
            got["s"] = v.detach()
        if case["train"]:
            loss = (y * flat["dy"][sl].double()).sum()
            if case["sum"]:
                loss = loss + (v * flat["ds"][sl].double()).sum()
            for k, g in zip(leaves, torch.autograd.grad(loss, list(leaves.values()))):
                if k in ("dw", "db"):
                    sums[k] = sums.get(k, 0) + g
                else:
                    got[k] = g
        for k, v in got.items():
            parts.setdefault(k, []).append(v)
    shape = (case["batch"], case["tokens"], d)
    return {**{k: torch.cat(v).view(shape) for k, v in parts.items()}, **sums}
