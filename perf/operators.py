"""The operators around a training step's products, as cases to measure and check.

Four operators, all on f32 tensors in device memory:

  linear          c = r + dropout(act(a b + bias)): the product with its epilogue, z = a b + bias kept on request
  linear_grad     its backward: da, db and dbias from dc and the kept z
  dropout         y = r + dropout(x), the mask a function of (seed, offset, row, column)
  linear_loss     softmax cross-entropy of x w^T over a vocabulary, without the logits, with dx and dw on request

Where `own` is false `run` computes them by elementary torch operations in 32 bits; where it is true it calls
this repository's library. `exact` computes them in 64 bits, apart from both.

Dropout draws from Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): the word
of row i, column j of an n-column tensor is word j % 4 of the block with counter
(i * ceil(n / 4) + j // 4, offset), key seed; it is dropped where the word is below p * 2^32.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ACTIVATIONS = ("none", "relu", "gelu", "silu")
MOST_FLOPS = 6 * 8192 * 32000 * 2048  # the largest listed case


def linear(m, k, n, act="none", bias=True, p=0.0, res=False, keep=False, b_t=False, pad=0):
    return {"op": "linear", "m": m, "k": k, "n": n, "act": act, "bias": bias, "p": p, "res": res, "keep": keep, "b_t": b_t, "pad": pad}


def linear_grad(m, k, n, act="none", bias=True, p=0.0, b_t=False, pad=0):
    return {"op": "linear_grad", "m": m, "k": k, "n": n, "act": act, "bias": bias, "p": p, "b_t": b_t, "pad": pad}


def dropout(m, n, p, res=False, pad=0):
    return {"op": "dropout", "m": m, "n": n, "p": p, "res": res, "pad": pad}


def linear_loss(m, v, d, grad=True, tied=True, ignored=False, pad=0):
    return {"op": "linear_loss", "m": m, "v": v, "d": d, "grad": grad, "tied": tied, "ignored": ignored, "pad": pad}


def listed():
    return [
        # one token through the large preset's up projection: latency and the reading of the weights
        {"name": "linear one token", **linear(1, 2048, 5632, act="silu")},
        # a short ragged batch, odd widths, every part of the epilogue, weights stored [out, in]
        {"name": "linear odd", **linear(37, 501, 1003, act="gelu", p=0.1, res=True, keep=True, b_t=True, pad=4)},
        # training forward of a mid-size decoder's up projection, z kept for the backward
        {"name": "linear up", **linear(8192, 1024, 2816, act="gelu", keep=True)},
        # the large preset's down projection into the residual stream, with dropout
        {"name": "linear down", **linear(8192, 5632, 2048, p=0.1, res=True)},
        # backward of the tiny preset's up projection, batch 8 x 256
        {"name": "linear grad tiny", **linear_grad(2048, 128, 344, act="gelu", p=0.1)},
        # backward of the large preset's up projection, batch 4 x 2048
        {"name": "linear grad large", **linear_grad(8192, 2048, 5632, act="silu")},
        # dropout of the tiny preset's activations: latency
        {"name": "dropout tiny", **dropout(2048, 128, 0.1)},
        # dropout of the large preset's residual branch, added to the stream
        {"name": "dropout large", **dropout(8192, 2048, 0.1, res=True)},
        # the tiny preset's tied head and loss with gradients, batch 8 x 256
        {"name": "loss tiny", **linear_loss(2048, 4096, 128)},
        # a few sequences of odd length, an odd vocabulary, an untied head stored [in, out], padded rows without a target
        {"name": "loss odd", **linear_loss(333, 50001, 516, tied=False, ignored=True, pad=4)},
        # evaluation of a mid-size decoder: the loss alone
        {"name": "loss eval", **linear_loss(8192, 32768, 1024, grad=False)},
        # the large preset's tied head and loss with gradients, batch 4 x 2048
        {"name": "loss large", **linear_loss(8192, 32000, 2048)},
    ]


def spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm; often odd."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("linear", "linear_grad", "dropout", "linear_loss"))
    pad = rng.choice((0, 0, 4, 12))
    if op == "dropout":
        return dropout(spread(rng, 1, 16384), spread(rng, 1, 8192), rng.choice((0.05, 0.1, 0.25, 0.5)), res=rng.random() < 0.5, pad=pad)
    while True:
        if op == "linear_loss":
            c = linear_loss(spread(rng, 1, 16384), spread(rng, 100, 131072), spread(rng, 32, 4096), grad=rng.random() < 0.7,
                            tied=rng.random() < 0.5, ignored=rng.random() < 0.5, pad=pad)
        else:
            m, k, n = spread(rng, 1, 16384), spread(rng, 8, 8192), spread(rng, 8, 8192)
            act, p, b_t = rng.choice(ACTIVATIONS), rng.choice((0.0, 0.0, 0.1, 0.5)), rng.random() < 0.5
            c = linear_grad(m, k, n, act, rng.random() < 0.7, p, b_t, pad)
            if op == "linear":
                c = linear(m, k, n, act, rng.random() < 0.7, p, rng.random() < 0.5, rng.random() < 0.5, b_t, pad)
        if work(c)["flops"] <= MOST_FLOPS and work(c)["bytes"] <= 4 << 30:
            return c


def work(c):
    m = c["m"]
    if c["op"] == "dropout":
        return {"bytes": 4 * m * c["n"] * (3 if c["res"] else 2), "flops": 2 * m * c["n"]}
    if c["op"] == "linear":
        k, n = c["k"], c["n"]
        outs = 1 + (1 if c["res"] else 0) + (1 if c["keep"] else 0)
        return {"bytes": 4 * (m * k + k * n + (n if c["bias"] else 0) + outs * m * n), "flops": 2 * m * n * k}
    if c["op"] == "linear_grad":
        k, n = c["k"], c["n"]
        ins = 1 + (1 if c["act"] != "none" else 0)
        return {"bytes": 4 * (2 * m * k + 2 * k * n + (n if c["bias"] else 0) + ins * m * n), "flops": 4 * m * n * k}
    v, d = c["v"], c["d"]
    both = 2 if c["grad"] else 1
    return {"bytes": 4 * (both * (m * d + v * d) + 2 * m), "flops": (6 if c["grad"] else 2) * m * v * d}


def wide(n, pad):
    """A row stride for n columns: a multiple of 4, with `pad` columns nobody reads or writes."""
    return (n + 3) // 4 * 4 + pad


def matrix(g, m, n, pad, scale=1.0):
    """[m, n] normal values in rows of a wider buffer, whose other columns hold NaN: they must not be used."""
    x = torch.full((m, wide(n, pad)), float("nan"), device="cuda")
    x[:, :n] = torch.randn(m, n, device="cuda", generator=g) * scale
    return x[:, :n]


def blank(m, n, pad):
    return torch.empty(m, wide(n, pad), device="cuda")[:, :n]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, pad = c["m"], c["pad"]
    s = {"case": c}
    if c["op"] != "linear_loss":
        # the generator's two words, {seed, offset}, on the device; the offset goes past 32 bits, as a long run's does
        s["rng"] = torch.tensor([seed * 2654435761 % (1 << 62), (seed % 1000) * 6700417 + (1 << 33)], dtype=torch.int64, device="cuda")
    if c["op"] == "dropout":
        n = c["n"]
        s["x"], s["r"], s["y"] = matrix(g, m, n, pad), matrix(g, m, n, pad) if c["res"] else None, blank(m, n, pad)
        return s
    if c["op"] in ("linear", "linear_grad"):
        k, n, b_t = c["k"], c["n"], c["b_t"]
        s["a"] = matrix(g, m, k, pad)  # a normalised activation
        s["b"] = matrix(g, n if b_t else k, k if b_t else n, pad, 1.0 / math.sqrt(k))
        s["bias"] = torch.randn(n, device="cuda", generator=g) * 0.1 if c["bias"] else None
        if c["op"] == "linear":
            s["r"] = matrix(g, m, n, pad) if c["res"] else None
            s["c"], s["z"] = blank(m, n, pad), blank(m, n, pad) if c["keep"] else None
        else:
            s["z"] = matrix(g, m, n, pad) if c["act"] != "none" else None
            s["dc"] = matrix(g, m, n, pad, 1e-3)  # a gradient's size
            s["da"], s["db"] = blank(m, k, pad), blank(*s["b"].shape, pad)
            s["dbias"] = torch.empty(n, device="cuda") if c["bias"] else None
        return s
    v, d = c["v"], c["d"]
    w = matrix(g, v, d, pad if c["tied"] else 0, 0.02 * math.sqrt(2048 / d))
    t = torch.randint(0, v, (m,), device="cuda", generator=g, dtype=torch.int32)
    # half of the rows know their target a little, as a model in training does
    x = matrix(g, m, d, pad)
    x += torch.randn(m, 1, device="cuda", generator=g).clamp(min=0) * 6 * torch.nn.functional.normalize(w[t.long()], dim=1)
    if c["ignored"]:  # rows behind a sequence's end: no target, values nobody vouches for
        gone = torch.rand(m, device="cuda", generator=g) < 0.2
        t[gone] = -1
        x[gone] *= 1e4
    s["x"], s["t"] = x, t
    if c["tied"]:
        s["w"] = w
    else:
        s["w"] = torch.full((d, wide(v, pad)), float("nan"), device="cuda")[:, :v]
        s["w"].copy_(w.T)
    s["scale"] = 1.0 / max(1, int((t >= 0).sum()))
    s["loss"], s["mean"] = torch.empty(m, device="cuda"), torch.empty(1, device="cuda")
    s["dx"] = blank(m, d, pad) if c["grad"] else None
    s["dw"] = blank(*s["w"].shape, pad) if c["grad"] else None
    return s


def library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "midman-ai_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import midman_b200
    return midman_b200


def stride(t):
    return 0 if t is None else t.stride(0)


def run_own(s):
    mm, c = library(), s["case"]
    m = c["m"]
    if c["op"] == "dropout":
        mm.dropout(s["x"], s["y"], rows=m, cols=c["n"], ldx=stride(s["x"]), ldy=stride(s["y"]), p=c["p"], rng=s["rng"], r=s["r"], ldr=stride(s["r"]))
        return {"y": s["y"]}
    if c["op"] == "linear":
        mm.linear_forward(s["a"], s["b"], s["c"], m=m, n=c["n"], k=c["k"], lda=stride(s["a"]), ldb=stride(s["b"]), ldc=stride(s["c"]),
                          b_mn_major=not c["b_t"], bias=s["bias"], activation=ACTIVATIONS.index(c["act"]), p=c["p"], rng=s["rng"],
                          r=s["r"], ldr=stride(s["r"]), z=s["z"], ldz=stride(s["z"]), precision=1)
        return {"c": s["c"], "z": s["z"]} if c["keep"] else {"c": s["c"]}
    if c["op"] == "linear_grad":
        mm.linear_backward(s["a"], s["b"], s["dc"], m=m, n=c["n"], k=c["k"], lda=stride(s["a"]), ldb=stride(s["b"]), lddc=stride(s["dc"]),
                           b_mn_major=not c["b_t"], activation=ACTIVATIONS.index(c["act"]), p=c["p"], rng=s["rng"], z=s["z"], ldz=stride(s["z"]),
                           da=s["da"], ldda=stride(s["da"]), db=s["db"], lddb=stride(s["db"]), dbias=s["dbias"], precision=1)
        return {"da": s["da"], "db": s["db"], **({"dbias": s["dbias"]} if c["bias"] else {})}
    mm.linear_cross_entropy(s["x"], s["w"], s["t"], s["loss"], rows=m, vocab=c["v"], dim=c["d"], ldx=stride(s["x"]), ldw=stride(s["w"]),
                            w_mn_major=not c["tied"], grad_scale=s["scale"], mean_loss=s["mean"], dx=s["dx"], lddx=stride(s["dx"]),
                            dw=s["dw"], lddw=stride(s["dw"]), precision=1)
    return {"loss": s["loss"], "mean": s["mean"], **({"dx": s["dx"], "dw": s["dw"]} if c["grad"] else {})}


LOW = 0xFFFFFFFF


def kept(rng, m, n, p):
    """The kept places of an [m, n] tensor, Philox4x32-10 in 64-bit whole numbers."""
    blocks = (n + 3) // 4
    at = torch.arange(m * blocks, device="cuda")
    c0, c1 = at & LOW, at >> 32
    c2, c3 = (rng[1] & LOW).expand_as(at), ((rng[1] >> 32) & LOW).expand_as(at)
    k0, k1 = rng[0] & LOW, (rng[0] >> 32) & LOW
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & LOW) ^ c1 ^ k0, p1 & LOW, ((p0 >> 32) & LOW) ^ c3 ^ k1, p0 & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack((c0, c1, c2, c3), 1).view(m, blocks * 4)[:, :n]
    return words >= int(p * 4294967296.0)


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z / (1 + torch.exp(-z)) if name == "silu" else z


def act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def run_plain(s):
    c = s["case"]
    m = c["m"]
    if c["op"] == "dropout":
        y = torch.where(kept(s["rng"], m, c["n"], c["p"]), s["x"] * (1 / (1 - c["p"])), 0.0)
        return {"y": y + s["r"] if c["res"] else y}
    if c["op"] == "linear":
        z = s["a"] @ (s["b"].T if c["b_t"] else s["b"])
        z = z + s["bias"] if c["bias"] else z
        y = act(z, c["act"])
        y = torch.where(kept(s["rng"], m, c["n"], c["p"]), y * (1 / (1 - c["p"])), 0.0) if c["p"] else y
        y = y + s["r"] if c["res"] else y
        return {"c": y, "z": z} if c["keep"] else {"c": y}
    if c["op"] == "linear_grad":
        dz = s["dc"]
        dz = torch.where(kept(s["rng"], m, c["n"], c["p"]), dz * (1 / (1 - c["p"])), 0.0) if c["p"] else dz
        dz = dz * act_slope(s["z"], c["act"]) if c["act"] != "none" else dz
        da = dz @ (s["b"] if c["b_t"] else s["b"].T)
        db = dz.T @ s["a"] if c["b_t"] else s["a"].T @ dz
        return {"da": da, "db": db, **({"dbias": dz.sum(0)} if c["bias"] else {})}
    w = s["w"] if c["tied"] else s["w"].T
    t, live = s["t"].long().clamp(min=0), s["t"] >= 0
    z = s["x"] @ w.T
    top = z.max(1, keepdim=True).values
    zt = z.gather(1, t[:, None])
    e = (z - top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(live, (top + total.log() - zt)[:, 0], 0.0)
    mean = (loss.double().sum() / live.sum().clamp(min=1)).float().view(1)
    if not c["grad"]:
        return {"loss": loss, "mean": mean}
    e *= live[:, None] * s["scale"] / total
    e[torch.arange(m, device="cuda"), t] -= live * s["scale"]
    dx = e @ w
    dw = e.T @ s["x"] if c["tied"] else s["x"].T @ e
    return {"loss": loss, "mean": mean, "dx": dx, "dw": dw}


def run(state):
    return run_own(state) if own else run_plain(state)


def philox_kept(seed, offset, m, n, p):
    """The kept places once more, in numpy's unsigned numbers."""
    blocks, low, u = -(-n // 4), np.uint64(LOW), np.uint64
    at = np.arange(m * blocks, dtype=np.uint64)
    ctr = [at & low, at >> u(32), np.full_like(at, offset & LOW), np.full_like(at, offset >> 32)]
    key = [seed & LOW, seed >> 32]
    for r in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        key_r = [u((key[0] + r * 0x9E3779B9) & LOW), u((key[1] + r * 0xBB67AE85) & LOW)]
        ctr = [(b >> u(32)) ^ ctr[1] ^ key_r[0], b & low, (a >> u(32)) ^ ctr[3] ^ key_r[1], a & low]
    out = np.empty((m * blocks, 4), np.uint64)
    for w in range(4):
        out[:, w] = ctr[w]
    return torch.from_numpy(out.reshape(m, blocks * 4)[:, :n] >= u(int(p * 2.0 ** 32))).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    m, f = c["m"], torch.float64
    mask = None
    if c["op"] != "linear_loss" and c["p"]:
        words = s["rng"].tolist()
        mask = philox_kept(words[0], words[1], m, c["n"], c["p"]).to(f) / (1 - c["p"])
    if c["op"] == "dropout":
        return {"y": s["x"].to(f) * mask + (s["r"].to(f) if c["res"] else 0)}
    gelu_half = lambda z: 0.5 * torch.special.erfc(-z / math.sqrt(2))  # noqa: E731: the normal distribution function
    if c["op"] == "linear":
        z = torch.einsum("mk,nk->mn" if c["b_t"] else "mk,kn->mn", s["a"].to(f), s["b"].to(f))
        if c["bias"]:
            z += s["bias"].to(f)
        y = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)), "gelu": lambda: z * gelu_half(z),
             "silu": lambda: z * torch.sigmoid(z)}[c["act"]]()
        y = y * mask if mask is not None else y
        y = y + s["r"].to(f) if c["res"] else y
        return {"c": y, "z": z} if c["keep"] else {"c": y}
    if c["op"] == "linear_grad":
        dz = s["dc"].to(f)
        dz = dz * mask if mask is not None else dz
        if c["act"] != "none":
            z = s["z"].to(f)
            dz = dz * {"relu": lambda: (z > 0).to(f), "gelu": lambda: gelu_half(z) + z * (-z.square() / 2).exp() / math.sqrt(2 * math.pi),
                       "silu": lambda: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)}[c["act"]]()
        a, b = s["a"].to(f), s["b"].to(f)
        da = torch.einsum("mn,nk->mk" if c["b_t"] else "mn,kn->mk", dz, b)
        db = torch.einsum("mn,mk->nk" if c["b_t"] else "mn,mk->kn", dz, a)
        return {"da": da, "db": db, **({"dbias": dz.sum(0)} if c["bias"] else {})}
    x, w = s["x"].to(f), s["w"].to(f)
    w = w if c["tied"] else w.T
    live = s["t"] >= 0
    loss, dx, dw = torch.zeros(m, dtype=f, device="cuda"), torch.zeros_like(x), torch.zeros(w.shape, dtype=f, device="cuda")
    rows = max(1, (1 << 28) // w.shape[0])  # blocks of rows whose logits fit 2 GiB
    for i in range(0, m, rows):
        xi, ti, li = x[i:i + rows], s["t"][i:i + rows].long(), live[i:i + rows]
        z = xi @ w.T
        lse = torch.logsumexp(z, 1)
        hot = torch.nn.functional.pad(ti, (0, 0)).clamp(min=0)[:, None]
        loss[i:i + rows] = torch.where(li, lse - z.gather(1, hot)[:, 0], 0.0)
        if c["grad"]:
            q = (z - lse[:, None]).exp().scatter_add_(1, hot, torch.full(hot.shape, -1.0, dtype=f, device="cuda"))
            q *= (li.to(f) * s["scale"])[:, None]
            dx[i:i + rows] = q @ w
            dw += q.T @ xi
    out = {"loss": loss, "mean": (loss.sum() / live.sum().clamp(min=1)).view(1)}
    return {**out, "dx": dx, "dw": dw if c["tied"] else dw.T} if c["grad"] else out
