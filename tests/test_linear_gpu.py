"""mm_gpu_linear_*, mm_gpu_dropout and mm_gpu_linear_cross_entropy against plain implementations in 64 bits.

Tolerances, element by element, before any run. A product's error is bounded by a share of S = |A| |B| (the sum of the
absolute products):
  exact mode   hi is x with 13 mantissa bits cut, so |lo| < 2^-10 |x|; lo is rounded to 11 bits (2^-11 of it): 2^-21 a
               factor, 2^-20 for two; the product of the lo parts is left out: 2^-20. Sums of 64 of K are truncated by the
               tensor core, 24 times at 2^-23, and added in f32, K / 64 times at 2^-24.
               => (2^-19 + 24 * 2^-23 + (K / 64 + 8) 2^-24) S  <=  (5.2e-6 + K * 1e-9) S
  one TF32 pass  both factors cut to 11 bits: 2 * 2^-10, sums as above over 1024 of K: (2^-9 + 2^-9) S at most
               (128 UMMAs at 2^-23 are far below it).
An activation passes an error on with its slope (at most 1.13) and adds its own: a few ulp of |z| + 1. Dropout multiplies by
1 / (1 - p), rounded (2^-24) twice.
"""
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

from philox import kept

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "silu"]
ULP = 2.0 ** -24
F = torch.float64


def product_tol(precision, s, k):
    return s * ((5.2e-6 + k * 1e-9) if precision == 1 else 2.0 ** -8) + 1e-37


def rng_words(seed, offset):
    return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    return z * torch.sigmoid(z) if name == "silu" else z


def slope64(z, name):
    if name == "relu":
        return (z > 0).to(F)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5
    if name == "silu":
        return torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))
    return torch.ones_like(z)


def padded(g, m, n, extra, scale=1.0):
    """[m, n] normal values in rows of a wider buffer that holds NaN elsewhere."""
    x = torch.full((m, (n + 3) // 4 * 4 + extra), float("nan"), device="cuda")
    x[:, :n] = torch.randn(m, n, device="cuda", generator=g) * scale
    return x


def check(got, want, tol, what):
    d = (got.to(F) - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (d / (tol + 1e-300)).max().item()
    assert (d <= tol).all(), f"{what}: {worst:.3g} times the tolerance"


def out_buffer(m, n, extra):
    return torch.full((m, (n + 3) // 4 * 4 + extra), 777.0, device="cuda")


def untouched(buf, n):
    assert (buf[:, n:] == 777.0).all(), "columns past the width were written"


# m, k, n, weights [n, k], activation, bias, p, residual, z kept, extra stride
FORWARD = [
    (1, 8, 8, False, "none", False, 0.0, False, False, 0),
    (1, 1, 1, False, "gelu", True, 0.0, True, True, 0),
    (1, 2048, 352, False, "silu", True, 0.1, True, True, 4),
    (3, 7, 5, True, "relu", True, 0.5, True, True, 4),
    (37, 501, 1003, True, "gelu", True, 0.1, True, True, 8),
    (128, 32, 64, False, "silu", False, 0.0, True, False, 0),
    (129, 33, 65, False, "none", True, 0.25, False, True, 0),
    (200, 1000, 130, True, "none", False, 0.0, True, False, 12),
    (640, 96, 1024, False, "gelu", True, 0.0, False, True, 0),
    (2048, 128, 344, False, "silu", True, 0.1, True, True, 0),
    (1537, 2052, 1031, False, "relu", True, 0.1, True, True, 4),
    (1537, 2052, 1031, True, "gelu", True, 0.1, True, True, 4),
    (2304, 768, 2304, False, "gelu", True, 0.05, True, True, 0),
    (4096, 4099, 513, True, "none", True, 0.0, True, False, 0),
    # few outputs over a long k
    (3, 20001, 41, False, "silu", True, 0.1, True, True, 4),
    (8, 9000, 64, True, "gelu", True, 0.1, True, True, 0),
    (8, 9001, 1000, False, "none", False, 0.0, False, False, 0),
    (37, 8196, 101, False, "gelu", True, 0.1, True, True, 4),
    (130, 16390, 70, True, "none", True, 0.0, True, False, 0),
]


@pytest.mark.parametrize("precision", [1, 0])
@pytest.mark.parametrize("m,k,n,b_t,act,bias,p,res,keep,extra", FORWARD)
def test_forward(mm, m, k, n, b_t, act, bias, p, res, keep, extra, precision):
    g = torch.Generator(device="cuda").manual_seed(m * 7 + k * 3 + n)
    a, b = padded(g, m, k, extra), padded(g, *((n, k) if b_t else (k, n)), extra, k ** -0.5)
    bs = torch.randn(n + 1, device="cuda", generator=g)[1:] if bias else None  # not 16-byte aligned
    r = padded(g, m, n, extra) if res else None
    c, z = out_buffer(m, n, extra), out_buffer(m, n, extra) if keep else None
    seed, offset = 0x123456789ABCDEF0, (5 << 40) + 3
    mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=a.stride(0), ldb=b.stride(0), ldc=c.stride(0), b_mn_major=not b_t, bias=bs,
                      activation=ACTS.index(act), p=p, rng=rng_words(seed, offset) if p else None, r=r,
                      ldr=r.stride(0) if res else 0, z=z, ldz=z.stride(0) if keep else 0, precision=precision)
    mm.device_status()
    A, B = a[:, :k].to(F), (b[:, :k].T if b_t else b[:, :n]).to(F)
    Z, S = A @ B, A.abs() @ B.abs()
    tol = product_tol(precision, S, k) + 2 * ULP * Z.abs()
    if bias:
        Z = Z + bs.to(F)
        tol = tol + 2 * ULP * Z.abs()
    if keep:
        check(z[:, :n], Z, tol, "z")
        untouched(z, n)
    Y = act64(Z, act)
    if act != "none":
        tol = 1.13 * tol + 8 * ULP * (Z.abs() + 1)
    if p:
        mask = torch.from_numpy(kept(seed, offset, m, n, p)).cuda()
        Y, tol = torch.where(mask, Y / (1 - p), 0.0), torch.where(mask, tol / (1 - p) + 4 * ULP * Y.abs() / (1 - p), 0.0)
    if res:
        Y = Y + r[:, :n].to(F)
        tol = tol + 2 * ULP * Y.abs()
    check(c[:, :n], Y, tol + 1e-37, "c")
    untouched(c, n)


def test_the_residual_may_be_the_output(mm):
    g = torch.Generator(device="cuda").manual_seed(1)
    for m, k, n in ((5, 64, 36), (300, 512, 1000), (2304, 256, 2304)):
        a, b, r = padded(g, m, k, 0), padded(g, k, n, 0), padded(g, m, n, 0)
        kw = dict(m=m, n=n, k=k, lda=a.stride(0), ldb=b.stride(0), ldc=r.stride(0), precision=1)
        c = torch.empty_like(r)
        mm.linear_forward(a, b, c, r=r, ldr=r.stride(0), **kw)
        mm.linear_forward(a, b, r, r=r, ldr=r.stride(0), **kw)
        assert torch.equal(c[:, :n], r[:, :n])
    mm.device_status()


BACKWARD = [(1, 8, 8, False, "none", True, 0.0, 0), (1, 1, 1, True, "silu", True, 0.0, 0), (3, 7, 5, True, "relu", True, 0.5, 4),
            (37, 501, 1003, True, "gelu", True, 0.1, 8), (65, 40, 129, False, "silu", True, 0.0, 4),
            (129, 2048, 352, False, "none", True, 0.25, 0), (2048, 128, 344, False, "gelu", True, 0.1, 0),
            (20000, 36, 68, False, "gelu", True, 0.1, 4), (9001, 3, 5, True, "relu", True, 0.1, 0), (20, 40, 12001, False, "silu", True, 0.0, 0),
            (2305, 1031, 1537, False, "gelu", True, 0.1, 4), (2305, 1031, 1537, True, "silu", False, 0.0, 4),
            (4096, 2304, 1536, False, "none", True, 0.0, 0)]


@pytest.mark.parametrize("precision", [1, 0])
@pytest.mark.parametrize("m,k,n,b_t,act,bias,p,extra", BACKWARD)
def test_backward(mm, m, k, n, b_t, act, bias, p, extra, precision):
    g = torch.Generator(device="cuda").manual_seed(m * 5 + k + n)
    a, b = padded(g, m, k, extra), padded(g, *((n, k) if b_t else (k, n)), extra, k ** -0.5)
    z, dc = padded(g, m, n, extra) if act != "none" else None, padded(g, m, n, extra)
    seed, offset = 99, 1 << 33
    da, db = out_buffer(m, k, extra), out_buffer(*((n, k) if b_t else (k, n)), extra)
    dbias = torch.full((n,), 777.0, device="cuda") if bias else None
    kw = dict(m=m, n=n, k=k, lda=a.stride(0), ldb=b.stride(0), lddc=dc.stride(0), b_mn_major=not b_t,
              activation=ACTS.index(act), p=p, rng=rng_words(seed, offset) if p else None, z=z,
              ldz=z.stride(0) if z is not None else 0, precision=precision)
    mm.linear_backward(a, b, dc, da=da, ldda=da.stride(0), db=db, lddb=db.stride(0), dbias=dbias, **kw)
    mm.device_status()
    A, B, D = a[:, :k].to(F), (b[:, :k].T if b_t else b[:, :n]).to(F), dc[:, :n].to(F)
    if p:
        D = D * torch.from_numpy(kept(seed, offset, m, n, p)).cuda() / (1 - p)
    rel = 0.0
    if p or act != "none":
        rel = 16 * ULP  # the slope's and the scale's own rounding, relative to |dc| (slopes reach 1.13)
    dtol = rel * D.abs()
    if act != "none":
        D = D * slope64(z[:, :n].to(F), act)
    da_w, da_s = D @ B.T, D.abs() @ B.abs().T
    check(da[:, :k], da_w, product_tol(precision, da_s, n) + dtol @ B.abs().T + 2 * ULP * da_w.abs(), "da")
    db_w, db_s = A.T @ D, A.abs().T @ D.abs()
    db_tol = product_tol(precision, db_s, m) + A.abs().T @ dtol + 2 * ULP * db_w.abs()
    db_got = (db[:, :k].T if b_t else db[:, :n])
    check(db_got, db_w, db_tol, "db")
    untouched(da, k)
    untouched(db, k if b_t else n)
    if bias:
        check(dbias, D.sum(0), 66 * ULP * D.abs().sum(0) + dtol.sum(0) + 1e-37, "dbias")
    # each output alone is the same, and accumulating adds the same values once more
    da2, db2 = torch.empty_like(da), torch.empty_like(db)
    mm.linear_backward(a, b, dc, da=da2, ldda=da.stride(0), **kw)
    mm.linear_backward(a, b, dc, db=db2, lddb=db.stride(0), **kw)
    assert torch.equal(da2[:, :k], da[:, :k]) and torch.equal(db2[:, :db_got.shape[1 - int(b_t)]], db[:, :k if b_t else n])
    again = [t.clone() if t is not None else None for t in (da, db, dbias)]
    mm.linear_backward(a, b, dc, da=again[0], ldda=da.stride(0), db=again[1], lddb=db.stride(0), dbias=again[2], accumulate=True,
                       **kw)
    mm.device_status()
    for got, once, width in ((again[0], da, k), (again[1], db, k if b_t else n)):
        # one more rounding: of the sum
        check(got[:, :width], 2 * once[:, :width].to(F), 4 * ULP * once[:, :width].to(F).abs() + 1e-37, "accumulated")
    if bias:
        check(again[2], 2 * dbias.to(F), 4 * ULP * dbias.to(F).abs() + 1e-37, "accumulated dbias")


def test_backward_agrees_with_differences(mm):
    """sum(c * u) along a direction of a, b and bias, by central differences in 64 bits of the formula's forward."""
    g = torch.Generator(device="cuda").manual_seed(4)
    m, k, n, p, seed, offset = 9, 12, 20, 0.25, 5, 6
    a, b, bias, u = (torch.randn(*s, device="cuda", generator=g) for s in ((m, k), (k, n), (n,), (m, n)))
    for act in ACTS[1:]:
        z, c = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        da, db, dbias = torch.empty_like(a), torch.empty_like(b), torch.empty_like(bias)
        kw = dict(m=m, n=n, k=k, lda=k, ldb=n, activation=ACTS.index(act), p=p, rng=rng_words(seed, offset), z=z, ldz=n, precision=1)
        mm.linear_forward(a, b, c, ldc=n, bias=bias, **kw)
        mm.linear_backward(a, b, u, lddc=n, da=da, ldda=k, db=db, lddb=n, dbias=dbias, **kw)
        mm.device_status()
        mask = torch.from_numpy(kept(seed, offset, m, n, p)).cuda() / (1 - p)

        def value(a_, b_, bias_):
            return (act64(a_ @ b_ + bias_, act) * mask * u.to(F)).sum()

        va, vb, vc = (torch.randn(t.shape, device="cuda", generator=g).to(F) for t in (a, b, bias))
        A, B, Bi, h = a.to(F), b.to(F), bias.to(F), 1e-6
        want = (value(A + h * va, B + h * vb, Bi + h * vc) - value(A - h * va, B - h * vb, Bi - h * vc)) / (2 * h)
        got = (da.to(F) * va).sum() + (db.to(F) * vb).sum() + (dbias.to(F) * vc).sum()
        # relu: no kink within h of these values; the gradients' own error is 1e-5 of their absolute sums at most
        size = (da.to(F) * va).abs().sum() + (db.to(F) * vb).abs().sum() + (dbias.to(F) * vc).abs().sum()
        assert abs(got - want) <= 1e-5 * size, act


def test_rows_that_are_not_finite_stay_alone(mm):
    """A NaN, an infinity and a very large row of a, as behind a sequence's end, leave the other rows as they are."""
    g = torch.Generator(device="cuda").manual_seed(2)
    for m, k, n in ((40, 96, 72), (2304, 512, 2304)):
        a, b = torch.randn(m, k, device="cuda", generator=g), torch.randn(k, n, device="cuda", generator=g)
        bad = a.clone()
        bad[3], bad[7, 5], bad[m - 1] = float("nan"), float("inf"), 1e30
        c, d = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        kw = dict(m=m, n=n, k=k, lda=k, ldb=n, ldc=n, precision=1)
        mm.linear_forward(a, b, c, **kw)
        mm.linear_forward(bad, b, d, **kw)
        mm.device_status()
        good = [i for i in range(m) if i not in (3, 7, m - 1)]
        assert torch.equal(c[good], d[good])
        assert torch.isnan(d[3]).all() and not torch.isfinite(d[7]).any() and torch.isfinite(d[m - 1]).all()
        want = bad[m - 1].to(F) @ b.to(F)
        check(d[m - 1], want, product_tol(1, bad[m - 1].to(F).abs() @ b.to(F).abs(), k) + 2 * ULP * want.abs(), "large row")


@pytest.mark.parametrize("precision", [1, 0])
@pytest.mark.parametrize("m,k,n", [(2, 64, 40), (40, 96, 72), (2304, 512, 2304)])
def test_activations_keep_a_nan(mm, m, k, n, precision):
    a, b = torch.ones(m, k, device="cuda"), torch.full((k, n), 0.5, device="cuda")
    a[1, 3] = float("nan")
    for act in range(4):
        c, z = (torch.zeros(m, n, device="cuda") for _ in range(2))
        mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=k, ldb=n, ldc=n, activation=act, z=z, ldz=n, precision=precision)
        mm.device_status()
        assert torch.isnan(c[1]).all() and torch.isnan(z[1]).all(), ACTS[act]
        rest = [i for i in range(m) if i != 1]
        assert torch.isfinite(c[rest]).all()


def test_entries_of_very_different_sizes(mm):
    """Rows of a and columns of b over 2^-40 .. 2^40: every element is held to its own row's and column's sizes."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for m, k, n in ((33, 200, 100), (2304, 256, 2304)):
        sa = 2.0 ** torch.randint(-40, 41, (m, 1), device="cuda", generator=g)
        sb = 2.0 ** torch.randint(-40, 41, (1, n), device="cuda", generator=g)
        a = torch.randn(m, k, device="cuda", generator=g) * sa
        b = torch.randn(k, n, device="cuda", generator=g) * sb
        c = torch.empty(m, n, device="cuda")
        mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=k, ldb=n, ldc=n, precision=1)
        mm.device_status()
        want = a.to(F) @ b.to(F)
        check(c, want, product_tol(1, a.to(F).abs() @ b.to(F).abs(), k) + 2 * ULP * want.abs(), "c")


@pytest.mark.parametrize("m,k,n", [(33, 200, 100), (2304, 256, 2304), (2304, 512, 2304)])  # direct, direct, pairs
@pytest.mark.parametrize("large_side", ["a", "b"])
def test_the_largest_entries_give_their_products(mm, m, k, n, large_side):
    """Entries of 2^100 to 2^127 on one side, 2^-100 to 2^-20 on the other: the products are ordinary numbers, and
    f32's order of multiplying a chunk's two scales must not lose them to infinity. A zero meets the largest too."""
    g = torch.Generator(device="cuda").manual_seed(6)
    rows, cols = (m, n) if large_side == "a" else (n, m)
    unit = lambda *s: torch.rand(*s, device="cuda", generator=g) * 0.5 + 0.5  # noqa: E731
    big = unit(rows, k) * 2.0 ** torch.randint(100, 128, (rows, 1), device="cuda", generator=g)
    big *= torch.randint(0, 2, (rows, k), device="cuda", generator=g) * 2 - 1
    small = unit(cols, k) * 2.0 ** torch.randint(-100, -19, (cols, 1), device="cuda", generator=g)
    big[:, 3], small[:, 4] = 0, 0
    a, b = (big, small) if large_side == "a" else (small, big)
    c = torch.empty(m, n, device="cuda")
    mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=k, ldb=k, ldc=n, b_mn_major=False, precision=1)
    mm.device_status()
    want = a.to(F) @ b.to(F).T
    check(c, want, product_tol(1, a.to(F).abs() @ b.to(F).abs().T, k) + 2 * ULP * want.abs(), "c")


@pytest.mark.parametrize("k", [256, 512])  # direct, pairs
@pytest.mark.parametrize("large_side", ["a", "b"])
def test_small_entries_against_large_ones(mm, large_side, k):
    """The other end: rows of 2^-120 to 2^-100, whose inverse scales reach the smallest there are."""
    g = torch.Generator(device="cuda").manual_seed(7)
    m = n = 2304
    big = torch.randn(m, k, device="cuda", generator=g) * 2.0 ** torch.randint(90, 111, (m, 1), device="cuda", generator=g)
    small = torch.randn(n, k, device="cuda", generator=g) * 2.0 ** torch.randint(-120, -99, (n, 1), device="cuda", generator=g)
    a, b = (big, small) if large_side == "a" else (small, big)
    c = torch.empty(m, n, device="cuda")
    mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=k, ldb=k, ldc=n, b_mn_major=False, precision=1)
    mm.device_status()
    want = a.to(F) @ b.to(F).T
    check(c, want, product_tol(1, a.to(F).abs() @ b.to(F).abs().T, k) + 2 * ULP * want.abs(), "c")


@pytest.mark.parametrize("below", [10, 17, 24, 31, 38, 45])
def test_small_entries_beside_a_large_one(mm, below):
    """Entries 2^-below of the largest of their 128 along the sum, which meets a zero: large exact products lose what the
    header says and no more (2^-39 of the largest an entry: lo's last bit is 2^-24 of a scaled unit, half of it 2^-25,
    and the largest is 2^14 at least), smaller ones nothing."""
    g = torch.Generator(device="cuda").manual_seed(below)
    for m, k, n in ((33, 256, 100), (2304, 256, 2304), (2304, 512, 2304)):  # direct, direct, pairs
        a, b = torch.randn(m, k, device="cuda", generator=g).clamp(-2, 2), torch.randn(k, n, device="cuda", generator=g)
        a *= 2.0 ** -below / 2
        a[:, ::128], b[::128] = 1, 0
        c = torch.empty(m, n, device="cuda")
        mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=k, ldb=n, ldc=n, precision=1)
        mm.device_status()
        want = a.to(F) @ b.to(F)
        tol = product_tol(1, a.to(F).abs() @ b.to(F).abs(), k) + 2 * ULP * want.abs()
        if k == 512:
            tol = tol + 2.0 ** -39 * b.to(F).abs().sum(0)
            assert below < 45 or (c == 0).all()
        check(c, want, tol, "c")


@pytest.mark.parametrize("m,n", [(128, 256), (2304, 2304)])  # direct, pairs
@pytest.mark.parametrize("b_t", [False, True])
def test_long_sums_of_one_sign_in_one_tf32_pass(mm, m, n, b_t):
    """Operands of 11 bits, so nothing of them is cut: what is left is the sums' error. An accumulation is 2048 of K at most,
    256 UMMAs that each cut less than 2^-23 of the sum so far: 2^-15. The accumulations are added in f32, at most K / 1024
    roundings of 2^-24, and up to 64 parts of K likewise."""
    k = 32768
    g = torch.Generator(device="cuda").manual_seed(n)
    eleven = lambda *s: ((torch.rand(*s, device="cuda", generator=g) + 1).view(torch.int32) & ~0x1FFF).view(torch.float32)  # noqa: E731
    a, b = eleven(m, k), eleven(*((n, k) if b_t else (k, n)))
    c = torch.empty(m, n, device="cuda")
    mm.linear_forward(a, b, c, m=m, n=n, k=k, lda=k, ldb=b.stride(0), ldc=n, b_mn_major=not b_t, precision=0)
    mm.device_status()
    want = a.to(F) @ (b.T if b_t else b).to(F)
    check(c, want, (2.0 ** -15 + (k / 1024 + 64) * ULP) * want, "c")
    # and a weight's gradient, whose sum is over the rows: a^T [k, m] plays the input, c's place is [k, n]
    db, dc = torch.empty(m, n, device="cuda"), eleven(k, n)
    x = a.T.contiguous()
    mm.linear_backward(x, None, dc, m=k, n=n, k=m, lda=m, ldb=n, lddc=n, db=db, lddb=n, precision=0)
    mm.device_status()
    want = a.to(F) @ dc.to(F)
    check(db, want, (2.0 ** -15 + (k / 1024 + 64) * ULP) * want, "db")


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("rows,cols,ldx,shift", [(1, 1, 1, 0), (3, 5, 5, 1), (7, 8, 12, 0), (100, 1001, 1001, 3), (33, 4096, 4096, 0),
                                                 (5000, 7, 8, 0), (257, 1030, 1032, 0)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5])
@pytest.mark.parametrize("res", [False, True])
def test_dropout(mm, rows, cols, ldx, shift, p, res):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    buf = torch.randn(2, rows * ldx + shift, device="cuda", generator=g)
    x, r = (t[shift:].view(rows, ldx) for t in buf)
    y = torch.full((rows * ldx + shift,), 777.0, device="cuda")[shift:].view(rows, ldx)
    seed, offset = (1 << 62) + 17, (1 << 50) + 1
    words = rng_words(seed, offset) if p else None
    mm.dropout(x, y, rows=rows, cols=cols, ldx=ldx, ldy=ldx, p=p, rng=words, r=r if res else None, ldr=ldx)
    mm.device_status()
    mask = torch.from_numpy(kept(seed, offset, rows, cols, p)).cuda()
    want = torch.where(mask, x[:, :cols].to(F) / (1 - p), 0.0)
    tol = 2 * ULP * want.abs()
    if res:
        want = want + r[:, :cols].to(F)
        tol = tol + ULP * want.abs()
    else:
        assert torch.equal(y[:, :cols] != 0, mask & (x[:, :cols] != 0))
    check(y[:, :cols], want, tol, "y")
    untouched(y, cols)
    # in place, and over r
    for out in (x.clone(), r.clone()):
        src, add = (out, r) if torch.equal(out, x) else (x, out)
        mm.dropout(src, out, rows=rows, cols=cols, ldx=ldx, ldy=ldx, p=p, rng=words, r=add if res else None, ldr=ldx)
        assert torch.equal(out[:, :cols], y[:, :cols])
    mm.device_status()


def test_dropout_drops_what_is_not_finite(mm):
    x = torch.full((64, 64), float("nan"), device="cuda")
    y = torch.empty_like(x)
    mm.dropout(x, y, rows=64, cols=64, ldx=64, ldy=64, p=0.5, rng=rng_words(1, 2))
    assert torch.equal(torch.isnan(y).cpu(), torch.from_numpy(kept(1, 2, 64, 64, 0.5)))


def test_a_captured_dropout_draws_anew(mm):
    x, y, words = torch.ones(33, 100, device="cuda"), torch.empty(33, 100, device="cuda"), rng_words(1, 0)
    kw = dict(rows=33, cols=100, ldx=100, ldy=100, p=0.5, rng=words)
    mm.dropout(x, y, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mm.dropout(x, y, **kw)
        words[1] += 1
    words[1] = 40
    for step in range(3):
        graph.replay()
        assert torch.equal((y != 0).cpu(), torch.from_numpy(kept(1, 40 + step, 33, 100, 0.5)))


# ------------------------------------------------------------------ linear cross-entropy
def loss64(x, w, t, scale, live):
    z = x.to(F) @ w.to(F).T
    lse = torch.logsumexp(z, 1)
    hot = t.long().clamp(0, w.shape[0] - 1)[:, None]
    loss = torch.where(live, lse - z.gather(1, hot)[:, 0], 0.0)
    q = (z - lse[:, None]).exp()
    gr = q.clone().scatter_add_(1, hot, torch.full(hot.shape, -1.0, dtype=F, device="cuda")) * live[:, None] * scale
    return z, lse, loss, q * live[:, None] * scale, gr


def loss_case(g, rows, vocab, dim, tied, extra):
    x = padded(g, rows, dim, extra)
    w = padded(g, *((vocab, dim) if tied else (dim, vocab)), extra, 2.0 * dim ** -0.5)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    return x, w, t


# rows, vocab, dim, tied, extra, rows left out
LOSS = [(1, 1, 4, True, 0, 0), (1, 5, 8, True, 0, 0), (3, 130, 33, False, 4, 1), (64, 1000, 64, True, 4, 5), (129, 4099, 96, False, 0, 0),
        (200, 513, 1030, True, 0, 199), (37, 32003, 260, True, 8, 3), (2049, 512, 128, False, 0, 100), (2304, 2305, 512, True, 0, 0),
        (700, 131072, 40, True, 0, 9), (600, 120001, 36, False, 4, 9), (5, 20001, 40, True, 4, 1), (64, 32000, 64, True, 0, 3), (1100, 131073, 132, True, 4, 9), (777, 65537, 260, False, 0, 9),
        (1100, 131073, 260, True, 4, 9), (900, 131072, 196, False, 0, 0)]


@pytest.mark.parametrize("precision", [1, 0])
@pytest.mark.parametrize("rows,vocab,dim,tied,extra,out", LOSS)
def test_linear_cross_entropy(mm, rows, vocab, dim, tied, extra, out, precision):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab + dim)
    x, w, t = loss_case(g, rows, vocab, dim, tied, extra)
    gone = torch.randperm(rows, device="cuda", generator=g)[:out]
    t[gone] = -1
    X, W = x[:, :dim].clone(), (w[:, :dim] if tied else w[:, :vocab].T)
    x[gone, :dim] = float("nan")  # whatever a row without a target holds
    live = t >= 0
    X[gone] = 0
    scale = 1.0 / max(1, rows - out)
    row_loss, mean = torch.full((rows,), 777.0, device="cuda"), torch.full((1,), 777.0, device="cuda")
    dx, dw = out_buffer(rows, dim, extra), out_buffer(*((vocab, dim) if tied else (dim, vocab)), extra)
    kw = dict(rows=rows, vocab=vocab, dim=dim, ldx=x.stride(0), ldw=w.stride(0), w_mn_major=not tied, grad_scale=scale,
              precision=precision)
    mm.linear_cross_entropy(x, w, t, row_loss, mean_loss=mean, dx=dx, lddx=dx.stride(0), dw=dw, lddw=dw.stride(0), **kw)
    mm.device_status()
    z, lse, loss, q, gr = loss64(X, W, t, scale, live)
    S = X.to(F).abs() @ W.to(F).abs().T
    tz = product_tol(precision, S, dim).max(1).values  # a row's logits' worst error
    # lse moves by tz at most; its sum (vocab terms in f32, pairwise and in 128s: 32 roundings) and log by a few ulp, and an
    # exponential's argument is rounded relative to the logits' range
    spread = z.max(1).values - z.min(1).values
    t_exp = 2 * tz + (64 + 2 * spread) * ULP
    check(row_loss, loss, torch.where(live, t_exp + 4 * ULP * (lse.abs() + z.abs().max(1).values), 0.0), "row_loss")
    m = loss.sum() / max(1, rows - out)
    check(mean, m.view(1), (torch.where(live, t_exp, 0.0).sum() / max(1, rows - out) + 8 * ULP * (lse.abs().max() + 1)).view(1), "mean")
    gtol = q * t_exp[:, None] + 4 * ULP * gr.abs() + 2 * ULP * scale * (q > 0)
    gtol[torch.arange(rows, device="cuda"), t.long().clamp(min=0)] += 2 * ULP * scale
    dxw, dww = gr @ W.to(F), gr.T @ X.to(F)
    check(dx[:, :dim], dxw, product_tol(precision, gr.abs() @ W.to(F).abs(), vocab) + gtol @ W.to(F).abs() + 2 * ULP * dxw.abs(), "dx")
    got = dw[:, :dim] if tied else dw[:, :vocab].T
    dw_tol = product_tol(precision, gr.abs().T @ X.to(F).abs(), rows) + gtol.T @ X.to(F).abs() + 2 * ULP * dww.abs()
    check(got, dww, dw_tol, "dw")
    untouched(dx, dim)
    untouched(dw, dim if tied else vocab)
    assert (dx[gone, :dim] == 0).all() and (row_loss[gone] == 0).all()
    # the loss alone
    alone = torch.full((rows,), 777.0, device="cuda")
    mm.linear_cross_entropy(x, w, t, alone, mean_loss=mean, **kw)
    mm.device_status()
    check(alone, loss, torch.where(live, t_exp + 4 * ULP * (lse.abs() + z.abs().max(1).values), 0.0), "the loss alone")
    # each gradient alone is the same
    bx, bw = torch.empty_like(dx), torch.empty_like(dw)
    mm.linear_cross_entropy(x, w, t, alone, dx=bx, lddx=dx.stride(0), **kw)
    mm.linear_cross_entropy(x, w, t, alone, dw=bw, lddw=dw.stride(0), **kw)
    assert torch.equal(bx[:, :dim], dx[:, :dim]) and torch.equal(bw[:, :dim if tied else vocab], dw[:, :dim if tied else vocab])
    # added to what the gradients hold
    ax, aw = dx.clone(), dw.clone()
    mm.linear_cross_entropy(x, w, t, row_loss, dx=ax, lddx=dx.stride(0), dw=aw, lddw=dw.stride(0), accumulate=True, **kw)
    mm.device_status()
    check(ax[:, :dim], 2 * dxw, 2 * (product_tol(precision, gr.abs() @ W.to(F).abs(), vocab) + gtol @ W.to(F).abs()) + 6 * ULP * dxw.abs(), "dx + dx")
    check(aw[:, :dim] if tied else aw[:, :vocab].T, 2 * dww, 2 * dw_tol + 6 * ULP * dww.abs(), "dw + dw")


def test_loss_gradients_agree_with_differences(mm):
    g = torch.Generator(device="cuda").manual_seed(8)
    rows, vocab, dim = 11, 300, 24
    x, w, t = loss_case(g, rows, vocab, dim, True, 0)
    row_loss, dx, dw = torch.empty(rows, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    mm.linear_cross_entropy(x, w, t, row_loss, rows=rows, vocab=vocab, dim=dim, ldx=dim, ldw=dim, grad_scale=0.5, dx=dx, lddx=dim,
                            dw=dw, lddw=dim, precision=1)
    mm.device_status()
    vx, vw = torch.randn(x.shape, device="cuda", generator=g).to(F), torch.randn(w.shape, device="cuda", generator=g).to(F)
    live, h = t >= 0, 1e-6

    def value(s):
        return 0.5 * loss64(x.to(F) + s * vx, w.to(F) + s * vw, t, 1.0, live)[2].sum()

    want = (value(h) - value(-h)) / (2 * h)
    got = (dx.to(F) * vx).sum() + (dw.to(F) * vw).sum()
    assert abs(got - want) <= 1e-5 * ((dx.to(F) * vx).abs().sum() + (dw.to(F) * vw).abs().sum())


def test_a_target_that_is_no_class(mm):
    g = torch.Generator(device="cuda").manual_seed(9)
    x, w, t = loss_case(g, 6, 40, 16, True, 0)
    t[1], t[4] = 40, -2
    row_loss, dx, dw, mean = torch.empty(6, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty(1, device="cuda")
    kw = dict(rows=6, vocab=40, dim=16, ldx=16, ldw=16, precision=1)
    for grads in (dict(dx=dx, lddx=16, dw=dw, lddw=16), {}):
        mm.linear_cross_entropy(x, w, t, row_loss, mean_loss=mean, **grads, **kw)
        with pytest.raises(mm.MidmanGpuError, match="outside"):
            mm.device_status()
        assert torch.isnan(row_loss[[1, 4]]).all() and torch.isfinite(row_loss[[0, 2, 3, 5]]).all() and torch.isnan(mean).all()
    assert (dx[[1, 4]] == 0).all() and torch.isfinite(dw).all()


# direct; direct gradients of logits on pairs; pairs; several blocks on pairs
@pytest.mark.parametrize("precision", [1, 0])
@pytest.mark.parametrize("rows,vocab,dim,tied", [(300, 1000, 64, True), (2304, 4096, 128, True), (2304, 2305, 512, False), (1100, 131073, 260, True)])
def test_targets_that_are_no_class_leave_the_other_rows_alone(mm, rows, vocab, dim, tied, precision):
    """Their rows' loss is NaN, their gradients are 0 and they have no share in dw, whatever x holds there; every other row's
    outputs, and dw, are those of a call that leaves these rows out."""
    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    x, w, t = loss_case(g, rows, vocab, dim, tied, 0)
    bad = torch.tensor([0, 1, 129, rows // 2, rows - 1], device="cuda")
    t[bad] = torch.tensor([vocab, -2, 2 ** 31 - 1, -2 ** 31, vocab + 127], dtype=torch.int32, device="cuda")
    x[bad, :dim] = float("nan")
    out = t.clone()
    out[bad] = -1
    kw = dict(rows=rows, vocab=vocab, dim=dim, ldx=x.stride(0), ldw=w.stride(0), w_mn_major=not tied, grad_scale=1 / rows, precision=precision)
    got, want = ([torch.full((rows,), 777.0, device="cuda"), out_buffer(rows, dim, 0), out_buffer(*((vocab, dim) if tied else (dim, vocab)), 0),
                  torch.empty(1, device="cuda")] for _ in range(2))
    for outs, targets in ((got, t), (want, out)):
        row_loss, dx, dw, mean = outs
        mm.linear_cross_entropy(x, w, targets, row_loss, mean_loss=mean, dx=dx, lddx=dx.stride(0), dw=dw, lddw=dw.stride(0), **kw)
        if targets is t:
            with pytest.raises(mm.MidmanGpuError, match="outside"):
                mm.device_status()
    mm.device_status()
    assert torch.isnan(got[0][bad]).all() and torch.isnan(got[3]).all() and (want[0][bad] == 0).all()
    good = torch.ones(rows, dtype=torch.bool, device="cuda").index_fill(0, bad, False)
    assert torch.equal(got[0][good], want[0][good]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert (got[1][bad, :dim] == 0).all() and torch.isfinite(got[2]).all()
    # the loss alone
    mm.linear_cross_entropy(x, w, t, got[0], mean_loss=got[3], **kw)
    mm.linear_cross_entropy(x, w, out, want[0], mean_loss=want[3], **kw)
    with pytest.raises(mm.MidmanGpuError, match="outside"):
        mm.device_status()
    assert torch.isnan(got[0][bad]).all() and torch.isnan(got[3]).all() and torch.equal(got[0][good], want[0][good])


@pytest.fixture
def room():
    """room(gb) skips a test where the device has less memory; what the test took is given back."""
    def need(gb):
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info()[0] < gb << 30:
            pytest.skip(f"needs {gb} GB of device memory")
    yield need
    torch.cuda.empty_cache()


@pytest.mark.parametrize("precision", [1, 0])
def test_a_vocabulary_of_more_segments_than_a_grid_has(mm, room, precision):
    """65,536 segments of 4096 classes and four classes: 268 million of width 4, one row. Off the target every gradient is
    softmax's share; the sums' tolerances are test_linear_cross_entropy's, with their S over this vocabulary."""
    room(40)
    vocab, dim, scale = (65536 << 12) + 4, 4, 1.0
    g = torch.Generator(device="cuda").manual_seed(12)
    x, w = torch.randn(1, dim, device="cuda", generator=g), torch.randn(vocab, dim, device="cuda", generator=g)
    t = torch.tensor([vocab - 2], dtype=torch.int32, device="cuda")
    row_loss, mean, dx, dw = torch.empty(1, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    mm.linear_cross_entropy(x, w, t, row_loss, rows=1, vocab=vocab, dim=dim, ldx=dim, ldw=dim, grad_scale=scale, mean_loss=mean, dx=dx,
                            lddx=dim, dw=dw, lddw=dim, precision=precision)
    mm.device_status()
    X, z = x.to(F)[0], w.to(F) @ x.to(F)[0]
    lse = torch.logsumexp(z, 0)
    tz = product_tol(precision, (w.abs().to(F) @ X.abs()).max(), dim)
    # the sum of 2^28 exponentials: 128 at a time, then 2^21 pairs by 256 threads, 2^13 roundings each in f32
    t_exp = 2 * tz + (8192 + 64 + 2 * (z.max() - z.min())) * ULP
    check(row_loss, (lse - z[-2]).view(1), t_exp + 4 * ULP * (lse.abs() + z.abs().max()), "row_loss")
    assert mean.item() == row_loss.item()
    q = (z - lse).exp()
    q[-2] -= 1
    for part in (slice(0, 1 << 20), slice(vocab - (1 << 20), vocab)):  # the first segments and the last
        want = q[part, None] * X
        tol = (t_exp + 8 * ULP) * want.abs() + product_tol(precision, want.abs(), 1) + 4 * ULP * X.abs() * (q[part, None] < 0)
        check(dw[part], want, tol, "dw")
    assert (dw[:, 0] != 0).all()  # no segment was left out
    # dx: up to eight rows are f32 multiply-adds, 2^28 of them by 512 blocks of 32 at a time: 2^14 roundings each
    size = q.abs() @ w.abs().to(F)
    check(dx[0], q @ w.to(F), (t_exp + (16384 + 1024) * ULP) * size, "dx")


LONGEST = 2 ** 31 - 512


def test_the_mean_over_the_most_rows(mm, room):
    """The rows' loop ends at the last row: a step past it is beyond 32 bits."""
    room(80)
    x, w = torch.zeros(LONGEST, 4, device="cuda"), torch.eye(4, device="cuda")
    t = torch.full((LONGEST,), -1, dtype=torch.int32, device="cuda")
    row_loss, mean = torch.empty(LONGEST, device="cuda"), torch.empty(1, device="cuda")
    at = torch.tensor([0, 1023, 1 << 30, LONGEST - 1025, LONGEST - 1], device="cuda")
    t[at], x[at, 1] = 1, torch.arange(1.0, 6.0, device="cuda")
    mm.linear_cross_entropy(x, w, t, row_loss, rows=LONGEST, vocab=4, dim=4, ldx=4, ldw=4, mean_loss=mean, precision=0)
    mm.device_status()
    z = torch.arange(1.0, 6.0, device="cuda", dtype=F)
    want = torch.log(z.exp() + 3) - z  # whole numbers pass a TF32 product as they are; a few ulp of the exponentials and of lse
    check(row_loss[at], want, 16 * ULP * (z + 1), "row_loss")
    check(mean, want.mean().view(1), 16 * ULP * (z + 1).mean() + 4 * ULP, "mean")
    assert torch.count_nonzero(row_loss) == 5


def test_the_gradient_of_the_widest_rows(mm, room):
    """The copy of x for dw ends at the last column, likewise."""
    room(120)
    x, w, dw = torch.zeros(1, LONGEST, device="cuda"), torch.zeros(4, LONGEST, device="cuda"), torch.empty(4, LONGEST, device="cuda")
    at = torch.tensor([0, 1023, 1024, 1 << 30, LONGEST - 1025, LONGEST - 1024, LONGEST - 1], device="cuda")
    x[0, at] = torch.arange(1.0, 8.0, device="cuda")
    t, row_loss = torch.tensor([2], dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda")
    mm.linear_cross_entropy(x, w, t, row_loss, rows=1, vocab=4, dim=LONGEST, ldx=LONGEST, ldw=LONGEST, dw=dw, lddw=LONGEST, precision=0)
    mm.device_status()
    want = torch.tensor([0.25, 0.25, -0.75, 0.25], device="cuda")[:, None] * torch.arange(1.0, 8.0, device="cuda")
    assert torch.equal(dw[:, at], want)  # exact: quarters of whole numbers
    assert torch.count_nonzero(dw) == 28
    check(row_loss, torch.tensor([4.0], device="cuda", dtype=F).log(), 4 * ULP, "row_loss")


@pytest.mark.parametrize("precision", [1, 0])
@pytest.mark.parametrize("rows,vocab,dim,tied", [(300, 1000, 64, True), (2304, 4096, 128, False), (2304, 2305, 512, True), (2304, 2305, 512, False)])
def test_gradients_scale_with_grad_scale(mm, rows, vocab, dim, tied, precision):
    """A power of two changes nothing but the exponents, of either sign and near the largest: losses and dw bit for bit. dx too,
    but on pairs, where a chunk of 128 classes takes softmax's factor (no power of two) and w's scale in the order that does not
    overflow: factor first, it is rounded (2^-24 of the chunk's sum) before it is added, scale first, it is not; so the chunks'
    sums and the running sums differ by 2^-24 of what they hold, twice a chunk."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x, w, t = loss_case(g, rows, vocab, dim, tied, 0)
    t[::7] = -1
    outs = []
    for scale in (1.0, -(2.0 ** 120), 2.0 ** 120, -(2.0 ** -40)):
        row_loss, dx, dw = torch.empty(rows, device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
        mm.linear_cross_entropy(x, w, t, row_loss, rows=rows, vocab=vocab, dim=dim, ldx=x.stride(0), ldw=w.stride(0), w_mn_major=not tied,
                                grad_scale=scale, dx=dx, lddx=dx.stride(0), dw=dw, lddw=dw.stride(0), precision=precision)
        mm.device_status()
        outs.append([row_loss] + [o[:, :n].to(F) / scale for o, n in ((dx, dim), (dw, dim if tied else vocab))])
    W = (w[:, :dim] if tied else w[:, :vocab].T).to(F)
    gr = loss64(x[:, :dim], W, t, 1.0, t >= 0)[4]
    tol = 2 * (-(-vocab // 128) + 1) * ULP * (gr.abs() @ W.abs()) if dim == 512 and precision == 1 else torch.zeros_like(x[:, :dim])
    for other in outs[1:]:
        assert torch.equal(outs[0][0], other[0]) and torch.equal(outs[0][2], other[2])
        check(other[1], outs[0][1], tol, "dx")


def test_no_row_has_a_target(mm):
    x, w, t = torch.randn(9, 8, device="cuda"), torch.randn(50, 8, device="cuda"), torch.full((9,), -1, dtype=torch.int32, device="cuda")
    row_loss, mean, dx, dw = torch.empty(9, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    mm.linear_cross_entropy(x, w, t, row_loss, rows=9, vocab=50, dim=8, ldx=8, ldw=8, mean_loss=mean, dx=dx, lddx=8, dw=dw, lddw=8)
    mm.device_status()
    for out in (row_loss, mean, dx, dw):
        assert (out == 0).all()


def test_no_rows(mm):
    w, dw = torch.randn(50, 8, device="cuda"), torch.ones(50, 8, device="cuda")
    e, t, mean = torch.empty(0, 8, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda")
    mm.linear_cross_entropy(e, w, t, e[:, 0], rows=0, vocab=50, dim=8, ldx=8, ldw=8, mean_loss=mean, dx=e, lddx=8, dw=dw, lddw=8)
    assert (dw == 0).all() and mean.item() == 0
    mm.linear_forward(e, w, torch.empty(0, 52, device="cuda"), m=0, n=50, k=8, lda=8, ldb=8, ldc=52, b_mn_major=False)
    db, dbias = torch.ones(50, 8, device="cuda"), torch.ones(50, device="cuda")
    kw = dict(m=0, n=50, k=8, lda=8, ldb=8, lddc=52, b_mn_major=False, da=e, ldda=8, db=db, lddb=8, dbias=dbias)
    mm.linear_backward(e, w, torch.empty(0, 52, device="cuda"), accumulate=True, **kw)
    assert (db == 1).all() and (dbias == 1).all()
    mm.linear_backward(e, w, torch.empty(0, 52, device="cuda"), **kw)
    assert (db == 0).all() and (dbias == 0).all()
    mm.dropout(e, e, rows=0, cols=8, ldx=8, ldy=8, p=0.5, rng=rng_words(1, 2))
    mm.device_status()


# ------------------------------------------------------------------ streams, graphs, repeats
def all_of_them(mm, s, stream=None):
    """The operators one after another on the tensors of `s`; every output."""
    m, k, n, v = s["sizes"]
    kw = dict(m=m, n=n, k=k, lda=k, ldb=n, activation=2, p=0.1, rng=s["rng"], z=s["z"], ldz=n, precision=s["precision"], stream=stream)
    mm.linear_forward(s["a"], s["b"], s["c"], ldc=n, bias=s["bias"], r=s["r"], ldr=n, **kw)
    mm.linear_cross_entropy(s["c"], s["w"], s["t"], s["loss"], rows=m, vocab=v, dim=n, ldx=n, ldw=n, grad_scale=1 / m,
                            mean_loss=s["mean"], dx=s["dc"], lddx=n, dw=s["dw"], lddw=n, precision=s["precision"], workspace=s["ws"],
                            stream=stream)
    mm.linear_backward(s["a"], s["b"], s["dc"], lddc=n, da=s["da"], ldda=k, db=s["db"], lddb=n, dbias=s["dbias"],
                       workspace=s["ws"], **kw)
    mm.dropout(s["da"], s["y"], rows=m, cols=k, ldx=k, ldy=k, p=0.1, rng=s["rng"], stream=stream)
    return [s[o] for o in ("c", "z", "loss", "mean", "dc", "dw", "da", "db", "dbias", "y")]


def tensors_for(mm, seed, m, k, n, v, precision):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s = {"sizes": (m, k, n, v), "precision": precision, "a": new(m, k), "b": new(k, n) * k ** -0.5, "bias": new(n), "r": new(m, n), "w": new(v, n) * 0.1,
         "t": torch.randint(0, v, (m,), device="cuda", generator=g, dtype=torch.int32), "rng": rng_words(seed, 7)}
    for name, shape in dict(c=(m, n), z=(m, n), loss=(m,), mean=(1,), dc=(m, n), dw=(v, n), da=(m, k), db=(k, n), dbias=(n,),
                            y=(m, k)).items():
        s[name] = torch.empty(*shape, device="cuda")
    need = max(mm.linear_workspace(m, n, k, backward=True, precision=precision), mm.linear_workspace(m, n, k, precision=precision),
               mm.linear_cross_entropy_workspace(m, v, n, precision=precision))
    s["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    return s


# few rows, direct products, slices of a long sum, pairs; both precisions
SIZES = [(5, 96, 200, 1000, 1), (300, 96, 200, 1000, 1), (300, 96, 200, 1000, 0), (40, 36, 68, 20001, 1), (2304, 256, 2304, 2305, 1),
         (2304, 256, 2304, 2305, 0)]


@pytest.mark.parametrize("sizes", SIZES)
def test_repeats_are_bit_identical(mm, sizes):
    s = tensors_for(mm, 1, *sizes)
    first = [t.clone() for t in all_of_them(mm, s)]
    s["ws"].fill_(255)  # whatever the workspace holds before
    assert all(torch.equal(x, y) for x, y in zip(first, all_of_them(mm, s)))
    mm.device_status()


@pytest.mark.parametrize("sizes", SIZES)
def test_two_streams_at_once(mm, sizes):
    pair = [tensors_for(mm, seed, *sizes) for seed in (1, 2)]
    want = [[t.clone() for t in all_of_them(mm, s)] for s in pair]
    for s in pair:
        for o in ("c", "z", "dc", "da", "db", "dw", "y"):
            s[o].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pair]
    for _ in range(3):
        for s, st in zip(pair, streams):
            with torch.cuda.stream(st):
                all_of_them(mm, s)
    torch.cuda.synchronize()
    for s, w in zip(pair, want):
        assert all(torch.equal(s[o], x) for o, x in zip(("c", "z", "loss", "mean", "dc", "dw", "da", "db", "dbias", "y"), w))
    mm.device_status()


@pytest.mark.parametrize("sizes", SIZES)
def test_calls_back_to_back_on_one_workspace(mm, sizes):
    """Launches overlap: nothing of a call may start before what it reads is there, or write what is still read."""
    pair = [tensors_for(mm, seed, *sizes) for seed in (1, 2)]
    pair[1]["ws"] = pair[0]["ws"]
    names = ("c", "z", "loss", "mean", "dc", "dw", "da", "db", "dbias", "y")
    m, k, n, v = sizes[:4]
    kw = dict(rows=m, vocab=v, dim=n, ldx=n, ldw=n, grad_scale=1 / m, precision=sizes[4], workspace=pair[0]["ws"])
    # The loss without gradients joins a row's sums in another order than the loss with them: outputs of its own
    names += ("alone", "mean alone")
    want = []
    for s in pair:
        s["alone"], s["mean alone"] = torch.empty(m, device="cuda"), torch.empty(1, device="cuda")
        all_of_them(mm, s)
        torch.cuda.synchronize()
        mm.linear_cross_entropy(s["c"], s["w"], s["t"], s["alone"], mean_loss=s["mean alone"], **kw)
        torch.cuda.synchronize()
        want.append([s[o].clone() for o in names])
    one_by_one = []
    for s in pair:  # a gradient alone, with the mean and without, the loss alone
        for grads in (dict(dx="dc"), dict(dw="dw"), dict(dx="dc", dw="dw"), {}):
            for mean in (True, False):
                one_by_one.append((s, {a: s[t] for a, t in grads.items()}, mean))
    for s in pair:
        for o in names:
            s[o].zero_()
    torch.cuda.synchronize()
    for _ in range(8):
        for s in pair:
            all_of_them(mm, s)
    for s, grads, mean in one_by_one:
        mm.linear_cross_entropy(s["c"], s["w"], s["t"], s["loss"] if grads else s["alone"], **grads, lddx=n, lddw=n,
                                mean_loss=(s["mean"] if grads else s["mean alone"]) if mean else None, **kw)
        bw = dict(m=m, n=n, k=k, lda=k, ldb=n, lddc=n, activation=2, p=0.1, rng=s["rng"], z=s["z"], ldz=n, precision=sizes[4],
                  workspace=pair[0]["ws"])
        mm.linear_backward(s["a"], s["b"], s["dc"], da=s["da"], ldda=k, **bw)
        mm.linear_backward(s["a"], s["b"], s["dc"], db=s["db"], lddb=n, dbias=s["dbias"], **bw)
        mm.linear_backward(s["a"], s["b"], s["dc"], dbias=s["dbias"], **bw)
        mm.dropout(s["da"], s["y"], rows=m, cols=k, ldx=k, ldy=k, p=0.1, rng=s["rng"])
    torch.cuda.synchronize()
    for s, w in zip(pair, want):
        for o, x in zip(names, w):
            assert torch.equal(s[o], x), o
    mm.device_status()


@pytest.mark.parametrize("sizes", SIZES)
def test_captured_and_replayed(mm, sizes):
    s, other = tensors_for(mm, 1, *sizes), tensors_for(mm, 2, *sizes)
    all_of_them(mm, s)
    want = [t.clone() for t in all_of_them(mm, other)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = all_of_them(mm, s)
    for name in ("a", "b", "bias", "r", "w", "t", "rng"):  # new inputs in the captured addresses
        s[name].copy_(other[name])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))
    mm.device_status()


@pytest.mark.parametrize("m,k,n,precision", [(4, 64, 40, 1), (40, 96, 72, 1), (40, 96, 72, 0), (2304, 512, 2304, 1), (2304, 512, 2304, 0)])
def test_a_host_thread_whose_first_call_it_is(mm, m, k, n, precision):
    a, b = torch.randn(m, k, device="cuda"), torch.randn(k, n, device="cuda")
    c, d = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    ws = torch.empty(mm.linear_workspace(m, n, k, precision=precision) + 256, dtype=torch.uint8, device="cuda")
    stream, failed = torch.cuda.current_stream().cuda_stream, []
    call = [m, n, k, a.data_ptr(), k, b.data_ptr(), n, 1, None, 0, 0.0, None, None, 0, None, 0]
    end = [n, precision, ws.data_ptr(), ws.numel(), stream]
    assert mm.load().mm_gpu_linear_forward(*call, c.data_ptr(), *end) == 0
    thread = threading.Thread(target=lambda: failed.append(mm.load().mm_gpu_linear_forward(*call, d.data_ptr(), *end)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert failed == [0] and torch.equal(c, d)
    mm.device_status()


def test_a_callers_context_stays_current():
    """A product's tensor maps need a current context; one that the caller made is left in its place. The sizes pass the
    checks and the maps, and are refused before anything is launched. In a process of its own, as contexts outlive tests."""
    code = """
import ctypes, sys, threading
sys.path.insert(0, sys.argv[1])
import torch, midman_b200 as mm
cuda = ctypes.CDLL("libcuda.so.1")
x = torch.zeros(64, device="cuda")
mm.device_status()
seen = []
def work():
    mine, now, dev = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int()
    assert cuda.cuDeviceGet(ctypes.byref(dev), 0) == 0
    assert cuda.cuCtxCreate_v2(ctypes.byref(mine), 0, dev) == 0
    n = 2 ** 31 - 512
    rc = mm.load().mm_gpu_linear_forward(n, n, 4, x.data_ptr(), 4, x.data_ptr(), 4, 0, None, 0, 0.0, None, None, 0, None, 0,
                                         x.data_ptr() + 128, n, 1, None, 0, None)
    assert cuda.cuCtxGetCurrent(ctypes.byref(now)) == 0
    seen.extend([rc, mine.value, now.value])
    assert cuda.cuCtxDestroy_v2(mine) == 0
t = threading.Thread(target=work)
t.start()
t.join()
torch.cuda.synchronize()
assert seen[0] == -1, seen
assert seen[1] == seen[2], "another context was made current"
print("stays")
"""
    run = subprocess.run([sys.executable, "-c", code, str(Path(__file__).resolve().parent.parent / "midman-ai_b200")], capture_output=True,
                         text=True, timeout=120)
    assert run.returncode == 0 and "stays" in run.stdout, run.stderr


@pytest.mark.parametrize("sizes", SIZES)
def test_two_host_threads_on_one_stream(mm, sizes):
    pair = [tensors_for(mm, seed, *sizes) for seed in (1, 2)]
    want = [[t.clone() for t in all_of_them(mm, s)] for s in pair]
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    start, failed = threading.Barrier(2), []

    def work(s, w):
        start.wait()
        try:
            for _ in range(20):
                all_of_them(mm, s, stream)
        except Exception as e:  # noqa: BLE001 - shown by the assertion
            failed.append(e)

    threads = [threading.Thread(target=work, args=p) for p in zip(pair, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for s, w in zip(pair, want):
        assert all(torch.equal(s[o], x) for o, x in zip(("c", "z", "loss", "mean", "dc", "dw", "da", "db", "dbias", "y"), w))
    mm.device_status()


def test_captured_on_streams_that_part_and_meet(mm):
    """Overlapping launches beside event waits, copies and fills of a captured graph."""
    pair = [tensors_for(mm, seed, 300, 96, 200, 1000, 1) for seed in (1, 2)]
    mm.device_status()
    want = [[t.clone() for t in all_of_them(mm, s)] for s in pair]
    torch.cuda.synchronize()
    kept_a = [s["a"].clone() for s in pair]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        pair[1]["a"].copy_(kept_a[1])
        side.wait_stream(main)
        with torch.cuda.stream(side):
            all_of_them(mm, pair[1])
            pair[1]["y"].add_(0)
        pair[0]["a"].copy_(kept_a[0])
        all_of_them(mm, pair[0])
        main.wait_stream(side)
        mm.dropout(pair[1]["y"], pair[1]["y"], rows=300, cols=96, ldx=96, ldy=96, p=0.0)
    for s in pair:
        for o in ("c", "z", "dc", "dw", "da", "db", "y", "a"):
            s[o].zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for s, w in zip(pair, want):
        assert all(torch.equal(s[o], x) for o, x in zip(("c", "z", "loss", "mean", "dc", "dw", "da", "db", "dbias", "y"), w))
    mm.device_status()


def test_linear_and_dropout_share_their_mask(mm):
    m, k, n = 50, 20, 70
    words = rng_words(3, 4)
    a, b = torch.randn(m, k, device="cuda"), torch.randn(k, 72, device="cuda")
    c, d, y = (torch.empty(m, 72, device="cuda") for _ in range(3))
    kw = dict(m=m, n=n, k=k, lda=k, ldb=72, ldc=72, precision=1)
    mm.linear_forward(a, b, c, **kw)
    mm.dropout(c, y, rows=m, cols=n, ldx=72, ldy=72, p=0.3, rng=words)
    mm.linear_forward(a, b, d, p=0.3, rng=words, **kw)
    assert torch.equal(d[:, :n], y[:, :n])


def test_wrong_types_and_places_are_refused(mm):
    x, h = torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda", dtype=torch.float16)
    with pytest.raises(TypeError, match="float32"):
        mm.dropout(h, x, rows=4, cols=8, ldx=8, ldy=8, p=0.5, rng=rng_words(1, 2))
    with pytest.raises(ValueError, match="cpu"):
        mm.dropout(x.cpu(), x, rows=4, cols=8, ldx=8, ldy=8, p=0.5, rng=rng_words(1, 2))
    with pytest.raises(TypeError, match="int64"):
        mm.dropout(x, x, rows=4, cols=8, ldx=8, ldy=8, p=0.5, rng=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="int32"):
        mm.linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64, device="cuda"), x[:, 0], rows=4, vocab=4, dim=8, ldx=8, ldw=8)
    with pytest.raises(mm.MidmanGpuError, match="workspace"):
        mm.linear_backward(x, x, x, m=4, n=8, k=4, lda=8, ldb=8, lddc=8, da=x, ldda=8, workspace=torch.empty(256, dtype=torch.uint8, device="cuda")[:8])


def test_workspaces_and_words_in_wrong_places_are_refused(mm):
    """Host memory, pieces and a single word, each before anything is queued: the kernels would follow their addresses."""
    m, k, n, v = 300, 96, 200, 1000
    s = tensors_for(mm, 1, m, k, n, v, 1)
    kw = dict(m=m, n=n, k=k, lda=k, ldb=n, precision=1)
    forward = lambda **c: mm.linear_forward(s["a"], s["b"], s["c"], ldc=n, **kw, **c)  # noqa: E731
    backward = lambda **c: mm.linear_backward(s["a"], s["b"], s["dc"], lddc=n, da=s["da"], ldda=k, **kw, **c)  # noqa: E731
    loss = lambda **c: mm.linear_cross_entropy(s["c"], s["w"], s["t"], s["loss"], rows=m, vocab=v, dim=n, ldx=n, ldw=n, dx=s["dc"],  # noqa: E731
                                               lddx=n, precision=1, **c)
    dropout = lambda **c: mm.dropout(s["a"], s["y"], rows=m, cols=k, ldx=k, ldy=k, p=0.1, **c)  # noqa: E731
    host = torch.empty(s["ws"].numel(), dtype=torch.uint8)
    for call in (forward, backward, loss):
        for ws in (host, host.pin_memory(), torch.empty(2 * s["ws"].numel(), dtype=torch.uint8, device="cuda")[::2]):
            with pytest.raises(ValueError, match="workspace"):
                call(workspace=ws)
    words = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda **c: forward(p=0.1, **c), lambda **c: backward(p=0.1, **c), dropout):
        for rng in (words[:1], words[::2], words.cpu()):
            with pytest.raises(ValueError):
                call(rng=rng)
        call(rng=words[2:])
    mm.device_status()
