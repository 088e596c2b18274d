"""mm_op_linear, mm_op_dropout and mm_op_linear_cross_entropy on the autograd tape: a decoder's MLP branch, residual stream
and loss as they are used together, against float64 PyTorch autograd with the same dropout masks; the fused operations
against the tape's separate ones; refusals.

The gradient gates are those of the tape's other tests: 1e-5 relative L2 in the exact mode, 1e-2 with one TF32 pass.
"""
import numpy as np
import pytest

from philox import kept

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


@pytest.fixture(params=[1, 0])
def tape(mm, request):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    t = mm.Tape(precision=request.param)
    t.tol = 1e-5 if request.param else 1e-2
    yield t
    t.close()


@pytest.mark.parametrize("rows,d,ff,vocab", [(1, 4, 8, 4), (37, 64, 176, 256), (300, 128, 344, 4096)])
def test_a_block_and_its_loss(mm, tape, rows, d, ff, vocab):
    rs = np.random.default_rng(rows)
    p, seed = 0.2, 11
    v = {n: (rs.standard_normal(s) * f).astype(np.float32) for n, s, f in [
        ("x", (rows, d), 1), ("g", (d,), 1), ("w1", (d, ff), d ** -0.5), ("b1", (ff,), 0.1), ("w2", (ff, d), ff ** -0.5),
        ("b2", (d,), 0.1), ("e", (vocab, d), 0.3)]}
    targets = rs.integers(0, vocab, rows).astype(np.int32)
    if rows > 1:
        targets[::5] = -1
    h = {n: tape.tensor(a, requires_grad=True) for n, a in v.items()}
    x = tape.dropout(h["x"], p, seed, 1)
    a = tape.linear(tape.rms_norm(x, h["g"]), h["w1"], bias=h["b1"], activation=mm.ACT_GELU, p=p, seed=seed, offset=2)
    y = tape.linear(a, h["w2"], bias=h["b2"], p=p, seed=seed, offset=3, residual=x)  # x is used twice
    loss = tape.linear_cross_entropy(y, h["e"], targets, w_transposed=True)
    tape.backward(loss)

    t = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in v.items()}
    drop = lambda z, offset: z * torch.from_numpy(kept(seed, offset, *z.shape, p)) / (1 - p)  # noqa: E731
    X = drop(t["x"], 1)
    A = drop(torch.nn.functional.gelu(X * torch.rsqrt(X.square().mean(1, keepdim=True) + 1e-5) * t["g"] @ t["w1"] + t["b1"]), 2)
    Y = X + drop(A @ t["w2"] + t["b2"], 3)
    L = torch.nn.functional.cross_entropy(Y @ t["e"].T, torch.tensor(targets, dtype=torch.long), ignore_index=-1)
    L.backward()
    assert rel(tape.read(y), Y.detach()) <= tape.tol
    assert abs(tape.read(loss)[0] - L.item()) <= tape.tol * max(1.0, abs(L.item()))
    for n in v:
        assert rel(tape.grad(h[n]), t[n].grad) <= tape.tol, n


def test_the_fused_operations_are_the_separate_ones(mm, tape):
    rs = np.random.default_rng(3)
    xv, wv, tv = rs.standard_normal((50, 64)), rs.standard_normal((64, 96)) * 0.2, rs.integers(0, 96, 50)
    x, w, r = tape.tensor(xv, requires_grad=True), tape.tensor(wv, requires_grad=True), tape.tensor(rs.standard_normal((50, 96)))
    fused, apart = tape.linear(x, w, residual=r), tape.add(tape.matmul(x, w), r)
    assert rel(tape.read(fused), tape.read(apart)) <= tape.tol
    one, two = tape.linear_cross_entropy(x, w, tv), tape.cross_entropy(tape.matmul(x, w), tv)
    grads = []
    for loss in (one, two):
        tape.backward(loss)
        grads.append([tape.grad(x), tape.grad(w)])
    assert abs(tape.read(one)[0] - tape.read(two)[0]) <= tape.tol
    assert all(rel(a, b) <= tape.tol for a, b in zip(*grads))
    # the transposed forms
    wt = tape.tensor(np.ascontiguousarray(wv.T), requires_grad=True)
    assert rel(tape.read(tape.linear(x, wt, w_transposed=True, activation=mm.ACT_SILU)),
               tape.read(tape.linear(x, w, activation=mm.ACT_SILU))) <= tape.tol
    tape.backward(tape.linear_cross_entropy(tape.linear(x, wt, w_transposed=True), tape.tensor(np.eye(96)), tv))
    assert rel(tape.grad(wt).T, grads[0][1]) <= tape.tol


def test_one_tensor_in_every_place(mm, tape):
    """x as input, weight and residual of one call: its gradient is the sum of the three."""
    v = np.random.default_rng(5).standard_normal((64, 64)).astype(np.float32) * 0.3
    x = tape.tensor(v, requires_grad=True)
    tape.backward(tape.linear_cross_entropy(tape.linear(x, x, activation=mm.ACT_SILU, residual=x), x, np.arange(64) % 7))
    t = torch.tensor(v, dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.silu(t @ t) + t
    torch.nn.functional.cross_entropy(y @ t, torch.arange(64) % 7).backward()
    assert rel(tape.grad(x), t.grad) <= tape.tol


@pytest.mark.parametrize("n", [64, 256, 1024, 2048])  # one direct tile a product, four, many, pairs
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_one_tensor_as_input_and_weight(mm, tape, n, transposed, bias):
    """x x and x x^T: both products add to the one gradient, in an order that does not change from run to run.

    The tolerance is the tape's relative one for the sum of the two products, which are each within it."""
    rs = np.random.default_rng(n)
    v = rs.standard_normal((n, n)).astype(np.float32) * np.float32(n ** -0.5)
    head, targets = rs.standard_normal((n, 8)).astype(np.float32), (np.arange(n) % 8).astype(np.int32)
    b = np.zeros(n, np.float32)
    x, w, bh = tape.tensor(v, requires_grad=True), tape.tensor(head), tape.tensor(b, requires_grad=True)
    loss = tape.linear_cross_entropy(tape.linear(x, x, w_transposed=transposed, bias=bh if bias else 0, activation=mm.ACT_SILU), w, targets)
    tape.backward(loss)
    first = tape.grad(x)
    for _ in range(10):
        tape.backward(loss)
        assert np.array_equal(tape.grad(x), first)
    t = torch.tensor(v, dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.silu(t @ (t.T if transposed else t))
    torch.nn.functional.cross_entropy(y @ torch.tensor(head, dtype=torch.float64), torch.tensor(targets, dtype=torch.long)).backward()
    assert rel(first, t.grad) <= tape.tol


def test_constants_get_no_gradient(mm, tape):
    rs = np.random.default_rng(6)
    x, w = tape.tensor(rs.standard_normal((8, 8))), tape.tensor(rs.standard_normal((8, 8)))
    b = tape.tensor(rs.standard_normal(8), requires_grad=True)
    loss = tape.linear_cross_entropy(tape.linear(x, w, bias=b, activation=mm.ACT_RELU), w, np.zeros(8, np.int32))
    tape.backward(loss)
    assert tape.grad(b).any() and not tape.grad(x).any() and not tape.grad(w).any()
    with pytest.raises(mm.MidmanGpuError, match="does not track"):
        tape.backward(tape.linear_cross_entropy(x, w, np.zeros(8, np.int32)))


@pytest.mark.parametrize("m,k,n", [(1, 8, 12), (37, 64, 176), (2304, 256, 2304), (2304, 512, 2304)])  # few rows, direct, pairs
@pytest.mark.parametrize("act", range(4))
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_only_the_residual_tracks(mm, tape, m, k, n, act, p):
    """Constant input, weight and bias, as of a frozen layer: no z is kept, and the residual's gradient is dc."""
    rs = np.random.default_rng(m + act)
    x, w, b = tape.tensor(rs.standard_normal((m, k))), tape.tensor(rs.standard_normal((k, n)) * 0.1), tape.tensor(rs.standard_normal(n))
    r, head = tape.tensor(rs.standard_normal((m, n)), requires_grad=True), tape.tensor(rs.standard_normal((n, 8)) * 0.1)
    y = tape.linear(x, w, bias=b, activation=act, p=p, seed=3, offset=1, residual=r)
    leaf = tape.tensor(tape.read(y), requires_grad=True)
    targets = (np.arange(m) % 8).astype(np.int32)
    tape.backward(tape.linear_cross_entropy(y, head, targets))
    got = tape.grad(r)
    tape.backward(tape.linear_cross_entropy(leaf, head, targets))
    assert got.any() and np.array_equal(got, tape.grad(leaf))
    assert not tape.grad(x).any() and not tape.grad(w).any() and not tape.grad(b).any()


def test_the_call_after_one_without_memory_is_unharmed(mm, tape):
    """[2^20, 2^20] outputs do not fit; the error belongs to the call that met it."""
    wide, tall = tape.tensor(np.ones((4, 1 << 20))), tape.tensor(np.ones((1 << 20, 4)))
    a, c = torch.ones(256, 256, device="cuda"), torch.empty(256, 256, device="cuda")
    for call in (lambda: tape.linear(tall, wide), lambda: tape.linear(tall, wide, activation=mm.ACT_GELU, p=0.5), lambda: tape.matmul(tall, wide)):
        with pytest.raises(mm.MidmanGpuError, match="out of memory"):
            call()
        mm.gemm(a, a, c, m=256, n=256, k=256, lda=256, ldb=256, ldc=256, a_mn_major=False, b_mn_major=False)
        assert (c == 256).all()
        with pytest.raises(mm.MidmanGpuError, match="out of memory"):
            call()
        assert (tape.read(tape.linear(tape.tensor(np.ones((8, 8))), tape.tensor(np.ones((8, 8))))) == 8).all()


def test_refusals(mm, tape):
    x, w = tape.tensor(np.ones((4, 8))), tape.tensor(np.ones((8, 12)))
    odd = tape.tensor(np.ones((8, 6)))
    for call, what in [(lambda: tape.linear(x, x), "inner dimensions"), (lambda: tape.linear(x, odd), "multiples of 4"),
                       (lambda: tape.linear(x, w, bias=x), "bias"), (lambda: tape.linear(x, w, residual=x), "residual"),
                       (lambda: tape.linear(x, w, activation=9), "activation"), (lambda: tape.linear(x, w, p=1.0), "p must lie"),
                       (lambda: tape.dropout(x, -0.5), "p must lie"), (lambda: tape.dropout(x, float("nan")), "p must lie"),
                       (lambda: tape.linear_cross_entropy(x, w, [0, 1, 2, 12]), "outside"),
                       (lambda: tape.linear_cross_entropy(x, w, [0, 1, 2, -2]), "outside"),
                       (lambda: tape.linear_cross_entropy(x, w, [0, 1]), "one target per row"),
                       (lambda: tape.linear_cross_entropy(x, odd, [0, 1, 2, 3]), "multiples of 4"),
                       (lambda: tape.linear(x, 424242), "not live")]:
        with pytest.raises(mm.MidmanGpuError, match=what):
            call()
