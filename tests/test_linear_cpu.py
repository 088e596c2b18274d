"""The products with an epilogue, dropout and the linear cross-entropy without a GPU: the generator's published test
vectors, workspace sizes, and the refusals, which all come before anything is queued (the pointers here are numbers
that nothing may follow)."""
import numpy as np
import pytest

from philox import kept, philox4x32_10

P = 0x1000  # a 256-byte aligned address that is never read


def test_the_generator_has_the_published_vectors():
    # Random123's known answers for philox4x32-10
    ones = 0xFFFFFFFF
    for ctr, key, want in [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                           ((ones,) * 4, (ones, ones), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                            (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]:
        assert tuple(int(w) for w in philox4x32_10(ctr, key)) == want


def test_the_mask_keeps_the_share_it_says():
    n = 512 * 1001
    for p in (0.05, 0.5):
        share = kept(7, 1 << 40, 512, 1001, p).mean()
        assert abs(share - (1 - p)) < 5 * np.sqrt(p * (1 - p) / n)
    assert (kept(7, 3, 8, 8, 0.5) != kept(7, 4, 8, 8, 0.5)).any()


def test_workspaces(mm):
    assert mm.linear_workspace(0, 1, 1) >= 0
    assert mm.linear_workspace(100, 30, 8, backward=True) >= 100 * 32 * 4
    # A block's logits take 384 MiB at most: 3146 rows of 32000. A row needs besides 250 (maximum, sum) pairs, three
    # numbers and its 256 inputs: 3036 bytes, under 10 MB in all. A last wave's parts: at most 74 tiles of 256 KiB.
    for rows in (8192, 65536, 1 << 20):
        assert mm.linear_cross_entropy_workspace(rows, 32000, 256) < (384 << 20) + 10_000_000 + 74 * (256 << 10)
    assert mm.linear_cross_entropy_workspace(8192, 32000, 256, gradients=False) < 128 << 20
    for bad in ((-1, 4, 4), (1, 0, 4), (1, 4, 0)):
        with pytest.raises(mm.MidmanGpuError):
            mm.linear_workspace(*bad)
        with pytest.raises(mm.MidmanGpuError):
            mm.linear_cross_entropy_workspace(*bad)


def forward(mm, **change):
    v = dict(m=4, n=8, k=8, a=P, lda=8, b=P, ldb=8, mn=1, bias=None, act=0, p=0.0, rng=None, r=None, ldr=0, z=None, ldz=0,
             c=P, ldc=8, precision=1, ws=P, bytes=1 << 30, stream=None)
    assert set(change) <= set(v)
    rc = mm.load().mm_gpu_linear_forward(*{**v, **change}.values())
    return rc, mm.load().mm_gpu_last_error().decode()


def backward(mm, **change):
    v = dict(m=4, n=8, k=8, a=P, lda=8, b=P, ldb=8, mn=1, act=0, p=0.0, rng=None, z=None, ldz=0, dc=P, lddc=8, da=P, ldda=8,
             db=P, lddb=8, dbias=None, accumulate=0, precision=1, ws=P, bytes=1 << 30, stream=None)
    assert set(change) <= set(v)
    rc = mm.load().mm_gpu_linear_backward(*{**v, **change}.values())
    return rc, mm.load().mm_gpu_last_error().decode()


def loss(mm, **change):
    v = dict(rows=4, vocab=8, dim=8, x=P, ldx=8, w=P, ldw=8, mn=0, targets=P, scale=1.0, row_loss=P, mean=None, dx=P, lddx=8,
             dw=P, lddw=8, accumulate=0, precision=1, ws=P, bytes=1 << 40, stream=None)
    assert set(change) <= set(v)
    rc = mm.load().mm_gpu_linear_cross_entropy(*{**v, **change}.values())
    return rc, mm.load().mm_gpu_last_error().decode()


def dropout(mm, **change):
    v = dict(rows=4, cols=8, x=P, ldx=8, r=None, ldr=0, y=P, ldy=8, p=0.5, rng=P, stream=None)
    assert set(change) <= set(v)
    rc = mm.load().mm_gpu_dropout(*{**v, **change}.values())
    return rc, mm.load().mm_gpu_last_error().decode()


NAN = float("nan")
SHAPE, ARGUMENT = -3, -1


@pytest.mark.parametrize("call,change,status", [
    (forward, dict(m=-1), SHAPE), (forward, dict(n=0), SHAPE), (forward, dict(k=0), SHAPE),
    (forward, dict(a=None), ARGUMENT), (forward, dict(a=P + 4), ARGUMENT), (forward, dict(lda=7), SHAPE),
    (forward, dict(k=7, lda=7), SHAPE), (forward, dict(ldb=4), SHAPE), (forward, dict(c=P + 8), ARGUMENT),
    (forward, dict(ldc=4), SHAPE), (forward, dict(r=P, ldr=4), SHAPE), (forward, dict(z=P + 4, ldz=8), ARGUMENT),
    (forward, dict(act=4), ARGUMENT), (forward, dict(act=-1), ARGUMENT), (forward, dict(precision=2), ARGUMENT),
    (forward, dict(p=1.0), ARGUMENT), (forward, dict(p=-0.1), ARGUMENT), (forward, dict(p=NAN), ARGUMENT),
    (forward, dict(p=0.1), ARGUMENT), (forward, dict(p=0.1, rng=P + 4), ARGUMENT),
    (forward, dict(n=16, mn=0, ldb=8, ldc=8), SHAPE), (forward, dict(r=P, ldr=12), SHAPE),
    (forward, dict(z=P, ldz=8), ARGUMENT), (forward, dict(z=2 * P, ldz=8, r=2 * P, ldr=8), ARGUMENT),
    (backward, dict(m=-1), SHAPE), (backward, dict(dc=None), ARGUMENT), (backward, dict(act=2), ARGUMENT),
    (backward, dict(act=2, z=P, ldz=4), SHAPE), (backward, dict(b=None), ARGUMENT), (backward, dict(a=None), ARGUMENT),
    (backward, dict(ldda=4), SHAPE), (backward, dict(db=P + 4), ARGUMENT), (backward, dict(ws=None), ARGUMENT),
    (backward, dict(bytes=16), ARGUMENT), (backward, dict(ws=P + 16), ARGUMENT),
    (loss, dict(rows=-1), SHAPE), (loss, dict(vocab=0), SHAPE), (loss, dict(targets=None), ARGUMENT),
    (loss, dict(row_loss=None), ARGUMENT), (loss, dict(scale=NAN), ARGUMENT), (loss, dict(scale=float("inf")), ARGUMENT),
    (loss, dict(x=P + 4), ARGUMENT), (loss, dict(ldw=4), SHAPE), (loss, dict(vocab=12, mn=1), SHAPE),
    (loss, dict(lddx=6), SHAPE), (loss, dict(dw=P + 4), ARGUMENT), (loss, dict(bytes=0), ARGUMENT),
    (loss, dict(precision=7), ARGUMENT),
    (dropout, dict(rows=-1), SHAPE), (dropout, dict(cols=0), SHAPE), (dropout, dict(x=None), ARGUMENT),
    (dropout, dict(ldx=7), SHAPE), (dropout, dict(r=P, ldr=7), SHAPE), (dropout, dict(p=1.0), ARGUMENT),
    (dropout, dict(rng=None), ARGUMENT), (dropout, dict(ldy=9), SHAPE), (dropout, dict(r=2 * P, ldr=9, y=2 * P), SHAPE),
])
def test_refusals(mm, call, change, status):
    rc, message = call(mm, **change)
    assert rc == status and message


Q, R, S, T = (P * i for i in (2, 3, 4, 5))


@pytest.mark.parametrize("call,change", [
    (forward, dict(a=Q, b=R, c=Q)), (forward, dict(a=Q, b=R, c=R)), (forward, dict(a=Q, b=R, c=S, bias=S)),
    (forward, dict(a=Q, b=R, c=S, z=S, ldz=8)), (forward, dict(a=Q, b=R, c=S, z=R, ldz=8)),
    (backward, dict(a=Q, b=R, dc=S, da=S, db=T)), (backward, dict(a=Q, b=R, dc=S, da=T, db=T)),
    (backward, dict(a=Q, b=R, dc=S, da=None, db=Q)), (backward, dict(a=Q, b=R, dc=S, da=R, db=None)),
    (backward, dict(a=Q, b=R, dc=S, z=T, ldz=8, act=1, da=P, db=T)),
    (backward, dict(a=Q, b=R, dc=S, da=P, db=T, dbias=T)),
    (loss, dict(x=Q, w=R, targets=S, dx=Q, dw=T)), (loss, dict(x=Q, w=R, targets=S, dx=None, dw=R)),
    (loss, dict(x=Q, w=R, targets=S, dx=T, dw=T)), (loss, dict(x=Q, w=R, targets=S, dx=T, dw=6 * P, mean=P)),
])
def test_outputs_that_are_inputs_or_one_another_are_refused(mm, call, change):
    rc, message = call(mm, **change)
    assert rc == ARGUMENT and "buffer of its own" in message


LONG = 2 ** 31 - 511


@pytest.mark.parametrize("call,change", [
    (forward, dict(m=LONG)), (forward, dict(n=LONG, ldb=2 ** 31, ldc=2 ** 31)), (forward, dict(k=LONG, lda=2 ** 31)),
    (backward, dict(m=LONG)), (loss, dict(rows=LONG)), (loss, dict(vocab=LONG)), (dropout, dict(cols=LONG, ldx=LONG, ldy=LONG)),
])
def test_dimensions_whose_tiles_pass_32_bits_are_refused(mm, call, change):
    rc, message = call(mm, **change)
    assert rc == SHAPE and "longer than" in message


@pytest.mark.parametrize("change", [dict(rows=2 ** 62), dict(rows=2 ** 60, ldx=2 ** 4, ldy=2 ** 4), dict(rows=2 ** 40, ldx=2 ** 40),
                                    dict(rows=2 ** 40, r=P, ldr=2 ** 40)])
def test_more_rows_than_addresses_are_refused(mm, change):
    """Their count of quads passes 64 bits: nothing would run, and the call would say that all is well."""
    rc, message = dropout(mm, **change)
    assert rc == SHAPE and "addresses" in message


def test_workspaces_of_the_longest_dimensions(mm):
    longest = LONG - 1
    for sizes in ((longest, 4, 4), (4, longest, 4), (4, 4, longest)):
        for backward_too in (False, True):
            assert mm.linear_workspace(*sizes, backward=backward_too, precision=1) >= 0
        assert mm.linear_cross_entropy_workspace(*sizes) > 0
    for too_long in ((LONG, 4, 4), (4, LONG, 4), (4, 4, LONG)):
        with pytest.raises(mm.MidmanGpuError):
            mm.linear_workspace(*too_long)
        with pytest.raises(mm.MidmanGpuError):
            mm.linear_cross_entropy_workspace(*too_long)


def test_no_rows_is_nothing_to_do(mm):
    assert forward(mm, m=0, a=None, c=None)[0] == 0
