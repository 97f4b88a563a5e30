"""Ring products whose columns exceed what a 32-bit sum holds; exact against the formula in 64-bit integers.

A workgroup of the tile kernel adds up 131071 // digits_of_the_weights // 64 steps of 64 columns in 32 bits (a segment), stores,
and goes on with the next.  Without scratch columns are not split, so one workgroup walks all of them."""
import ctypes as C

import numpy as np
import pytest

from tests.ring_fixtures import DIGITS_LOW, mask, words

pytestmark = pytest.mark.gpu
SEED = 0x4C4F4E47
FULL = 8      # as many digits as the ring has


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int64) if a.dtype == np.uint64 else a).cuda()


def host(t):
    return t.cpu().numpy().view(np.uint64)


def encoded(w, bw):
    from openmm_amd.ring_fc_ss import RingFCSS
    f = RingFCSS()
    f.setUp(bw)
    return f, f.encodeWeights(dev(w))


def digits_x(bw):
    return 4 if bw <= 32 else 5 if bw <= 40 else 6 if bw <= 48 else 8


def low_weights(bw, digits):
    """the weight whose `digits` balanced bytes are all -128 (the highest of as many has 127 in each)"""
    return -128 * ((256 ** digits - 1) // 255) if digits < 8 else int(DIGITS_LOW.view(np.int64))


def raw(rw, x, ldx, tokens, n, out, ldo, x1=None, ldx1=0, rows=None, off=None, add=None, ldadd=0, zero=0):
    """mmh_ring_matmul without scratch"""
    from openmm_amd.lib import check, load_library
    p = lambda t: None if t is None else C.c_void_p(t.data_ptr())
    check(load_library().mmh_ring_matmul(rw.handle, p(x), ldx, p(x1), ldx1, tokens, p(rows), p(off), n, p(add), ldadd, p(out), ldo,
                                         zero, None, 0, None))


def product(x, w, bw):
    """x [n, cols], w [rows, cols] -> [n, rows] mod 2^bw; numpy's uint64 arithmetic wraps"""
    return (x @ w.astype(np.int64).view(np.uint64).T) & mask(bw)


def long_case(bw, digits, cols, tokens):
    """rows of all -128 digits, where every product has the same sign and sums come nearest to their bound, and of random words"""
    x = words(SEED + cols, (tokens, cols))
    x[0] = DIGITS_LOW
    low = low_weights(bw, digits)
    w = np.random.default_rng(SEED + digits).integers(low, -low // 128 * 127, (3, cols), dtype=np.int64, endpoint=True) \
        if digits < FULL else words(SEED, (3, cols)).view(np.int64)
    w[0] = low
    return x, w


SEGMENTS = [(64, 1), (64, 2), (64, 3), (64, 4), (64, FULL), (44, 2), (44, FULL), (37, 1), (37, 3), (37, FULL), (32, 1), (32, 2), (32, FULL)]


# one column short of a segment, a segment, one column more (a step that mostly repeats), three steps more, two and a bit
@pytest.mark.parametrize("segments,extra", [(1, -1), (1, 0), (1, 1), (1, 192), (2, 65)])
@pytest.mark.parametrize("bw,digits", SEGMENTS)
def test_segments(bw, digits, segments, extra):
    import torch
    nx = digits_x(bw)
    stored = digits if digits <= 4 and digits < nx else nx
    cols, tokens, rows = segments * (131071 // stored // 64) * 64 + extra, 10, 3
    x, w = long_case(bw, min(digits, nx), cols, tokens)
    f, rw = encoded(w, bw)
    assert rw.digits == stored
    dx, add = dev(x), words(SEED + 3, (tokens, rows))
    idx = np.arange(tokens)[::-1].copy()
    idx[4] = -1
    xr = x[np.maximum(idx, 0)]
    xr[4] = 0
    want = product(xr, w, bw)
    out, didx, dadd = torch.full((tokens, rows), -1, dtype=torch.int64, device="cuda"), dev(idx), dev(add)
    raw(rw, dx, cols, tokens, tokens, out, rows, rows=didx)
    assert np.array_equal(host(out), want)
    raw(rw, dx, cols, tokens, tokens, out, rows, rows=didx, add=dadd, ldadd=rows)
    assert np.array_equal(host(out), (want + add) & mask(bw))
    raw(rw, dx, cols, tokens, tokens, dadd, rows, rows=didx, add=dadd, ldadd=rows)      # in place
    assert np.array_equal(host(dadd), (want + add) & mask(bw))
    # the second share, one row of it for all
    one = words(SEED + 4, (1, cols))
    raw(rw, dx, cols, tokens, tokens, out, rows, x1=dev(one), ldx1=0, rows=didx)
    xr = (x + one)[np.maximum(idx, 0)]
    xr[4] = 0
    assert np.array_equal(host(out), product(xr, w, bw))


# tiles of twice the outputs: 256 row tiles of one row of words
@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("bw,digits", [(32, 1), (32, 2), (37, 1), (37, 2), (44, 1)])
def test_segments_of_wide_tiles(bw, digits, two):
    import torch
    cols, tokens, rows = 131071 // digits // 64 * 64 + 65, 8192, 3
    x, w = long_case(bw, digits, cols, 2)
    f, rw = encoded(w, bw)
    out, add = torch.empty((tokens, rows), dtype=torch.int64, device="cuda"), words(SEED + 3, (tokens, rows))
    for row in range(2):
        if two:     # shares of the row
            share = words(SEED + 5, (1, cols))
            raw(rw, dev(x[row:row + 1] - share), 0, tokens, tokens, out, rows, x1=dev(share), ldx1=0, add=dev(add), ldadd=rows)
        else:
            raw(rw, dev(x[row:row + 1]), 0, tokens, tokens, out, rows, add=dev(add), ldadd=rows)
        assert np.array_equal(host(out), (product(x[row:row + 1], w, bw) + add) & mask(bw))


# 64-bit sums of a few rows: the most columns that their kernel takes (16 waves, a segment each), and one more
@pytest.mark.parametrize("digits", [1, 4, FULL])
def test_few_rows_at_their_bound(digits):
    stored = min(digits, 8)
    most = (131071 // stored // 64) * 1024 - 1
    for cols in (most, most + 1):
        x, w = long_case(64, digits, cols, 2)
        f, rw = encoded(w[:2], 64)
        y = f.matMul(rw, dev(x))
        assert np.array_equal(host(y), product(x, w[:2], 64)), cols


def test_one_row_of_more_outputs_than_the_kernel_for_few_rows_counts():
    """2^26 outputs: its grid would have 2^32 lanes"""
    import torch
    from openmm_amd.ring_fc_ss import RingFCSS
    outputs, cols = 1 << 26, 4
    w = torch.randint(-128, 128, (outputs, cols), dtype=torch.int8, device="cuda", generator=torch.Generator("cuda").manual_seed(SEED))
    x = words(SEED, (1, cols))
    f = RingFCSS()
    f.setUp(64)
    y = f.matMul(f.encodeWeights(w), dev(x))
    want = (w.to(torch.int64) * dev(x)).sum(dim=1)
    assert torch.equal(y[0], want)
