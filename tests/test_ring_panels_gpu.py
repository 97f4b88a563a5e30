"""Ring products of many outputs (more than one panel of output tiles), and with a second share at every digit count; exact against
the formula in 64-bit integers.  Output tiles are 256 or 512 outputs, a panel is 16 of them."""
import numpy as np
import pytest

from tests.ring_fixtures import DIGITS_LOW, mask, words
from tests.test_ring_long_gpu import dev, encoded, host, product

pytestmark = pytest.mark.gpu
SEED = 0x50414E45


def grouped(x, w, bw, off, idx, x1, add):
    out = np.zeros((len(idx), w.shape[1]), np.uint64)
    xs = x if x1 is None else x + x1
    for g in range(len(off) - 1):
        r = slice(off[g], off[g + 1])
        out[r] = product(xs[idx[r]], w[g], bw) if add is None else (product(xs[idx[r]], w[g], bw) + add[r]) & mask(bw)
    return out


@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("bw,dtype,n,outputs,cols", [
    (64, np.int16, 200, 4096, 40), (64, np.int16, 200, 4097, 40), (64, np.int16, 90, 4352, 65), (64, np.int16, 200, 8200, 5),
    (37, np.int16, 150, 4400, 70), (44, np.int32, 60, 8200, 6), (64, np.int64, 60, 4352, 40),
    (64, np.int16, 50, 4352, 1500),                                                   # columns split as well
    (32, np.int8, 470, 8200, 40), (32, np.int16, 470, 8193, 70), (37, np.int8, 470, 8705, 6), (44, np.int8, 470, 8200, 40),   # 512 across
    (32, np.int8, 4100, 600, 40), (32, np.int16, 4100, 513, 64), (37, np.int16, 4100, 1030, 40), (64, np.int16, 300, 70000, 4)])
def test_panels(bw, dtype, n, outputs, cols, two):
    """groups of odd sizes, one of them empty, rows in front of the first group and behind the last"""
    import torch
    r = np.random.default_rng(SEED + outputs)
    groups, tokens = 4, 50
    off = np.array([3, n // 5, n // 5, n // 2 + 1, n - 7])
    lo, hi = (-32896, 32639) if dtype == np.int16 else (np.iinfo(dtype).min, np.iinfo(dtype).max)
    w = r.integers(max(lo, np.iinfo(dtype).min), hi, (groups, outputs, cols), dtype=dtype, endpoint=True)
    x, x1 = words(SEED, (tokens, cols)), words(SEED + 1, (tokens, cols)) if two else None
    idx, add = r.integers(0, tokens, n), words(SEED + 2, (n, outputs), bw)
    f, rw = encoded(w, bw)
    args = dict(rows=dev(idx), share1=dev(x1) if two else None)
    want = grouped(x, w, bw, off, idx, x1, None)
    got = f.matMul(rw, dev(x), dev(off), **args)        # a new result has zeros where no group is
    assert np.array_equal(host(got), want)
    kept = torch.full((n, outputs), 5, dtype=torch.int64, device="cuda")
    f.matMul(rw, dev(x), dev(off), add=dev(add), out=kept, **args)
    want = grouped(x, w, bw, off, idx, x1, add)
    want[:off[0]], want[off[-1]:] = 5, 5
    assert np.array_equal(host(kept), want)


# every digit count of both operands in the tile kernels and in the one for few rows, with the second share
@pytest.mark.parametrize("tokens", [3, 7, 40])
@pytest.mark.parametrize("bw", [31, 32, 37, 40, 44, 48, 49, 64])
@pytest.mark.parametrize("dtype,top", [(np.int8, None), (np.int16, 32639), (np.int32, 1 << 22), (np.int32, 1 << 30), (np.int64, None)])
def test_second_share_with_every_digit_count(tokens, bw, dtype, top):
    r = np.random.default_rng(SEED + bw)
    lo, hi = (np.iinfo(dtype).min, np.iinfo(dtype).max) if top is None else (-top, top)
    w = r.integers(lo, hi, (37, 150), dtype=dtype, endpoint=True)
    w[0, :3] = lo, hi, 0
    x, x1 = words(SEED + 2, (tokens, 150)), words(SEED + 3, (tokens, 150))
    x[0, :4], x1[0, :4] = [0, 1, (1 << 64) - 1, int(DIGITS_LOW)], [0, (1 << 64) - 1, (1 << 64) - 1, 0]
    f, rw = encoded(w, bw)
    assert np.array_equal(host(f.matMul(rw, dev(x), share1=dev(x1))), product(x + x1, w, bw))
