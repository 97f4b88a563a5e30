"""CPU checks of the ring products and rotary positions: refusals of the C ABI (they come before anything touches a GPU) and
the phase steps against extended precision."""
import ctypes as C
import math

import numpy as np
import pytest

from openmm_amd import lib as L
from openmm_amd.rotary import rotary_phases
from tests.ring_fixtures import DIGITS_LOW

P = C.c_void_p(0x1000)   # never read: the calls below fail before a launch


def test_ring_product_refusals_without_gpu():
    lib = L.load_library()
    h = C.c_void_p()
    make = lambda w=P, eb=2, g=1, rows=4, cols=4, bw=37: lib.mmh_ring_weights_create(w, eb, g, rows, cols, bw, None, C.byref(h))
    assert lib.mmh_ring_weights_create(P, 2, 1, 4, 4, 37, None, None) == 2
    assert make(w=None) == 2
    assert make(eb=3) == 7 and make(bw=1) == 7 and make(bw=65) == 7
    assert make(g=0) == 3 and make(rows=0) == 3 and make(cols=0) == 3
    assert make(g=1 << 24) == 6 and make(rows=1 << 30) == 6 and make(cols=1 << 30) == 6
    assert not h and b"mmh_ring_weights_create" in lib.mmh_last_error()
    assert lib.mmh_ring_weights_info(None, None, None, None, None, None) == 2
    assert lib.mmh_ring_weights_destroy(None) == 0
    assert lib.mmh_ring_matmul(None, P, 4, None, 0, 1, None, None, 1, None, 0, P, 4, 0, None, 0, None) == 2
    assert lib.mmh_ring_matmul_workspace(None, 1, C.byref(C.c_size_t())) == 2


def test_rotary_refusals_without_gpu():
    lib = L.load_library()

    def call(x=P, xt=64, xh=16, t=2, h=4, d=16, pos=P, ph=P, rot=16, inter=0, amp=1.0, frac=12, bw=64, out=P, ot=64, oh=16):
        return lib.mmh_rotary(x, xt, xh, t, h, d, pos, ph, rot, inter, amp, frac, bw, out, ot, oh, None)

    assert call(t=0) == 0 and call(h=0) == 0      # nothing to do
    assert call(x=None) == 2 and call(out=None) == 2 and call(pos=None) == 2 and call(ph=None) == 2
    assert call(rot=15) == 3 and call(rot=18) == 3 and call(d=0, rot=0) == 3
    assert call(oh=15) == 3 and call(ot=15) == 3  # rows of the result would overlap
    assert call(oh=16, ot=63) == 3 and call(oh=31, ot=16) == 3 and call(oh=0, ot=0) == 3 and call(oh=0, ot=64) == 3
    assert call(t=1, oh=15) == 3 and call(h=1, ot=15) == 3 and call(h=1, ot=0) == 3
    assert call(frac=25) == 7 and call(frac=-1) == 7 and call(bw=1) == 7 and call(bw=65) == 7
    assert call(amp=0.0) == 7 and call(amp=17.0) == 7 and call(amp=float("nan")) == 7 and call(amp=-1.0) == 7
    assert call(d=4097) == 6 and call(h=65537) == 6 and call(t=1 << 31) == 6

    def pre(party=1, bw=64, heur=1):
        return lib.mmh_rotary_trunc_pre(party, P, 64, 16, 0, 4, 16, P, P, 16, 0, 1.0, 12, bw, 1, heur, P, None, None)

    assert pre() == 0
    assert pre(party=0) == 7 and pre(party=3) == 7 and pre(bw=3) == 7 and pre(bw=3, heur=0) == 0


def _thetas(rot, base=10000.0):
    return [np.longdouble(base) ** (np.longdouble(-2 * i) / rot) for i in range(rot // 2)]


TWO_PI = np.longdouble("6.28318530717958647692528676655900576839")


def _close(phases, thetas):
    """extended precision keeps 64 bits: the powers and quotients are a few units of 2^-63 off, relative"""
    for p, th in zip(phases, thetas):
        want = th / TWO_PI * np.longdouble(2) ** 64
        assert abs(np.longdouble(p) - want) <= 1 + want * np.longdouble(2) ** -58


@pytest.mark.parametrize("rot,base", [(2, 10000), (48, 10000), (128, 500000), (30, 10000)])
def test_phases(rot, base):
    p = rotary_phases(rot, base)
    assert len(p) == rot // 2 and all(0 <= v < 1 << 64 for v in p)
    assert p[0] == 2935890503282001226      # 2^64 / (2 pi), to the nearest integer
    _close(p, _thetas(rot, base))


def test_phases_scaled_for_long_contexts():
    th = _thetas(64)
    _close(rotary_phases(64, linear=4), [t / 4 for t in th])
    ntk = rotary_phases(64, ntk=8)
    _close(ntk, _thetas(64, np.longdouble(10000) * np.longdouble(8) ** (np.longdouble(64) / 62)))
    assert abs(ntk[-1] * 8 - rotary_phases(64)[-1]) <= 8      # the slowest pair is divided by the factor
    y = rotary_phases(64, yarn=(16, 4096))
    keep = [min(1, max(0, (t / TWO_PI * 4096 - 1) / 31)) for t in th]
    _close(y, [t * k + t / 16 * (1 - k) for t, k in zip(th, keep)])
    assert keep[0] == 1 and y[0] == rotary_phases(64)[0] and keep[-1] == 0 and any(0 < k < 1 for k in keep)
    assert rotary_phases(0) == []
    for bad in (dict(rot_dim=3), dict(rot_dim=-2), dict(rot_dim=4, base=0), dict(rot_dim=4, linear=0),
                dict(rot_dim=4, linear=2, ntk=2), dict(rot_dim=2, ntk=2), dict(rot_dim=4, yarn=(0, 4096)),
                dict(rot_dim=4, yarn=(2, 4096, 3, 3))):
        with pytest.raises(L.MMHError):
            rotary_phases(**bad)


def test_digits_low_is_all_minus_128():
    assert (int(DIGITS_LOW) - sum(-128 * 256 ** i for i in range(8))) % (1 << 64) == 0
