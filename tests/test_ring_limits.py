"""CPU check: weights that no product call could take are refused before anything is allocated or read."""
import ctypes as C

from openmm_amd import lib as L

P = C.c_void_p(0x1000)   # never read


def test_weights_of_too_many_groups_are_refused():
    lib, h = L.load_library(), C.c_void_p()
    for groups in (32768, 65536, 1 << 24):
        assert lib.mmh_ring_weights_create(P, 2, groups, 1, 1, 37, None, C.byref(h)) == 6 and not h
