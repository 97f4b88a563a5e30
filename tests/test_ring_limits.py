"""CPU check: weights that no product call could take are refused before anything is allocated or read."""
import ctypes as C

from openmm_amd import lib as L

P = C.c_void_p(0x1000)   # never read


def test_weights_of_too_many_groups_are_refused():
    lib, h = L.load_library(), C.c_void_p()
    for groups in (32768, 65536, 1 << 24):
        assert lib.mmh_ring_weights_create(P, 2, groups, 1, 1, 37, None, C.byref(h)) == 6 and not h


def test_turns_of_two_to_the_32_lanes_are_refused():
    """heads of more than 4096 words take a workgroup of 256 lanes for each token"""
    lib = L.load_library()
    for tokens in (1 << 24, (1 << 31) - 1):
        assert lib.mmh_rotary(P, 4224, 128, tokens, 33, 128, P, P, 128, 0, 1.0, 12, 64, P, 4224, 128, None) == 6
        assert lib.mmh_rotary_trunc_pre(1, P, 4224, 128, tokens, 33, 128, P, P, 128, 0, 1.0, 12, 64, 1, 1, P, None, None) == 6
