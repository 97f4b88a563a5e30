"""Ring products at the ends of what their launches can count: layouts of more workgroups than one launch has, calls whose grid
would have 2^32 lanes."""
import ctypes as C

import numpy as np
import pytest

from tests.ring_fixtures import product, words

pytestmark = pytest.mark.gpu
SEED = 0x4C494D


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int64) if a.dtype == np.uint64 else a).cuda()


def fc(bw):
    from openmm_amd.ring_fc_ss import RingFCSS
    f = RingFCSS()
    f.setUp(bw)
    return f


# a layout launch has at most 2^24 lanes, one for 16 columns of an output: 2^25 of them here, and one output more
@pytest.mark.parametrize("groups,rows,cols", [(1, (1 << 23) + 1, 1), (3, 1 << 18, 120)])
def test_layout_of_several_rounds(groups, rows, cols):
    import torch
    r = np.random.default_rng(SEED)
    w = r.integers(-128, 127, (groups, rows, cols), dtype=np.int8, endpoint=True)
    x = words(SEED, (groups, cols))
    f = fc(64)
    rw = f.encodeWeights(dev(w))
    off = dev(np.arange(groups + 1))
    y = f.matMul(rw, dev(x), off).cpu().numpy().view(np.uint64)
    at = np.unique(np.concatenate([r.integers(0, rows, 5000), [0, rows - 1, rows // 2]]))
    assert np.array_equal(y[:, at], product(x, w[:, at], 64, np.arange(groups + 1)))


# 2^19 rows are 2^14 row tiles: with 2^9 output tiles the grid would have 2^23 workgroups of 512 lanes.  Nothing is launched.
@pytest.mark.parametrize("bw,rows", [(64, 131072), (32, 262144)])
def test_grids_of_two_to_the_32_lanes_are_refused(bw, rows):
    import torch
    from openmm_amd.lib import load_library
    f = fc(bw)
    rw = f.encodeWeights(torch.ones((rows, 4), dtype=torch.int8, device="cuda"))
    word = torch.zeros(1, dtype=torch.int64, device="cuda")
    p, n = C.c_void_p(word.data_ptr()), 1 << 19
    call = lambda n_rows: load_library().mmh_ring_matmul(rw.handle, p, 0, None, 0, n, None, None, n_rows, None, 0, p, rows, 0, None, 0, None)
    assert call(n) == 6
    assert int(word) == 0
