"""PreparedFCSS end to end on the GPU where one object serves several contexts, matrices and batches; values against the product
in 64-bit integers (tests/ring_fixtures.py)."""
import numpy as np
import pytest

from tests.ring_fixtures import mask, product, words

pytestmark = pytest.mark.gpu
SEED = 0x50524550
BW = 37


@pytest.fixture(scope="module")
def mm():
    import torch
    assert torch.cuda.is_available()
    import openmm_amd
    openmm_amd.load_library()
    return openmm_amd


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int64) if a.dtype == np.uint64 else a).cuda()


def host(t):
    return t.cpu().numpy().view(np.uint64)


def parties(mm, N, bob, alice, exact=True):
    from openmm_amd.lib import Sampler
    ctx = mm.Context(N, (60, 49), 1 << BW)
    smp = Sampler(ctx, key=bytes(range(32)))
    sk, pk = smp.keygen()
    bob.setUp(ctx, smp, sk_ntt=sk)
    alice.setUp(ctx, smp, pk_ntt=pk, exact=exact)


def weights(seed, groups, rows, cols, dtype=np.int64):
    w = np.random.default_rng(seed).integers(-1 << 12, 1 << 12, (groups, rows, cols), dtype=dtype)
    w[w == 0] = 1      # a block of zeros is refused (hom_fc_ss.cc:414-422)
    return w


def run(bob, alice, w, off, seed, meta=None):
    """one batch through both parties: the shares add up to W (x0 + x1) exactly"""
    from openmm_amd.hom_fc_ss import Meta
    rows, cols = w.shape[1:]
    meta = meta or Meta((rows, cols), (cols,), True)
    x0, x1 = words(seed, (off[-1], cols), BW), words(seed + 1, (off[-1], cols), BW)
    bob.finishMasks(alice.prepareRows(bob.prepareMasks(off[-1], meta), off))
    opened, y0 = bob.openInput(dev(x0))
    y1 = alice.online(opened, dev(x1))
    want = product((x0 + x1) & mask(BW), w, BW, off)
    assert np.array_equal((host(y0) + host(y1)) & mask(BW), want)


def test_one_object_over_several_contexts(mm):
    """N = 8192, then 4096 and back: plans, masks and weights are those of the current context"""
    from openmm_amd.hom_fc_ss import Meta
    from openmm_amd.ring_fc_ss import PreparedFCSS
    bob, alice = PreparedFCSS(), PreparedFCSS()
    rows, cols = 12, 5000
    w, meta = weights(SEED, 2, rows, cols), Meta((rows, cols), (cols,), True)
    for i, N in enumerate((8192, 4096, 8192)):
        parties(mm, N, bob, alice)
        alice.prepareWeights(dev(w), meta)
        run(bob, alice, w, [0, 2, 3], SEED + 10 * i)


def test_weights_replaced_between_rows_and_input(mm):
    from openmm_amd.hom_fc_ss import Meta
    from openmm_amd.lib import MMHError
    from openmm_amd.ring_fc_ss import PreparedFCSS
    bob, alice = PreparedFCSS(), PreparedFCSS()
    parties(mm, 4096, bob, alice)
    rows, cols, off = 7, 30, [0, 1, 1, 4]
    meta = Meta((rows, cols), (cols,), True)
    first, second = weights(SEED, 3, rows, cols), weights(SEED + 1, 3, rows, cols)
    alice.prepareWeights(dev(first), meta)
    bob.finishMasks(alice.prepareRows(bob.prepareMasks(4, meta), off))
    alice.prepareWeights(dev(second), meta)
    opened, _ = bob.openInput(dev(words(SEED, (4, cols), BW)))
    with pytest.raises(MMHError) as e:
        alice.online(opened, opened)
    assert e.value.code == 1
    run(bob, alice, second, off, SEED + 2)      # and the new weights serve rows prepared with them
    run(bob, alice, second, [0, 0, 0, 0], SEED + 3)     # no rows at all


def test_input_shape_is_checked_each_time(mm):
    from openmm_amd.hom_fc_ss import Meta
    from openmm_amd.lib import MMHError
    from openmm_amd.ring_fc_ss import PreparedFCSS
    bob, alice = PreparedFCSS(), PreparedFCSS()
    parties(mm, 4096, bob, alice)
    bob.prepareMasks(1, Meta((7, 30), (30,), True))
    with pytest.raises(MMHError) as e:
        bob.prepareMasks(1, Meta((7, 30), (20,), True))
    assert e.value.code == 7
