"""Rotary positions on shares (mmh_rotary, mmh_rotary_trunc_pre, Rotary) against the formula in integers with coefficients from
extended precision: every value must be equal.  The kernel's coefficients are a few units of 2^-53 off before they are rounded to
at most 24 + 4 fraction bits, so one of them differs from the correctly rounded one with a chance below 2^-20; the seeds are
fixed."""
import numpy as np
import pytest

from tests.ring_fixtures import coefficients, mask, product, rotary, words

pytestmark = pytest.mark.gpu
SEED = 0x524F5459


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
    return t.contiguous().cpu().numpy().view(np.uint64)


def positions(seed, n):
    """near, far, and the ends of 64 bits"""
    r = np.random.default_rng(seed)
    p = np.where(r.random(n) < 0.5, r.integers(0, 5000, n), r.integers(-1 << 62, 1 << 62, n))
    ends = np.array([0, -1, (1 << 63) - 1, -1 << 63, 1 << 31, (1 << 32) + 1, 1], np.int64)
    p[:min(n, 7)] = ends[:min(n, 7)]
    return p


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 40, 128, 128), (3, 5, 7, 6), (9, 3, 80, 30), (2, 2, 96, 48), (5, 1, 64, 0),
                                                  (4, 3, 130, 2), (300, 2, 16, 16), (2, 1, 1030, 1026), (33, 7, 3, 2)])
def test_shapes(mm, interleaved, tokens, heads, dim, rot):
    from openmm_amd.rotary import Rotary, rotary_phases
    bw, frac = 64, 12
    x, pos, ph = words(SEED + dim, (tokens, heads, dim)), positions(SEED, tokens), rotary_phases(rot)
    y = Rotary(ph, dim, frac, bw, interleaved).rotate(dev(x), dev(pos))
    assert np.array_equal(host(y), rotary(x, pos, ph, frac, bw, interleaved))


@pytest.mark.parametrize("bw", [2, 13, 32, 37, 41, 63, 64])
@pytest.mark.parametrize("frac,amplitude", [(0, 1.0), (10, 1.0), (24, 1.0), (16, 1.25), (24, 16.0), (12, 0.01)])
def test_rings_and_scales(mm, bw, frac, amplitude):
    from openmm_amd.rotary import Rotary, rotary_phases
    x, pos = words(SEED + bw, (20, 3, 24)), positions(SEED + 1, 20)
    ph = rotary_phases(20, 500000, yarn=(8, 2048))
    y = Rotary(ph, 24, frac, bw, amplitude=amplitude).rotate(dev(x), dev(pos))
    assert np.array_equal(host(y), rotary(x, pos, ph, frac, bw, amplitude=amplitude))


def test_quadrants_and_ties(mm):
    """phases at and next to multiples of an eighth of a turn; 30 degrees has a sine of exactly one half"""
    from openmm_amd.rotary import Rotary
    eighth = 1 << 61
    ph = [(k * eighth + d) % (1 << 64) for k in range(8) for d in (-1, 0, 1)] + [(1 << 64) // 12]
    pos = np.array([1, -1, 0, 3, 5], np.int64)
    x = np.zeros((5, 1, 2 * len(ph)), np.uint64)
    x[:, :, :len(ph)] = 1      # the result is the coefficients themselves
    for frac in (1, 11, 24):
        got = host(Rotary(ph, 2 * len(ph), frac, 64).rotate(dev(x), dev(pos)))[:, 0]
        c, s = coefficients(pos, ph, frac)
        assert np.array_equal(got[:, :len(ph)], c) and np.array_equal(got[:, len(ph):], s)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(32, 32), (33, 20), (24, 12)])
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 0), (0, 1), (0, 2), (1, 3)])
def test_strides(mm, interleaved, dim, rot, shift, pad):
    """heads of wider rows, odd strides, data at 8 modulo 16, in place, and nothing written between the rows"""
    import torch
    from openmm_amd.rotary import Rotary, rotary_phases
    t, h, bw, frac = 6, 3, 44, 9
    x, pos, ph = words(SEED, (t, h, dim), bw), positions(SEED, t), rotary_phases(rot)
    want = rotary(x, pos, ph, frac, bw, interleaved)
    r = Rotary(ph, dim, frac, bw, interleaved)

    def wide():
        buf = torch.full((shift + t * ((h + 1) * (dim + pad) + pad),), 77, dtype=torch.int64, device="cuda")
        return buf, buf[shift:].view(t, -1)[:, :h * (dim + pad)].unflatten(1, (h, dim + pad))[:, :, :dim]

    _, v = wide()
    v.copy_(dev(x))
    assert np.array_equal(host(r.rotate(v, dev(pos))), want)
    buf, out = wide()
    r.rotate(v, dev(pos), out=out)
    assert np.array_equal(host(out), want)
    out.fill_(77)
    assert bool((buf == 77).all())
    assert r.rotate(v, dev(pos), out=v) is v and np.array_equal(host(v), want)
    # heads-first storage: a transposed view
    y = dev(np.ascontiguousarray(x.transpose(1, 0, 2))).transpose(0, 1)
    assert np.array_equal(host(r.rotate(y, dev(pos))), want)


def test_far_tokens(mm):
    """tokens further apart than 32 bits count"""
    import torch
    from openmm_amd.rotary import Rotary, rotary_phases
    far = (1 << 29) + 16
    x, pos, ph = words(SEED, (9, 2, 16)), positions(SEED, 9), rotary_phases(16)
    buf = torch.empty(8 * far + 64, dtype=torch.int64, device="cuda")     # 34 GB, of which nine rows are touched
    wide = buf.as_strided((9, 2, 16), (far, 16, 1))
    wide.copy_(dev(x))
    r = Rotary(ph, 16, 12, 64)
    want = rotary(x, pos, ph, 12, 64)
    assert np.array_equal(host(r.rotate(wide, dev(pos))), want)
    assert np.array_equal(host(r.rotate(wide, dev(pos), out=wide)), want)


@pytest.mark.parametrize("party", [1, 2])
@pytest.mark.parametrize("signed_arith", [True, False])
@pytest.mark.parametrize("heuristic", [True, False])
@pytest.mark.parametrize("bw", [4, 37, 64])
@pytest.mark.parametrize("interleaved,dim,rot", [(False, 32, 32), (True, 31, 10), (False, 31, 10), (True, 32, 16)])
def test_truncate_pre(mm, party, signed_arith, heuristic, bw, interleaved, dim, rot):
    """bit for bit the turn followed by mmh_trunc_pre"""
    import torch
    from openmm_amd.lib import check, dptr, load_library
    from openmm_amd.rotary import Rotary, rotary_phases
    r = Rotary(rotary_phases(rot), dim, 8, bw, interleaved)
    x, pos = dev(words(SEED + bw, (11, 3, dim))), dev(positions(SEED, 11))
    adj, cmp = r.truncate_pre(party, x, pos, signed_arith, heuristic)
    y = r.rotate(x, pos)
    a, c = torch.empty_like(y), torch.empty_like(y)
    check(load_library().mmh_trunc_pre(party, dptr(y), y.numel(), bw, int(signed_arith), int(heuristic), dptr(a), dptr(c), None))
    assert torch.equal(adj, a)
    assert cmp is None if heuristic else torch.equal(cmp, c)


def test_streams_and_replays(mm):
    import torch
    from openmm_amd.rotary import Rotary, rotary_phases
    ph, bw = rotary_phases(64), 64
    r = Rotary(ph, 64, 12, bw)
    x, pos = [words(SEED + i, (50, 8, 64)) for i in range(2)], [positions(SEED + i, 50) for i in range(2)]
    want = [rotary(x[i], pos[i], ph, 12, bw) for i in range(2)]
    dx, dp, streams = [dev(v) for v in x], [dev(v) for v in pos], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(r.rotate(dx[i], dp[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(np.array_equal(host(y), want[i]) for y in got[i])
    out = torch.zeros_like(dx[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.rotate(dx[0], dp[0], out=out)
    for i in (0, 1, 0, 1):
        dx[0].copy_(dx[1] if i else dev(x[0]))
        dp[0].copy_(dp[1] if i else dev(pos[0]))
        out.fill_(-1)
        graph.replay()
        eager = r.rotate(dx[0], dp[0])
        torch.cuda.synchronize()
        assert np.array_equal(host(out), want[i]) and torch.equal(out, eager)


def test_refusals(mm):
    import torch
    from openmm_amd.lib import MMHError
    from openmm_amd.rotary import Rotary, rotary_phases
    from openmm_amd.truncation import Truncation
    ph = rotary_phases(16)
    r = Rotary(ph, 16, 12, 64)
    z = lambda *s: torch.zeros(s, dtype=torch.int64, device="cuda")
    x, pos = z(4, 2, 16), z(4)
    assert r.rotate(x[:0], pos[:0]).shape == (0, 2, 16) and r.rotate(x[:, :0], pos).shape == (4, 0, 16)
    bad = [
        (3, lambda: Rotary(ph, 15, 12, 64)), (7, lambda: Rotary(ph, 16, 25, 64)), (7, lambda: Rotary(ph, 16, 12, 65)),
        (7, lambda: Rotary(ph, 16, 12, 64, amplitude=0.0)), (7, lambda: Rotary(ph, 16, 12, 64, amplitude=float("nan"))),
        (7, lambda: Rotary(z(8).cpu(), 16, 12, 64)), (7, lambda: Rotary(z(8).int(), 16, 12, 64)),
        (7, lambda: Rotary(z(16)[::2], 16, 12, 64)),
        (7, lambda: r.rotate(x.cpu(), pos)), (7, lambda: r.rotate(x.int(), pos)), (7, lambda: r.rotate(x[0], pos)),
        (3, lambda: r.rotate(z(4, 2, 15), pos)), (7, lambda: r.rotate(z(4, 16, 2).transpose(1, 2), pos)),
        (3, lambda: r.rotate(x, z(3))), (7, lambda: r.rotate(x, pos.int())), (7, lambda: r.rotate(x, pos.cpu())),
        (7, lambda: r.rotate(x, z(8)[::2])), (3, lambda: r.rotate(x, pos, out=z(4, 3, 16))),
        (3, lambda: r.rotate(x, pos, out=z(1, 2, 16).expand(4, 2, 16))),      # rows of the result on top of each other
        (7, lambda: Truncation(1, None).truncate_rotary(r, x, pos, 0)), (7, lambda: Truncation(2, None).truncate_rotary(r, x, pos, 62)),
        (7, lambda: r.truncate_pre(3, x, pos)), (7, lambda: Rotary(ph, 16, 0, 3).truncate_pre(1, x, pos)),
    ]
    for code, call in bad:
        with pytest.raises(MMHError) as e:
            call()
        assert e.value.code == code


def _two_parties(run):
    import threading
    import torch
    got, failed = [None, None, None], []

    def go(party):
        try:
            got[party] = run(party)
            torch.cuda.synchronize()
        except BaseException as e:      # noqa: BLE001 - reported by the main thread
            failed.append(e)

    threads = [threading.Thread(target=go, args=(p,)) for p in (1, 2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    if failed:
        raise failed[0]
    return got


def test_two_party_projection_turn_truncation(mm):
    """A query projection in two adapters' weights, the turn and one truncation, between two parties: the ciphertext product of
    the client's masks runs ahead and the online product takes opened inputs (PreparedFCSS), then Truncation.truncate_rotary.
    The shares add up to the turned projection within the one unit the truncation gives up, plus the unit of its floor."""
    from openmm_amd.hom_fc_ss import Meta
    from openmm_amd.lib import MMHError, Sampler
    from openmm_amd.ring_fc_ss import PreparedFCSS
    from openmm_amd.rotary import Rotary, rotary_phases
    from openmm_amd.truncation import IdealAux, Truncation
    bw, scale, frac = 44, 8, 10
    tokens, cols, heads, dim = 9, 48, 2, 16
    rows, groups = heads * dim, 2
    off, ring = np.array([0, 4, 9]), 1 << bw
    r = np.random.default_rng(SEED)
    xs = r.integers(-1 << scale, 1 << scale, (tokens, cols))                # values in (-1, 1)
    w = r.integers(-1 << scale, 1 << scale, (groups, rows, cols))
    w[w == 0] = 1                                                           # HomFCSS refuses blocks of zeros
    pos = r.integers(0, 100000, tokens)
    x0 = words(SEED, (tokens, cols), bw)
    x1 = (xs.astype(np.int64).view(np.uint64) - x0) & mask(bw)
    ctx = mm.Context(4096, (60, 49), ring)
    smp = Sampler(ctx, key=bytes(range(32)))
    sk, pk = smp.keygen()
    meta = Meta((rows, cols), (cols,), True)
    want = product(xs.astype(np.int64).view(np.uint64), w, bw, off)
    signed = lambda v: ((v.astype(object) + ring // 2) % ring - ring // 2)
    for exact in (False, True):
        bob, alice = PreparedFCSS(), PreparedFCSS()
        bob.setUp(ctx, smp, sk_ntt=sk)
        alice.setUp(ctx, smp, pk_ntt=pk, exact=exact)
        alice.prepareWeights(dev(w), meta)
        bob.finishMasks(alice.prepareRows(bob.prepareMasks(tokens, meta), off))
        opened, y0 = bob.openInput(dev(x0))
        y1 = alice.online(opened, dev(x1))
        err = signed((host(y0) + host(y1) - want) & mask(bw)).astype(np.int64)
        assert np.abs(err).max() <= (0 if exact else 1)
        for again in (lambda: bob.openInput(dev(x0)), lambda: alice.online(opened, dev(x1))):   # masks serve once
            with pytest.raises(MMHError) as e:
                again()
            assert e.value.code == 1
    # each party turns and truncates its own share: one truncation takes off the product's and the turn's scale
    ph, aux = rotary_phases(dim), IdealAux()
    share = {1: y1, 2: y0}

    def party(p):
        rot = Rotary(ph, dim, frac, bw)
        return Truncation(p, None, aux=aux).truncate_rotary(rot, share[p].view(tokens, heads, dim), dev(pos), scale + frac)

    got = _two_parties(party)
    total = (host(got[1]) + host(got[2])) & mask(bw)
    turned = rotary(want.reshape(tokens, heads, dim), pos, ph, frac, bw)
    exact = signed(turned) // (1 << (scale + frac))
    assert np.abs((signed(total) - exact).astype(np.int64)).max() <= 1
    # and without the heuristic, through the comparison
    aux = IdealAux()

    def party2(p):
        rot = Rotary(ph, dim, frac, bw)
        return Truncation(p, None, aux=aux).truncate_rotary(rot, share[p].view(tokens, heads, dim), dev(pos), scale + frac,
                                                            apply_msb0_heuristic=False)

    got = _two_parties(party2)
    total = (host(got[1]) + host(got[2])) & mask(bw)
    assert np.abs((signed(total) - exact).astype(np.int64)).max() <= 1
