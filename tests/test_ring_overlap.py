"""CPU checks of which results of a ring product or a turn are refused because they lie on top of an operand: workgroups read
operands while others write, so such a call has no defined result."""
import random
from types import SimpleNamespace

import pytest
import torch

from openmm_amd.lib import MMHError, rows_overlap
from openmm_amd import ring_fc_ss

WORD = 8


def test_rows_overlap_against_sets_of_words():
    rng, seen = random.Random(1), [0, 0]

    def words(p, width, dims):
        at = [p // WORD]
        for n, s in dims:
            at = [v + i * s for v in at for i in range(n)]
        return {v + k for v in at for k in range(width)}

    for _ in range(20000):
        depth = rng.choice([1, 1, 1, 2])
        one = lambda: (WORD * rng.randint(0, 60), rng.randint(rng.random() > 0.05, 6),
                       tuple((rng.randint(rng.random() > 0.03, 5), rng.choice([0, 1, 3, 7, 8, 10, 20])) for _ in range(depth)))
        a, b = one(), one()
        if rng.random() < 0.5:
            b = (b[0], b[1], tuple((n, s) for (n, _), (_, s) in zip(b[2], a[2])))
        want = bool(words(*a) & words(*b))
        seen[want] += 1
        assert rows_overlap(a, b) == want, (a, b)
    assert min(seen) > 1000


@pytest.fixture
def call(monkeypatch):
    """matMul on host tensors: returns what it would have launched"""
    launched = []
    w = ring_fc_ss.RingWeights.__new__(ring_fc_ss.RingWeights)
    w.handle, w.ring_bw, w.device, w.groups, w.rows, w.cols, w._words = 1, 64, -1, 1, 6, 6, {n: 0 for n in range(100)}
    w.lib = SimpleNamespace(mmh_ring_matmul=lambda *a: launched.append(a) or 0, mmh_ring_weights_destroy=lambda h: 0)
    monkeypatch.setattr(ring_fc_ss, "_stream_of", lambda dev: 0)
    f = ring_fc_ss.RingFCSS()
    f.setUp(64)

    def run(*args, **kwargs):
        launched.clear()
        f.matMul(w, *args, **kwargs)
        assert len(launched) == 1
    return run


def z(*shape):
    return torch.zeros(shape, dtype=torch.int64)


def test_product_results_beside_their_operands_are_taken(call):
    x, wide = z(5, 6), z(5, 24)
    call(x, out=z(5, 6))
    call(wide[:, :6], share1=wide[:, 6:12], add=wide[:, 12:18], out=wide[:, 18:])
    call(wide[:, :6], add=wide[:, 6:12], out=wide[:, 6:12])      # add is out
    buf = z(10, 6)
    call(buf[:5], out=buf[5:], offsets=z(2), rows=z(5))
    call(buf[:5], add=buf[7], out=buf[:0].new_zeros(5, 6))
    call(buf[:1], add=buf[1], out=buf[1:2])                      # one row: the same as add is out
    call(buf[:1], add=buf[1:2], out=buf[1:2])


def test_product_results_on_top_of_operands_are_refused(call):
    x, buf, flat = z(5, 6), z(12, 6), z(400)
    bad = [
        lambda: call(x, out=x), lambda: call(buf[:5], out=buf[4:9]), lambda: call(x, share1=buf[:5], out=buf[3:8]),
        lambda: call(x, add=buf[:5], out=buf[1:6]),                                       # rows above: read and written by others
        lambda: call(x, add=buf[2], out=buf[:5]),                                         # one row for all
        lambda: call(x, add=flat[:60].view(5, 12)[:, :6], out=flat[:40].view(5, 8)[:, :6]),
        lambda: call(flat[:60].view(5, 12)[:, :6], out=flat[5:65].view(5, 12)[:, :6]),
        lambda: call(x, rows=flat[3:8], out=flat[:30].view(5, 6)), lambda: call(x, offsets=flat[28:30], out=flat[:30].view(5, 6)),
    ]
    for i, b in enumerate(bad):
        with pytest.raises(MMHError) as e:
            b()
            pytest.fail(f"case {i} was accepted")
        assert e.value.code == 7, i


@pytest.fixture
def turn(monkeypatch):
    """rotate on host tensors of heads of 4 words: returns what it would have launched"""
    from openmm_amd import rotary
    launched = []
    r = rotary.Rotary.__new__(rotary.Rotary)
    r.head_dim, r._dev, r.phases = 4, -1, z(2)
    r._pairs = (r.phases.data_ptr(), 4, False, 1.0, 12, 64)
    r.lib = SimpleNamespace(mmh_rotary=None)
    r._call = lambda fn, args: launched.append(args)

    def run(x, positions, out):
        launched.clear()
        r.rotate(x, positions, out=out)
        assert len(launched) == 1
    run.phases = r.phases
    return run


def test_turns_beside_their_operands_are_taken(turn):
    x, wide, pos = z(5, 3, 4), z(5, 9, 4), z(5)
    turn(x, pos, z(5, 3, 4))
    turn(x, pos, x)
    turn(wide[:, :3], pos, wide[:, :3])
    turn(wide[:, :3], pos, wide[:, 3:6])
    turn(wide[:, ::2][:, :3], pos, wide[:, 1::2][:, :3])          # heads of two turns between one another
    turn(wide[:, 0:1], pos, wide[:, 8:9])
    turn(x.expand(5, 3, 4)[:1].expand(5, 3, 4), pos, z(5, 3, 4))  # one token for all
    turn(x[:0], pos[:0], x[:0])


def test_turns_on_top_of_operands_are_refused(turn):
    wide, flat, pos = z(5, 9, 4), z(200), z(5)
    bad = [
        lambda: turn(wide[:, :3], pos, wide[:, 2:5]), lambda: turn(wide[:4, :3], pos[:4], wide[1:, :3]),
        lambda: turn(flat[:60].view(5, 3, 4), pos, flat[1:61].view(5, 3, 4)),
        lambda: turn(flat[:60].view(5, 3, 4), pos, flat[:60].view(3, 5, 4).transpose(0, 1)),     # the same words in another order
        lambda: turn(wide[:1, :3].expand(5, 3, 4), pos, wide[:, :3]),
        lambda: turn(wide[:, :3], flat[30:35], flat[:60].view(5, 3, 4)),
    ]
    for i, b in enumerate(bad):
        with pytest.raises(MMHError) as e:
            b()
            pytest.fail(f"case {i} was accepted")
        assert e.value.code == 7, i


def test_one_operand_in_place_does_not_excuse_another(call, turn):
    """the addend may be the result and x may be turned in place, but nothing else that starts at the same word"""
    acc, x = z(5, 6), z(5, 6)
    flat = z(60)
    same = flat.view(5, 3, 4)
    for bad in (lambda: call(acc, add=acc, out=acc), lambda: call(x, share1=acc, add=acc, out=acc),
                lambda: call(x, rows=acc.view(-1)[:5], add=acc, out=acc), lambda: turn(same, flat[:5], same)):
        with pytest.raises(MMHError) as e:
            bad()
        assert e.value.code == 7
