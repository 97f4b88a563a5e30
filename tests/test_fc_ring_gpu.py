"""Grouped ring products with cleartext weights (mmh_ring_matmul, RingFCSS) against the formula in 64-bit integers: every value
must be equal, the arithmetic is exact modulo 2^l."""
import ctypes as C

import numpy as np
import pytest

from tests.ring_fixtures import DIGITS_LOW, mask, product, words

pytestmark = pytest.mark.gpu
SEED = 0x52494E47


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


def weights(seed, shape, dtype, top=None):
    """whole range of the type by default, both ends and zero among them"""
    r = np.random.default_rng(seed)
    lo, hi = (np.iinfo(dtype).min, np.iinfo(dtype).max) if top is None else (-top, top)
    w = r.integers(lo, hi, shape, dtype=dtype, endpoint=True)
    ends = np.array([lo, hi, 0, -1, 1], dtype)
    flat = w.reshape(-1)
    flat[:min(5, flat.size)] = ends[:min(5, flat.size)]
    return w


def fc(bw):
    from openmm_amd.ring_fc_ss import RingFCSS
    f = RingFCSS()
    f.setUp(bw)
    return f


def digits_of(w, bw):
    """balanced base-256 digits that the widest weight needs (the representative next to zero, modulo 2^bw)"""
    need = 1
    for v in np.unique(w.astype(np.int64)):
        v = (int(v) + (1 << (bw - 1))) % (1 << bw) - (1 << (bw - 1))
        n = 1
        while not -128 * (256 ** n - 1) // 255 <= v <= 127 * (256 ** n - 1) // 255:
            n += 1
        need = max(need, n)
    return need


# one group: few and many rows, sizes around the tiles' 16 outputs and 64 columns, every ring's digit count and weight type
@pytest.mark.parametrize("tokens", [1, 4, 5, 8, 9, 31, 32, 33, 70])
@pytest.mark.parametrize("cols,rows", [(1, 1), (3, 300), (4, 16), (5, 31), (6, 32), (33, 33), (63, 15), (64, 16), (65, 17), (127, 256), (130, 300),
                                       (700, 257)])
def test_sizes(mm, tokens, cols, rows):
    w = weights(SEED + rows, (1, rows, cols), np.int16)
    x = words(SEED + cols, (tokens, cols))
    f = fc(64)
    y = f.matMul(f.encodeWeights(dev(w[0])), dev(x))
    assert np.array_equal(host(y), product(x, w, 64))


@pytest.mark.parametrize("tokens", [3, 40])
@pytest.mark.parametrize("bw", [2, 8, 31, 32, 33, 37, 40, 41, 44, 48, 49, 63, 64])
@pytest.mark.parametrize("dtype,top", [(np.int8, None), (np.int16, 32639), (np.int16, None), (np.int32, 1 << 22), (np.int32, 1 << 30),
                                       (np.int32, None), (np.int64, None)])
def test_rings_and_weight_types(mm, tokens, bw, dtype, top):
    w = weights(SEED + bw, (1, 21, 100), dtype, top)
    x = words(SEED + 2, (tokens, 100))      # bits above the ring in the inputs: taken modulo 2^bw
    x[0, :4] = [0, 1, (1 << 64) - 1, int(DIGITS_LOW)]
    f = fc(bw)
    rw = f.encodeWeights(dev(w))
    nx = 4 if bw <= 32 else 5 if bw <= 40 else 6 if bw <= 48 else 8
    need = digits_of(w, bw)
    assert rw.digits == (need if need <= 4 and need < nx else nx)
    assert np.array_equal(host(f.matMul(rw, dev(x))), product(x, w, bw))


# sums as large as they get: every digit of both operands -128, more columns than 32-bit sums hold
@pytest.mark.parametrize("tokens", [2, 33])
@pytest.mark.parametrize("dtype,value,cols", [(np.int8, -128, 131200), (np.int16, -32896 + 256, 65600), (np.int64, None, 16500)])
def test_largest_sums(mm, tokens, dtype, value, cols):
    w = np.full((1, 3, cols), DIGITS_LOW.view(np.int64) if value is None else value, dtype)
    x = np.full((tokens, cols), DIGITS_LOW, np.uint64)
    x[1] = words(SEED, cols)
    w[0, 1] = weights(SEED, cols, dtype)
    f = fc(64)
    assert np.array_equal(host(f.matMul(f.encodeWeights(dev(w)), dev(x))), product(x, w, 64))


# ragged groups, gathered rows, both shares, addends: few rows per group and many
@pytest.mark.parametrize("counts", [[1], [0, 5, 0], [3, 0, 1, 40, 16], [0, 0, 129, 31], [1] * 70 + [0] * 5 + [2] * 60, [0, 0]])
@pytest.mark.parametrize("bw", [37, 64])
def test_groups(mm, counts, bw):
    import torch
    g, n, cols, rows = len(counts), sum(counts), 77, 35
    w = weights(SEED + g, (g, rows, cols), np.int16, 32639)
    tokens = 13
    x, x1 = words(SEED + 3, (tokens, cols), bw), words(SEED + 4, (tokens, cols), bw)
    r = np.random.default_rng(SEED)
    idx = r.integers(0, tokens, n)
    add = words(SEED + 5, (n, rows), bw)
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    f = fc(bw)
    rw = f.encodeWeights(dev(w))
    y = f.matMul(rw, dev(x), dev(off), rows=dev(idx), share1=dev(x1), add=dev(add))
    assert np.array_equal(host(y), product(x, w, bw, off, idx, x1, add))
    # the same rows twice over, a bias for all rows, in place
    bias = words(SEED + 6, rows, bw)
    y = f.matMul(rw, dev(x), dev(off), rows=dev(idx), add=dev(bias))
    assert np.array_equal(host(y), product(x, w, bw, off, idx, None, bias))
    acc = dev(add)
    assert f.matMul(rw, dev(x), dev(off), rows=dev(idx), add=acc, out=acc) is acc
    assert np.array_equal(host(acc), product(x, w, bw, off, idx, None, add))


# rows behind the last group stay; offsets and row indices that lead outside stay inside
@pytest.mark.parametrize("scale", [1, 9])
def test_padding_and_bad_indices(mm, scale):
    import torch
    cols, rows, bw = 64, 20, 44
    counts = np.array([4, 0, 7]) * scale
    n = int(counts.sum()) + 10
    w = weights(SEED, (3, rows, cols), np.int16)
    x = words(SEED + 1, (n, cols))
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    f = fc(bw)
    rw = f.encodeWeights(dev(w))
    out = torch.full((n, rows), -7, dtype=torch.int64, device="cuda")
    f.matMul(rw, dev(x), dev(off), out=out)
    keep = np.full((n, rows), np.uint64(2 ** 64 - 7))
    assert np.array_equal(host(out), product(x, w, bw, off, out=keep))
    assert not host(f.matMul(rw, dev(x), dev(off)))[off[-1]:].any()      # a new tensor has zeros there
    idx = np.arange(n)
    idx[2], idx[5], idx[6] = -1, n, 1 << 62
    assert np.array_equal(host(f.matMul(rw, dev(x), dev(off), rows=dev(idx))), product(x, w, bw, off, idx))
    over = off.copy()
    over[-1] = n + 1000
    cut = off.copy()
    cut[-1] = n
    assert np.array_equal(host(f.matMul(rw, dev(x), dev(over))), product(x, w, bw, cut))
    under = off.copy()
    under[0] = -5
    assert np.array_equal(host(f.matMul(rw, dev(x), dev(under))), product(x, w, bw, off))


# offsets that no caller may pass (decreasing, overlapping, far outside): whatever comes out, nothing but the result is written
@pytest.mark.parametrize("cols,n", [(1, 70), (40, 6), (130, 70), (2048, 70)])
def test_offsets_out_of_order(mm, cols, n):
    import torch
    g, rows = 100, 37
    f = fc(64)
    rw = f.encodeWeights(dev(weights(SEED, (g, rows, cols), np.int16)))
    x = dev(words(SEED, (n, cols)))
    r = np.random.default_rng(SEED)
    for off in (r.integers(-5, n + 5, g + 1), r.integers(-1 << 62, 1 << 62, g + 1), np.where(np.arange(g + 1) % 2, n, 0)):
        buf = torch.full((n + 20, rows), 9, dtype=torch.int64, device="cuda")
        f.matMul(rw, x, dev(off.astype(np.int64)), out=buf[10:10 + n])
        f.matMul(rw, x, dev(off.astype(np.int64)))
        assert bool((buf[:10] == 9).all()) and bool((buf[10 + n:] == 9).all())


# strides and alignment: rows of wider arrays, odd strides, data at 8 modulo 16
@pytest.mark.parametrize("tokens", [5, 50])
@pytest.mark.parametrize("pad,shift", [(3, 0), (4, 1), (0, 1), (2, 0)])
def test_strides(mm, tokens, pad, shift):
    import torch
    cols, rows, bw = 90, 33, 64
    w = weights(SEED, (1, rows, cols), np.int16)
    f = fc(bw)
    rw = f.encodeWeights(dev(w))

    def wide(a, fill):
        buf = torch.full((a.shape[0] * (a.shape[1] + pad) + shift + 8,), fill, dtype=torch.int64, device="cuda")
        v = buf[shift:shift + a.shape[0] * (a.shape[1] + pad)].view(a.shape[0], a.shape[1] + pad)[:, :a.shape[1]]
        v.copy_(dev(a))
        return buf, v

    x, x1, add = words(SEED, (tokens, cols)), words(SEED + 1, (tokens, cols)), words(SEED + 2, (tokens, rows))
    buf, out = wide(np.zeros((tokens, rows), np.uint64), 77)
    out.fill_(77)
    f.matMul(rw, wide(x, 1)[1], share1=wide(x1, 2)[1], add=wide(add, 3)[1], out=out)
    assert np.array_equal(host(out.contiguous()), product(x, w, bw, None, None, x1, add))
    out.fill_(77)
    assert bool((buf == 77).all())      # nothing written between the rows
    # one row for all of them
    y = f.matMul(rw, dev(x[:1]).expand(tokens, cols), share1=dev(x1), add=dev(add[:1]).expand(tokens, rows))
    assert np.array_equal(host(y), product(np.repeat(x[:1], tokens, 0), w, bw, None, None, x1, add[0]))
    y = f.matMul(rw, dev(x), share1=dev(x1[:1]).expand(tokens, cols))
    assert np.array_equal(host(y), product(x, w, bw, None, None, np.repeat(x1[:1], tokens, 0)))


# k over several workgroups, whose sums a second launch joins (a few rows against long columns), and the same without scratch
@pytest.mark.parametrize("tokens,cols,rows", [(9, 2048, 40), (48, 1500, 300), (200, 4096, 33)])
@pytest.mark.parametrize("bw,dtype,top", [(64, np.int16, 32639), (37, np.int8, None), (64, np.int32, 1 << 29)])
def test_split_columns(mm, tokens, cols, rows, bw, dtype, top):
    import torch
    from openmm_amd.lib import check, load_library
    f = fc(bw)
    g, off = 3, np.array([0, tokens // 3, tokens // 3, tokens - 2])
    w, x, x1 = weights(SEED, (g, rows, cols), dtype, top), words(SEED, (tokens, cols)), words(SEED + 1, (tokens, cols))
    add = words(SEED + 2, (tokens, rows), bw)
    idx = np.random.default_rng(SEED).integers(0, tokens, tokens)
    idx[1] = -1
    rw = f.encodeWeights(dev(w))
    assert rw.workspace(tokens) > 0
    want = product(x, w, bw, off, idx, x1, add)
    args = dev(x), dev(x1), dev(idx), dev(off), dev(add)
    y = f.matMul(rw, args[0], args[3], rows=args[2], share1=args[1], add=args[4])
    assert np.array_equal(host(y), want)       # rows that no group has: zeros
    keep = torch.full((tokens, rows), 5, dtype=torch.int64, device="cuda")
    f.matMul(rw, args[0], args[3], rows=args[2], share1=args[1], add=args[4], out=keep)
    assert np.array_equal(host(keep)[:off[-1]], want[:off[-1]]) and bool((keep[off[-1]:] == 5).all())
    keep.fill_(5)
    p = [C.c_void_p(a.data_ptr()) for a in args]
    check(load_library().mmh_ring_matmul(rw.handle, p[0], cols, p[1], cols, tokens, p[2], p[3], tokens, p[4], rows,
                                         C.c_void_p(keep.data_ptr()), rows, 0, None, 0, None))
    assert np.array_equal(host(keep)[:off[-1]], want[:off[-1]]) and bool((keep[off[-1]:] == 5).all())


# many rows: tiles of twice the outputs for the digit counts that have them
@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("cols", [40, 200])
@pytest.mark.parametrize("bw,dtype", [(32, np.int8), (32, np.int16), (37, np.int8), (37, np.int16), (44, np.int8), (64, np.int8), (64, np.int16)])
def test_many_rows(mm, bw, dtype, cols, two):
    rows, tokens = 43, 8300
    off = np.array([0, 17, 17, 8290])
    w = weights(SEED, (3, rows, cols), dtype, None if dtype == np.int8 else 32639)
    x, x1 = words(SEED, (tokens, cols)), words(SEED + 1, (tokens, cols)) if two else None
    f = fc(bw)
    y = f.matMul(f.encodeWeights(dev(w)), dev(x), dev(off), share1=dev(x1) if two else None)
    assert np.array_equal(host(y), product(x, w, bw, off, None, x1))


def test_far_rows(mm):
    """rows further apart than 32 bits count, in words as in bytes"""
    import torch
    cols, rows, bw, far = 70, 20, 64, (1 << 29) + 8
    w = weights(SEED, (1, rows, cols), np.int16)
    x = words(SEED, (10, cols))
    f = fc(bw)
    rw = f.encodeWeights(dev(w))
    buf = torch.empty(9 * far + 128, dtype=torch.int64, device="cuda")     # 39 GB, of which ten rows are touched
    wide = buf.as_strided((10, cols), (far, 1))
    wide.copy_(dev(x))
    assert np.array_equal(host(f.matMul(rw, wide)), product(x, w, bw))
    assert np.array_equal(host(f.matMul(rw, wide[:5])), product(x[:5], w, bw))
    out = buf.as_strided((10, rows), (far, 1), 100)
    f.matMul(rw, dev(x), out=out)
    assert np.array_equal(host(out.contiguous()), product(x, w, bw))


@pytest.mark.parametrize("cols", [200, 2048])      # one launch, and two with scratch between them
def test_streams_and_replays(mm, cols):
    """two calls at once on two streams; captured calls replayed among eager work, each graph with scratch of its own"""
    import torch
    rows, bw = 100, 64
    f = fc(bw)
    w = [weights(SEED + i, (2, rows, cols), np.int16) for i in range(2)]
    x = [words(SEED + i, (60, cols)) for i in range(2)]
    off = np.array([0, 20, 60])
    rw, dx, doff = [f.encodeWeights(dev(v)) for v in w], [dev(v) for v in x], dev(off)
    want = [product(x[i], w[i], bw, off) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(f.matMul(rw[i], dx[i], doff))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(np.array_equal(host(y), want[i]) for y in got[i])
    assert (rw[0].workspace(60) > 0) == (cols == 2048)
    outs = [torch.zeros((60, rows), dtype=torch.int64, device="cuda") for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for k in range(2):
        with torch.cuda.graph(graphs[k]):
            f.matMul(rw[k], dx[0], doff, out=outs[k])
    expect = [[product(v, u, bw, off) for v in x] for u in w]
    for i in (0, 1, 0, 1):
        dx[0].copy_(dx[1] if i else dev(x[0]))
        for o in outs:
            o.fill_(-1)
        torch.cuda.synchronize()
        for k, s in enumerate(streams):      # both graphs at once
            with torch.cuda.stream(s):
                graphs[k].replay()
        eager = f.matMul(rw[0], dx[0], doff)
        torch.cuda.synchronize()
        assert all(np.array_equal(host(outs[k]), expect[k][i]) for k in range(2)) and torch.equal(outs[0], eager)


def test_refusals(mm):
    import torch
    from openmm_amd.lib import MMHError, load_library
    from openmm_amd.ring_fc_ss import RingFCSS
    f = fc(37)
    w = dev(weights(SEED, (2, 8, 12), np.int16))
    rw = f.encodeWeights(w)
    assert (rw.groups, rw.rows, rw.cols, rw.ring_bw) == (2, 8, 12, 37)
    x, off = dev(words(SEED, (4, 12))), dev(np.array([0, 1, 4]))
    z = lambda *s, **k: torch.zeros(s, dtype=k.get("dtype", torch.int64), device=k.get("device", "cuda"))
    assert f.matMul(rw, x[:0], dev(np.array([0, 0, 0]))).shape == (0, 8)
    bad = [
        (7, lambda: f.encodeWeights(w.cpu())), (7, lambda: f.encodeWeights(w.float())), (3, lambda: f.encodeWeights(w[0, 0])),
        (1, lambda: RingFCSS().encodeWeights(w)), (1, lambda: RingFCSS().matMul(rw, x, off)), (7, lambda: RingFCSS().setUp(65)),
        (7, lambda: fc(38).matMul(rw, x, off)), (7, lambda: f.matMul(None, x, off)),
        (2, lambda: f.matMul(rw, x)),                                  # two groups need offsets
        (3, lambda: f.matMul(rw, z(4, 11), off)), (7, lambda: f.matMul(rw, x.cpu(), off)), (7, lambda: f.matMul(rw, x.int(), off)),
        (7, lambda: f.matMul(rw, z(12, 4).t(), off)),                  # rows are not contiguous
        (3, lambda: f.matMul(rw, x, z(2))), (7, lambda: f.matMul(rw, x, off.int())), (7, lambda: f.matMul(rw, x, off.cpu())),
        (7, lambda: f.matMul(rw, x, off, rows=z(8)[::2])), (3, lambda: f.matMul(rw, x, off, share1=z(3, 12))),
        (3, lambda: f.matMul(rw, x, off, add=z(3, 8))), (3, lambda: f.matMul(rw, x, off, add=z(4, 7))),
        (3, lambda: f.matMul(rw, x, off, out=z(3, 8))), (3, lambda: f.matMul(rw, x, off, out=z(4, 9))),
    ]
    for code, call in bad:
        with pytest.raises(MMHError) as e:
            call()
        assert e.value.code == code
    lib, vp = load_library(), C.c_void_p
    px, po, y = vp(x.data_ptr()), vp(off.data_ptr()), z(4, 8)
    py = vp(y.data_ptr())
    raw = lambda x=px, ldx=12, x1=None, ldx1=0, t=4, rows=None, off=po, n=4, add=None, lda=0, out=py, ldo=8: \
        lib.mmh_ring_matmul(rw.handle, x, ldx, x1, ldx1, t, rows, off, n, add, lda, out, ldo, 0, None, 0, None)
    assert raw() == 0 and raw(n=0, x=None, out=None) == 0
    assert raw(x=None) == 2 and raw(out=None) == 2 and raw(off=None) == 2
    assert raw(t=0, rows=po) == 3 and raw(t=3) == 3 and raw(ldx=11) == 3 and raw(x1=px, ldx1=11) == 3 and raw(ldo=7) == 3 and raw(add=py, lda=7) == 3
    assert raw(n=(1 << 19) + 1, t=1 << 20) == 6
    rw.close()
    with pytest.raises(MMHError):
        f.matMul(rw, x, off)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(MMHError) as e:
        with torch.cuda.graph(graph):
            f.encodeWeights(w)          # allocates and waits
    assert e.value.code == 7
    torch.cuda.synchronize()
