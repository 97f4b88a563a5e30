"""CPU checks of PreparedFCSS's phases: nothing prepared for one set-up, matrix or batch of rows serves the next."""
from types import SimpleNamespace

import pytest
import torch

from openmm_amd.hom_fc_ss import Meta
from openmm_amd.lib import MMHError
from openmm_amd.ring_fc_ss import PreparedFCSS

META = Meta((3, 4), (4,), True)


def context(N=4096, t=1 << 20, q=(97, 193), device=0):
    return SimpleNamespace(N=N, L=len(q), t=t, q=list(q), device=device)


def sampler(ctx):
    return SimpleNamespace(ctx=ctx)


def ready(layer, rows=2):
    """as after prepareMasks, finishMasks, prepareWeights and prepareRows"""
    layer._meta = META
    layer._masks, layer._y0 = torch.zeros((rows, 4), dtype=torch.int64), torch.zeros((rows, 3), dtype=torch.int64)
    layer.weights, layer._plain = SimpleNamespace(groups=1, rows=3), [None]
    layer._s, layer._offsets = torch.zeros((rows, 3), dtype=torch.int64), torch.tensor([0, rows])
    return layer


def code_of(call):
    with pytest.raises(MMHError) as e:
        call()
    return e.value.code


@pytest.fixture
def layer():
    p = PreparedFCSS()
    p.setUp(context(), sampler(context()))
    p.ring.encodeWeights = lambda w: SimpleNamespace(groups=w.shape[0], rows=w.shape[1])
    p.fc.encodeWeightMatrix = lambda m, meta: None
    return p


x = torch.zeros((2, 4), dtype=torch.int64)


def test_setup_drops_what_was_prepared(layer):
    ready(layer)
    other = context(N=8192)
    layer.setUp(other, sampler(other))
    assert code_of(lambda: layer.online(x, x)) == 1
    assert code_of(lambda: layer.openInput(x)) == 1
    assert code_of(lambda: layer.finishMasks([None, None])) == 3
    assert code_of(lambda: layer.prepareRows([None, None], [0, 2])) == 1


def test_new_weights_drop_prepared_rows(layer):
    """otherwise W2 (x0 - r + x1) + s would come out, where the client holds W1 r - s"""
    ready(layer)
    layer.prepareWeights(torch.ones((1, 3, 4), dtype=torch.int64), META)
    assert code_of(lambda: layer.online(x, x)) == 1


def test_failed_preparations_leave_nothing_behind(layer):
    ready(layer)

    def fails(*a, **k):
        raise MMHError(4, "no memory")

    layer.fc.plan = lambda meta: SimpleNamespace(n_in=1, n_out=1)
    layer.fc.matVecMul = fails
    layer.sampler.reshare = lambda n: None
    assert code_of(lambda: layer.prepareRows([None, None], [0, 2])) == 4
    assert code_of(lambda: layer.online(x, x)) == 1
    layer.sampler.words = fails
    assert code_of(lambda: layer.prepareMasks(2, META)) == 4
    assert code_of(lambda: layer.openInput(x)) == 1
    layer.fc.encodeWeightMatrix = fails
    assert code_of(lambda: layer.prepareWeights(torch.ones((1, 3, 4), dtype=torch.int64), META)) == 4
    assert code_of(lambda: layer.prepareRows([None, None], [0, 2])) == 1


@pytest.mark.parametrize("other", [dict(N=8192), dict(q=(97, 113)), dict(q=(97,)), dict(device=1)])
def test_sampler_of_another_context_is_refused(other):
    assert code_of(lambda: PreparedFCSS().setUp(context(), sampler(context(**other)))) == 7


@pytest.mark.parametrize("t", [1 << 15, 1 << 30, 1 << 37])
@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.int32, torch.int64])
def test_weights_of_every_type_reach_the_encoder_as_words(dtype, t):
    """the ciphertext half reads 64-bit words modulo t, whatever type the other half lays out"""
    p, ctx, seen = PreparedFCSS(), context(t=t), []
    p.setUp(ctx, sampler(ctx))
    p.ring.encodeWeights = lambda w: SimpleNamespace(groups=w.shape[0], rows=w.shape[1])
    p.fc.encodeWeightMatrix = lambda m, meta: seen.append(m)
    w = torch.tensor([[[-1, 2, -3, 4], [5, -128, 127, 0], [1, 1, 1, 1]]], dtype=dtype)
    p.prepareWeights(w, META)
    assert seen[0].dtype == torch.int64 and seen[0].tolist() == [[v % t for v in row] for row in w[0].tolist()]


def test_every_step_makes_the_layers_device_current(monkeypatch):
    """draws, ciphertext work and its verdicts go to the current device's stream: that has to be the context's device"""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *a):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    p, ctx, seen = PreparedFCSS(), context(device=1), []
    p.setUp(ctx, sampler(ctx))
    ready(p)

    def stop(name):
        def call(*a, **k):
            seen.append((name, current[-1]))
            raise MMHError(8, name)
        return call

    p._mask_meta, p.sampler.words = META, stop("words")
    p.fc.plan, p.fc.decryptToVector, p.ring.encodeWeights = (lambda meta: SimpleNamespace(n_in=1, n_out=1)), stop("decrypt"), stop("encode")
    p.fc.matVecMul, p.sampler.reshare, p.ring.matMul = stop("matVecMul"), lambda n: None, stop("matMul")
    rows = [None, None]
    for call in (lambda: p.finishMasks(rows), lambda: p.online(x, x), lambda: p.prepareRows(rows, [0, 2]), lambda: p.prepareMasks(2, META),
                 lambda: p.prepareWeights(torch.ones((1, 3, 4), dtype=torch.int64), META)):
        assert code_of(call) == 8
    assert seen == [("decrypt", 1), ("matMul", 1), ("matVecMul", 1), ("words", 1), ("encode", 1)] and current == [0]
