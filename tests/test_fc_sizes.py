"""CPU checks that HomFCSS refuses operands smaller than the words the device reads through their pointers."""
from types import SimpleNamespace

import pytest
import torch

from openmm_amd import hom_fc_ss
from openmm_amd.lib import MMHError

N, L = 64, 2


@pytest.fixture
def fc(monkeypatch):
    """a set-up HomFCSS whose plan has 2 input and 3 output ciphertexts; a call that reaches the device library fails the test"""
    class NoDevice:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(hom_fc_ss, "Plan", lambda ctx, meta: SimpleNamespace(n_in=2, n_out=3, split=(4, 8), handle=None))
    monkeypatch.setattr(hom_fc_ss.L, "_stream_ptr", lambda: None)
    monkeypatch.setattr(hom_fc_ss.L, "dptr", lambda t: None)
    monkeypatch.setattr(hom_fc_ss.L, "DeferredFlag", lambda flag: flag)      # pinned memory needs a GPU
    ctx = SimpleNamespace(N=N, L=L, t=1 << 20, lib=NoDevice(), _empty=lambda *s: torch.empty(s, dtype=torch.int64))
    h = hom_fc_ss.HomFCSS()
    keys = torch.zeros((2, L, N), dtype=torch.int64)
    h.setUp(ctx, sk_ntt=keys[0], pk_ntt=keys)
    return h


META = hom_fc_ss.Meta((10, 16), (16,), True)


def z(*shape, dtype=torch.int64):
    return torch.zeros(shape, dtype=dtype)


def test_good_calls_reach_the_device(fc):
    for call in (lambda: fc.encryptInputVector(z(16), META, (z(2, L, N), z(2, N))), lambda: fc.encodeInputVector(z(16), META),
                 lambda: fc.encodeWeightMatrix(z(10, 16), META), lambda: fc.decryptToVector(z(3, 2, 1, N), META),
                 lambda: fc.matVecMul(z(3, 2, N), z(2, 2, L, N), z(2, N), META, (z(3, N),) * 3)):
        with pytest.raises(AssertionError, match="was reached"):
            call()


def test_short_operands_are_refused(fc):
    i32 = torch.int32
    bad = [
        (3, lambda: fc.encryptInputVector(z(16), META, (z(2, L, N // 2), z(2, N)))),      # a sampler of another degree
        (3, lambda: fc.encryptInputVector(z(16), META, (z(2, L, N), z(2, N // 2)))),
        (3, lambda: fc.encryptInputVector(z(16), META, (z(2, 1, N), z(2, N)))),
        (3, lambda: fc.encryptInputVector(z(16), META, (z(1, L, N), z(1, N)))),
        (7, lambda: fc.encryptInputVector(z(16, dtype=i32), META, (z(2, L, N), z(2, N)))),
        (7, lambda: fc.encryptInputVector(z(16), META, (z(2, L, N, dtype=i32), z(2, N)))),
        (7, lambda: fc.encryptInputVector(z(16), META, (z(2, L, N), z(2, N, dtype=i32)))),
        (7, lambda: fc.encodeInputVector(z(16, dtype=i32), META)),
        (7, lambda: fc.encodeWeightMatrix(z(10, 16, dtype=torch.int16), META)),
        (7, lambda: fc.matVecMul(z(3, 2, N, dtype=i32), z(2, 2, L, N), z(2, N), META, (z(3, N),) * 3)),
        (7, lambda: fc.matVecMul(z(3, 2, N), z(2, 2, L, N, dtype=i32), z(2, N), META, (z(3, N),) * 3)),
        (7, lambda: fc.matVecMul(z(3, 2, N), z(2, 2, L, N), z(2, N, dtype=i32), META, (z(3, N),) * 3)),
        (7, lambda: fc.matVecMul(z(3, 2, N), z(2, 2, L, N), z(2, N), META, (z(3, N), z(3, N, dtype=i32), z(3, N)))),
        (7, lambda: fc.decryptToVector(z(3, 2, 1, N // 2), META)),                         # ciphertexts of another degree
        (7, lambda: fc.decryptToVector(z(3, 1, 1, N), META)),
        (7, lambda: fc.decryptToVector(z(3, 2, 1, N, dtype=i32), META)),
    ]
    for i, (code, call) in enumerate(bad):
        with pytest.raises(MMHError) as e:
            call()
            pytest.fail(f"case {i} was accepted")
        assert e.value.code == code, i


def test_more_randomness_than_a_call_takes_is_accepted(fc):
    """a caller may draw for its largest layer once, in any shape that holds the words in order"""
    for a, e in ((z(5, L, N), z(3, N)), (z(2 * L * N), z(2 * N)), (z(2 * L, N), z(2, 1, N))):
        with pytest.raises(AssertionError, match="was reached"):
            fc.encryptInputVector(z(16), META, (a, e))
    for a, e in ((z(5, L, 2 * N), z(3, N)), (z(5, L, N), z(3, 2 * N)), (z(5, 1, N), z(3, N))):      # of another context
        with pytest.raises(MMHError) as err:
            fc.encryptInputVector(z(16), META, (a, e))
        assert err.value.code == 3
