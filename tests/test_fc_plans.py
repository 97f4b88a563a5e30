"""CPU checks of which plan the layer classes hand to the device: a plan carries its context's degree and limbs and its layer's
columns, by which kernels index buffers that are sized by the current context and the call's tensors."""
from types import SimpleNamespace

import pytest

from openmm_amd import hom_fc_ss
from openmm_amd.lib import MMHError


class Made:
    """stands for a plan: what it was made from"""

    def __init__(self, ctx, meta):
        self.ctx, self.meta = ctx, meta


def context(N):
    return SimpleNamespace(N=N, L=2, t=1 << 37)


def test_fc_plan_follows_the_context(monkeypatch):
    monkeypatch.setattr(hom_fc_ss, "Plan", Made)
    h, meta = hom_fc_ss.HomFCSS(), hom_fc_ss.Meta((10, 20), (20,))
    first, second = context(8192), context(4096)
    h.setUp(first)
    p = h.plan(meta)
    assert p.ctx is first and h.plan(meta) is p
    h.setUp(first)
    assert h.plan(meta) is p            # the same context again: the plan stays
    h.setUp(second)
    assert h.plan(meta).ctx is second


def test_fc_plan_checks_every_meta(monkeypatch):
    """an input shape that does not fit the weights is refused also where a plan for these weights is there already"""
    class Checked(hom_fc_ss.Plan):
        def __init__(self, ctx, meta):
            if meta.input_shape[0] == meta.weight_shape[1]:
                return                  # a valid one: nothing is asked of a device here
            super().__init__(ctx, meta)

        def __del__(self):
            pass

    monkeypatch.setattr(hom_fc_ss, "Plan", Checked)
    h = hom_fc_ss.HomFCSS()
    h.setUp(context(4096))
    h.plan(hom_fc_ss.Meta((10, 20), (20,)))
    with pytest.raises(MMHError) as e:
        h.plan(hom_fc_ss.Meta((10, 20), (12,)))
    assert e.value.code == 7
