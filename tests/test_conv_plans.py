"""CPU check of which plan HomConv2DSS hands to the device: a plan carries its context's degree and limbs, by which kernels index
buffers that are sized by the current context."""
from types import SimpleNamespace

from openmm_amd import hom_conv2d_ss


def test_conv_plan_follows_the_context(monkeypatch):
    monkeypatch.setattr(hom_conv2d_ss, "Plan", lambda ctx, meta: SimpleNamespace(ctx=ctx, meta=meta))
    h, meta = hom_conv2d_ss.HomConv2DSS(), hom_conv2d_ss.Meta((3, 8, 8), (3, 1, 1), 2)
    first, second = (SimpleNamespace(N=N, L=2, t=1 << 37) for N in (8192, 4096))
    h.setUp(first)
    p = h.plan(meta)
    h.setUp(first)
    assert p.ctx is first and h.plan(meta) is p
    h.setUp(second)
    assert h.plan(meta).ctx is second
