"""CPU check of the device that truncate_rotary works on: the turn runs on the share's device, so the steps behind it have to run
there too, on that device's stream, whichever device is current."""
from types import SimpleNamespace

import torch

from openmm_amd import lib as L
from openmm_amd.truncation import ALICE, Truncation


def test_truncate_rotary_makes_its_device_current(monkeypatch):
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *a):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    seen = []

    def call(name):
        def launch(*a):
            seen.append((name, current[-1], a[-1]))
            return 0
        return launch

    monkeypatch.setattr(L, "_stream_ptr", lambda: f"stream of {current[-1]}")
    monkeypatch.setattr(L, "dptr", lambda t: None)
    monkeypatch.setattr(L, "to_device", lambda a, device: a)
    t = Truncation(ALICE, None, device=1, aux=SimpleNamespace(wrap=lambda *a: 0, B2A=lambda *a: 0))
    t.lib = SimpleNamespace(mmh_trunc_post=call("post"))
    t._out = lambda dim: torch.zeros(dim, dtype=torch.int64)

    def turn(party, x, positions, signed, heuristic):
        seen.append(("turn", current[-1], f"stream of {current[-1]}"))
        return torch.zeros((2, 1, 4), dtype=torch.int64), None

    x = SimpleNamespace(numel=lambda: 8, get_device=lambda: 1, shape=(2, 1, 4))
    out = t.truncate_rotary(SimpleNamespace(ring_bw=37, truncate_pre=turn), x, None, 10)
    assert seen == [("turn", 1, "stream of 1"), ("post", 1, "stream of 1")] and out.shape == (2, 1, 4) and current == [0]
