"""CPU checks of arguments of the rotary layer that used to be taken without effect."""
import pytest

from openmm_amd.lib import MMHError
from openmm_amd.rotary import rotary_phases


def test_yarn_takes_both_bounds_or_none():
    full = rotary_phases(64, yarn=(16, 4096, 1, 32))
    assert rotary_phases(64, yarn=(16, 4096)) == full
    assert rotary_phases(64, yarn=(16, 4096, 2, 32)) != full
    for yarn in ((16, 4096, 2), (16,), (16, 4096, 1, 32, 0)):      # a lone lower bound was ignored
        with pytest.raises(MMHError) as e:
            rotary_phases(64, yarn=yarn)
        assert e.value.code == 7
