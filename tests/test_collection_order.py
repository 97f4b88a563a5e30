"""CPU check of the order tests are collected in: programs that could not be built here run last."""
import os
from types import SimpleNamespace

from tests import conftest


def test_programs_that_were_not_built_run_last(monkeypatch):
    names = ["test_a", "test_reference_sources_run_on_the_device_library[ref_gemini_test]", "test_b", "test_c"]
    monkeypatch.setattr(os.path, "isdir", lambda p: False)
    items = [SimpleNamespace(name=n) for n in names]
    conftest.pytest_collection_modifyitems(items)
    assert [i.name for i in items] == [names[0], names[2], names[3], names[1]]
    monkeypatch.setattr(os.path, "isdir", lambda p: True)       # built: the order stays
    items = [SimpleNamespace(name=n) for n in names]
    conftest.pytest_collection_modifyitems(items)
    assert [i.name for i in items] == names
