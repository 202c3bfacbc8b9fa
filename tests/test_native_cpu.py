"""Whether a built kernel library counts as current."""
import pytest

from r9700_stack_b200 import _native


@pytest.mark.parametrize("name", ["NVCC_FLAGS", "CXX_FLAGS", "CXX_RUNTIME"])
def test_a_library_built_with_other_flags_is_not_current(monkeypatch, name):
    before = _native._source_hash()
    was = getattr(_native, name)
    monkeypatch.setattr(_native, name, was + ["-DX"] if isinstance(was, list) else was + "X")
    assert _native._source_hash() != before
