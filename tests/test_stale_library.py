"""A library built before an entry point was added is refused when it is loaded, whatever its version says (CPU)."""

import pytest

from hilberta_amd import _lib, ops


def test_library_without_an_entry_point(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setitem(_lib.SIGNATURES, "hb_of_a_later_build", (None, []))
    with pytest.raises(RuntimeError, match=r"lacks hb_of_a_later_build.*rebuild the HIP library \(python -m hilberta_amd.build\)"):
        _lib.load()
    monkeypatch.delitem(_lib.SIGNATURES, "hb_of_a_later_build")
    assert _lib.load().hb_version() == _lib.header_abi_version()


def test_operator_library_without_an_operator(monkeypatch):
    monkeypatch.setattr(ops, "_NAMES", (*ops._NAMES, "op_of_a_later_build"))
    with pytest.raises(RuntimeError, match=r"lacks op_of_a_later_build.*rebuild the libraries \(python -m hilberta_amd.build\)"):
        ops._load()


def test_every_signature_is_declared():
    assert set(_lib.SIGNATURES) <= set(_lib.header_symbols())
