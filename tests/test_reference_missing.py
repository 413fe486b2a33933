"""Without the reference's sources and without a library built from them, tests that compare with the reference are
skipped; a library that is there but does not load is still an error."""
import unittest

import pytest

import oracle as O


@pytest.fixture
def no_reference(tmp_path, monkeypatch):
    monkeypatch.setattr(O, "REF_ROOT", tmp_path)
    for so, held in (("REF_SO", "_ref"), ("REF_B200_SO", "_ref_b200")):
        monkeypatch.setattr(O, so, tmp_path / f"{so}.so")
        monkeypatch.setattr(O, held, None)
    return tmp_path


@pytest.mark.parametrize("call", [lambda: O.ref(), lambda: O.ref_b200(), lambda: O._port_lib("b200")])
def test_missing_reference_skips(no_reference, call):
    assert not O.ref_available()
    with pytest.raises(unittest.SkipTest):
        call()


def test_broken_library_is_an_error(no_reference):
    O.REF_SO.write_bytes(b"no library")
    with pytest.raises(OSError) as e:
        O.ref()
    assert not isinstance(e.value, unittest.SkipTest)
