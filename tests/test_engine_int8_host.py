"""The engine's 8-bit prompt option without a GPU."""

import pytest

from opac1ty_b200.engine import Engine, EngineError, lib


@pytest.mark.parametrize("bits", [0, 4, 32, "8"])
def test_other_widths_are_refused(tmp_path, bits):
    with pytest.raises(ValueError, match="prompt_bits"):
        Engine(tmp_path / "none.bf2", prompt_bits=bits)


def test_a_missing_file_is_an_error(tmp_path):
    with pytest.raises(EngineError, match="Cannot open"):
        Engine(tmp_path / "none.bf2", prompt_bits=8)


def test_unknown_options_are_an_error():
    assert not lib().bf_engine_create_with(None, 0, 0, 0)
    h = lib().bf_engine_create_with(b"none.bf2", 0, 0, 4)
    assert b"unknown engine options 0x4" in lib().bf_engine_get_error(h)
    lib().bf_engine_destroy(h)
