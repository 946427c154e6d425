"""What the 4-bit cache's engine and the `score` command refuse without a GPU."""

import pytest
from click.testing import CliRunner

from opac1ty_b200.cli import cli
from opac1ty_b200.engine import Engine, EngineError, lib


@pytest.mark.parametrize("bits", [0, 2, 8, 5, "4"])
def test_engine_refuses_other_cache_widths(tmp_path, bits):
    with pytest.raises(ValueError, match="kv_bits"):
        Engine(tmp_path / "none.bf2", kv_bits=bits)


def test_missing_file_is_an_error(tmp_path):
    with pytest.raises(EngineError):
        Engine(tmp_path / "none.bf2", kv_bits=4)


def test_score_without_an_engine():
    assert lib().bf_engine_score(None, None, 0, None, None, 0, None, None) != 0
    assert not lib().bf_engine_create_kv4(None, 0, 0)


@pytest.mark.parametrize("args,msg", [([], "either"), (["--tokens", "1,2", "--text", "ab"], "either"),
                                      (["--tokens", "1"], "two tokens"), (["--text", ""], "two tokens"),
                                      (["--tokens", "1,x"], "token ids")])
def test_score_command_refusals(tmp_path, args, msg):
    p = tmp_path / "x.bf2"
    p.write_bytes(b"")
    res = CliRunner().invoke(cli, ["score", str(p), *args])
    assert res.exit_code == 2 and msg in res.output
