"""`python -m rustane_b200.generate --help` (CPU only)."""
import pytest

pytest.importorskip("torch")

from rustane_b200 import generate  # noqa: E402


@pytest.mark.parametrize("argv", [["--help"], ["-h"], ["--prompt", "1", "--help"]])
def test_help(argv, capsys):
    assert generate.main(argv) == 0
    out = capsys.readouterr()
    assert all(flag in out.out for flag in generate._FLAGS) and "--prompt" in out.out and not out.err
