"""Argument handling of `python -m rustane_b200.generate` (CPU only)."""
import pytest

pytest.importorskip("torch")

from rustane_b200 import generate  # noqa: E402
from rustane_b200.train import UsageError  # noqa: E402


def test_defaults_and_lists():
    a = generate.parse_args(["--prompt", "1,2,3", "--prompt", "4", "--bias", "5:1.5,9:-2", "--forbid", "0,1", "--cache", "int8"])
    assert a.prompts == [[1, 2, 3], [4]] and a.bias == {5: 1.5, 9: -2.0} and a.forbid == [0, 1] and a.cache == "int8"
    assert (a.model, a.max_new, a.answers, a.chunk, a.page_size, a.max_pos) == ("gpt_karpathy", 64, 1, 512, 16, 4096)


@pytest.mark.parametrize("argv", [[], ["--prompt", ""], ["--prompt"], ["--prompt", "1", "--model", "nope"], ["--prompt", "8192"],
                                  ["--prompt", "-1"], ["--prompt", "x"], ["--prompt", "1", "--cache", "fp4"],
                                  ["--prompt", "1", "--max-new", "0"], ["--prompt", "1", "--answers", "0"],
                                  ["--prompt", "1", "--max-new", "4096"], ["--prompt", "1", "--bias", "9000:1"],
                                  ["--prompt", "1", "--speed", "9"]])
def test_refusals(argv):
    with pytest.raises(UsageError):
        generate.parse_args(argv)
    assert generate.main(argv) == 1
