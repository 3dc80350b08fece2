"""`python -m rustane_b200.generate --page-size` takes the cache's page sizes only (CPU only)."""
import pytest

pytest.importorskip("torch")

from rustane_b200 import generate  # noqa: E402
from rustane_b200.train import UsageError  # noqa: E402


@pytest.mark.parametrize("size", ["0", "8", "24", "256", "-16"])
def test_page_sizes(size):
    with pytest.raises(UsageError, match="page-size"):
        generate.parse_args(["--prompt", "1", "--page-size", size])
    assert generate.main(["--prompt", "1", "--page-size", size]) == 1
