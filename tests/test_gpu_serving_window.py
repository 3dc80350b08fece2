"""Windows as large as the argument takes."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import Paged  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 1, 1 << 40])
@pytest.mark.parametrize("q_lens,kv_lens", [([6], [3]), ([60, 2], [10, 2]), ([300], [7]), ([1], [50])])
def test_a_window_past_every_length_is_none(q_lens, kv_lens, window, int8):
    """Also where the first rows see nothing (fewer cached tokens than new ones)."""
    p = Paged(q_lens, kv_lens, 4, 2, 128, 16, int8, seed=51)
    exp, exp_l = p.run()
    p.check()
    got, lse = p.run(window=window)
    p.cache.check()
    assert torch.equal(got, exp) and torch.equal(lse, exp_l)
