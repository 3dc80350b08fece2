"""Rows that are done over because a NaN met them, alone and one warp each: what they give and how long they take."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import Paged, close  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,ps", [(128, 16), (64, 64)])
@pytest.mark.parametrize("n,ctx", [(2, 9), (5, 100), (9, 1003), (150, 700), (300, 300)])
def test_rows_before_a_nan_value(n, ctx, hd, ps):
    """Windows and lengths that begin and end inside a step of keys; every page but the sequence's holds NaN."""
    p = Paged([n], [ctx], 4, 2, hd, ps, False, seed=n)
    at = ctx - 1  # only the last row sees it
    p.cache.v[int(p.table[0, at // ps]), :, at % ps] = float("nan")
    for window in (0, 1, 5, 37):
        got, lse = p.run(window)
        p.cache.check()
        o, a, l = p.exact(window)
        got = got.view(n, 4, hd)
        close(got[:n - 1], o[:n - 1], 2.0**-8 * (o.abs() + a)[:n - 1] + 1e-30)
        close(lse[:n - 1], l[:n - 1], 1e-4 + 1e-5 * torch.where(l.isfinite(), l.abs(), 0)[:n - 1])
        assert torch.isnan(got[n - 1]).all()


def test_a_nan_token_does_not_stall_a_chunk():
    """4 x 509 rows of 20 heads over 4091 keys, all of one request's done over: 1e4 rows x 4e3 keys on 148 x 8 warps are
    3.6e4 keys a warp.  With a key at a time, each waiting for the last one's loads, that took 76 ms; a third of it is
    the limit."""
    p = Paged([509] * 4, [4091] * 4, 20, 20, 128, 16, False, seed=1)
    p.run()
    at = 4091 - 509
    p.cache.v[int(p.table[0, at // 16]), :, at % 16] = float("nan")
    times = []
    for _ in range(3):
        start, end = torch.cuda.Event(True), torch.cuda.Event(True)
        start.record()
        p.run()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    p.cache.check()
    assert min(times) < 25, times
