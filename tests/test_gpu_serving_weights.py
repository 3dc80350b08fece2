"""How many bits attention over the paged cache keeps of its weights for single tokens and other few rows.

Tolerances, derived before the first run.  The output's own rounding to bf16 (8 bits) is 2^-8 |o| at most.
A bf16 cache's weights go into the product as the sum of two bf16 numbers, 2^-15 of each weight off;
scores are sums of 128 fp32 products of size about 1 scaled by 1 / sqrt(128), a few 2^-24 of 81 off, and
ex2 adds 2^-22: together under 2^-13 of sum p |v| / sum p.  An int8 cache's weights times scales are
rounded to fp16 (11 bits), 2^-11 of each; with the same noise under 2^-10.
"""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import Paged, close  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8,bits", [(False, 13), (True, 10)])
@pytest.mark.parametrize("H,Hk,hd,n", [(4, 4, 128, 1), (8, 2, 128, 1), (16, 1, 128, 1), (6, 2, 64, 1), (12, 1, 64, 1), (4, 2, 128, 3)])
def test_weights_of_few_rows(H, Hk, hd, n, int8, bits):
    lens = [n + 1, 17, 33, 64, 127, 500, 1025]
    p = Paged([n] * len(lens), lens, H, Hk, hd, 16, int8, seed=H + n)
    for window in (0, 40):
        got, _ = p.run(window)
        o, a, _ = p.exact(window)
        p.cache.check()
        close(got.view(p.T, H, hd), o, 2.0**-8 * o.abs() + 2.0**-bits * a + 1e-30)


@pytest.mark.parametrize("int8,bits", [(False, 13), (True, 10)])
def test_weights_of_split_contexts(int8, bits):
    p = Paged([1, 1], [20011, 700], 4, 2, 128, 64, int8, seed=3)
    got, _ = p.run()
    o, a, _ = p.exact()
    p.cache.check()
    close(got.view(2, 4, 128), o, 2.0**-8 * o.abs() + 2.0**-bits * a + 1e-30)


@pytest.mark.parametrize("H,Hk,hd", [(2, 2, 128), (16, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_an_infinite_value_gives_an_infinite_output(H, Hk, hd, bad):
    """Equal weights, whose bits end early: v's infinity in one column gives the same in that column of every row."""
    p = Paged([1], [64], H, Hk, hd, 16, False, seed=6)
    p.q.zero_()
    p.cache.v[int(p.table[0, 1]), :, 3, 5] = bad
    got, _ = p.run()
    p.cache.check()
    got = got.view(H, hd)
    assert (got[:, 5] == bad).all()
    assert torch.isfinite(got[:, torch.arange(hd, device="cuda") != 5]).all()
