"""Arguments of the serving operators that are views: parts of wider tensors, single rows, shared rows."""
import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import RustaneError, ops  # noqa: E402
from test_gpu_serving import Paged, randn, rope_case  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 40])
def test_page_table_that_is_part_of_a_wider_one(n):
    """Only the part's own entries are read: a length that they do not hold is reported, whatever stands next to them."""
    p = Paged([n, n, n], [300, 70, 90], 4, 2, 128, 16, False, seed=41)
    exp, exp_l = p.run()
    own = p.table
    w = own.shape[1]
    wide = torch.zeros(3, w + 5, dtype=torch.int32, device="cuda")  # the neighbours are valid pages
    wide[:, 3:3 + w] = own
    p.table = wide[:, 3:3 + w]
    got, lse = p.run()
    p.cache.check()
    assert torch.equal(got, exp) and torch.equal(lse, exp_l)
    for s in (0, 2):
        old = p.kv_lens[s].clone()
        p.kv_lens[s] = w * 16 + 1
        got, lse = p.run()
        with pytest.raises(RustaneError):
            p.cache.check()
        rows = slice(s * n, (s + 1) * n)
        assert (got[rows] == 0).all() and torch.isinf(lse[rows]).all()
        p.kv_lens[s] = old
    one = Paged([n], [200], 4, 2, 128, 16, False, seed=42)
    one.table = torch.cat((one.table, one.table), 1)[:, :13]  # a single row of a longer one
    one.kv_lens[0] = 13 * 16 + 1
    got, lse = one.run()
    with pytest.raises(RustaneError):
        one.cache.check()
    assert (got == 0).all() and torch.isinf(lse).all()


@pytest.mark.parametrize("n", [1, 40])
def test_page_table_row_shared_by_all_sequences(n):
    p = Paged([n] * 3, [200] * 3, 4, 2, 128, 16, False, seed=43)
    p.table = p.table[:1].repeat(3, 1)
    exp, exp_l = p.run()
    p.table = p.table[:1].expand(3, -1)
    got, lse = p.run()
    p.cache.check()
    assert torch.equal(got, exp) and torch.equal(lse, exp_l)


def test_a_single_row_of_any_stride():
    """torch leaves the stride of a lone row as it was in the wider tensor: it is no row stride and has no rule."""
    H, Hk, hd = 4, 2, 64
    g, qkv, pos, rope, gq, gk = rope_case(1, H, Hk, hd, 64, "half", True, seed=44)

    def lone(x):  # [1, n] with an odd stride
        wide = torch.zeros(3, x.shape[1] + 3, dtype=x.dtype, device="cuda")
        wide.as_strided((1, x.shape[1]), (wide.shape[1], 1)).copy_(x)
        return wide[:1, :x.shape[1]]

    assert torch.equal(ops.qk_norm_rope(lone(qkv), pos, rope, H, Hk, gq, gk), ops.qk_norm_rope(qkv, pos, rope, H, Hk, gq, gk))
    none = lone(qkv)[:0]
    assert ops.qk_norm_rope(none, pos[:0], rope, H, Hk, gq, gk).shape == none.shape
    p = Paged([1], [50], 4, 2, 64, 16, False, seed=45)
    exp, exp_l = p.run()
    got, lse = p.run(q=lone(p.q), out=lone(p.q))
    assert torch.equal(got, exp) and torch.equal(lse, exp_l)
    x = randn(g, 1, 1000)
    mask = torch.full((1, 32), -1, dtype=torch.int32, device="cuda")
    a, b = ops.logits_adjust(lone(x), mask=mask.t().contiguous().t()), ops.logits_adjust(x, mask=mask)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
