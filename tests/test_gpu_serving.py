"""The serving operators on the GPU (rustane_b200.ops over rt_kernel_*), against plain
64-bit implementations written here from the formulas.

Tolerances, derived before the first run.  A bf16 result is half a unit off at most, 2^-9 of
its value; fp32 arithmetic adds a few 2^-24 of the row's largest term: 2^-8 |y| + 1e-5 max|row|
holds both.  Attention rounds each weight to bf16 (2^-9 of it) before the weighted sum, so
its error is within 2^-8 |o| + 2^-8 sum p |v| / sum p.  int8 rows: the code may differ by one
where y / scale lies within fp32 noise of a half: one step (amax / 127) at the few places,
half a step plus the bf16 rounding elsewhere, so: 0.51 steps + 2^-8 |y|.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import RustaneError, ops  # noqa: E402

pytestmark = pytest.mark.gpu
F8 = torch.float64


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def close(got, exp, tol):
    got, exp = got.to(F8), exp.to(F8)
    assert got.shape == exp.shape
    assert torch.equal(torch.isnan(got), torch.isnan(exp))
    bad = ~(((got - exp).abs() <= tol) | (got == exp) | torch.isnan(exp))
    assert not bad.any(), (int(bad.sum()), got[bad][:4], exp[bad][:4])


def row_tol(exp):
    top = exp.abs().flatten(1).amax(1) if exp.numel() else exp.new_zeros(exp.shape[0])
    return exp.abs() * 2.0**-8 + 1e-5 * top.view(-1, *[1] * (exp.dim() - 1))


# ----------------------------------------------------------- rope, plain form
def rot_matrix(cos, sin, rot, hd, layout):
    """[T, hd, hd] rotation of each position's tables."""
    T = cos.shape[0]
    m = torch.eye(hd, device="cuda", dtype=F8).repeat(T, 1, 1)
    i = torch.arange(rot // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + rot // 2)
    m[:, a, a], m[:, b, b] = cos.to(F8), cos.to(F8)
    m[:, a, b], m[:, b, a] = -sin.to(F8), sin.to(F8)
    return m


def plain_vectors(x, gamma, m, eps):
    """y [T, H, hd] of x [T, H, hd] in 64 bits."""
    if gamma is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gamma
    return torch.einsum("tij,thj->thi", m, x)


def rope_case(T, H, Hk, hd, rot, layout, norm, seed, scale=1.0):
    g = gen(seed)
    qkv = (scale * randn(g, T, (H + 2 * Hk) * hd)).bfloat16()
    pos = torch.randint(0, 50, (T,), generator=g, device="cuda", dtype=torch.int32)
    rope = ops.Rope.tables(50, rot, "cuda", layout=layout)
    gq, gk = (1 + 0.3 * randn(g, hd), 1 + 0.3 * randn(g, hd)) if norm else (None, None)
    return g, qkv, pos, rope, gq, gk


def exact_rope(qkv, pos, rope, gq, gk, H, Hk, hd, eps=1e-5):
    T = qkv.shape[0]
    x = qkv.to(F8).view(T, -1, hd).clone().requires_grad_(True)
    m = rot_matrix(rope.cos[pos.long().clamp(0, rope.n_pos - 1)], rope.sin[pos.long().clamp(0, rope.n_pos - 1)], rope.rot, hd, rope.layout)
    gq, gk = ((None if g is None else g.to(F8).clone().requires_grad_(True)) for g in (gq, gk))
    y = torch.cat((plain_vectors(x[:, :H], gq, m, eps), plain_vectors(x[:, H:H + Hk], gk, m, eps), x[:, H + Hk:]), 1)
    return x, gq, gk, y


ROPE_CASES = [(1, 1, 1, 128, 128, "interleaved", True), (7, 12, 12, 128, 128, "interleaved", False),
              (33, 6, 2, 64, 64, "half", True), (65, 5, 1, 128, 64, "half", True), (130, 32, 8, 128, 32, "interleaved", True),
              (3, 7, 7, 64, 16, "half", False), (1025, 4, 4, 64, 48, "interleaved", True), (2, 8, 8, 128, 16, "half", True)]


@pytest.mark.parametrize("T,H,Hk,hd,rot,layout,norm", ROPE_CASES)
def test_qk_norm_rope_forward_and_backward(T, H, Hk, hd, rot, layout, norm):
    g, qkv, pos, rope, gq, gk = rope_case(T, H, Hk, hd, rot, layout, norm, seed=T)
    x, xq, xk, y = exact_rope(qkv, pos, rope, gq, gk, H, Hk, hd)
    out = ops.qk_norm_rope(qkv, pos, rope, H, Hk, gq, gk)
    close(out.view(T, -1, hd), y.detach(), row_tol(y.detach()))
    assert torch.equal(out[:, (H + Hk) * hd:], qkv[:, (H + Hk) * hd:])
    dout = randn(g, *qkv.shape).bfloat16()
    y.backward(dout.to(F8).view(T, -1, hd))
    dqkv, dgq, dgk = ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk)
    close(dqkv.view(T, -1, hd), x.grad, row_tol(x.grad))
    if norm:
        # fp32 sums of T * heads terms of size about 1
        close(dgq, xq.grad, 1e-5 * math.sqrt(T * H) + 1e-5 * xq.grad.abs())
        close(dgk, xk.grad, 1e-5 * math.sqrt(T * Hk) + 1e-5 * xk.grad.abs())
        again = ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk)
        assert all(torch.equal(a, b) for a, b in zip(again, (dqkv, dgq, dgk)))  # fixed order of sums
        base = torch.ones(hd, device="cuda"), 2 * torch.ones(hd, device="cuda")
        ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk, dgamma_q=base[0], dgamma_k=base[1])
        close(base[0], dgq + 1, 1e-6 * (dgq.abs() + 1))
        close(base[1], dgk + 2, 1e-6 * (dgk.abs() + 2))
    else:
        assert dgq is None and dgk is None


def test_qk_norm_rope_nonfinite_v_stays_in_v():
    """v passes through; its NaN and Inf, forward and backward, reach nothing of q, k or the gammas."""
    T, H, Hk, hd = 9, 5, 1, 128
    g, qkv, pos, rope, gq, gk = rope_case(T, H, Hk, hd, 64, "half", True, seed=2)
    dout = randn(g, *qkv.shape).bfloat16()
    exp, exp_d = ops.qk_norm_rope(qkv, pos, rope, H, Hk, gq, gk), ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk)
    cut = (H + Hk) * hd
    for t in (qkv, dout):
        t[3, cut] = float("nan")
        t[4, cut + 7] = float("inf")
    out, d = ops.qk_norm_rope(qkv, pos, rope, H, Hk, gq, gk), ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk)
    assert torch.equal(out[:, :cut], exp[:, :cut]) and torch.equal(d[0][:, :cut], exp_d[0][:, :cut])
    assert torch.equal(d[1], exp_d[1]) and torch.equal(d[2], exp_d[2])
    assert torch.equal(out[:, cut:].view(torch.int16), qkv[:, cut:].view(torch.int16))
    assert torch.equal(d[0][:, cut:].view(torch.int16), dout[:, cut:].view(torch.int16))


def test_qk_norm_rope_gradient_against_differences():
    """d(sum w . y)/dx and /dgamma by central differences of the 64-bit forward: a check of the formula
    that shares nothing with autograd."""
    T, H, Hk, hd = 3, 2, 1, 64
    g, qkv, pos, rope, gq, gk = rope_case(T, H, Hk, hd, 32, "half", True, seed=9)
    w = randn(g, *qkv.shape).bfloat16()
    dqkv, dgq, dgk = ops.qk_norm_rope_backward(w, qkv, pos, rope, H, Hk, gq, gk)
    m = rot_matrix(rope.cos[pos.long()], rope.sin[pos.long()], 32, hd, "half")

    def loss(x, a, b):
        x = x.view(T, -1, hd)
        y = torch.cat((plain_vectors(x[:, :H], a, m, 1e-5), plain_vectors(x[:, H:H + Hk], b, m, 1e-5), x[:, H + Hk:]), 1)
        return float((y.reshape(T, -1) * w.to(F8)).sum())

    x, a, b = qkv.to(F8), gq.to(F8), gk.to(F8)
    h = 1e-5
    rng = np.random.default_rng(0)
    for t, c in zip(rng.integers(0, T, 24), rng.integers(0, qkv.shape[1], 24)):
        e = torch.zeros_like(x)
        e[t, c] = h
        d = (loss(x + e, a, b) - loss(x - e, a, b)) / (2 * h)
        assert abs(float(dqkv[t, c]) - d) <= 2**-8 * abs(d) + 1e-4
    for i in rng.integers(0, hd, 8):
        e = torch.zeros_like(a)
        e[i] = h
        assert abs(float(dgq[i]) - (loss(x, a + e, b) - loss(x, a - e, b)) / (2 * h)) < 1e-4
        assert abs(float(dgk[i]) - (loss(x, a, b + e) - loss(x, a, b - e)) / (2 * h)) < 1e-4


def test_qk_norm_rope_in_place_strided_and_other_stream():
    T, H, Hk, hd = 37, 4, 2, 128
    g, qkv, pos, rope, gq, gk = rope_case(T, H, Hk, hd, 128, "half", True, seed=3)
    exp = ops.qk_norm_rope(qkv, pos, rope, H, Hk, gq, gk)
    wide = torch.full((T, qkv.shape[1] + 72), 7.0, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:8 + qkv.shape[1]] = qkv
    view = wide[:, 8:8 + qkv.shape[1]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.qk_norm_rope(view, pos, rope, H, Hk, gq, gk, out=view)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(view, exp)
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + qkv.shape[1]:] == 7).all()
    no_v = ops.qk_norm_rope(qkv[:, :(H + Hk) * hd], pos, rope, H, Hk, gq, gk)
    assert torch.equal(no_v, exp[:, :(H + Hk) * hd])
    dout = randn(g, *qkv.shape).bfloat16()
    exp_d = ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk)[0]
    assert torch.equal(ops.qk_norm_rope_backward(dout, qkv, pos, rope, H, Hk, gq, gk, dqkv=dout)[0], exp_d)


def test_qk_norm_rope_bad_position_zero_rows_and_zero_tokens():
    T, H, Hk, hd = 5, 2, 2, 64
    g, qkv, pos, rope, gq, gk = rope_case(T, H, Hk, hd, 64, "interleaved", True, seed=4)
    qkv[2] = 0  # r = 1 / sqrt(eps): finite
    pos[1], pos[3] = 50, -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.qk_norm_rope(qkv, pos, rope, H, Hk, gq, gk, err=err)
    assert err.item() == 6
    pos0 = pos.clone()
    pos0[1] = pos0[3] = 0
    assert torch.equal(out, ops.qk_norm_rope(qkv, pos0, rope, H, Hk, gq, gk))
    assert (out[2] == 0).all()
    empty = ops.qk_norm_rope(qkv[:0], pos[:0], rope, H, Hk, gq, gk)
    assert empty.shape == (0, qkv.shape[1])
    d, dgq, dgk = ops.qk_norm_rope_backward(qkv[:0], qkv[:0], pos[:0], rope, H, Hk, gq, gk)
    assert d.shape[0] == 0 and (dgq == 0).all() and (dgk == 0).all()


def test_rope_matches_the_models_own_rotation():
    """Interleaved tables at theta 10000 are the fused QKV epilogue's."""
    import pyoracle as po
    from rustane_b200.model import ModelConfig
    _, _, cb, sb = po.Oracle(ModelConfig.custom(256, 256, 2, 1, seq=64, vocab=256), 1).rope_tables()
    rope = ops.Rope.tables(64, 128, "cuda")
    # the reference takes cos of an fp32 angle: p * 2^-24 off at most
    assert np.abs(rope.cos.cpu().numpy() - cb.T).max() < 64 * 2**-22
    assert np.abs(rope.sin.cpu().numpy() - sb.T).max() < 64 * 2**-22


# ---------------------------------------------------------------- paged cache
def new_cache(pages, ps, Hk, hd, int8):
    return ops.KvCache.empty(pages, ps, Hk, hd, torch.int8 if int8 else torch.bfloat16, "cuda")


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,H,Hk,hd,ps,norm,layout", [(1, 12, 12, 128, 16, False, "interleaved"), (19, 8, 2, 128, 64, True, "half"),
                                                      (130, 6, 3, 64, 32, True, "interleaved"), (300, 4, 4, 64, 128, False, "half")])
def test_kv_append_and_gather(T, H, Hk, hd, ps, norm, layout, int8):
    g, qkv, pos, rope, gq, gk = rope_case(T, H, Hk, hd, hd // 2, layout, norm, seed=T + ps, scale=3.0)
    if T > 2:
        qkv[1] = 0  # an all-zero row: scale 0
        if int8:
            qkv[2, (H + Hk) * hd] = 1e-38  # a denormal scale
            qkv[2, (H + Hk) * hd + 1:(H + Hk + 1) * hd] = 0
    pages = -(-T // ps) + 3
    cache = new_cache(pages, ps, Hk, hd, int8)
    for t in (cache.k, cache.v):
        t.fill_(5)
    slots = torch.randperm(pages * ps, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 5:
        slots[5] = -1
    _, _, _, y = exact_rope(qkv, pos, rope, gq, gk, H, Hk, hd)
    y = y.detach()
    q = ops.kv_append(qkv, pos, slots, rope, cache, H, gq, gk)
    close(q.view(T, H, hd), y[:, :H], row_tol(y)[:, :H])
    k, v = ops.kv_gather(cache, slots)
    cache.check()
    for got, exp in ((k, y[:, H:H + Hk]), (v, y[:, H + Hk:])):
        exp = exp.clone()
        if T > 5:
            assert (got[5] == 0).all()
            exp[5] = 0
        tol = 0.51 * exp.abs().amax(-1, keepdim=True) / 127 + 2.0**-8 * exp.abs() + 1e-42 if int8 else row_tol(exp)
        close(got, exp, tol.expand_as(exp))
    # only the named slots were written
    untouched = torch.ones(pages * ps, dtype=torch.bool, device="cuda")
    untouched[slots[slots >= 0].long()] = False
    for t in (cache.k, cache.v):
        rows = t.transpose(1, 2).reshape(pages * ps, -1)
        assert (rows[untouched] == 5).all()
    if not int8:
        at = slots[slots >= 0].long()
        assert torch.equal(cache.k[at // ps, :, at % ps], k[slots >= 0])


def test_kv_append_nonfinite_rows_and_bad_slots():
    T, H, Hk, hd, ps = 6, 2, 2, 64, 16
    g, qkv, pos, rope, _, _ = rope_case(T, H, Hk, hd, 64, "half", False, seed=1)
    qkv[0, (H + Hk) * hd + 3] = float("inf")
    qkv[1, (H + Hk + 1) * hd + 5] = float("nan")
    cache = new_cache(2, ps, Hk, hd, True)
    slots = torch.tensor([0, 1, 2, 32, -2, 31], dtype=torch.int32, device="cuda")
    ops.kv_append(qkv, pos, slots, rope, cache, H)
    with pytest.raises(RustaneError):
        cache.check()
    cache.check()  # cleared
    good = torch.tensor([0, 1, 2, 31], dtype=torch.int32, device="cuda")
    _, v = ops.kv_gather(cache, good)
    assert torch.isnan(v[0, 0]).all() and torch.isfinite(v[0, 1]).all()
    assert torch.isnan(v[1, 1]).all() and torch.isfinite(v[1, 0]).all()
    assert torch.isfinite(v[2:]).all()
    ops.kv_gather(cache, slots)
    with pytest.raises(RustaneError):
        cache.check()


def test_large_offsets_in_a_long_cache():
    """Rows past 2^31 elements and 2^32 bytes of one cache tensor."""
    Hk, hd, ps = 32, 128, 128
    pages = (5 << 30) // (Hk * hd * ps)  # 5 Gi elements of int8
    cache = ops.KvCache(torch.empty((pages, Hk, ps, hd), dtype=torch.int8, device="cuda"),
                        torch.empty((pages, Hk, ps, hd), dtype=torch.int8, device="cuda"),
                        torch.zeros((pages, Hk, ps), device="cuda"), torch.zeros((pages, Hk, ps), device="cuda"))
    T = 40
    g, qkv, pos, rope, _, _ = rope_case(T, Hk, Hk, hd, 128, "half", False, seed=8)
    last = pages * ps - ps
    slots = torch.arange(last, last + T, dtype=torch.int32, device="cuda")
    q = ops.kv_append(qkv, pos, slots, rope, cache, Hk)
    k, v = ops.kv_gather(cache, slots)
    near = new_cache(1, ps, Hk, hd, True)
    here = torch.arange(T, dtype=torch.int32, device="cuda")
    ops.kv_append(qkv, pos, here, rope, near, Hk)
    kn, vn = ops.kv_gather(near, here)
    assert torch.equal(k, kn) and torch.equal(v, vn)
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    ws = ops.AttentionWorkspace("cuda")
    far_t = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    for n in (1, T):
        start[1] = n
        a, _ = ops.attention_paged(q[:n], cache, far_t, lens, start, Hk, ws, max_q=n, max_kv=T)
        b, _ = ops.attention_paged(q[:n], near, torch.zeros_like(far_t), lens, start, Hk, ws, max_q=n, max_kv=T)
        assert torch.equal(a, b)
    cache.check()


# ------------------------------------------------------------------ attention
class Paged:
    """Sequences of q_lens new tokens over kv_lens cached ones, in a shuffled cache whose every other
    place (unused pages, page tails, stale scales) holds `stale`."""

    def __init__(self, q_lens, kv_lens, H, Hk, hd, ps, int8, seed, stale=float("nan"), amp=1.0):
        g = gen(seed)
        self.q_lens, self.kv_lens_l, self.H, self.Hk, self.hd, self.ps = q_lens, kv_lens, H, Hk, hd, ps
        per = [-(-n // ps) for n in kv_lens]
        pages, width = sum(per) + 2, max(per + [1]) + 1
        kd = [(amp * randn(g, n, Hk, hd)).bfloat16() for n in kv_lens]
        vd = [randn(g, n, Hk, hd).bfloat16() for n in kv_lens]
        self.cache = new_cache(pages, ps, Hk, hd, int8)
        if int8:
            self.cache.k.fill_(127), self.cache.v.fill_(-128)
            self.cache.k_scale.fill_(stale), self.cache.v_scale.fill_(stale)
        else:
            self.cache.k.fill_(stale), self.cache.v.fill_(stale)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(kv_lens), width), -1, dtype=torch.int32, device="cuda")
        self.k, self.v, at = [], [], 0
        for i, n in enumerate(kv_lens):
            mine = order[at:at + per[i]]
            self.table[i, :per[i]] = mine
            at += per[i]
            where = (mine.long()[:, None] * ps + torch.arange(ps, device="cuda")).reshape(-1)[:n]
            ks, vs = [], []
            for t, s, data, keep in ((self.cache.k, self.cache.k_scale, kd[i], ks), (self.cache.v, self.cache.v_scale, vd[i], vs)):
                page, off = where // ps, where % ps
                if int8:
                    sc = data.float().abs().amax(-1) / 127 if n else data.float().sum(-1)
                    codes = (data.float() / sc[..., None]).round().clamp(-127, 127)
                    t[page, :, off], s[page, :, off] = codes.to(torch.int8), sc
                    keep.append(codes.to(F8) * sc.to(F8)[..., None])
                else:
                    t[page, :, off] = data
                    keep.append(data.to(F8))
            self.k += ks
            self.v += vs
        self.T = sum(q_lens)
        self.q = randn(g, self.T, H * hd).bfloat16()
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        self.q_start = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
        self.ws = ops.AttentionWorkspace("cuda")

    def run(self, window=0, q=None, out=None, max_q=None, max_kv=None, scale=None):
        return ops.attention_paged(self.q if q is None else q, self.cache, self.table, self.kv_lens, self.q_start, self.H, self.ws,
                                   max_q=max(self.q_lens + [1]) if max_q is None else max_q,
                                   max_kv=max(self.kv_lens_l + [1]) if max_kv is None else max_kv, window=window, out=out,
                                   want_lse=True, scale=scale)

    def exact(self, window=0, scale=None):
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        G, at = self.H // self.Hk, 0
        o, a, l = (torch.zeros(self.T, self.H, self.hd, dtype=F8, device="cuda") for _ in "oal")
        l = torch.full((self.T, self.H), -math.inf, dtype=F8, device="cuda")
        for n, L, k, v in zip(self.q_lens, self.kv_lens_l, self.k, self.v):
            for i in range(n):
                hi = L - n + i + 1
                lo = max(0, hi - window) if window else 0
                if hi <= lo:
                    continue
                q = self.q[at + i].to(F8).view(self.Hk, G, self.hd)
                s = torch.einsum("hgd,khd->hgk", q, k[lo:hi]) * scale
                l[at + i] = torch.logsumexp(s, -1).reshape(-1) / math.log(2)
                p = torch.softmax(s, -1)
                o[at + i] = torch.einsum("hgk,khd->hgd", p, v[lo:hi]).reshape(self.H, self.hd)
                a[at + i] = torch.einsum("hgk,khd->hgd", p, v[lo:hi].abs()).reshape(self.H, self.hd)
            at += n
        return o, a, l

    def check(self, window=0, scale=None, **kw):
        got, lse = self.run(window, scale=scale, **kw)
        o, a, l = self.exact(window, scale)
        self.cache.check()
        close(got.view(self.T, self.H, self.hd), o, 2.0**-8 * (o.abs() + a) + 1e-30)
        # fp32 scores: 128 products of size about amp, each 2^-24 off
        close(lse, l, 1e-4 + 1e-5 * torch.where(l.isfinite(), l.abs(), 0))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,Hk,hd", [(4, 4, 128), (8, 2, 128), (6, 2, 64), (16, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("ps", [16, 64])
def test_attention_single_tokens_ragged(H, Hk, hd, ps, int8):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1025]
    p = Paged([1] * len(lens), lens, H, Hk, hd, ps, int8, seed=H + ps)
    p.check()
    p.check(window=1)
    p.check(window=100)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,Hk,hd,ps", [(3, 3, 128, 16), (8, 2, 128, 32), (6, 1, 64, 128), (4, 4, 64, 16)])
@pytest.mark.parametrize("q_lens,kv_lens", [([2], [2]), ([5, 3], [5, 400]), ([16, 1, 0, 9], [33, 1, 70, 9]), ([40], [300]),
                                            ([130, 7], [130, 7]), ([128], [256]), ([129, 257, 1], [1000, 257, 64]),
                                            ([6, 3], [4, 0])])
def test_attention_chunks(q_lens, kv_lens, H, Hk, hd, ps, int8):
    p = Paged(q_lens, kv_lens, H, Hk, hd, ps, int8, seed=sum(q_lens) + sum(kv_lens) + hd)
    p.check()
    p.check(window=37)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("q_lens,kv_lens,H,Hk", [([1], [20011], 2, 2), ([1, 1], [9000, 30], 8, 1), ([64], [5000], 2, 1),
                                                 ([700], [3500], 1, 1)])
def test_attention_long_contexts_split_and_joined(q_lens, kv_lens, H, Hk, int8):
    p = Paged(q_lens, kv_lens, H, Hk, 128, 16, int8, seed=7)
    p.check()
    a = p.run()
    b = p.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # joined in a fixed order


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [1, 500])
def test_attention_with_cold_caches(n, int8):
    """Slow K and V loads (L2 flushed before every call) shift the kernel's roles against one another: no
    wait runs out, and the results are the same bits."""
    p = Paged([n] * 3, [4000, 2500, n], 4, 2, 128, 16, int8, seed=21)
    exp, exp_l = p.run()
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for i in range(10):
        flush.fill_(i)
        got, lse = p.run()
        assert torch.equal(got, exp) and torch.equal(lse, exp_l)
    p.cache.check()


@pytest.mark.parametrize("n", [1, 300])
def test_attention_rising_scores(n):
    """Scores that grow along the keys force the running maximum up again and again."""
    p = Paged([n], [1200], 2, 2, 128, 16, False, seed=2, amp=4.0)
    order = torch.argsort(p.k[0][:, 0, :] @ p.q[0].to(F8).view(2, 128)[0])
    ks = p.k[0][order]
    where = (p.table[0, :75].long()[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)[:1200]
    p.cache.k[where // 16, :, where % 16] = ks.bfloat16()
    p.k[0] = ks
    p.check()
    p.check(scale=0.5)


@pytest.mark.parametrize("n", [1, 200])
def test_attention_infinite_and_lowest_scores(n):
    """Keys whose scores are -inf or near the lowest finite value; a row whose every score is -inf
    has no weight and gives the empty row's result."""
    p = Paged([n], [300], 2, 2, 128, 16, False, seed=5)
    p.q.fill_(1.0)
    k = p.k[0]
    k[:150] = 0
    k[:150, :, 0] = -math.inf
    k[150:200, :, 0] = -3e38
    where = (p.table[0, :19].long()[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)[:300]
    p.cache.k[where // 16, :, where % 16] = k.bfloat16()
    p.k[0] = p.cache.k[where // 16, :, where % 16].to(F8)
    got, lse = p.run()
    p.cache.check()
    o, a, l = p.exact()
    o = torch.where(l[..., None] > -math.inf, o, 0.0).nan_to_num(0.0)
    a = a.nan_to_num(0.0)
    close(got.view(n, 2, 128), o, 2.0**-8 * (o.abs() + a) + 1e-30)
    close(lse, l, 1e-4 + 1e-5 * torch.where(l.isfinite(), l.abs(), 0))


@pytest.mark.parametrize("n", [1, 2, 150])
@pytest.mark.parametrize("q_amp,v_lo,v_hi", [(1.0, -12, 12), (2.0**40, -20, 0), (2.0**-30, 0, 30), (0.0, -60, -60), (1.0, 40, 40)])
def test_attention_int8_rows_of_very_different_scales(n, q_amp, v_lo, v_hi):
    """k and v rows whose scales differ by powers of two, up and down along the keys, and q far from 1: the
    scores stay ordinary (k's scale undoes q's), the weighted rows of v span the whole range."""
    p = Paged([n], [700], 4, 2, 128, 16, True, seed=31)
    where = (p.table[0, :44].long()[:, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)[:700]
    page, off = where // 16, where % 16
    step = (torch.arange(700, device="cuda") * 37 % 101).double() / 100
    up = torch.exp2((v_lo + (v_hi - v_lo) * step).round())
    p.q.mul_(q_amp)
    if q_amp:
        p.cache.k_scale[page, :, off] /= q_amp
        p.k[0] /= q_amp
    p.cache.v_scale[page, :, off] *= up[:, None].float()
    p.v[0] *= up[:, None, None]
    p.check()


@pytest.mark.parametrize("n,H,Hk", [(2, 2, 2), (3, 4, 2), (8, 4, 2), (4, 8, 1), (150, 2, 2)])
def test_attention_int8_later_keys_of_any_scale_stay_masked(n, H, Hk):
    """The last token's v is 2^60 times the others', or its scales are NaN or infinite: the rows before it do not
    see it and stay exact, whatever range the last row needs."""
    for bad in (2.0**60, float("nan"), float("inf")):
        p = Paged([n], [n + 9], H, Hk, 128, 16, True, seed=33)
        at = n + 8
        page, off = int(p.table[0, at // 16]), at % 16
        p.cache.v_scale[page, :, off] *= bad
        if bad == bad and bad < math.inf:
            p.v[0][at] *= bad
            p.check()
            continue
        p.cache.k_scale[page, :, off] *= bad
        got, lse = p.run()
        o, a, l = p.exact()
        got = got.view(n, H, 128)
        close(got[:n - 1], o[:n - 1], 2.0**-8 * (o.abs() + a)[:n - 1])
        close(lse[:n - 1], l[:n - 1], 1e-4 + 1e-5 * l.abs()[:n - 1])
        assert not torch.isfinite(got[n - 1]).any()


@pytest.mark.parametrize("n,H,Hk", [(1, 8, 1), (1, 16, 1), (2, 8, 2), (40, 4, 2)])
def test_attention_int8_query_heads_of_very_different_sizes(n, H, Hk):
    """Query heads that share a key head, every other one 2^-25 of the rest: with keys of size 2^25 the small
    ones have ordinary scores and stay exact."""
    p = Paged([n], [300], H, Hk, 128, 16, True, seed=34)
    small = torch.arange(H, device="cuda") % 2 == 1
    p.q.view(n, H, 128)[:, small] *= 2.0**-25
    p.cache.k_scale *= 2.0**25
    p.k[0] *= 2.0**25
    got, lse = p.run()
    o, a, l = p.exact()
    close(got.view(n, H, 128)[:, small], o[:, small], 2.0**-8 * (o.abs() + a)[:, small])
    close(lse[:, small], l[:, small], 1e-4 + 1e-5 * l.abs()[:, small])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n,H,Hk", [(3, 2, 2), (4, 8, 1), (150, 2, 2)])
def test_attention_nonfinite_values_of_later_keys_stay_masked(n, H, Hk, bad):
    """A later token's k and v hold NaN / Inf: earlier rows of the same tile, which must not see it, stay exact;
    the rows that see it are not finite."""
    p = Paged([n], [n + 70], H, Hk, 128, 16, False, seed=11)
    at = 70 + n // 2  # key of row n // 2
    page, off = int(p.table[0, at // 16]), at % 16
    p.cache.v[page, :, off, 5] = bad
    p.cache.k[page, :, off, 7] = bad
    got, lse = p.run()
    o, a, l = p.exact()
    close(got.view(n, H, 128)[:n // 2], o[:n // 2], 2.0**-8 * (o.abs() + a)[:n // 2])
    close(lse[:n // 2], l[:n // 2], 1e-4 + 1e-5 * l.abs()[:n // 2])
    assert not torch.isfinite(got.view(n, H, 128)[n // 2:, :, 5]).any()
    # v alone: the rows that see it are off in that column only
    p.cache.k[page, :, off, 7] = 0.5
    p.k[0][at, :, 7] = 0.5
    got, lse = p.run()
    o, a, l = p.exact()
    keep = torch.arange(128, device="cuda") != 5
    close(got.view(n, H, 128)[..., keep], o[..., keep], 2.0**-8 * (o.abs() + a)[..., keep])
    close(got.view(n, H, 128)[:n // 2, :, 5], o[:n // 2, :, 5], 2.0**-8 * (o.abs() + a)[:n // 2, :, 5])
    assert not torch.isfinite(got.view(n, H, 128)[n // 2:, :, 5]).any()
    close(lse, l, 1e-4 + 1e-5 * l.abs())


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [1, 3, 140])
def test_attention_freed_pages_before_the_window_are_not_read(n, int8):
    p = Paged([n], [900], 4, 2, 128, 16, int8, seed=13)
    exp, exp_l = p.run(window=200)
    first = 900 - n + 1 - 200  # the first row's first visible key
    p.table[0, :max(0, first // 16)] = -1  # pages wholly before it are gone
    got, lse = p.run(window=200)
    p.cache.check()
    assert torch.equal(got, exp) and torch.equal(lse, exp_l)


@pytest.mark.parametrize("n", [1, 140])
def test_attention_bad_pages_and_lengths_are_reported(n):
    p = Paged([n], [400], 2, 2, 128, 16, False, seed=14, stale=0.0)
    good = p.table[0, 7].clone()
    p.table[0, 7] = 1 << 30
    p.run()
    with pytest.raises(RustaneError):
        p.cache.check()
    p.table[0, 7] = good
    for bad in (-5, p.table.shape[1] * 16 + 1):
        p.kv_lens[0] = bad
        out, lse = p.run()
        with pytest.raises(RustaneError):
            p.cache.check()
        assert (out == 0).all() and torch.isinf(lse).all()
    p.kv_lens[0] = 400
    p.check()


def test_attention_strided_rows_hints_and_streams():
    p = Paged([1, 40, 3], [77, 200, 3], 4, 2, 128, 32, True, seed=15)
    exp, exp_l = p.run()
    wide = torch.zeros(p.T, 4 * 128 + 24, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:8 + 512] = p.q
    out = torch.full((p.T, 600), 3.0, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse = p.run(q=wide[:, 8:520], out=out[:, 16:528])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, exp) and torch.equal(lse, exp_l)
    assert (out[:, :16] == 3).all() and (out[:, 528:] == 3).all()
    # the bounds are hints: larger ones, and a max_q below the truth, give results within tolerance
    p.check(max_q=4096, max_kv=100000)
    p.check(max_q=1, max_kv=1)


def test_attention_in_a_cuda_graph_follows_the_lengths():
    p = Paged([1, 1], [300, 40], 4, 4, 128, 16, False, seed=16)
    out = torch.empty(2, 512, device="cuda", dtype=torch.bfloat16)
    p.run(out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.run(out=out, max_kv=512)
    for lens in ([300, 40], [17, 33], [1, 0]):
        p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        p.kv_lens_l = lens
        graph.replay()
        o, a, _ = p.exact()
        close(out.view(2, 4, 128), o, 2.0**-8 * (o.abs() + a) + 1e-30)


# --------------------------------------------------------------------- logits
def plain_logits(x, hist, n_prompt, rep, pres, freq, bias, allowed):
    """One row in 64 bits: hist and bias as lists, allowed a bool array or None."""
    x = x.astype(np.float64).copy()
    for t in set(hist):
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
    made = hist[n_prompt:]
    for t in set(made):
        x[t] -= freq * made.count(t) + pres
    for t, b in bias:
        x[t] += b
    if allowed is not None:
        x[~allowed] = -np.inf
    top = np.nanmax(np.where(np.isnan(x), -np.inf, x))
    return x, (int(np.flatnonzero(x == top)[0]) if top > -np.inf else -1)


@pytest.mark.parametrize("B,V,L,masked,pad", [(1, 1, 0, False, 0), (3, 33, 5, True, 0), (2, 1000, 40, True, 24), (5, 8192, 700, True, 0),
                                              (1, 50001, 3000, True, 3), (2, 140000, 100, False, 0), (300, 517, 9, True, 7),
                                              (1, 300000, 20, True, 4)])
def test_logits_adjust(B, V, L, masked, pad):
    rng = np.random.default_rng(V + L)
    store = np.full((B, V + pad), 99.0, np.float32)
    store[:, :V] = 3 * rng.standard_normal((B, V))
    x = torch.from_numpy(store).cuda()[:, :V]
    lens = rng.integers(0, L + 1, B)
    hist = [[int(t) for t in (rng.random(n) ** 2 * V).astype(np.int64)] for n in lens]
    n_prompt = [int(rng.integers(0, n + 1)) for n in lens]
    nb = [int(rng.integers(0, min(V, 70) + 1)) for _ in range(B)]
    bias = [[(int(t), float(np.float32(4 * rng.standard_normal()))) for t in rng.integers(0, V, n)] for n in nb]  # with repeats
    rep, pres, freq = (rng.random((3, B)) + [[1.0], [0.0], [0.0]]).astype(np.float32)
    allowed = rng.random((B, V)) < 0.5 if masked else None
    bits = None
    if masked:
        padded = np.zeros((B, -(-V // 32) * 32), np.uint8)
        padded[:, :V] = allowed
        bits = torch.from_numpy(np.packbits(padded, axis=1, bitorder="little").view(np.int32).copy()).cuda()

    def flat(rows, dtype):
        return torch.tensor([t for r in rows for t in r], dtype=dtype, device="cuda")

    def starts(ns):
        return torch.tensor(np.concatenate([[0], np.cumsum(ns)]), dtype=torch.int32, device="cuda")

    T = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(hist=flat(hist, torch.int32), hist_start=starts(lens), n_prompt=torch.tensor(n_prompt, dtype=torch.int32, device="cuda"),
              repetition=T(rep), presence=T(pres), frequency=T(freq), bias_ids=flat([[t for t, _ in r] for r in bias], torch.int32),
              bias_vals=flat([[b for _, b in r] for r in bias], torch.float32), bias_start=starts(nb), mask=bits)
    out, token = ops.logits_adjust(x, **kw)
    for b in range(B):
        e, t = plain_logits(store[b, :V], hist[b], n_prompt[b], float(rep[b]), float(pres[b]), float(freq[b]), bias[b],
                            allowed[b] if masked else None)
        # a handful of fp32 operations on values up to about 4 * 70 (repeated biases)
        close(out[b], torch.from_numpy(e).cuda(), 1e-5 + 1e-6 * torch.from_numpy(np.nan_to_num(np.abs(e), posinf=0, neginf=0)).cuda())
        got = int(token[b])
        assert (got == -1) == (t == -1)
        if t >= 0:
            assert got == int(np.flatnonzero(out[b].cpu().numpy() == out[b].max().item())[0])
            assert e[got] >= e[t] - 1e-4
    same, token2 = ops.logits_adjust(x, out=x, **kw)
    assert torch.equal(same, out) and torch.equal(token2, token)
    if pad:
        assert (same.as_strided((B, V + pad), (V + pad, 1))[:, V:] == 99.0).all()


def test_logits_edge_rows():
    V = 40000
    x = torch.zeros(6, V, device="cuda")
    x[0, 17] = x[0, 9] = x[0, 39999] = 2.0   # ties: the lowest index
    x[1, :] = float("nan")                   # NaN is never chosen
    x[1, 30001] = -5.0
    x[2, :] = -float("inf")                  # nothing above -inf
    x[3, 5] = float("inf")
    x[4, :] = float("nan")
    out, token = ops.logits_adjust(x)
    assert token.tolist() == [9, 30001, -1, 5, -1, 0]
    assert torch.equal(torch.nan_to_num(out, nan=3.0), torch.nan_to_num(x, nan=3.0))
    mask = torch.zeros(6, V // 32, dtype=torch.int32, device="cuda")
    mask[0, 0] = 1 << 17
    mask[1] = -1
    mask[5, 1000] = -(1 << 31)
    out, token = ops.logits_adjust(x, mask=mask)
    assert token.tolist() == [17, 30001, -1, -1, -1, 1000 * 32 + 31]
    assert torch.isinf(out[4]).all()  # forbidden NaN becomes -inf
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    hist = torch.tensor([3, -1, V, 3], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 0, 0, 0, 0, 0, 4], dtype=torch.int32, device="cuda")
    out, token = ops.logits_adjust(x, hist=hist, hist_start=start, frequency=torch.full((6,), 2.0, device="cuda"), err=err)
    assert err.item() == 4 and out[5, 3].item() == -4.0 and token[5].item() == 0
    out, token = ops.logits_adjust(x[:0])
    assert out.shape == (0, V) and token.shape == (0,)


# ------------------------------------------------------------------- refusals
def test_refusals():
    L = __import__("rustane_b200")._lib.lib()
    g, qkv, pos, rope, gq, gk = rope_case(4, 2, 2, 64, 64, "half", True, seed=0)
    cache = new_cache(2, 16, 2, 64, False)
    for bad in (lambda: ops.qk_norm_rope(qkv.float(), pos, rope, 2, 2), lambda: ops.qk_norm_rope(qkv, pos.long(), rope, 2, 2),
                lambda: ops.qk_norm_rope(qkv, pos[:3], rope, 2, 2), lambda: ops.qk_norm_rope(qkv, pos, rope, 3, 2),
                lambda: ops.qk_norm_rope(qkv, pos, rope, 2, 2, gq), lambda: ops.qk_norm_rope(qkv.cpu(), pos, rope, 2, 2),
                lambda: ops.qk_norm_rope(qkv, pos, rope, 2, 2, gq.bfloat16(), gk),
                lambda: ops.qk_norm_rope(qkv.t().contiguous().t(), pos, rope, 2, 2),
                lambda: ops.qk_norm_rope_backward(qkv, None, pos, rope, 2, 2, gq, gk),
                lambda: ops.kv_append(qkv, pos, pos.long(), rope, cache, 2), lambda: ops.kv_gather(cache, pos.long()),
                lambda: ops.KvCache(cache.k, cache.v, cache.k[..., 0].float()), lambda: ops.KvCache(cache.k, cache.v[:1]),
                lambda: ops.Rope(rope.cos, rope.sin, "sideways"), lambda: ops.Rope.tables(4, 64, "cuda", scaling="much"),
                lambda: ops.logits_adjust(qkv), lambda: ops.logits_adjust(qkv.float(), hist=pos),
                lambda: ops.logits_adjust(qkv.float(), mask=pos[None])):
        with pytest.raises(ValueError):
            bad()
    odd = torch.empty(4, 6 * 64 + 4, device="cuda", dtype=torch.bfloat16)[:, 4:]  # rows not on 16 bytes
    for bad in (lambda: ops.qk_norm_rope(odd, pos, rope, 2, 2), lambda: ops.kv_append(odd, pos, pos, rope, cache, 2),
                lambda: ops.Rope.tables(4, 63, "cuda"), lambda: ops.Rope.tables(0, 64, "cuda"),
                lambda: ops.qk_norm_rope(qkv, pos, ops.Rope.tables(4, 24, "cuda"), 2, 2),
                lambda: ops.kv_gather(new_cache(2, 24, 2, 64, False), pos), lambda: ops.kv_gather(new_cache(2, 8, 2, 64, False), pos),
                lambda: ops.kv_gather(new_cache(2, 16, 2, 32, False), pos)):
        with pytest.raises(RustaneError) as e:
            bad()
        assert e.value.code == -2
    ws = ops.AttentionWorkspace("cuda")
    lens, start, table = pos[:1].clone(), torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    q = qkv[:, :128].contiguous()
    for bad in (lambda: ops.attention_paged(q, cache, table, lens, start, 3, ws, 4, 32),
                lambda: ops.attention_paged(q.float(), cache, table, lens, start, 2, ws, 4, 32),
                lambda: ops.attention_paged(q, cache, table[0], lens, start, 2, ws, 4, 32),
                lambda: ops.attention_paged(q, cache, table, lens, start[:1], 2, ws, 4, 32)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.attention_paged(torch.cat((q, q[:, :64]), 1), cache, table, lens, start, 3, ws, 4, 32),
                lambda: ops.attention_paged(q, cache, table, lens, start, 2, ws, 4, 32, window=-1)):
        with pytest.raises(RustaneError) as e:
            bad()
        assert e.value.code == -2
    st = torch.cuda.current_stream().cuda_stream
    args = [q.data_ptr(), 128, q.data_ptr(), 128, None, cache.ref, table.data_ptr(), 2, lens.data_ptr(), start.data_ptr(), 1, 4, 4, 32, 2, 0,
            0.1, ws.buf.data_ptr(), ws.buf.numel(), None, st]
    for i, rc in ((0, -1), (2, -1), (5, -1), (6, -1), (8, -1), (17, -1)):
        a = list(args)
        a[i] = None
        assert L.rt_kernel_attention_paged(*a) == rc
    a = list(args)
    a[18] = 16
    assert L.rt_kernel_attention_paged(*a) == -2
    assert L.rt_kernel_kv_gather(None, None, None, None, 0, 1, None, st) == -1
    assert L.rt_kernel_logits_adjust(None, 4, None, 4, None, 1, 4, None, None, st) == -1
    torch.cuda.synchronize()
