"""Requests one after another on one Generator: those that fail, those that share a past, and their errors."""
import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import RustaneError, generate  # noqa: E402
from test_gpu_generate import model  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def test_a_request_that_does_not_fit_changes_nothing_for_the_next(model):  # noqa: F811
    cfg, w, tok, _, _ = model
    prompts = [tok[0, :37].tolist(), tok[1, :20].tolist()]
    g = generate.Generator(cfg, w, capacity=160, max_pos=256)
    exp = g.generate(prompts, max_new=9, answers=2)
    for big in (dict(prompts=[tok[0, :200].tolist()], max_new=2), dict(prompts=prompts, max_new=200),
                dict(prompts=prompts, max_new=2, answers=4)):
        with pytest.raises(RustaneError):
            g.generate(**big)
        assert all(n == 0 for n in g.uses)
    assert g.generate(prompts, max_new=9, answers=2) == exp


def test_a_request_past_the_rotary_tables_is_reported_once(model):  # noqa: F811
    cfg, w, tok, _, _ = model
    g = generate.Generator(cfg, w, capacity=400, max_pos=64)
    prompt = tok[0, :30].tolist()
    exp = g.generate([prompt], max_new=5)
    with pytest.raises(RustaneError):
        g.generate([tok[1, :80].tolist()], max_new=3)  # every layer's cache reports it
    assert g.generate([prompt], max_new=5) == exp


def test_forbidden_tokens_start_no_answer(model):  # noqa: F811
    cfg, w, tok, _, _ = model
    g = generate.Generator(cfg, w, capacity=400, max_pos=256)
    p = [tok[0, :9].tolist(), tok[1, :21].tolist()]
    out = g.generate(p, max_new=3, answers=3, forbid=[t for t in range(cfg.vocab) if t not in (5, 17, 900, 1000)])
    for answers in out:
        firsts = [a[0] for a in answers]
        assert len(set(firsts)) == 3 and all(t in (5, 17, 900, 1000) for a in answers for t in a)
    with pytest.raises(ValueError):
        g.generate(p, max_new=3, answers=3, forbid=[t for t in range(cfg.vocab) if t not in (5, 900)])
    assert not any(g.uses)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_a_forked_sequence_has_the_same_past(model, dtype):  # noqa: F811
    """Bit for bit, codes and scales, also of an infinite key; and what follows does not touch the source."""
    cfg, w, tok, _, _ = model
    g = generate.Generator(cfg, w, capacity=200, cache_dtype=dtype, max_pos=256)
    (seq,), _ = g.prefill([tok[0, :37].tolist()])
    if dtype == torch.bfloat16:
        g.caches[0].k[seq.pages[2], :, 3, 8] = float("inf")
    new = g.fork(seq)
    assert new.pages[:2] == seq.pages[:2] and new.pages[2] != seq.pages[2] and new.cached == 37

    def rows(s):  # the last page's 5 tokens
        return [t[s.pages[2], :, :5] for c in g.caches for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None]

    before = [r.clone() for r in rows(seq)]
    assert all(torch.equal(a, b) for a, b in zip(rows(new), before))
    g.forward(torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), [new], [3])
    assert all(torch.equal(a, b) for a, b in zip(rows(seq), before))
    assert all(torch.equal(a, b) for a, b in zip(rows(new), before))
    g.free(seq)
    g.free(new)
    assert not any(g.uses)


def test_score_of_a_text_that_just_fits_the_rotary_tables(model):  # noqa: F811
    cfg, w, tok, _, _ = model
    text = tok[0, :150].tolist()
    exp = generate.Generator(cfg, w, capacity=64, max_pos=256).score(text)
    g = generate.Generator(cfg, w, capacity=64, max_pos=150)
    assert torch.equal(g.score(text), exp)
    assert g.score(text[:1]).shape == (0,)
    with pytest.raises(RustaneError):
        g.score(text + [1])
