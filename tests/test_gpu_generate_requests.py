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
