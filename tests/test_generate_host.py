"""What rustane_b200.generate.Generator does on the host, on the CPU: the library's and the operators' calls are replaced by
functions that record them, and the device by the CPU."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import ModelConfig, RustaneError, generate, ops  # noqa: E402
from rustane_b200._lib import RT_ERR_DEVICE, RT_ERR_OOM, RT_ERR_TOKEN  # noqa: E402


class Current:
    """Stands for torch.cuda.device: which device is current inside."""
    now = None

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.before, Current.now = Current.now, self.device

    def __exit__(self, *_):
        Current.now = self.before


@pytest.fixture
def host(monkeypatch):
    """(make, calls): make(pages) gives a Generator; calls are (name, current device)."""
    calls = []
    Current.now = None

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, Current.now)) or 0

    monkeypatch.setattr(generate, "lib", lambda: Lib())
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=0))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: None)

    def append(qkv, pos, slots, rope, cache, heads, *a):
        calls.append(("kv_append", Current.now))
        return torch.zeros(qkv.shape[0], heads * 128, dtype=torch.bfloat16)

    monkeypatch.setattr(ops, "kv_append", append)
    monkeypatch.setattr(ops, "attention_paged", lambda q, *a, **k: (torch.zeros_like(q), None))
    monkeypatch.setattr(ops, "qk_norm_rope", lambda qkv, *a, **k: qkv)

    def make(pages=8, page_size=16, int8=False):
        c = ModelConfig.custom(128, 256, 1, 2, seq=64, vocab=64)
        g = object.__new__(generate.Generator)
        g.cfg, g.page_size, g.softcap, g.device = c, page_size, 0.0, torch.device("cpu")
        w = torch.zeros(1, 1)
        g.embed = g.embed_b = g.gamma_final = w
        g.layers = [dict(wqkv=w, wo=w, w13=w, w2=w, gamma1=w, gamma2=w) for _ in range(c.nlayers)]
        g.rope = None

        def cache():
            shape = (pages, c.kv_heads, page_size, c.hd)
            x = SimpleNamespace(err=torch.zeros(1, dtype=torch.int32), device=torch.device("cpu"),
                                k=torch.zeros(shape, dtype=torch.int8 if int8 else torch.bfloat16), k_scale=None, v_scale=None)
            x.v = x.k.clone()
            x.check = lambda: ops.KvCache.check(x)
            if int8:
                x.k_scale, x.v_scale = torch.zeros(shape[:3]), torch.zeros(shape[:3])
            return x

        g.caches = [cache() for _ in range(c.nlayers)]
        g.uses, g.workspace, g.err, g.alpha = [0] * pages, None, torch.zeros(1, dtype=torch.int32), 0.5
        return g

    return make, calls


def test_the_librarys_calls_run_on_the_generators_device(host):
    """The library launches on the current device: whichever that is outside, it is the generator's inside."""
    make, calls = host
    g = make()
    seq = generate.Sequence()
    g.forward(torch.zeros(5, dtype=torch.int32), [seq], [5])
    g.prefill([[1, 2, 3]])
    g.score([1, 2, 3])
    assert {n for n, _ in calls} >= {"rt_kernel_gemm", "rt_kernel_rmsnorm_fwd", "rt_kernel_embed_gather", "rt_kernel_attention_fwd"}
    assert all(d == g.device for _, d in calls)
    assert Current.now is None


def adjust(logits, **k):
    return logits, torch.zeros(logits.shape[0], dtype=torch.int32)


@pytest.mark.parametrize("prompts,max_new,answers", [([[1] * 40], 20, 1), ([[1] * 20, [2] * 40], 1, 1), ([[1] * 33], 1, 2),
                                                     ([[1] * 17], 2, 4)])
def test_a_request_that_does_not_fit_leaves_no_page_behind(host, monkeypatch, prompts, max_new, answers):
    """It runs out while answering, while the second prompt is fed, and while an answer is forked."""
    make, _ = host
    monkeypatch.setattr(ops, "logits_adjust", adjust)
    g = make(pages=3)
    with pytest.raises(RustaneError) as e:
        g.generate(prompts, max_new, answers=answers)
    assert e.value.code == RT_ERR_OOM
    assert g.uses == [0, 0, 0]
    assert len(g.generate([[1] * 30], 10)[0][0]) == 10


def test_a_reported_error_leaves_no_page_behind(host, monkeypatch):
    make, _ = host
    monkeypatch.setattr(ops, "logits_adjust", adjust)
    g = make()
    g.err[0] = 4
    with pytest.raises(RustaneError):
        g.generate([[1, 2]], 3)
    assert g.uses == [0] * 8


def test_forward_that_fails_leaves_its_sequences_as_they_were(host, monkeypatch):
    make, _ = host
    g = make(pages=3)
    a, b = generate.Sequence(), generate.Sequence()
    g.forward(torch.zeros(3, dtype=torch.int32), [a, b], [1, 2])
    with pytest.raises(RustaneError):
        g.forward(torch.zeros(60, dtype=torch.int32), [a, b], [20, 40])
    assert (len(a.pages), a.cached, len(b.pages), b.cached) == (1, 1, 1, 2) and sum(g.uses) == 2
    monkeypatch.setattr(ops, "attention_paged", lambda *x, **k: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        g.forward(torch.zeros(21, dtype=torch.int32), [a, b], [20, 1])
    assert (len(a.pages), a.cached, len(b.pages), b.cached) == (1, 1, 1, 2) and sum(g.uses) == 2


def test_check_clears_every_word_that_it_reports(host):
    """One request's errors are not the next one's."""
    make, _ = host
    g = make()
    for word, code in ((g.err, 4), (g.caches[0].err, 6), (g.caches[1].err, 6)):
        word[0] = code
    with pytest.raises(RustaneError) as e:
        g.check()
    assert e.value.code == RT_ERR_TOKEN
    assert not any(int(w) for w in (g.err, g.caches[0].err, g.caches[1].err))
    g.check()
    g.caches[1].err[0] = 6
    with pytest.raises(RustaneError) as e:
        g.check()
    assert e.value.code == RT_ERR_DEVICE
    g.check()


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("row,answers,exp", [([1, 3, 2, 3], 3, [1, 3, 2]),          # equal values: the lower index first
                                             ([NAN, 1, NAN, 2], 2, [3, 1]),         # NaN is never chosen
                                             ([0, INF, -5, -INF], 3, [1, 0, 2])])
def test_first_tokens_of_several_answers(host, monkeypatch, row, answers, exp):
    """The best ones by the greedy token's own rule."""
    make, _ = host
    g = make(pages=40)
    logits = torch.full((1, 64), -INF)
    logits[0, :4] = torch.tensor(row)
    monkeypatch.setattr(g, "_logits", lambda x: logits.expand(x.shape[0], -1).clone())
    monkeypatch.setattr(ops, "logits_adjust", adjust)
    out = g.generate([[1, 2], [3]], 2, answers=answers)
    assert [[a[0] for a in p] for p in out] == [exp, exp]


@pytest.mark.parametrize("max_new", [1, 3])
def test_fewer_tokens_than_answers_are_refused(host, monkeypatch, max_new):
    make, _ = host
    g = make(pages=40)
    logits = torch.full((1, 64), -INF)
    logits[0, :3] = torch.tensor([1, 2, NAN])
    monkeypatch.setattr(g, "_logits", lambda x: logits.expand(x.shape[0], -1).clone())
    monkeypatch.setattr(ops, "logits_adjust", adjust)
    assert [a[0] for a in g.generate([[1]], max_new, answers=2)[0]] == [1, 0]
    with pytest.raises(ValueError, match="answer"):
        g.generate([[1]], max_new, answers=3)
    assert not any(g.uses)


@pytest.mark.parametrize("n", [0, 1])
def test_score_of_a_text_without_a_second_token_is_empty(host, n):
    make, calls = host
    assert make().score([5] * n).shape == (0,)
    assert not calls


@pytest.mark.parametrize("n", [2, 77, 128, 290])
def test_score_uses_no_position_past_its_text(host, monkeypatch, n):
    """Whatever the training form's attention pads a text to."""
    make, _ = host
    seen = []
    monkeypatch.setattr(ops, "qk_norm_rope", lambda qkv, pos, *a, **k: seen.append(pos) or qkv)
    assert make().score([5] * n).shape == (n - 1,)
    assert len(seen) == 2
    for pos in seen:
        assert torch.equal(pos[:n], torch.arange(n, dtype=torch.int32)) and int(pos.max()) == n - 1 and int(pos.min()) == 0


@pytest.mark.parametrize("rules", [dict(forbid=[-1]), dict(forbid=[3, 64]), dict(bias={-1: 2.0}), dict(bias={64: 2.0})])
def test_rules_for_ids_outside_the_vocabulary_are_refused(host, monkeypatch, rules):
    """(-1 forbade the vocabulary's last token.)"""
    make, calls = host
    monkeypatch.setattr(ops, "logits_adjust", adjust)
    with pytest.raises(ValueError, match="ids"):
        make().generate([[1]], 2, **rules)
    assert not calls
