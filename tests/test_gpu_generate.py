"""Generation through the paged cache against a 64-bit decoder on the same bf16 weights, measured by how
far the model's own forward (rt_forward) is from it.

Both run the same bf16 kernels but for the attention and the rotation, which rounds q and k once more,
so the generator's logits may be twice as far from the 64-bit ones as the forward's.  An int8 cache's
k and v are 0.021 / sqrt(12) = 0.006 of a row's rms off (step amax / 127, amax about 2.7 rms at 128
entries), 5.5 times bf16's rounding, at 2 of a layer's about 10 roundings: sqrt(0.8 + 0.2 * 30) = 2.6,
with the factor 2 again under 6 times as far.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import CompiledKernels, ModelConfig, generate  # noqa: E402
from rustane_b200.tensors import ModelTensors  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = ModelConfig.custom(512, 1024, 4, 3, seq=256, vocab=1024)
    w = ModelTensors.normal(cfg, seed=5, std=0.08)
    k = CompiledKernels.compile(cfg, max_batch=2, device=0)
    k.upload_weights(w)
    rng = np.random.default_rng(3)
    tok = rng.integers(0, cfg.vocab, 2 * cfg.seq).astype(np.uint32)
    tgt = np.roll(tok, -1)
    _, losses = k.forward(tok, tgt, per_token=True)
    logits = k.logits().reshape(2, cfg.seq, cfg.vocab)
    k.close()
    return cfg, w, tok.reshape(2, cfg.seq), losses.reshape(2, cfg.seq), logits


def exact_logits(cfg, w, tok):
    """[tokens, vocab] of one sequence in 64 bits, weights rounded to bf16 (the embedding's rows are not)."""
    def up(a, half=True):
        x = torch.from_numpy(a).cuda()
        return (x.bfloat16() if half else x).double()

    def norm(x, gamma):
        return x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * up(gamma, False)

    n, alpha = len(tok), 1 / np.sqrt(2 * cfg.nlayers)
    x = up(w.embed, False)[torch.from_numpy(tok.astype(np.int64)).cuda()]
    ang = torch.arange(n, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(64, device="cuda").double() / 64)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def turn(v):
        a, b = v[..., 0::2], v[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)

    later = torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1)
    for L in w.layers:
        h = norm(x, L.gamma1)
        q, k, v = ((h @ up(m)).view(n, cfg.heads, 128) for m in (L.wq, L.wk, L.wv))
        s = torch.einsum("ihd,jhd->hij", turn(q), turn(k)) / np.sqrt(128)
        p = torch.softmax(s.masked_fill(later, -np.inf), -1)
        x = x + alpha * torch.einsum("hij,jhd->ihd", p, v).flatten(1) @ up(L.wo)
        h = norm(x, L.gamma2)
        x = x + alpha * (torch.nn.functional.silu(h @ up(L.w1)) * (h @ up(L.w3))) @ up(L.w2).T
    return (norm(x, w.gamma_final) @ up(w.embed).T).cpu().numpy()


@pytest.mark.parametrize("dtype,times,page", [(torch.bfloat16, 2, 16), (torch.int8, 6, 64)])
def test_chunks_and_steps_are_as_near_as_the_forward(model, dtype, times, page):
    cfg, w, tok, _, logits = model
    exact = [exact_logits(cfg, w, t) for t in tok]
    off = max(np.abs(logits[i] - exact[i]).max() for i in range(2))
    g = generate.Generator(cfg, w, capacity=2 * 256 + 2 * page, page_size=page, cache_dtype=dtype, max_pos=256)
    dev = torch.from_numpy(tok.astype(np.int32)).cuda()
    a, b = generate.Sequence(), generate.Sequence()
    at = [0, 0]
    for na, nb in [(33, 1), (100, 64), (1, 150), (1, 1), (17, 3), (1, 1)]:
        new = torch.cat((dev[0, at[0]:at[0] + na], dev[1, at[1]:at[1] + nb])).contiguous()
        got = g.forward(new, [a, b], [na, nb]).cpu().numpy()
        at = [at[0] + na, at[1] + nb]
        assert np.abs(got[0] - exact[0][at[0] - 1]).max() <= times * off
        assert np.abs(got[1] - exact[1][at[1] - 1]).max() <= times * off
    g.check()


def test_score_is_the_training_forwards_loss(model):
    cfg, w, tok, losses, _ = model
    g = generate.Generator(cfg, w, capacity=64, max_pos=256)
    got = g.score(tok[0].tolist()).cpu().numpy()
    # a loss is a difference of logits of size about 10, each within bf16 products' noise
    assert np.abs(got - losses[0, :-1]).max() < 2e-2 * max(1.0, np.abs(losses[0]).max())
    short = g.score(tok[0, :77].tolist()).cpu().numpy()
    assert np.abs(short - losses[0, :76]).max() < 2e-2 * max(1.0, np.abs(losses[0]).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_generate_is_greedy_over_its_own_logits(model, dtype):
    cfg, w, tok, _, _ = model
    g = generate.Generator(cfg, w, capacity=700, cache_dtype=dtype, max_pos=256)
    prompts = [tok[0, :37].tolist(), tok[1, :5].tolist(), [7]]
    out = g.generate(prompts, max_new=12, chunk=16)
    assert [len(p) for p in out] == [1, 1, 1] and all(len(a[0]) == 12 for a in out)
    assert all(n == 0 for n in g.uses)  # every page was handed back
    assert out == g.generate(prompts, max_new=12, chunk=16)
    # each token is the best one after what precedes it, or within the noise of another chunking of it
    for p, (a,) in zip(prompts, out):
        for i in (0, 5, 11):
            _, logits = g.prefill([p + a[:i]])
            top = logits[0].max().item()
            assert top - logits[0, a[i]].item() <= 2e-2 * max(1.0, abs(top)) * (3 if dtype == torch.int8 else 1)
        g.uses = [0] * len(g.uses)


def test_answers_penalties_biases_and_forbidden_tokens(model):
    cfg, w, tok, _, _ = model
    g = generate.Generator(cfg, w, capacity=2000, max_pos=256)
    p = [tok[0, :21].tolist(), tok[1, :40].tolist()]
    out = g.generate(p, max_new=8, answers=3)
    assert [len(a) for a in out] == [3, 3]
    for prompt, answers in zip(p, out):
        _, logits = g.prefill([prompt])
        assert [a[0] for a in answers] == logits[0].topk(3).indices.tolist()
        g.uses = [0] * len(g.uses)
        # an answer from a forked cache continues as one that was fed whole
        again = g.generate([prompt + answers[1][:1]], max_new=7)[0][0]
        _, l2 = g.prefill([prompt + answers[1][:1]])
        gap = l2[0].topk(2).values
        if (gap[0] - gap[1]).item() > 2e-2 * gap[0].abs().item():
            assert again[0] == answers[1][1]
        g.uses = [0] * len(g.uses)
    forced = g.generate(p, max_new=6, bias={9: 1e4})
    assert all(a == [9] * 6 for (a,) in forced)
    banned = g.generate(p, max_new=6, bias={9: 1e4}, forbid=[9])
    assert all(9 not in a for (a,) in banned)
    once = g.generate(p, max_new=6, bias={t: 100.0 for t in range(6)}, presence=1e3)
    assert all(sorted(a) == list(range(6)) for (a,) in once)
    with pytest.raises(ValueError):
        g.generate([[]], max_new=2)


def test_cli_prints_one_line_per_answer(capsys):
    lines = []
    a = generate.parse_args(["--model", "custom:256,512,2,128", "--prompt", "1,2,3", "--prompt", "4", "--max-new", "5", "--answers", "2",
                             "--cache", "int8", "--repetition", "1.2"])
    generate.run(a, out=lines.append)
    assert len(lines) == 4 and all(len(ln.split(",")) == 5 for ln in lines)
