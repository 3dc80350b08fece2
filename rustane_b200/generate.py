"""Answers from a trained model: greedy generation over a paged key/value cache.

    python -m rustane_b200.generate --model gpt_karpathy --ckpt ckpt.bin --prompt 11,42,7 [--prompt 5,6 ...] \\
        [--max-new 64] [--answers 1] [--chunk 512] [--cache bf16|int8] [--page-size 16] [--max-pos 4096]
        [--rope-linear F] [--repetition 1.0] [--presence 0] [--frequency 0] [--forbid 0,1] [--bias 5:1.5,9:-2]
        [--softcap 0] [--device 0]

Prompts are token ids (the training data's own ids; the reference has no tokenizer).  All prompts are
served together: fed in chunks of --chunk tokens each, then one token of every answer a step.  With
--answers N an answer starts from each of a prompt's N best first tokens; the answers share the
prompt's full pages and copy its last one.  One line per answer: the ids, comma separated.

`Generator` is the same as a library: the model's own kernels (embedding, RMSNorm, fused GEMMs) with
the serving operators of `rustane_b200.ops` around the attention.  `Generator.score` runs the training
form (rotation out of place, causal attention without a cache) and returns per-token losses.
"""
from __future__ import annotations

import functools
import math
import sys
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib, ops
from ._lib import RustaneError, lib
from .data import load_checkpoint
from .engine import random_weights
from .model import ModelConfig
from .tensors import ModelTensors
from .train import UsageError, model_config


@dataclass
class Sequence:
    """A request: its pages of the cache and the tokens cached so far."""
    pages: list[int] = field(default_factory=list)
    cached: int = 0


def _on_device(method):
    """The library launches on the current device: the generator's, while `method` runs."""
    @functools.wraps(method)
    def call(self, *args, **kw):
        with torch.cuda.device(self.device):
            return method(self, *args, **kw)
    return call


def _best(logits: torch.Tensor, n: int) -> torch.Tensor:
    """The n best tokens of each row by the greedy token's rule: equal values by index, never NaN or -inf."""
    values, tokens = logits.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).sort(dim=1, descending=True, stable=True)
    if not (values[:, :n] > -math.inf).all():
        raise ValueError(f"fewer than {n} tokens may start an answer")
    return tokens[:, :n]


class Generator:
    """A model's weights on one GPU and a paged cache for `capacity` tokens of all requests together."""

    def __init__(self, cfg: ModelConfig, weights: ModelTensors, capacity: int, page_size: int = 16,
                 cache_dtype: torch.dtype = torch.bfloat16, max_pos: int | None = None, device: int = 0, softcap: float = 0.0,
                 **rope):
        self.cfg, self.page_size, self.softcap = cfg, page_size, softcap
        self.device = torch.device("cuda", device)

        def up(a, dtype=torch.bfloat16):
            return torch.from_numpy(np.ascontiguousarray(a)).to(self.device).to(dtype)

        self.embed, self.embed_b = up(weights.embed, torch.float32), up(weights.embed)
        self.gamma_final = up(weights.gamma_final, torch.float32)
        self.layers = [dict(wqkv=up(np.concatenate([w.wq, w.wk, w.wv], 1)), wo=up(w.wo),
                            w13=up(np.concatenate([w.w1, w.w3], 1)), w2=up(w.w2), gamma1=up(w.gamma1, torch.float32),
                            gamma2=up(w.gamma2, torch.float32)) for w in weights.layers]
        self.rope = ops.Rope.tables(max_pos or max(cfg.seq, 4096), cfg.hd, self.device, **rope)
        pages = -(-capacity // page_size)
        self.caches = [ops.KvCache.empty(pages, page_size, cfg.kv_heads, cfg.hd, cache_dtype, self.device)
                       for _ in range(cfg.nlayers)]
        self.uses = [0] * pages  # sequences that hold each page
        self.workspace = ops.AttentionWorkspace(self.device)
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.alpha = 1.0 / math.sqrt(2.0 * cfg.nlayers)

    # ------------------------------------------------------------- the model's kernels
    def _call(self, name: str, *args) -> None:
        rc = getattr(lib(), name)(*args, torch.cuda.current_stream(self.device).cuda_stream)
        if rc != _lib.RT_OK:
            raise RustaneError(rc, name)

    def _gemm(self, x, w, n: int, epi: int, b_mn: bool, aux=None, out2=None, n_half: int = 0, alpha: float = 1.0):
        M, K = x.shape
        wide = 2 * n if epi == _lib.EPI_SWIGLU else n
        out = torch.empty((M, wide), device=self.device,
                          dtype=torch.float32 if epi in (_lib.EPI_RESIDUAL, _lib.EPI_F32) else torch.bfloat16)
        self._call("rt_kernel_gemm", x.data_ptr(), K, 0, w.data_ptr(), w.shape[1], int(b_mn), M, n, K, epi, out.data_ptr(), wide,
                   None if out2 is None else out2.data_ptr(), n, None if aux is None else aux.data_ptr(), n, alpha, 0, None, None,
                   1, 0, n_half, 0, self.err.data_ptr())
        return out

    def _norm(self, x, gamma):
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=self.device)
        rms = torch.empty(x.shape[0], device=self.device)
        self._call("rt_kernel_rmsnorm_fwd", x.data_ptr(), gamma.data_ptr(), out.data_ptr(), rms.data_ptr(), *x.shape)
        return out

    def _blocks(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """The decoder over token ids [T] int32; attend(layer index, qkv) -> [T, q_dim] bf16."""
        c = self.cfg
        x = torch.empty((tokens.shape[0], c.dim), device=self.device)
        self._call("rt_kernel_embed_gather", self.embed.data_ptr(), tokens.data_ptr(), x.data_ptr(), x.shape[0], c.dim, c.vocab,
                   self.err.data_ptr())
        for i, w in enumerate(self.layers):
            qkv = self._gemm(self._norm(x, w["gamma1"]), w["wqkv"], c.q_dim + 2 * c.kv_dim, _lib.EPI_BF16, True)
            x = self._gemm(attend(i, qkv), w["wo"], c.dim, _lib.EPI_RESIDUAL, True, aux=x, alpha=self.alpha)
            gate = torch.empty((x.shape[0], c.hidden), dtype=torch.bfloat16, device=self.device)
            self._gemm(self._norm(x, w["gamma2"]), w["w13"], c.hidden, _lib.EPI_SWIGLU, True, out2=gate, n_half=c.hidden)
            x = self._gemm(gate, w["w2"], c.dim, _lib.EPI_RESIDUAL, False, aux=x, alpha=self.alpha)
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        logits = self._gemm(self._norm(x, self.gamma_final), self.embed_b, self.cfg.vocab, _lib.EPI_F32, False)
        return logits if self.softcap <= 0 else self.softcap * torch.tanh(logits / self.softcap)

    def check(self) -> None:
        """Wait for the calls so far, of every stream; clear what they reported and raise the first of it."""
        torch.cuda.synchronize(self.device)
        words = [self.err] + [cache.err for cache in self.caches]
        codes = [c for c in torch.cat(words).tolist() if c]
        if codes:
            for w in words:
                w.zero_()
            raise RustaneError(_lib.RT_ERR_TOKEN if codes[0] == 4 else _lib.RT_ERR_DEVICE, f"device error code {codes[0]}")

    # ---------------------------------------------------------------------- serving
    def _page(self) -> int:
        for i, n in enumerate(self.uses):
            if n == 0:
                self.uses[i] = 1
                return i
        raise RustaneError(_lib.RT_ERR_OOM, "no free page in the cache")

    def free(self, seq: Sequence) -> None:
        self._back_to(seq, 0, 0)

    def _back_to(self, seq: Sequence, pages: int, cached: int) -> None:
        """Give back what the sequence took since it had this many pages and cached tokens."""
        for p in seq.pages[pages:]:
            self.uses[p] -= 1
        del seq.pages[pages:]
        seq.cached = cached

    @_on_device
    def forward(self, tokens: torch.Tensor, seqs: list[Sequence], counts: list[int]) -> torch.Tensor:
        """Append counts[s] >= 1 new tokens to each sequence (`tokens` int32, concatenated) and return the
        logits [sequences, vocab] after each one's last token.  If it raises, the sequences are as before."""
        before = [(s, len(s.pages), s.cached) for s in seqs]
        try:
            return self._forward(tokens, seqs, counts)
        except BaseException:
            for s, pages, cached in before:
                self._back_to(s, pages, cached)
            raise

    def _forward(self, tokens: torch.Tensor, seqs: list[Sequence], counts: list[int]) -> torch.Tensor:
        c, ps = self.cfg, self.page_size
        pos, slots, lens = [], [], []
        for s, n in zip(seqs, counts):
            while len(s.pages) * ps < s.cached + n:
                s.pages.append(self._page())
            at = np.arange(s.cached, s.cached + n)
            pos.append(at)
            slots.append(np.asarray(s.pages)[at // ps] * ps + at % ps)
            s.cached += n
            lens.append(s.cached)
        table = np.zeros((len(seqs), max(len(s.pages) for s in seqs)), np.int32)
        for i, s in enumerate(seqs):
            table[i, :len(s.pages)] = s.pages
        ends = np.cumsum(counts)
        # one upload for everything that the step's kernels read
        parts = [np.concatenate(pos), np.concatenate(slots), np.concatenate([[0], ends]), np.asarray(lens), ends - 1, table.ravel()]
        flat = torch.from_numpy(np.concatenate(parts).astype(np.int32)).to(self.device)
        d_pos, d_slots, d_start, d_lens, d_last, d_table = flat.split([p.size for p in parts])
        d_table = d_table.view(table.shape)

        def attend(i: int, qkv: torch.Tensor) -> torch.Tensor:
            q = ops.kv_append(qkv, d_pos, d_slots, self.rope, self.caches[i], c.heads)
            return ops.attention_paged(q, self.caches[i], d_table, d_lens, d_start, c.heads, self.workspace,
                                       max_q=max(counts), max_kv=max(lens))[0]

        return self._logits(self._blocks(tokens, attend)[d_last.long()].contiguous())

    @_on_device
    def prefill(self, prompts: list[list[int]], chunk: int = 512) -> tuple[list[Sequence], torch.Tensor]:
        """Feed prompts, `chunk` tokens of each at a time; (sequences, logits after each prompt)."""
        seqs = [Sequence() for _ in prompts]
        logits = torch.empty((len(prompts), self.cfg.vocab), device=self.device)
        try:
            for at in range(0, max(len(p) for p in prompts), chunk):
                on = [i for i, p in enumerate(prompts) if len(p) > at]
                new = [prompts[i][at:at + chunk] for i in on]
                tok = torch.tensor([t for n in new for t in n], dtype=torch.int32, device=self.device)
                logits[on] = self.forward(tok, [seqs[i] for i in on], [len(n) for n in new])
        except BaseException:
            for s in seqs:
                self.free(s)
            raise
        return seqs, logits

    @_on_device
    def fork(self, seq: Sequence) -> Sequence:
        """A second sequence with the same past: full pages are shared, the last one is copied as it is."""
        full, rest = divmod(seq.cached, self.page_size)
        new = Sequence(seq.pages[:full], seq.cached)
        for p in new.pages:
            self.uses[p] += 1
        if not rest:
            return new
        try:
            new.pages.append(self._page())
            for c in self.caches:
                for t in (c.k, c.v, c.k_scale, c.v_scale):
                    if t is not None:
                        t[new.pages[full]].copy_(t[seq.pages[full]])
        except BaseException:
            self.free(new)
            raise
        return new

    @_on_device
    def generate(self, prompts: list[list[int]], max_new: int, chunk: int = 512, answers: int = 1, repetition: float = 1.0,
                 presence: float = 0.0, frequency: float = 0.0, bias: dict[int, float] | None = None,
                 forbid: list[int] | None = None) -> list[list[list[int]]]:
        """answers greedy answers of max_new tokens to each prompt, as [prompt][answer][token].  ValueError where
        more answers are asked for than there are tokens to start one with."""
        if not prompts or any(not p for p in prompts) or max_new < 1 or not 1 <= answers <= self.cfg.vocab:
            raise ValueError("prompts of one token at least, max_new >= 1, answers from 1 to the vocabulary")
        if any(not 0 <= t < self.cfg.vocab for t in [*(forbid or []), *(bias or {})]):
            raise ValueError(f"bias and forbid take ids from 0 to {self.cfg.vocab - 1}")
        held, logits = self.prefill(prompts, chunk)
        try:
            return self._answer(prompts, held, logits, max_new, answers, repetition, presence, frequency, bias, forbid)
        finally:
            for s in held:
                self.free(s)

    def _answer(self, prompts, held, logits, max_new, answers, repetition, presence, frequency, bias, forbid):
        """generate() after the prompts, whose sequences are `held`; the forked ones join them there."""
        V, dev = self.cfg.vocab, self.device
        n = len(prompts) * answers
        cap = max(len(p) for p in prompts) + max_new
        hist = torch.full((n, cap), -1, dtype=torch.int32, device=dev)  # -1: not yet written
        lens = []
        for i in range(n):
            p = prompts[i // answers]
            hist[i, :len(p)] = torch.tensor(p, dtype=torch.int32, device=dev)
            lens.append(len(p))
        rules = dict(hist=hist.view(-1), hist_start=torch.arange(0, n * cap + 1, cap, dtype=torch.int32, device=dev),
                     n_prompt=torch.tensor(lens, dtype=torch.int32, device=dev),
                     repetition=torch.full((n,), repetition, device=dev), presence=torch.full((n,), presence, device=dev),
                     frequency=torch.full((n,), frequency, device=dev))
        if bias:
            ids, vals = list(bias), list(bias.values())
            rules |= dict(bias_ids=torch.tensor(ids * n, dtype=torch.int32, device=dev),
                          bias_vals=torch.tensor(vals * n, dtype=torch.float32, device=dev),
                          bias_start=torch.arange(0, n * len(ids) + 1, len(ids), dtype=torch.int32, device=dev))
        if forbid:
            bits = np.zeros((1, (V + 31) // 32 * 32), np.uint8)
            bits[0, :V] = 1
            bits[0, forbid] = 0
            words = np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()
            rules["mask"] = torch.from_numpy(words).to(dev).expand(n, -1).contiguous()
        seqs = []
        for s in list(held):
            seqs.append(s)
            for _ in range(1, answers):
                seqs.append(self.fork(s))
                held.append(seqs[-1])
        logits = logits.repeat_interleave(answers, 0)
        rows, at = torch.arange(n, device=dev), torch.tensor(lens, device=dev)
        for step in range(max_new):
            logits, token = ops.logits_adjust(logits, err=self.err, **rules)
            if step == 0 and answers > 1:  # answer k of a prompt starts with the k-th best token
                token = _best(logits[::answers], answers).reshape(-1).to(torch.int32)
            hist[rows, at + step] = token
            if step + 1 < max_new:
                logits = self.forward(token, seqs, [1] * n)
        out = hist.cpu().numpy()
        self.check()
        return [[out[i * answers + k, lens[i * answers]:lens[i * answers] + max_new].tolist() for k in range(answers)]
                for i in range(len(prompts))]

    # ---------------------------------------------------------------- training form
    @_on_device
    def score(self, tokens: list[int]) -> torch.Tensor:
        """Losses [len - 1] of a text's tokens 1.. given those before, without the cache."""
        c, n = self.cfg, len(tokens)
        if n < 2:
            return torch.empty(0, device=self.device)
        S = -(-n // 128) * 128
        tok = torch.tensor(tokens + [0] * (S - n), dtype=torch.int32, device=self.device)
        pos = torch.arange(S, dtype=torch.int32, device=self.device).clamp_(max=n - 1)  # the padding takes none of its own

        def attend(i: int, qkv: torch.Tensor) -> torch.Tensor:
            qkv = ops.qk_norm_rope(qkv, pos, self.rope, c.heads, c.kv_heads, err=self.err)
            out = torch.empty((S, c.q_dim), dtype=torch.bfloat16, device=self.device)
            lse2 = torch.empty((c.heads, S), device=self.device)
            self._call("rt_kernel_attention_fwd", qkv.data_ptr(), out.data_ptr(), lse2.data_ptr(), 1, S, c.heads)
            return out

        logits = self._logits(self._blocks(tok, attend)[:n - 1].contiguous())
        self.check()
        return torch.logsumexp(logits, -1) - logits.gather(1, tok[1:n, None].long())[:, 0]


# ------------------------------------------------------------------------------- CLI
@dataclass
class Args:
    model: str = "gpt_karpathy"
    ckpt: str | None = None
    prompts: list = field(default_factory=list)
    max_new: int = 64
    answers: int = 1
    chunk: int = 512
    cache: str = "bf16"
    page_size: int = 16
    max_pos: int = 4096
    rope_linear: float = 0.0
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    forbid: list = field(default_factory=list)
    bias: dict = field(default_factory=dict)
    softcap: float = 0.0
    device: int = 0


def _ids(text: str) -> list[int]:
    return [int(t) for t in text.split(",") if t.strip()]


def _bias(text: str) -> dict[int, float]:
    return {int(k): float(v) for k, v in (t.split(":") for t in text.split(","))}


_FLAGS = {"--model": ("model", str), "--ckpt": ("ckpt", str), "--max-new": ("max_new", int), "--answers": ("answers", int),
          "--chunk": ("chunk", int), "--cache": ("cache", str), "--page-size": ("page_size", int), "--max-pos": ("max_pos", int),
          "--rope-linear": ("rope_linear", float), "--repetition": ("repetition", float), "--presence": ("presence", float),
          "--frequency": ("frequency", float), "--forbid": ("forbid", _ids), "--bias": ("bias", _bias),
          "--softcap": ("softcap", float), "--device": ("device", int)}


def parse_args(argv: list[str]) -> Args:
    a = Args()
    for i in range(0, len(argv), 2):
        flag = argv[i]
        if flag not in _FLAGS and flag != "--prompt":
            raise UsageError(f"Unknown arg: {flag}")
        if i + 1 >= len(argv):
            raise UsageError(f"{flag} needs a value")
        try:
            if flag == "--prompt":
                a.prompts.append(_ids(argv[i + 1]))
            else:
                setattr(a, _FLAGS[flag][0], _FLAGS[flag][1](argv[i + 1]))
        except ValueError as e:
            raise UsageError(f"{flag}: {e}") from None
    cfg = model_config(a.model)
    if not a.prompts or any(not p for p in a.prompts):
        raise UsageError("--prompt required (token ids, comma separated)")
    if any(not 0 <= t < cfg.vocab for p in a.prompts + [a.forbid, list(a.bias)] for t in p):
        raise UsageError(f"token ids of {a.model} are 0 to {cfg.vocab - 1}")
    if a.cache not in ("bf16", "int8"):
        raise UsageError("--cache: bf16 or int8")
    if a.page_size not in (16, 32, 64, 128):
        raise UsageError("--page-size: 16, 32, 64 or 128")
    if a.max_new < 1 or a.chunk < 1 or not 1 <= a.answers <= cfg.vocab:
        raise UsageError("--max-new, --chunk and --answers are 1 at least")
    if max(len(p) for p in a.prompts) + a.max_new > a.max_pos:
        raise UsageError(f"prompt and answer pass --max-pos {a.max_pos}")
    return a


def run(a: Args, out=print) -> None:
    cfg = model_config(a.model)
    weights = load_checkpoint(a.ckpt, cfg, with_opt=False)[0] if a.ckpt else random_weights(cfg)
    room = -(-(max(len(p) for p in a.prompts) + a.max_new) // a.page_size) * a.page_size
    rope = dict(scaling="linear", factor=a.rope_linear) if a.rope_linear > 0 else {}
    g = Generator(cfg, weights, capacity=room * len(a.prompts) * a.answers, page_size=a.page_size, max_pos=a.max_pos,
                  cache_dtype=torch.int8 if a.cache == "int8" else torch.bfloat16, device=a.device, softcap=a.softcap, **rope)
    for prompt in g.generate(a.prompts, a.max_new, a.chunk, a.answers, a.repetition, a.presence, a.frequency, a.bias, a.forbid):
        for answer in prompt:
            out(",".join(str(t) for t in answer))


def main(argv: list[str] | None = None) -> int:
    argv = sys.argv[1:] if argv is None else argv
    if "--help" in argv or "-h" in argv:
        print(__doc__)
        return 0
    try:
        a = parse_args(argv)
    except UsageError as e:
        print(e, file=sys.stderr)
        return 1
    run(a, out=lambda s: print(s, flush=True))
    return 0


if __name__ == "__main__":
    sys.exit(main())
