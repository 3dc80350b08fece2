"""Measured cases of the serving operators and of the q/k norm + rotation that training shares with them.

Every case names one operator (`op`):

* ``rope``    per-head RMSNorm and rotary position of q and k, forward and backward (a training step's use);
* ``append``  the same pass writing k and v into a paged cache, bf16 or 8-bit, and (8-bit) reading the tokens back;
* ``gather``  reading a long stretch of a cache back;
* ``attn``    attention of each sequence's new tokens over its paged cache;
* ``logits``  repetition / presence / frequency penalties, biases, a grammar mask and the greedy token.

With ``own`` false the operators run in plain torch operations in 32 bits, rounded once at the end; with ``own`` true
they are the framework's (``rustane_b200.ops``).
"""
import math

import torch

own = False

DEV = "cuda"
THETA = 10000.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # 5B configuration's heads, one training batch of 4 x 512: interleaved rotation of the whole head, with norms
        dict(name="rope_5b_batch", op="rope", tokens=2048, heads=20, kv_heads=20, hd=128, rot=128, layout="interleaved",
             norm=True, max_pos=512),
        # a long training batch with shared k heads and half-rotated heads, an odd token count
        dict(name="rope_gqa_long", op="rope", tokens=16389, heads=32, kv_heads=8, hd=128, rot=64, layout="half", norm=True,
             max_pos=8192),
        # one decode step of 48 requests written into an 8-bit cache (7B heads)
        dict(name="append_step_int8", op="append", tokens=48, heads=32, kv_heads=32, hd=128, rot=128, layout="interleaved",
             norm=False, max_pos=4096, pages=1024, int8=True, page=16),
        # a long prompt written into a bf16 cache (7B heads), norms on
        dict(name="append_prompt_bf16", op="append", tokens=8209, heads=32, kv_heads=32, hd=128, rot=128, layout="half",
             norm=True, max_pos=16384, pages=130, int8=False, page=64),
        # one request's 8-bit cache read back whole
        dict(name="gather_int8", op="gather", tokens=30011, kv_heads=32, hd=128, pages=1900, int8=True, page=16),
        # the smallest serving call: one token of one request of the 600M configuration
        dict(name="attn_step_600m", op="attn", seqs=1, q=1, ctx=512, spread=0.0, heads=12, kv_heads=12, hd=128, window=0,
             int8=False, pad=0, page=16),
        # a decode step of 48 requests of ragged length over an 8-bit cache (7B heads), two slots of the batch unused
        dict(name="attn_batch_int8", op="attn", seqs=48, q=1, ctx=6011, spread=0.9, heads=32, kv_heads=32, hd=128, window=0,
             int8=True, pad=2, page=16),
        # a decode step of 8 long requests with shared k heads
        dict(name="attn_long_gqa", op="attn", seqs=8, q=1, ctx=40037, spread=0.3, heads=32, kv_heads=8, hd=128, window=0,
             int8=False, pad=0, page=64),
        # prompts fed in chunks: 4 requests, 509 new tokens each over up to 4091 (5B heads)
        dict(name="attn_chunk_bf16", op="attn", seqs=4, q=509, ctx=4091, spread=0.6, heads=20, kv_heads=20, hd=128, window=0,
             int8=False, pad=0, page=32),
        # one long prompt's chunk over an 8-bit cache with shared k heads
        dict(name="attn_chunk_int8_gqa", op="attn", seqs=1, q=1531, ctx=20011, spread=0.0, heads=32, kv_heads=8, hd=128,
             window=0, int8=True, pad=0, page=16),
        # one request's next token, this repository's vocabulary
        dict(name="logits_one", op="logits", rows=1, vocab=8192, history=700, prompt=500, biases=8, mask=True),
        # a full batch over a large, odd vocabulary
        dict(name="logits_batch", op="logits", rows=192, vocab=128003, history=2000, prompt=1500, biases=40, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "gather", "attn", "attn", "attn", "logits"])
    heads, kv = rng.choice([(6, 6), (12, 12), (16, 16), (20, 20), (32, 32), (32, 8), (16, 2), (8, 1), (14, 14), (12, 4)])
    hd = rng.choice([128, 128, 64])
    layout = rng.choice(["interleaved", "half"])
    page = rng.choice([16, 16, 32, 64, 128])
    rot = rng.choice([hd, hd, hd // 2, hd // 4])
    if op == "rope":
        tokens = min(_log(rng, 1, 20000), 16389 * 48 // (heads + 2 * kv))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, hd=hd, rot=rot, layout=layout,
                    norm=rng.random() < 0.7, max_pos=rng.choice([512, 4096, 131072]))
    if op == "append":
        tokens = min(_log(rng, 1, 8209), 8209 * 96 // (heads + 2 * kv))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, hd=hd, rot=rot, layout=layout, norm=rng.random() < 0.5,
                    max_pos=16384, page=page, pages=-(-tokens // page) + rng.randrange(20),
                    int8=rng.random() < 0.5)
    if op == "gather":
        tokens = _log(rng, 1, 30011)
        return dict(op=op, tokens=tokens, kv_heads=kv, hd=hd, page=page, pages=-(-tokens // page) + rng.randrange(20),
                    int8=rng.random() < 0.5)
    if op == "logits":
        vocab = rng.choice([8192, 8192, _log(rng, 1000, 200000)])
        rows = min(_log(rng, 1, 192), max(1, 192 * 128003 // vocab))
        prompt = _log(rng, 1, 1500)
        return dict(op=op, rows=rows, vocab=vocab, history=prompt + rng.randrange(500), prompt=prompt,
                    biases=rng.choice([0, 1, 40]), mask=rng.random() < 0.5)
    q = rng.choice([1, 1, 1, rng.randrange(2, 17), _log(rng, 17, 1531)])
    seqs = _log(rng, 1, 48) if q < 17 else _log(rng, 1, 6)
    int8 = rng.random() < 0.5
    ctx = _log(rng, max(q, 16), 40037)
    ctx = max(q, min(ctx, (4_500_000 if int8 else 2_250_000) // (kv * seqs)))  # the cache within the listed cases'
    while heads * q * seqs * ctx > 800_000_000 and seqs > 1:
        seqs -= 1
    ctx = max(q, min(ctx, 800_000_000 // (heads * q * seqs)))
    return dict(op=op, seqs=seqs, q=q, ctx=ctx, spread=rng.choice([0.0, 0.5, 0.9]), heads=heads, kv_heads=kv, hd=hd,
                window=rng.choice([0, 0, 0, max(1, ctx // 3)]), int8=int8,
                pad=rng.choice([0, 0, 1]) if seqs > 2 else 0, page=page)


# ------------------------------------------------------------------ inputs
def _lens(c):
    """(new tokens, cached tokens) of every sequence: a ragged batch that depends on the case alone."""
    n = c["seqs"]
    kv = [max(c["q"], int(round(c["ctx"] * (1.0 - c["spread"] * ((i * 37) % n) / n)))) for i in range(n - c["pad"])]
    return [c["q"]] * n, kv + [0] * c["pad"]  # `pad` slots of a fixed batch hold no request


def _tables(c):
    f = THETA ** (-torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64) * 2 / c["rot"])
    a = torch.arange(c["max_pos"], device=DEV, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _quantise(x):
    """8-bit rows with one 32-bit scale each: amax / 127, codes rounded to the nearest."""
    x = x.float()
    s = x.abs().amax(-1) / 127.0
    codes = torch.where(s[..., None] > 0, x / s[..., None], torch.zeros_like(x)).round().clamp_(-127, 127)
    return codes.to(torch.int8), s


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"c": c, "seed": seed}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def perm(n):
        return torch.randperm(n, generator=g, device=DEV).to(torch.int32)

    def gammas():
        s["gq"] = 1 + 0.2 * randn(c["hd"]) if c["norm"] else None
        s["gk"] = 1 + 0.2 * randn(c["hd"]) if c["norm"] else None

    def new_cache(pages, fill):
        shape = (pages, c["kv_heads"], c["page"], c["hd"])
        if not fill:
            s["k"], s["v"] = (torch.zeros(shape, device=DEV, dtype=torch.int8 if c["int8"] else torch.bfloat16) for _ in "kv")
            s["ks"], s["vs"] = (torch.zeros(shape[:3], device=DEV) if c["int8"] else None for _ in "kv")
        else:
            k, v = randn(*shape).bfloat16(), randn(*shape).bfloat16()
            if c["int8"]:
                (s["k"], s["ks"]), (s["v"], s["vs"]) = _quantise(k), _quantise(v)
            else:
                s["k"], s["v"], s["ks"], s["vs"] = k, v, None, None

    if c["op"] in ("rope", "append"):
        cols = (c["heads"] + 2 * c["kv_heads"]) * c["hd"]
        s["qkv"] = (1.5 * randn(c["tokens"], cols)).bfloat16()
        s["pos"] = torch.randint(0, c["max_pos"], (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        s["cos"], s["sin"] = _tables(c)
        gammas()
    if c["op"] == "rope":
        s["dout"] = randn(c["tokens"], cols).bfloat16()
    if c["op"] in ("append", "gather"):
        new_cache(c["pages"], c["op"] == "gather")
        whole = perm(c["pages"])[:, None] * c["page"] + torch.arange(c["page"], device=DEV, dtype=torch.int32)
        # a prompt's tokens fill pages in order; a step's tokens go to a place each
        s["slots"] = (perm(whole.numel()) if c["tokens"] < 64 else whole.reshape(-1))[: c["tokens"]].contiguous()
    if c["op"] == "attn":
        qn, kn = _lens(c)
        per = [-(-k // c["page"]) for k in kn]
        total, width = max(1, sum(per)), max(1, max(per))
        new_cache(total, True)
        order, at = perm(total), 0
        table = torch.zeros(c["seqs"], width, device=DEV, dtype=torch.int32)
        for i, p in enumerate(per):
            table[i, :p] = order[at:at + p]
            at += p
        s["table"], s["kv_lens"] = table, torch.tensor(kn, device=DEV, dtype=torch.int32)
        s["q_start"] = torch.tensor([0] + [sum(qn[: i + 1]) for i in range(len(qn))], device=DEV, dtype=torch.int32)
        s["max_kv"] = max(kn)
        s["q"] = randn(sum(qn), c["heads"] * c["hd"]).bfloat16()
    if c["op"] == "logits":
        b, v = c["rows"], c["vocab"]
        s["logits"] = 3 * randn(b, v)
        u = torch.rand(b, c["history"], generator=g, device=DEV)
        s["hist"] = (u * u * v).to(torch.int32).clamp_(max=v - 1).reshape(-1)  # low ids repeat
        s["hist_start"] = (torch.arange(b + 1, device=DEV) * c["history"]).to(torch.int32)
        s["n_prompt"] = torch.full((b,), c["prompt"], device=DEV, dtype=torch.int32)
        s["rep"] = 1 + 0.5 * torch.rand(b, generator=g, device=DEV)
        s["pres"] = torch.rand(b, generator=g, device=DEV)
        s["freq"] = 0.5 * torch.rand(b, generator=g, device=DEV)
        s["bias_start"] = s["bias_ids"] = s["bias_vals"] = s["bits"] = None
        if c["biases"]:
            s["bias_ids"] = torch.rand(b, v, generator=g, device=DEV).topk(c["biases"]).indices.to(torch.int32).reshape(-1)
            s["bias_vals"] = 5 * randn(b * c["biases"])
            s["bias_start"] = (torch.arange(b + 1, device=DEV) * c["biases"]).to(torch.int32)
        if c["mask"]:
            s["bits"] = torch.randint(-(1 << 31), 1 << 31, (b, -(-v // 32)), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    if own:
        from rustane_b200 import ops
        if "cos" in s:
            s["rope"] = ops.Rope(s["cos"], s["sin"], layout=c["layout"])
        if "k" in s:
            s["cache"] = ops.KvCache(s["k"], s["v"], s["ks"], s["vs"])
        if c["op"] == "attn":
            s["ws"] = ops.AttentionWorkspace(DEV)
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, c, back=False):
    """Rotates the first `rot` columns of x [T, H, hd] by the tables' angles (`back`: by their opposite)."""
    r = c["rot"]
    cos, sin = cos[:, None, :], -sin[:, None, :] if back else sin[:, None, :]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["layout"] == "interleaved" else (x[..., : r // 2], x[..., r // 2: r])
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((u, w), -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat((u, w), -1)
    return torch.cat((y, x[..., r:]), -1)


def _norm(x, gamma):
    return x if gamma is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * gamma


def _split(x, c):
    x = x.view(x.shape[0], -1, c["hd"]).float()
    h, k = c["heads"], c["kv_heads"]
    return x[:, :h], x[:, h:h + k], x[:, h + k:]


def _norm_back(dn, x, gamma):
    if gamma is None:
        return dn, None
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    xh = x * r
    dg = dn * gamma
    return r * (dg - xh * (dg * xh).mean(-1, keepdim=True)), (dn * xh).sum((0, 1))


def _plain_rope(s):
    c = s["c"]
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    q, k, v = _split(s["qkv"], c)
    out = torch.cat((_rotate(_norm(q, s["gq"]), cos, sin, c), _rotate(_norm(k, s["gk"]), cos, sin, c), v), 1)
    dq, dk, dv = _split(s["dout"], c)
    dq, dgq = _norm_back(_rotate(dq, cos, sin, c, True), q, s["gq"])
    dk, dgk = _norm_back(_rotate(dk, cos, sin, c, True), k, s["gk"])
    return {"out": out.flatten(1).bfloat16(), "dqkv": torch.cat((dq, dk, dv), 1).flatten(1).bfloat16(), "dgq": dgq, "dgk": dgk}


def _plain_gather(s):
    at = s["slots"].long()
    page, off = at // s["c"]["page"], at % s["c"]["page"]
    k, v = s["k"][page, :, off].float(), s["v"][page, :, off].float()
    if s["ks"] is not None:
        k, v = k * s["ks"][page, :, off][..., None], v * s["vs"][page, :, off][..., None]
    return {"k": k.bfloat16(), "v": v.bfloat16()}


def _plain_append(s):
    c = s["c"]
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    q, k, v = _split(s["qkv"], c)
    q, k = _rotate(_norm(q, s["gq"]), cos, sin, c), _rotate(_norm(k, s["gk"]), cos, sin, c)
    at = s["slots"].long()
    page, off = at // s["c"]["page"], at % s["c"]["page"]
    q = q.flatten(1).bfloat16()
    if not c["int8"]:
        s["k"][page, :, off], s["v"][page, :, off] = k.bfloat16(), v.bfloat16()
        return {"q": q, "k": s["k"], "v": s["v"]}
    (s["k"][page, :, off], s["ks"][page, :, off]), (s["v"][page, :, off], s["vs"][page, :, off]) = _quantise(k), _quantise(v)
    return {"q": q, **_plain_gather(s)}


def _plain_attn(s):
    c = s["c"]
    n, h, hk, hd, dev = c["seqs"], c["heads"], c["kv_heads"], c["hd"], s["q"].device
    lens, width = s["kv_lens"].long(), s["table"].shape[1] * c["page"]
    table = s["table"].long()

    def dense(x, scale):  # [n, kv_heads, keys, hd]
        y = x[table].float()
        if scale is not None:
            y = y * scale[table][..., None]
        return y.permute(0, 2, 1, 3, 4).reshape(n, hk, width, hd)

    q = s["q"].float().view(n, c["q"], hk, h // hk, hd).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, hd)
    sc = torch.matmul(q, dense(s["k"], s["ks"]).transpose(-1, -2)).mul_(1.0 / math.sqrt(hd))
    sc = sc.view(n, hk, h // hk, c["q"], width)
    key = torch.arange(width, device=dev)
    pos = lens[:, None] - c["q"] + torch.arange(c["q"], device=dev)  # [n, q]
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hk, -1, width), dense(s["v"], s["vs"])).view(n, hk, h // hk, c["q"], hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse2 = (top + total.log())[..., 0] * (1 / math.log(2.0))
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(n * c["q"], h * hd).bfloat16(),
            "lse2": lse2.permute(0, 3, 1, 2).reshape(n * c["q"], h)}


def _plain_logits(s):
    b, v = s["logits"].shape
    row = torch.arange(b, device=DEV).repeat_interleave(s["hist_start"].diff().long(), output_size=s["hist"].numel())
    nth = torch.arange(s["hist"].numel(), device=DEV) - s["hist_start"].long()[row]
    made = nth >= s["n_prompt"].long()[row]
    at = row * v + s["hist"].long()
    seen = torch.zeros(b * v, device=DEV).index_fill_(0, at, 1.0).view(b, v) > 0
    count = torch.zeros(b * v, device=DEV).index_add_(0, at, made.float()).view(b, v)
    x = s["logits"]
    rep = s["rep"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["freq"][:, None] * count - s["pres"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        brow = torch.arange(b, device=DEV).repeat_interleave(s["bias_start"].diff().long(), output_size=s["bias_ids"].numel())
        x = x.reshape(-1).index_add(0, brow * v + s["bias_ids"].long(), s["bias_vals"]).view(b, v)
    if s["bits"] is not None:
        word = s["bits"][:, torch.arange(v, device=DEV) // 32]
        x = torch.where((word >> (torch.arange(v, device=DEV, dtype=torch.int32) % 32)) & 1 == 1, x, torch.full_like(x, float("-inf")))
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(v, device=DEV), v).amin(-1)
    return {"logits": x, "token": torch.where(top[:, 0] > float("-inf"), first, -1).to(torch.int32)}


# ------------------------------------------------------------------ the framework's
def _own(s):
    from rustane_b200 import ops
    c = s["c"]
    if c["op"] == "rope":
        out = ops.qk_norm_rope(s["qkv"], s["pos"], s["rope"], c["heads"], c["kv_heads"], gamma_q=s["gq"], gamma_k=s["gk"])
        dqkv, dgq, dgk = ops.qk_norm_rope_backward(s["dout"], s["qkv"], s["pos"], s["rope"], c["heads"], c["kv_heads"],
                                                   gamma_q=s["gq"], gamma_k=s["gk"])
        return {"out": out, "dqkv": dqkv, "dgq": dgq, "dgk": dgk}
    if c["op"] == "append":
        q = ops.kv_append(s["qkv"], s["pos"], s["slots"], s["rope"], s["cache"], c["heads"], gamma_q=s["gq"], gamma_k=s["gk"])
        if not c["int8"]:
            return {"q": q, "k": s["k"], "v": s["v"]}
        k, v = ops.kv_gather(s["cache"], s["slots"])
        return {"q": q, "k": k, "v": v}
    if c["op"] == "gather":
        k, v = ops.kv_gather(s["cache"], s["slots"])
        return {"k": k, "v": v}
    if c["op"] == "attn":
        out, lse2 = ops.attention_paged(s["q"], s["cache"], s["table"], s["kv_lens"], s["q_start"], c["heads"], s["ws"],
                                        max_q=c["q"], max_kv=s["max_kv"], window=c["window"], want_lse=True)
        return {"out": out, "lse2": lse2}
    out, token = ops.logits_adjust(s["logits"], hist=s["hist"], hist_start=s["hist_start"], n_prompt=s["n_prompt"],
                                   repetition=s["rep"], presence=s["pres"], frequency=s["freq"], bias_ids=s["bias_ids"],
                                   bias_vals=s["bias_vals"], bias_start=s["bias_start"], mask=s["bits"])
    return {"logits": out, "token": token}


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "append": _plain_append, "gather": _plain_gather, "attn": _plain_attn,
            "logits": _plain_logits}[state["c"]["op"]](state)


# ------------------------------------------------------------------ least work
def work(case):
    c = dict(case)
    op = c["op"]
    if op == "rope":
        t, hd = c["tokens"], c["hd"]
        qk, v = t * (c["heads"] + c["kv_heads"]) * hd, t * c["kv_heads"] * hd
        tables = 2 * min(t, c["max_pos"]) * c["rot"] // 2 * 4
        # forward: qkv in, out; backward: dout and the q, k inputs in, dqkv out
        return {"bytes": 4 * (qk + v) + 6 * qk + 4 * v + 2 * tables + 8 * t, "flops": 25 * qk}
    if op in ("append", "gather"):
        t, hd = c["tokens"], c["hd"]
        kv = 2 * t * c["kv_heads"]
        held = kv * (hd + 4 if c["int8"] else 2 * hd)
        if op == "gather":
            return {"bytes": held + 2 * kv * hd + 4 * t, "flops": kv * hd}
        q = t * c["heads"] * hd
        tables = 2 * min(t, c["max_pos"]) * c["rot"] // 2 * 4
        back = held + 2 * kv * hd + 4 * t if c["int8"] else 0
        return {"bytes": 4 * q + 2 * kv * hd + held + back + tables + 8 * t, "flops": 12 * (q + kv * hd)}
    if op == "attn":
        qn, kn = _lens(c)
        pairs = keys = 0
        for n, k in zip(qn, kn):
            seen = [min(max(k - n + i + 1, 0), c["window"] or k) for i in range(n)]
            pairs += sum(seen)
            keys += min(k, (c["window"] or k) + n - 1)
        row = c["hd"] + 4 if c["int8"] else 2 * c["hd"]
        io = sum(qn) * c["heads"] * (4 * c["hd"] + 4)
        return {"bytes": 2 * keys * c["kv_heads"] * row + io, "flops": 4 * c["hd"] * c["heads"] * pairs}
    b, v = c["rows"], c["vocab"]
    return {"bytes": b * (8 * v + 4 * c["history"] + 8 * c["biases"] + (v // 8 if c["mask"] else 0)), "flops": 6 * b * v}


# ------------------------------------------------------------------ 64 bits
def _exact_rot(x, ang_cos, ang_sin, c, sign):
    y = x.clone()
    half, r = c["rot"] // 2, c["rot"]
    i = torch.arange(half, device=DEV)
    a, b = (2 * i, 2 * i + 1) if c["layout"] == "interleaved" else (i, i + half)
    cs, sn = ang_cos[:, None, :], sign * ang_sin[:, None, :]
    y[..., a] = x[..., a] * cs - x[..., b] * sn
    y[..., b] = x[..., a] * sn + x[..., b] * cs
    return y


def exact(case, seed):
    s = prepare(case, seed)
    c, f8 = s["c"], torch.float64
    if c["op"] in ("rope", "append"):
        t = c["tokens"]
        x = s["qkv"].to(f8).view(t, -1, c["hd"])
        cs, sn = s["cos"].to(f8)[s["pos"].long()], s["sin"].to(f8)[s["pos"].long()]
        h, hk = c["heads"], c["kv_heads"]
        parts, gs = [x[:, :h], x[:, h:h + hk], x[:, h + hk:]], [s["gq"], s["gk"]]
        rs = [1 / (p.pow(2).sum(-1, keepdim=True) / c["hd"] + 1e-5).sqrt() for p in parts[:2]]
        ys = [_exact_rot(p if g is None else p * r * g.to(f8), cs, sn, c, 1.0) for p, g, r in zip(parts, gs, rs)]
    if c["op"] == "rope":
        d = s["dout"].to(f8).view(t, -1, c["hd"])
        ds, dgs = [], []
        for p, g, r, dy in zip(parts, gs, rs, (d[:, :h], d[:, h:h + hk])):
            dn = _exact_rot(dy, cs, sn, c, -1.0)
            if g is None:
                ds.append(dn)
                dgs.append(None)
                continue
            dgs.append(torch.einsum("thd,thd->d", dn, p * r))
            w = dn * g.to(f8)
            ds.append(w * r - p * r.pow(3) * (w * p).sum(-1, keepdim=True) / c["hd"])
        return {"out": torch.cat(ys + [parts[2]], 1).reshape(t, -1), "dqkv": torch.cat(ds + [d[:, h + hk:]], 1).reshape(t, -1),
                "dgq": dgs[0], "dgk": dgs[1]}
    if c["op"] in ("append", "gather"):
        at = s["slots"].long()
        if c["op"] == "append" and not c["int8"]:
            k, v = s["k"].to(f8), s["v"].to(f8)
            k[at // c["page"], :, at % c["page"]], v[at // c["page"], :, at % c["page"]] = ys[1], parts[2]
            return {"q": ys[0].reshape(t, -1), "k": k, "v": v}
        if c["op"] == "append":
            back = []
            for y in (ys[1], parts[2]):
                step = (y.abs().max(-1, keepdim=True).values / 127).clamp_min(1e-300)
                back.append((y / step).round() * step)
            return {"q": ys[0].reshape(t, -1), "k": back[0], "v": back[1]}
        both = []
        for x, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            y = x.to(f8) if sc is None else x.to(f8) * sc.to(f8)[..., None]
            both.append(y[at // c["page"], :, at % c["page"]])
        return {"k": both[0], "v": both[1]}
    if c["op"] == "attn":
        qn, kn = _lens(c)
        h, hk, hd = c["heads"], c["kv_heads"], c["hd"]
        outs, lses, at = [], [], 0
        for i, (n, k) in enumerate(zip(qn, kn)):
            pages = s["table"][i, : -(-k // c["page"])].long()
            kk, vv = s["k"][pages].to(f8), s["v"][pages].to(f8)
            if s["ks"] is not None:
                kk, vv = kk * s["ks"][pages].to(f8)[..., None], vv * s["vs"][pages].to(f8)[..., None]
            kk, vv = (z.transpose(0, 1).reshape(hk, -1, hd)[:, :k] for z in (kk, vv))
            q = s["q"][at:at + n].to(f8).view(n, h, hd)
            at += n
            o, l = torch.zeros(n, h, hd, device=DEV, dtype=f8), torch.full((n, h), -math.inf, device=DEV, dtype=f8)
            place = torch.arange(k - n, k, device=DEV)[:, None] - torch.arange(k, device=DEV)
            off = (place < 0) | (place >= c["window"]) if c["window"] else place < 0
            for j in range(h if k else 0):
                z = (q[:, j] @ kk[j // (h // hk)].T / math.sqrt(hd)).masked_fill(off, -math.inf)
                l[:, j] = torch.logsumexp(z, -1)
                o[:, j] = (z - l[:, j:j + 1]).exp().nan_to_num(0.0) @ vv[j // (h // hk)]
            outs.append(o.reshape(n, -1))
            lses.append(l / math.log(2.0))
        return {"out": torch.cat(outs), "lse2": torch.cat(lses)}
    b, v = s["logits"].shape
    x = s["logits"].to(f8)
    for i in range(b):
        ids = s["hist"][s["hist_start"][i]:s["hist_start"][i + 1]].long()
        made = torch.bincount(ids[int(s["n_prompt"][i]):], minlength=v).to(f8)
        seen = torch.unique(ids)
        old, rep = x[i, seen], s["rep"][i].to(f8)
        x[i, seen] = torch.where(old > 0, old / rep, old * rep)
        x[i] -= s["freq"][i].to(f8) * made + s["pres"][i].to(f8) * (made > 0)
        if s["bias_ids"] is not None:
            lo, hi = int(s["bias_start"][i]), int(s["bias_start"][i + 1])
            x[i].index_add_(0, s["bias_ids"][lo:hi].long(), s["bias_vals"][lo:hi].to(f8))
    if s["bits"] is not None:
        allowed = ((s["bits"].long()[:, :, None] >> torch.arange(32, device=DEV)) & 1).reshape(b, -1)[:, :v]
        x = x.masked_fill(allowed == 0, -math.inf)
    return {"logits": x, "token": None}
