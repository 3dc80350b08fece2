"""Serving operators on torch tensors: rotary positions with per-head norms (and their
backward, for training), a paged key/value cache, attention over it, and the step from
logits to a token.

    rope = Rope.tables(n_pos=4096, rot=128, device="cuda")
    cache = KvCache.empty(num_pages=512, page_size=16, kv_heads=12, hd=128, dtype=torch.int8, device="cuda")
    ws = AttentionWorkspace("cuda")
    q = kv_append(qkv, positions, slots, rope, cache, heads=12)
    o, _ = attention_paged(q, cache, page_table, kv_lens, q_start, heads=12, workspace=ws, max_q=1, max_kv=4096)
    logits, token = logits_adjust(logits, hist=..., hist_start=..., repetition=..., mask=...)

Each function checks its tensors' types, shapes and strides on the host (ValueError), launches
on the tensors' device and torch's current stream there, and returns without waiting.  What
only the device sees (a position, slot, page, length or token id out of range) lands in an error
word: the cache's own, or the `err` argument; ``KvCache.check()`` waits for it and raises.
The kernels are librustane_cuda.so's rt_kernel_* entry points (include/rustane_cuda.h says
what each computes); there is no fallback.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib
from ._lib import RtKvPages, RtLogitRules, RtRope, RustaneError, lib


_DENSE = torch.contiguous_format
_raw_stream = torch._C._cuda_getCurrentRawStream
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _fail(msg: str):
    raise ValueError(msg)


def _rows(name: str, t: torch.Tensor, cols: int, dtype: torch.dtype, device: torch.device, rows: int | None = None) -> int:
    """Checks a row matrix; its row stride, which torch leaves arbitrary where there are fewer than two rows."""
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 2 or shape[1] != cols or (rows is not None and shape[0] != rows):
        _fail(f"{name}: expected a [{'T' if rows is None else rows}, {cols}] {dtype} tensor, got {tuple(shape)} {t.dtype}")
    ld, step = t.stride()
    if (step != 1 and shape[0]) or t.device != device:
        _fail(f"{name}: its rows have to be contiguous and on {device}")
    return ld if shape[0] > 1 else max(ld, cols)


def _vec(name: str, t: torch.Tensor, n: int | None, dtype: torch.dtype, device: torch.device) -> None:
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 1 or (n is not None and shape[0] != n):
        _fail(f"{name}: expected {'a vector' if n is None else n} of {dtype}, got {tuple(shape)} {t.dtype}")
    if t.device != device or not t.is_contiguous():
        _fail(f"{name}: has to be contiguous and on {device}")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _cuda(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        _fail("a CUDA tensor is needed")
    return t.device


def _call(name: str, device: torch.device, *args) -> None:
    # torch's raw handle of the current stream: the public Stream object costs 2 us to build, a
    # fifth of a small call
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = getattr(lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = getattr(lib(), name)(*args, _raw_stream(index))
    if rc:
        raise RustaneError(rc, name)


class Rope:
    """Rotary tables [n_pos, rot / 2] fp32; layout "interleaved" rotates (2i, 2i + 1), as the
    model's own forward does, "half" (i, i + rot / 2)."""

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, layout: str = "interleaved"):
        if layout not in ("interleaved", "half"):
            _fail(f"layout {layout!r}: interleaved or half")
        device = _cuda(cos)
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or \
                sin.device != device or not cos.is_contiguous() or not sin.is_contiguous():
            _fail("cos, sin: contiguous fp32 [n_pos, rot / 2] tensors of one device")
        self.cos, self.sin, self.layout, self.device = cos, sin, layout, device
        self.n_pos, self.rot = cos.shape[0], 2 * cos.shape[1]
        self.c = RtRope(cos.data_ptr(), sin.data_ptr(), self.n_pos, self.rot, int(layout == "half"))
        self.ref = ctypes.byref(self.c)

    @classmethod
    def tables(cls, n_pos: int, rot: int, device, theta: float = 10000.0, layout: str = "interleaved",
               scaling: str | None = None, factor: float = 1.0, low: float = 1.0, high: float = 32.0,
               trained_pos: int = 0) -> "Rope":
        """Tables for positions 0 .. n_pos - 1.  scaling None; "linear": every frequency / factor; "bands":
        frequencies with fewer than `low` turns over trained_pos positions / factor, those with more than
        `high` kept, blended between."""
        kinds = {None: _lib.RT_ROPE_PLAIN, "linear": _lib.RT_ROPE_LINEAR, "bands": _lib.RT_ROPE_BANDS}
        if scaling not in kinds:
            _fail(f"scaling {scaling!r}: None, linear or bands")
        cos, sin = (np.empty((max(n_pos, 0), max(rot, 0) // 2), np.float32) for _ in "cs")
        p = ctypes.POINTER(ctypes.c_float)
        rc = lib().rt_rope_tables(cos.ctypes.data_as(p), sin.ctypes.data_as(p), n_pos, rot, theta, kinds[scaling], factor,
                                  low, high, trained_pos)
        if rc != _lib.RT_OK:
            raise RustaneError(rc, "rt_rope_tables")
        return cls(torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device), layout)


class KvCache:
    """Paged cache over caller-owned tensors: k, v [num_pages, kv_heads, page_size, hd], bf16, or int8 with
    fp32 k_scale, v_scale [num_pages, kv_heads, page_size]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        device = _cuda(k)
        int8 = k.dtype == torch.int8
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.int8) or \
                v.device != device or not k.is_contiguous() or not v.is_contiguous():
            _fail("k, v: contiguous bf16 or int8 [num_pages, kv_heads, page_size, hd] tensors of one device")
        if int8 != (k_scale is not None) or int8 != (v_scale is not None):
            _fail("an int8 cache has scales, a bf16 cache none")
        for s in (k_scale, v_scale):
            if s is not None and (s.shape != k.shape[:3] or s.dtype != torch.float32 or s.device != device or
                                  not s.is_contiguous()):
                _fail("k_scale, v_scale: contiguous fp32 [num_pages, kv_heads, page_size]")
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, device
        self.num_pages, self.kv_heads, self.page_size, self.hd = k.shape
        self.scale = 1.0 / math.sqrt(self.hd)  # of attention scores, by default
        self.err = torch.zeros(1, dtype=_I32, device=device)
        self.err_ptr = self.err.data_ptr()
        self.c = RtKvPages(k.data_ptr(), v.data_ptr(), _ptr(k_scale), _ptr(v_scale), self.num_pages, self.page_size,
                           self.kv_heads, self.hd, int(int8))
        self.ref = ctypes.byref(self.c)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, hd: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "KvCache":
        shape = (num_pages, kv_heads, page_size, hd)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in "kv")
        scales = [torch.zeros(shape[:3], device=device) for _ in "kv"] if dtype == torch.int8 else [None, None]
        return cls(k, v, *scales)

    def check(self) -> None:
        """Wait for the error word of the calls so far; raise and clear it if one is set."""
        code = int(self.err.item())
        if code:
            self.err.zero_()
            raise RustaneError(_lib.RT_ERR_TOKEN if code == 4 else _lib.RT_ERR_DEVICE, f"device error code {code}")


class AttentionWorkspace:
    """Scratch of attention_paged; calls that share one run on one stream."""

    def __init__(self, device="cuda"):
        n = max(lib().rt_kernel_attention_paged_workspace_bytes(hd) for hd in (64, 128))
        self.buf = torch.zeros(n, dtype=torch.uint8, device=device)
        self.ptr, self.size, self.device = self.buf.data_ptr(), n, self.buf.device


def _gammas(gamma_q, gamma_k, hd, device):
    if (gamma_q is None) != (gamma_k is None):
        _fail("gamma_q and gamma_k: both or neither")
    if gamma_q is not None:
        _vec("gamma_q", gamma_q, hd, _F32, device)
        _vec("gamma_k", gamma_k, hd, _F32, device)


def _vectors(t: torch.Tensor, heads: int, kv_heads: int) -> tuple[int, int]:
    """(hd, v heads) of q | k | v rows: hd from the column count, with or without the v part (the count
    fits one of the four: 128 without v would be 64 with v only for heads == 0)."""
    cols = t.shape[-1] if t.dim() == 2 else 0
    for v in (kv_heads, 0):
        hd, rest = divmod(cols, max(1, heads + kv_heads + v))
        if not rest and (hd == 128 or hd == 64):
            return hd, v
    _fail(f"rows of {tuple(t.shape)} do not hold {heads} q and {kv_heads} k (and v) heads of 64 or 128")


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, rope: Rope, heads: int, kv_heads: int,
                 gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None, eps: float = 1e-5,
                 out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """q and k heads of qkv [T, (heads + kv_heads (+ kv_heads)) * hd] bf16 normed (with gammas) and rotated, v copied;
    out=qkv works in place."""
    device = _cuda(qkv)
    hd, nv = _vectors(qkv, heads, kv_heads)
    T, cols = qkv.shape
    ld = _rows("qkv", qkv, cols, _BF16, device)
    _vec("positions", positions, T, _I32, device)
    _gammas(gamma_q, gamma_k, hd, device)
    if rope.device != device:
        _fail(f"rope: its tables have to be on {device}")
    if out is None:
        out, ldo = torch.empty_like(qkv, memory_format=_DENSE), cols
    else:
        ldo = _rows("out", out, cols, _BF16, device, T)
    _call("rt_kernel_qk_norm_rope_fwd", device, qkv.data_ptr(), ld, out.data_ptr(), ldo, positions.data_ptr(),
          rope.ref, _ptr(gamma_q), _ptr(gamma_k), eps, T, heads, kv_heads, nv, hd, _ptr(err))
    return out


def qk_norm_rope_backward(dout: torch.Tensor, qkv: torch.Tensor | None, positions: torch.Tensor, rope: Rope, heads: int,
                          kv_heads: int, gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None,
                          eps: float = 1e-5, dqkv: torch.Tensor | None = None, dgamma_q: torch.Tensor | None = None,
                          dgamma_k: torch.Tensor | None = None, err: torch.Tensor | None = None):
    """(dqkv, dgamma_q, dgamma_k) of qk_norm_rope, from the gradient of its output and its input qkv (not read
    without gammas).  dqkv=dout works in place; dgammas given are added to, otherwise new (None without gammas)."""
    device = _cuda(dout)
    hd, nv = _vectors(dout, heads, kv_heads)
    T, cols = dout.shape
    ld = _rows("dout", dout, cols, _BF16, device)
    _vec("positions", positions, T, _I32, device)
    _gammas(gamma_q, gamma_k, hd, device)
    if rope.device != device:
        _fail(f"rope: its tables have to be on {device}")
    if dqkv is None:
        dqkv, lddx = torch.empty_like(dout, memory_format=_DENSE), cols
    else:
        lddx = _rows("dqkv", dqkv, cols, _BF16, device, T)
    accumulate, partials, ldx = 0, None, 0
    if gamma_q is not None:
        if qkv is None:
            _fail("the gammas' backward reads qkv")
        ldx = _rows("qkv", qkv, cols, _BF16, device, T)
        if (dgamma_q is None) != (dgamma_k is None):
            _fail("dgamma_q and dgamma_k: both or neither")
        accumulate = int(dgamma_q is not None)
        if accumulate:
            _vec("dgamma_q", dgamma_q, hd, _F32, device)
            _vec("dgamma_k", dgamma_k, hd, _F32, device)
        else:
            dgamma_q, dgamma_k = torch.empty_like(gamma_q), torch.empty_like(gamma_k)
        partials = gamma_q.new_empty(lib().rt_kernel_qk_norm_rope_bwd_partials(T, heads, kv_heads) * hd)
    _call("rt_kernel_qk_norm_rope_bwd", device, dout.data_ptr(), ld, _ptr(qkv), ldx, dqkv.data_ptr(), lddx, positions.data_ptr(), rope.ref, _ptr(gamma_q), _ptr(gamma_k), eps, _ptr(dgamma_q),
          _ptr(dgamma_k), accumulate, _ptr(partials), T, heads, kv_heads, nv, hd, _ptr(err))
    return dqkv, dgamma_q, dgamma_k


def kv_append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, rope: Rope, cache: KvCache, heads: int,
              gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None, eps: float = 1e-5,
              q_out: torch.Tensor | None = None) -> torch.Tensor:
    """qk_norm_rope that writes k and v of token t into cache slot slots[t] (-1: nowhere) and returns q."""
    device = cache.device
    T, hd = qkv.shape[0], cache.hd
    ld = _rows("qkv", qkv, (heads + 2 * cache.kv_heads) * hd, _BF16, device)
    _vec("positions", positions, T, _I32, device)
    _vec("slots", slots, T, _I32, device)
    _gammas(gamma_q, gamma_k, hd, device)
    if rope.device != device:
        _fail(f"rope: its tables have to be on {device}")
    if q_out is None:
        q_out, ldq = qkv.new_empty((T, heads * hd)), heads * hd
    else:
        ldq = _rows("q_out", q_out, heads * hd, _BF16, device, T)
    _call("rt_kernel_kv_append", device, qkv.data_ptr(), ld, q_out.data_ptr(), ldq, positions.data_ptr(),
          slots.data_ptr(), rope.ref, _ptr(gamma_q), _ptr(gamma_k), eps, cache.ref, T, heads, cache.err_ptr)
    return q_out


def kv_gather(cache: KvCache, slots: torch.Tensor, k_out: torch.Tensor | None = None,
              v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached tokens back as bf16: (k, v) [T, kv_heads, hd]; slot -1 gives zeros."""
    device, T = cache.device, slots.shape[0]
    _vec("slots", slots, T, _I32, device)
    shape = (T, cache.kv_heads, cache.hd)
    given = [x for x in (("k_out", k_out), ("v_out", v_out)) if x[1] is not None]
    k_out = torch.empty(shape, dtype=_BF16, device=device) if k_out is None else k_out
    v_out = torch.empty_like(k_out) if v_out is None else v_out
    for name, t in given:
        if t.shape != shape or t.dtype != torch.bfloat16 or t.device != device or not t.is_contiguous():
            _fail(f"{name}: a contiguous bf16 {shape} tensor on {device}")
    _call("rt_kernel_kv_gather", device, cache.ref, slots.data_ptr(), k_out.data_ptr(), v_out.data_ptr(),
          cache.kv_heads * cache.hd, T, cache.err_ptr)
    return k_out, v_out


def attention_paged(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    q_start: torch.Tensor, heads: int, workspace: AttentionWorkspace, max_q: int, max_kv: int,
                    window: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                    want_lse: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Causal attention of the new tokens q [T, heads * hd] over the cache: sequence s owns rows
    q_start[s] .. q_start[s + 1] and the first kv_lens[s] tokens of pages page_table[s], its new tokens last.
    Returns (out [T, heads * hd] bf16, lse2 [T, heads] fp32 or None)."""
    device, T, n = cache.device, q.shape[0], kv_lens.shape[0]
    cols = heads * cache.hd
    ldq = _rows("q", q, cols, _BF16, device)
    _vec("kv_lens", kv_lens, n, _I32, device)
    _vec("q_start", q_start, n + 1, _I32, device)
    ldt = _rows("page_table", page_table, page_table.shape[-1], _I32, device, n)
    if out is None:
        out, ldo = torch.empty_like(q, memory_format=_DENSE), cols
    else:
        ldo = _rows("out", out, cols, _BF16, device, T)
    if workspace.device != device:
        _fail(f"workspace: has to be on {device}")
    lse2 = q.new_empty((T, heads), dtype=_F32) if want_lse else None
    _call("rt_kernel_attention_paged", device, q.data_ptr(), ldq, out.data_ptr(), ldo, _ptr(lse2), cache.ref,
          page_table.data_ptr(), ldt, kv_lens.data_ptr(), q_start.data_ptr(), n, T, max_q, max_kv, heads, window,
          cache.scale if scale is None else scale, workspace.ptr, workspace.size,
          cache.err_ptr)
    return out, lse2


def logits_adjust(logits: torch.Tensor, hist: torch.Tensor | None = None, hist_start: torch.Tensor | None = None,
                  n_prompt: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_vals: torch.Tensor | None = None,
                  bias_start: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(logits after penalties, biases and the grammar mask, the greedy token) per row; out=logits works in place.
    hist (int32, rows by hist_start [B + 1], the first n_prompt[b] the prompt's), biases likewise, mask [B, ceil(V / 32)]
    int32 words.  token: int32 [B], -1 where every token is forbidden."""
    device = _cuda(logits)
    if logits.dim() != 2:
        _fail("logits: [B, V]")
    B, V = logits.shape
    ldl = _rows("logits", logits, V, _F32, device)
    r = RtLogitRules()
    if hist is not None:
        if hist_start is None:
            _fail("hist needs hist_start")
        _vec("hist", hist, None, _I32, device)
        _vec("hist_start", hist_start, B + 1, _I32, device)
        r.hist, r.hist_start, r.n_hist = hist.data_ptr(), hist_start.data_ptr(), hist.shape[0]
        if n_prompt is not None:
            _vec("n_prompt", n_prompt, B, _I32, device)
            r.n_prompt = n_prompt.data_ptr()
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            _vec(name, t, B, _F32, device)
            setattr(r, name, t.data_ptr())
    if bias_ids is not None:
        if bias_vals is None or bias_start is None:
            _fail("bias_ids needs bias_vals and bias_start")
        _vec("bias_ids", bias_ids, None, _I32, device)
        _vec("bias_vals", bias_vals, bias_ids.shape[0], _F32, device)
        _vec("bias_start", bias_start, B + 1, _I32, device)
        r.bias_ids, r.bias_vals, r.bias_start, r.n_bias = (bias_ids.data_ptr(), bias_vals.data_ptr(), bias_start.data_ptr(),
                                                           bias_ids.shape[0])
    if mask is not None:
        r.mask_ld = _rows("mask", mask, (V + 31) // 32, _I32, device, B)
        r.mask = mask.data_ptr()
    if out is None:
        out, ldo = torch.empty_like(logits, memory_format=_DENSE), V
    else:
        ldo = _rows("out", out, V, _F32, device, B)
    token = torch.empty(B, dtype=_I32, device=device)
    _call("rt_kernel_logits_adjust", device, logits.data_ptr(), ldl, out.data_ptr(), ldo, token.data_ptr(), B, V,
          ctypes.byref(r), _ptr(err))
    return out, token
