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
on the tensors' device and torch's current stream there, and returns without waiting (csrc_torch/ops.cpp).  What
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
from ._lib import RtKvPages, RtRope, RustaneError, lib

try:
    from . import _torch_ops as _ext
except ImportError as e:  # no fallback
    raise RuntimeError(f"rustane_b200/_torch_ops is missing or does not load ({e}): build it with "
                       "`python -m rustane_b200.build`") from None


def _fail(msg: str):
    raise ValueError(msg)


def _cuda(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        _fail("a CUDA tensor is needed")
    return t.device


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


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
        self.ref, self.addr, self.index = ctypes.byref(self.c), ctypes.addressof(self.c), device.index

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
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        self.err_ptr = self.err.data_ptr()
        self.c = RtKvPages(k.data_ptr(), v.data_ptr(), _ptr(k_scale), _ptr(v_scale), self.num_pages, self.page_size,
                           self.kv_heads, self.hd, int(int8))
        self.ref, self.addr, self.index = ctypes.byref(self.c), ctypes.addressof(self.c), device.index

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, hd: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "KvCache":
        shape = (num_pages, kv_heads, page_size, hd)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in "kv")
        scales = [torch.zeros(shape[:3], device=device) for _ in "kv"] if dtype == torch.int8 else [None, None]
        return cls(k, v, *scales)

    def check(self) -> None:
        """Wait for the calls so far, of every stream; clear the error word and raise if it is set."""
        torch.cuda.synchronize(self.device)
        code = int(self.err.item())
        if code:
            self.err.zero_()
            raise RustaneError(_lib.RT_ERR_TOKEN if code == 4 else _lib.RT_ERR_DEVICE, f"device error code {code}")


class AttentionWorkspace:
    """Scratch of attention_paged; calls that share one run on one stream."""

    def __init__(self, device="cuda"):
        n = max(lib().rt_kernel_attention_paged_workspace_bytes(hd) for hd in (64, 128))
        self.buf = torch.zeros(n, dtype=torch.uint8, device=device)
        self.ptr, self.size, self.index = self.buf.data_ptr(), n, self.buf.device.index


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, rope: Rope, heads: int, kv_heads: int,
                 gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None, eps: float = 1e-5,
                 out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """q and k heads of qkv [T, (heads + kv_heads (+ kv_heads)) * hd] bf16 normed (with gammas) and rotated, v copied;
    out=qkv works in place."""
    return _ext.qk_norm_rope(qkv, positions, rope.addr, rope.index, heads, kv_heads, gamma_q, gamma_k, eps, out, err)


def qk_norm_rope_backward(dout: torch.Tensor, qkv: torch.Tensor | None, positions: torch.Tensor, rope: Rope, heads: int,
                          kv_heads: int, gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None,
                          eps: float = 1e-5, dqkv: torch.Tensor | None = None, dgamma_q: torch.Tensor | None = None,
                          dgamma_k: torch.Tensor | None = None, err: torch.Tensor | None = None):
    """(dqkv, dgamma_q, dgamma_k) of qk_norm_rope, from the gradient of its output and its input qkv (not read
    without gammas).  dqkv=dout works in place; dgammas given are added to, otherwise new (None without gammas)."""
    return _ext.qk_norm_rope_backward(dout, qkv, positions, rope.addr, rope.index, heads, kv_heads, gamma_q, gamma_k, eps,
                                      dqkv, dgamma_q, dgamma_k, err)


def kv_append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, rope: Rope, cache: KvCache, heads: int,
              gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None, eps: float = 1e-5,
              q_out: torch.Tensor | None = None) -> torch.Tensor:
    """qk_norm_rope that writes k and v of token t into cache slot slots[t] (-1: nowhere) and returns q."""
    return _ext.kv_append(qkv, positions, slots, rope.addr, rope.index, cache.addr, cache.index, cache.err_ptr, heads, gamma_q,
                          gamma_k, eps, q_out)


def kv_gather(cache: KvCache, slots: torch.Tensor, k_out: torch.Tensor | None = None,
              v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached tokens back as bf16: (k, v) [T, kv_heads, hd]; slot -1 gives zeros."""
    return _ext.kv_gather(cache.addr, cache.index, cache.err_ptr, slots, k_out, v_out)


def attention_paged(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    q_start: torch.Tensor, heads: int, workspace: AttentionWorkspace, max_q: int, max_kv: int,
                    window: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                    want_lse: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Causal attention of the new tokens q [T, heads * hd] over the cache: sequence s owns rows
    q_start[s] .. q_start[s + 1] and the first kv_lens[s] tokens of pages page_table[s], its new tokens last.
    page_table may be a part of a wider tensor, or one row expanded over the sequences.  Weights keep 15 bits (int8
    cache: 11) for their product with v where max_q * heads / kv_heads <= 16, 8 where it is more.
    Returns (out [T, heads * hd] bf16, lse2 [T, heads] fp32 or None)."""
    return _ext.attention_paged(q, cache.addr, cache.index, cache.err_ptr, page_table, kv_lens, q_start, heads, workspace.ptr,
                                workspace.size, workspace.index, max_q, max_kv, window,
                                cache.scale if scale is None else scale, out, want_lse)


def logits_adjust(logits: torch.Tensor, hist: torch.Tensor | None = None, hist_start: torch.Tensor | None = None,
                  n_prompt: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_vals: torch.Tensor | None = None,
                  bias_start: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(logits after penalties, biases and the grammar mask, the greedy token) per row; out=logits works in place.
    hist (int32, rows by hist_start [B + 1], the first n_prompt[b] the prompt's, -1: not yet written), biases likewise,
    mask [B, ceil(V / 32)] int32 words.  token: int32 [B], -1 where every token is forbidden."""
    return _ext.logits_adjust(logits, hist, hist_start, n_prompt, repetition, presence, frequency, bias_ids, bias_vals,
                              bias_start, mask, out, err)
