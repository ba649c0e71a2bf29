"""Serving many requests from one paged 8-bit key/value cache.

The reference keeps one contiguous fp16 cache per sequence and rotates whole
heads (engine.py:100-158).  These operators serve a batch of requests of any
lengths from a shared pool of pages:

* :func:`page_plan`, :func:`page_release` -- block tables, positions and slot
  maps of a step, built on the GPU from the requests' lengths;
* :func:`rope_tables`, :func:`rope` -- rotary positions: neighbouring or half
  pairs, part of the head, frequencies scaled for long contexts;
* :func:`kv_append`, :func:`rope_append` -- the write of a step's keys and
  values: e4m3 with one power-of-two scale per page and head;
* :func:`paged_attention` -- causal attention of the step's rows over the pages;
* :class:`PagedKVCache` -- the pool, tables and lengths of a model's layers,
  with those calls as methods.

A step's tokens are rows: request r owns rows ``cu_q[r]..cu_q[r + 1]``.  All
functions take CUDA tensors, run on the current stream of their device, never
read the device from the host and can be captured in a CUDA graph.  ``status``
is an optional device int32 word that collects HC_ERR_* bits
(``hc_native.read_status``).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch

import hc_native as N

_DTYPES = {torch.float16: N.HC_F16, torch.bfloat16: N.HC_BF16}
PAGE_SIZES = (16, 32, 64, 128)


# ─── Argument checks ──────────────────────────────────────────────────────────
def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _tensor(t: torch.Tensor, name: str, dtype, shape, device):
    """t is a contiguous tensor of this dtype, shape (None: any size) and device."""
    if t.dtype != dtype or t.dim() != len(shape) or not t.is_contiguous() or t.device != device or \
            any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on {device}, got "
                         f"{t.dtype} {list(t.shape)} on {t.device}"
                         f"{'' if t.is_contiguous() else ', not contiguous'}")


def _heads(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None):
    """t is [rows, heads, dim] in fp16 or bf16 with contiguous dim (rows and heads may be strided)."""
    if not t.is_cuda:
        N.require_cuda(t)
    if t.dim() != 3 or t.dtype not in _DTYPES or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name} must be [rows, heads, dim] in float16 or bfloat16 with contiguous dim")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[0] != like.shape[0]
                             or t.shape[2] != like.shape[2]):
        raise ValueError(f"{name} must have the rows, dim, dtype and device of the other heads")


class _On:
    """The stream to launch on: the tensor's device made current for the call."""

    def __init__(self, device: torch.device):
        self.device = device

    def __enter__(self) -> int:
        self.back = torch.cuda.current_device()
        if self.device.index != self.back:
            torch.cuda.set_device(self.device)
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.device.index != self.back:
            torch.cuda.set_device(self.back)


# ─── Block tables and slot maps ───────────────────────────────────────────────
class PagePlan(NamedTuple):
    """A step's rows: offsets and lengths of the requests, position and slot of every row."""
    cu_q: torch.Tensor          # [requests + 1] int32
    kv_lens: torch.Tensor       # [requests] int32, cached tokens after the step
    positions: torch.Tensor     # [rows] int64, -1 behind the last token
    slots: torch.Tensor         # [rows] int64, -1 behind the last token


def page_plan(starts: torch.Tensor, q_lens: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor,
              n_free: torch.Tensor, page_size: int, n_rows: int, status: Optional[torch.Tensor] = None) -> PagePlan:
    """Places the next ``q_lens[r]`` tokens of every request behind its
    ``starts[r]`` cached ones (hc_page_plan).

    ``tables`` [requests, width] int32 holds page ids, -1 where a page is
    missing; pages that the new tokens need are popped from the stack
    ``free_pages[:n_free]``, in place.  ``n_rows`` (host) is the number of rows
    of the step's arrays, at least the new tokens; the rest is padding.  When
    the lengths, rows or free pages do not work out, nothing is taken, every
    row is padding and HC_ERR_RANGE is set in ``status``."""
    N.require_cuda(starts)
    dev, n = starts.device, starts.shape[0]
    _tensor(starts, "starts", torch.int32, (None,), dev)
    _tensor(q_lens, "q_lens", torch.int32, (n,), dev)
    _tensor(free_pages, "free_pages", torch.int32, (None,), dev)
    _tensor(n_free, "n_free", torch.int32, (1,), dev)
    _need(tables.dim() == 2 and tables.shape[0] == n and tables.dtype == torch.int32 and tables.device == dev
          and tables.stride(1) == 1, "tables must be int32 [requests, width] with contiguous rows")
    _need(n_rows >= 0, "n_rows must not be negative")
    both = torch.empty(2 * n + 1, dtype=torch.int32, device=dev)
    rows = torch.empty(2, n_rows, dtype=torch.int64, device=dev)
    cu_q, kv_lens = both[:n + 1], both[n + 1:]
    positions, slots = rows[0], rows[1]
    with _On(dev) as s:
        N.check(N.lib.hc_page_plan(starts.data_ptr(), q_lens.data_ptr(), n, tables.data_ptr(), tables.stride(0),
                                   tables.shape[1], free_pages.data_ptr(), free_pages.shape[0], n_free.data_ptr(),
                                   page_size, n_rows, cu_q.data_ptr(), kv_lens.data_ptr(), positions.data_ptr(),
                                   slots.data_ptr(), N.ptr(status), s), "hc_page_plan")
    return PagePlan(cu_q, kv_lens, positions, slots)


def page_release(done: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor,
                 status: Optional[torch.Tensor] = None):
    """Gives the pages of the requests with ``done[r]`` (bool) back to the
    stack and empties their table rows, in place (hc_page_release)."""
    N.require_cuda(done)
    dev, n = done.device, done.shape[0]
    _tensor(done, "done", torch.bool, (None,), dev)
    _tensor(free_pages, "free_pages", torch.int32, (None,), dev)
    _tensor(n_free, "n_free", torch.int32, (1,), dev)
    _need(tables.dim() == 2 and tables.shape[0] == n and tables.dtype == torch.int32 and tables.device == dev
          and tables.stride(1) == 1, "tables must be int32 [requests, width] with contiguous rows")
    with _On(dev) as s:
        N.check(N.lib.hc_page_release(done.data_ptr(), n, tables.data_ptr(), tables.stride(0), tables.shape[1],
                                      free_pages.data_ptr(), free_pages.shape[0], n_free.data_ptr(), N.ptr(status),
                                      s), "hc_page_release")


# ─── Rotary positions ─────────────────────────────────────────────────────────
def rope_frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None, max_seq_len: int = 0,
                     device=None):
    """(angle per position of each pair in 64 bits, factor on cos and sin).

    ``scaling`` is a model configuration's dictionary (``rope_type`` or
    ``type``): None or "default"; "linear" (positions divided by ``factor``);
    "dynamic" (base raised for ``max_seq_len`` beyond the original length);
    "yarn" (long wavelengths divided, short ones kept, a linear ramp between
    ``beta_fast`` and ``beta_slow`` turns over the original length, and the
    attention factor); "llama3" (the ramp between ``high_freq_factor`` and
    ``low_freq_factor`` wavelengths of the original length)."""
    _need(rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_dim must be even and positive")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    base = float(theta)
    kind = "default" if not scaling else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return base ** (-i / half), 1.0
    factor = float(scaling["factor"])
    if kind == "linear":
        return base ** (-i / half) / factor, 1.0
    original = scaling.get("original_max_position_embeddings")
    _need(original is not None and original > 0, f"{kind} scaling needs original_max_position_embeddings")
    if kind == "dynamic":
        length = max(int(max_seq_len), int(original))
        base *= (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
        return base ** (-i / half), 1.0
    freq = base ** (-i / half)
    if kind == "yarn":
        def pair(turns):           # the pair that makes so many turns over the original length
            return half * math.log(original / (turns * 2 * math.pi)) / math.log(base)
        low = max(math.floor(pair(float(scaling.get("beta_fast", 32)))), 0)
        high = min(math.ceil(pair(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)       # 0: kept, 1: divided
        attention = scaling.get("attention_factor")
        if attention is None:
            attention = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        return freq * (1 - ramp) + freq / factor * ramp, float(attention)
    if kind == "llama3":
        lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = original * freq / (2 * math.pi)
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)                 # 1: kept, 0: divided
        return freq * keep + freq / factor * (1 - keep), 1.0
    raise ValueError(f"rope scaling {kind!r} is not known")


def rope_tables(max_seq_len: int, rotary_dim: int, theta: float, scaling: Optional[dict] = None, device=None):
    """cos / sin [max_seq_len, rotary_dim // 2] in fp32.  Angles are computed
    in 64 bits: at position 131071 an angle in 32 bits is off by up to 2^-8."""
    freq, factor = rope_frequencies(rotary_dim, theta, scaling, max_seq_len, device)
    angle = torch.arange(max_seq_len, dtype=torch.float64, device=device)[:, None] * freq
    return (angle.cos() * factor).float(), (angle.sin() * factor).float()


def _rope_args(q, k, q_out, k_out, cos, sin, positions, interleaved) -> N.RopeArgs:
    _heads(q, "q")
    _heads(k, "k", q)
    _heads(q_out, "q_out", q)
    _need(q_out.shape == q.shape, "q_out must have the shape of q")
    if k_out is not None:
        _heads(k_out, "k_out", q)
        _need(k_out.shape == k.shape, "k_out must have the shape of k")
    dev, dim = q.device, q.shape[2]
    _tensor(cos, "cos", torch.float32, (None, None), dev)
    _tensor(sin, "sin", torch.float32, cos.shape, dev)
    _tensor(positions, "positions", torch.int64, (q.shape[0],), dev)
    _need(0 < 2 * cos.shape[1] <= dim, "cos and sin must cover at most the head")
    ko = k_out if k_out is not None else k
    return N.RopeArgs(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), ko.data_ptr(), q.stride(0), q.stride(1),
                      k.stride(0), k.stride(1), q_out.stride(0), q_out.stride(1), ko.stride(0), ko.stride(1),
                      cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), q.shape[0], q.shape[1],
                      k.shape[1], dim, 2 * cos.shape[1], int(bool(interleaved)), _DTYPES[q.dtype])


def rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
         interleaved: bool = False, q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
         status: Optional[torch.Tensor] = None):
    """q [rows, heads, dim] and k rotated by their rows' positions (hc_rope).

    ``cos`` / ``sin`` [positions, rotary_dim // 2] fp32; pairs are (i, i +
    rotary_dim / 2), or (2i, 2i + 1) when ``interleaved``; dims past rotary_dim
    pass through.  Returns (q_out, k_out), new tensors unless given (q and k
    themselves rotate in place).  Rows at position -1 are left alone."""
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    args = _rope_args(q, k, q_out, k_out, cos, sin, positions, interleaved)
    with _On(q.device) as s:
        N.check(N.lib.hc_rope(ctypes.byref(args), N.ptr(status), s), "hc_rope")
    return q_out, k_out


# ─── The cache: write and attention ───────────────────────────────────────────
def _pages(k_pages, v_pages, k_scale, v_scale) -> N.KVPages:
    if not k_pages.is_cuda:
        N.require_cuda(k_pages)
    dev = k_pages.device
    _tensor(k_pages, "k_pages", torch.uint8, (None, None, None, None), dev)
    n, h, p, d = k_pages.shape
    _tensor(v_pages, "v_pages", torch.uint8, (n, h, p, d), dev)
    _tensor(k_scale, "k_scale", torch.float32, (n, h), dev)
    _tensor(v_scale, "v_scale", torch.float32, (n, h), dev)
    return N.KVPages(k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, h, p, d)


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              k_scale: torch.Tensor, v_scale: torch.Tensor, status: Optional[torch.Tensor] = None):
    """Writes k and v [rows, kv heads, dim] into their slots of the cache, in
    place (hc_kv_append).  Pages are [pages, kv heads, page size, dim] uint8
    holding e4m3, scales [pages, kv heads] fp32.  The slots of a call are
    distinct, the rows of one page follow one another (as page_plan gives
    them); rows with a negative slot are padding."""
    pages = _pages(k_pages, v_pages, k_scale, v_scale)
    _heads(k, "k")
    _heads(v, "v", k)
    _need(k.shape == v.shape and k.shape[1] == pages.n_kv_heads and k.shape[2] == pages.head_dim
          and k.device == k_pages.device, "k and v must have the cache's heads, dim and device")
    _tensor(slots, "slots", torch.int64, (k.shape[0],), k.device)
    with _On(k.device) as s:
        N.check(N.lib.hc_kv_append(ctypes.byref(pages), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                   v.stride(0), v.stride(1), slots.data_ptr(), k.shape[0], _DTYPES[k.dtype],
                                   N.ptr(status), s), "hc_kv_append")


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor, *, interleaved: bool = False,
                q_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`rope` of q and k and :func:`kv_append` of the rotated k and of v
    in one launch (hc_rope_append), with the same results.  Returns q_out."""
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    args = _rope_args(q, k, q_out, None, cos, sin, positions, interleaved)
    pages = _pages(k_pages, v_pages, k_scale, v_scale)
    _heads(v, "v", k)
    _need(k.shape == v.shape and k.shape[1] == pages.n_kv_heads and k.shape[2] == pages.head_dim
          and k.device == k_pages.device, "k and v must have the cache's heads, dim and device")
    _tensor(slots, "slots", torch.int64, (k.shape[0],), k.device)
    with _On(q.device) as s:
        N.check(N.lib.hc_rope_append(ctypes.byref(args), ctypes.byref(pages), v.data_ptr(), v.stride(0), v.stride(1),
                                     slots.data_ptr(), N.ptr(status), s), "hc_rope_append")
    return q_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, tables: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
                    max_q: int, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    lse: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of q [rows, heads, dim] (rotated) over the requests'
    pages (hc_paged_attn): the row of request r at position pos sees its
    positions 0..pos, its last row sits at ``kv_lens[r] - 1``, and query head h
    reads key-value head h // (heads / kv heads).

    ``max_q`` (host) is the largest number of new tokens of a request: it
    chooses the kernels, any value gives right results.  ``scale`` defaults to
    dim ** -0.5.  ``lse`` (optional, [rows, heads] fp32) receives the logarithm
    of each softmax's sum.  A row that sees no key gives 0 and -inf; padding
    rows of ``out`` are left as they were."""
    pages = _pages(k_pages, v_pages, k_scale, v_scale)
    _heads(q, "q")
    dev = q.device
    rows, heads, dim = q.shape
    _need(dim == pages.head_dim and dev == k_pages.device and heads % pages.n_kv_heads == 0,
          "q must have the cache's dim and device, and a multiple of its heads")
    n = kv_lens.shape[0]
    _tensor(kv_lens, "kv_lens", torch.int32, (None,), dev)
    _tensor(cu_q, "cu_q", torch.int32, (n + 1,), dev)
    _need(tables.dim() == 2 and tables.shape[0] == n and tables.dtype == torch.int32 and tables.device == dev
          and tables.stride(1) == 1, "tables must be int32 [requests, width] with contiguous rows")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _heads(out, "out", q)
        _need(out.shape == q.shape, "out must have the shape of q")
    if lse is not None:
        _tensor(lse, "lse", torch.float32, (rows, heads), dev)
    args = N.AttnArgs(q.data_ptr(), out.data_ptr(), N.ptr(lse), q.stride(0), q.stride(1), out.stride(0),
                      out.stride(1), tables.data_ptr(), tables.stride(0), tables.shape[1], cu_q.data_ptr(),
                      kv_lens.data_ptr(), n, rows, int(max_q), heads,
                      dim ** -0.5 if scale is None else float(scale), _DTYPES[q.dtype])
    need = N.lib.hc_paged_attn_workspace_bytes(n, rows, heads, pages.n_kv_heads, dim)
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    with _On(dev) as s:
        N.check(N.lib.hc_paged_attn(ctypes.byref(args), ctypes.byref(pages), workspace.data_ptr(),
                                    workspace.numel(), N.ptr(status), s), "hc_paged_attn")
    return out


class PagedKVCache:
    """The pages, block tables and lengths of a model's layers.

    One table serves every layer (a page id names a page in each), so a step is
    planned once: ``plan`` places its tokens, ``rope_append`` (or ``append``)
    and ``attend`` run per layer, and ``commit`` makes the new lengths the
    cached ones.  Requests are table rows 0..max_requests-1; ``release`` empties
    rows whose request has ended.  Everything lives on the device, so a step of
    fixed ``n_rows`` can be captured in a CUDA graph.  Calls on one cache must
    be ordered (one stream, or events)."""

    def __init__(self, n_layers: int, n_kv: int, head_dim: int, n_pages: int, *, page_size: int = 64,
                 max_requests: int = 64, max_len: int = 8192, device="cuda"):
        _need(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}")
        _need(head_dim in (64, 128), "head_dim must be 64 or 128")
        _need(n_layers > 0 and n_kv > 0 and n_pages > 0 and max_requests > 0 and max_len > 0, "sizes must be positive")
        self.page_size, self.max_requests = page_size, max_requests
        self.k = torch.zeros(n_layers, n_pages, n_kv, page_size, head_dim, dtype=torch.uint8, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = torch.zeros(n_layers, n_pages, n_kv, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)
        self.tables = torch.full((max_requests, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(n_pages, dtype=torch.int32, device=device).flip(0).contiguous()
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=device)
        self.status = N.new_status(device)

    def __len__(self):
        return self.k.shape[0]

    def __getitem__(self, layer: int):
        """(k pages, v pages, k scales, v scales) of a layer."""
        return self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer]

    def plan(self, q_lens: torch.Tensor, n_rows: int) -> PagePlan:
        """Places ``q_lens[r]`` new tokens of every request (device int32 [max_requests])."""
        return page_plan(self.lens, q_lens, self.tables, self.free_pages, self.n_free, self.page_size, n_rows,
                         self.status)

    def commit(self, plan: PagePlan):
        """The planned tokens are in the cache: the step is over."""
        self.lens.copy_(plan.kv_lens)

    def release(self, done: torch.Tensor):
        """Frees the pages of the requests with ``done[r]`` (device bool [max_requests])."""
        page_release(done, self.tables, self.free_pages, self.n_free, self.status)
        self.lens.masked_fill_(done, 0)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: PagePlan):
        kv_append(k, v, plan.slots, *self[layer], status=self.status)

    def rope_append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, plan: PagePlan, *, interleaved: bool = False,
                    q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        return rope_append(q, k, v, cos, sin, plan.positions, plan.slots, *self[layer], interleaved=interleaved,
                           q_out=q_out, status=self.status)

    def attend(self, layer: int, q: torch.Tensor, plan: PagePlan, *, max_q: int, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        return paged_attention(q, *self[layer], self.tables, plan.cu_q, plan.kv_lens, max_q=max_q, scale=scale,
                               out=out, lse=lse, status=self.status)

    def check(self):
        """Raises HotColdError when a call reported an error (synchronises)."""
        N.read_status(self.status, "paged cache")
