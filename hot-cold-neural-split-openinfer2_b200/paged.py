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
import functools
import math
import struct
from typing import NamedTuple, Optional

import torch

import hc_native as N

_DTYPES = {torch.float16: N.HC_F16, torch.bfloat16: N.HC_BF16}
PAGE_SIZES = (16, 32, 64, 128)
MAX_REQUESTS = 2048             # of one call
# scalings of rope_frequencies and the numbers that each cannot do without, beside the original length
ROPE_SCALINGS = {"linear": ("factor",), "dynamic": ("factor",), "yarn": ("factor",),
                 "llama3": ("factor", "low_freq_factor", "high_freq_factor")}


# ─── Argument checks ──────────────────────────────────────────────────────────
# A step makes three calls a layer, so the checks are plain expressions; what
# is wrong is put into words only when one of them fails.
_I32, _I64, _F32, _U8 = torch.int32, torch.int64, torch.float32, torch.uint8
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
# The argument structs as bytes: packing takes half of the time that building the ctypes structures does.
_KV_PAGES, _ROPE_ARGS = struct.Struct("4P4i"), struct.Struct("4P8q2PqP7i0P")
_ATTN_ARGS = struct.Struct("3P4qPqi2P4ifi0P")
if (_KV_PAGES.size, _ROPE_ARGS.size, _ATTN_ARGS.size) != tuple(
        ctypes.sizeof(c) for c in (N.KVPages, N.RopeArgs, N.AttnArgs)):
    raise ImportError("the packed argument structs do not match hotcold.h")


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _bad(t: torch.Tensor, name: str, dtype, shape, dev: int):
    raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on cuda:{dev}, got {t.dtype} "
                     f"{list(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")


def _vector(t: torch.Tensor, name: str, dtype, n: Optional[int], dev: int) -> int:
    """t is a contiguous vector of n elements (None: any number) on device dev; its address."""
    if t.dtype is not dtype or t.get_device() != dev or t.dim() != 1 or not t.is_contiguous() or \
            (n is not None and t.shape[0] != n):
        _bad(t, name, dtype, [n], dev)
    return t.data_ptr()


def _matrix(t: torch.Tensor, name: str, dtype, n: Optional[int], m: Optional[int], dev: int) -> int:
    if t.dtype is not dtype or t.get_device() != dev or t.dim() != 2 or not t.is_contiguous() or \
            (n is not None and t.shape[0] != n) or (m is not None and t.shape[1] != m):
        _bad(t, name, dtype, [n, m], dev)
    return t.data_ptr()


def _table(t: torch.Tensor, n: int, dev: int) -> int:
    if t.dtype is not _I32 or t.get_device() != dev or t.dim() != 2 or t.shape[0] != n or t.stride(1) != 1:
        raise ValueError(f"tables must be int32 [{n}, width] with contiguous rows on cuda:{dev}")
    return t.data_ptr()


def _heads(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> int:
    """t is [rows, heads, dim] in fp16 or bf16 with contiguous dim (rows and heads may be strided); its address."""
    if not t.is_cuda:
        N.require_cuda(t)
    if t.dim() != 3 or t.dtype not in _DTYPES or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name} must be [rows, heads, dim] in float16 or bfloat16 with contiguous dim")
    if like is not None and (t.dtype is not like.dtype or t.get_device() != like.get_device()
                             or t.shape[0] != like.shape[0] or t.shape[2] != like.shape[2]):
        raise ValueError(f"{name} must have the rows, dim, dtype and device of the other heads")
    return t.data_ptr()


def _status(t: Optional[torch.Tensor], dev: int) -> Optional[int]:
    return None if t is None else _vector(t, "status", _I32, 1, dev)


def _call(fn, where: str, dev: int, *args):
    """fn(*args, stream) with ``dev`` current and its current stream."""
    if _current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        raise N.HotColdError(where, rc)


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
    dev, n = starts.get_device(), starts.shape[0]
    if dev < 0:
        N.require_cuda(starts)
    _need(n_rows >= 0, "n_rows must not be negative")
    device = starts.device
    cu_q = torch.empty(n + 1, dtype=_I32, device=device)
    kv_lens = torch.empty_like(starts)
    positions = torch.empty(n_rows, dtype=_I64, device=device)
    slots = torch.empty_like(positions)
    _call(N.lib.hc_page_plan, "hc_page_plan", dev, _vector(starts, "starts", _I32, None, dev),
          _vector(q_lens, "q_lens", _I32, n, dev), n, _table(tables, n, dev), tables.stride(0), tables.shape[1],
          _vector(free_pages, "free_pages", _I32, None, dev), free_pages.shape[0],
          _vector(n_free, "n_free", _I32, 1, dev), page_size, n_rows, cu_q.data_ptr(), kv_lens.data_ptr(),
          positions.data_ptr(), slots.data_ptr(), _status(status, dev))
    return PagePlan(cu_q, kv_lens, positions, slots)


def page_release(done: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor,
                 status: Optional[torch.Tensor] = None):
    """Gives the pages of the requests with ``done[r]`` (bool) back to the
    stack and empties their table rows, in place (hc_page_release)."""
    dev, n = done.get_device(), done.shape[0]
    if dev < 0:
        N.require_cuda(done)
    _call(N.lib.hc_page_release, "hc_page_release", dev, _vector(done, "done", torch.bool, None, dev), n,
          _table(tables, n, dev), tables.stride(0), tables.shape[1],
          _vector(free_pages, "free_pages", _I32, None, dev), free_pages.shape[0],
          _vector(n_free, "n_free", _I32, 1, dev), _status(status, dev))


# ─── Rotary positions ─────────────────────────────────────────────────────────
def rope_frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None, max_seq_len: int = 0,
                     device=None):
    """(angle per position of each pair in 64 bits, factor on cos and sin).

    ``scaling`` is a model configuration's dictionary (``rope_type`` or
    ``type``): None or "default"; "linear" (positions divided by ``factor``);
    "dynamic" (base raised for ``max_seq_len`` beyond the original length);
    "yarn" (long wavelengths divided, short ones kept, a linear ramp between
    ``beta_fast`` and ``beta_slow`` turns over the original length, and the
    attention factor: given, or from ``mscale`` and ``mscale_all_dim``);
    "llama3" (the ramp between ``high_freq_factor`` and ``low_freq_factor``
    wavelengths of the original length)."""
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
        _need(rotary_dim > 2, "dynamic scaling needs more than one pair")
        length = max(int(max_seq_len), int(original))
        base *= (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
        return base ** (-i / half), 1.0
    freq = base ** (-i / half)
    if kind == "yarn":
        def pair(turns):           # the pair that makes so many turns over the original length
            return half * math.log(original / (turns * 2 * math.pi)) / math.log(base)
        low, high = pair(float(scaling.get("beta_fast", 32))), pair(float(scaling.get("beta_slow", 1)))
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)       # 0: kept, 1: divided
        attention = scaling.get("attention_factor")
        if attention is None:
            def temper(weight):
                return 0.1 * weight * math.log(factor) + 1.0 if factor > 1 else 1.0
            every = scaling.get("mscale_all_dim")                     # given: the model's scale has this part already
            attention = temper(float(scaling.get("mscale") or 1)) / (temper(float(every)) if every else 1.0)
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


def _rope_args(q, k, q_out, k_out, cos, sin, positions, interleaved) -> bytes:
    qp, kp = _heads(q, "q"), _heads(k, "k", q)
    rows, nq, dim = q.shape
    dev = q.get_device()
    if q_out is not q:
        _heads(q_out, "q_out", q)
        _need(q_out.shape[1] == nq, "q_out must have the shape of q")
    if k_out is not k:
        _heads(k_out, "k_out", q)
        _need(k_out.shape[1] == k.shape[1], "k_out must have the shape of k")
    cp = _matrix(cos, "cos", _F32, None, None, dev)
    length, half = cos.shape
    sp = _matrix(sin, "sin", _F32, length, half, dev)
    _need(0 < 2 * half <= dim, "cos and sin must cover at most the head")
    q0, q1, _ = q.stride()
    k0, k1, _ = k.stride()
    r0, r1, _ = q_out.stride()
    t0, t1, _ = k_out.stride()
    return _ROPE_ARGS.pack(qp, kp, q_out.data_ptr(), k_out.data_ptr(), q0, q1, k0, k1, r0, r1, t0, t1, cp, sp, length,
                           _vector(positions, "positions", _I64, rows, dev), rows, nq, k.shape[1], dim, 2 * half,
                           1 if interleaved else 0, _DTYPES[q.dtype])


def rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
         interleaved: bool = False, q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
         status: Optional[torch.Tensor] = None):
    """q [rows, heads, dim] and k rotated by their rows' positions (hc_rope).

    ``cos`` / ``sin`` [positions, rotary_dim // 2] fp32; pairs are (i, i +
    rotary_dim / 2), or (2i, 2i + 1) when ``interleaved``; dims past rotary_dim
    pass through.  Returns (q_out, k_out), new tensors unless given (q and k
    themselves rotate in place; outputs must not overlap the inputs otherwise).
    Rows at position -1 are left alone."""
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    args = _rope_args(q, k, q_out, k_out, cos, sin, positions, interleaved)
    dev = q.get_device()
    _call(N.lib.hc_rope, "hc_rope", dev, args, _status(status, dev))
    return q_out, k_out


# ─── The cache: write and attention ───────────────────────────────────────────
def _pages(k_pages, v_pages, k_scale, v_scale) -> bytes:
    dev = k_pages.get_device()
    if dev < 0:
        N.require_cuda(k_pages)
    shape = k_pages.shape
    if k_pages.dtype is not _U8 or len(shape) != 4 or not k_pages.is_contiguous():
        _bad(k_pages, "k_pages", _U8, "[pages, kv heads, page size, dim]", dev)
    if v_pages.dtype is not _U8 or v_pages.shape != shape or not v_pages.is_contiguous() or \
            v_pages.get_device() != dev:
        _bad(v_pages, "v_pages", _U8, list(shape), dev)
    n, h, p, d = shape
    return _KV_PAGES.pack(k_pages.data_ptr(), v_pages.data_ptr(), _matrix(k_scale, "k_scale", _F32, n, h, dev),
                          _matrix(v_scale, "v_scale", _F32, n, h, dev), n, h, p, d)


def _fits(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, dev: int):
    pages = k_pages.shape
    if k.shape != v.shape or k.shape[1] != pages[1] or k.shape[2] != pages[3] or k.get_device() != dev:
        raise ValueError("k and v must have the cache's heads, dim and device")


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              k_scale: torch.Tensor, v_scale: torch.Tensor, status: Optional[torch.Tensor] = None):
    """Writes k and v [rows, kv heads, dim] into their slots of the cache, in
    place (hc_kv_append).  Pages are [pages, kv heads, page size, dim] uint8
    holding e4m3, scales [pages, kv heads] fp32.  The slots of a call are
    distinct, the rows of one page follow one another (as page_plan gives
    them); rows with a negative slot are padding."""
    pages = _pages(k_pages, v_pages, k_scale, v_scale)
    kp, vp, dev = _heads(k, "k"), _heads(v, "v", k), k_pages.get_device()
    _fits(k, v, k_pages, dev)
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    rows = k.shape[0]
    _call(N.lib.hc_kv_append, "hc_kv_append", dev, pages, kp, k0, k1, vp, v0, v1,
          _vector(slots, "slots", _I64, rows, dev), rows, _DTYPES[k.dtype], _status(status, dev))


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor, *, interleaved: bool = False,
                q_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`rope` of q and k and :func:`kv_append` of the rotated k and of v
    in one call (hc_rope_append), with the same results.  Returns q_out."""
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    args = _rope_args(q, k, q_out, k, cos, sin, positions, interleaved)
    pages = _pages(k_pages, v_pages, k_scale, v_scale)
    vp, dev = _heads(v, "v", k), k_pages.get_device()
    _fits(k, v, k_pages, dev)
    v0, v1, _ = v.stride()
    _call(N.lib.hc_rope_append, "hc_rope_append", dev, args, pages, vp, v0, v1,
          _vector(slots, "slots", _I64, k.shape[0], dev), _status(status, dev))
    return q_out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(requests: int, rows: int, heads: int, kv_heads: int, dim: int) -> int:
    return int(N.lib.hc_paged_attn_workspace_bytes(requests, rows, heads, kv_heads, dim))


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
    rows of ``out`` are left as they were.  ``out`` may be ``q`` itself, but not
    overlap it otherwise."""
    pages = _pages(k_pages, v_pages, k_scale, v_scale)
    qp, dev = _heads(q, "q"), k_pages.get_device()
    rows, heads, dim = q.shape
    nkv = k_pages.shape[1]
    if dim != k_pages.shape[3] or q.get_device() != dev or nkv == 0 or heads % nkv:
        raise ValueError("q must have the cache's dim and device, and a multiple of its heads")
    n = kv_lens.shape[0]
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op = out.data_ptr()
    else:
        op = _heads(out, "out", q)
        _need(out.shape[1] == heads, "out must have the shape of q")
    q0, q1, _ = q.stride()
    o0, o1, _ = out.stride()
    args = _ATTN_ARGS.pack(qp, op, 0 if lse is None else _matrix(lse, "lse", _F32, rows, heads, dev), q0, q1, o0, o1,
                           _table(tables, n, dev), tables.stride(0), tables.shape[1],
                           _vector(cu_q, "cu_q", _I32, n + 1, dev), _vector(kv_lens, "kv_lens", _I32, None, dev), n,
                           rows, max_q, heads, dim ** -0.5 if scale is None else scale, _DTYPES[q.dtype])
    need = max(_workspace_bytes(n, rows, heads, nkv, dim), 16)
    workspace = torch.empty(need, dtype=_U8, device=q.device)
    _call(N.lib.hc_paged_attn, "hc_paged_attn", dev, args, pages, workspace.data_ptr(),
          need, _status(status, dev))
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
        _need(max_requests <= MAX_REQUESTS, f"max_requests must be at most {MAX_REQUESTS}")
        _need(n_layers > 0 and n_kv > 0 and n_pages > 0 and max_requests > 0 and max_len > 0, "sizes must be positive")
        self.page_size, self.max_requests, self.max_len = page_size, max_requests, max_len
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
        """Places ``q_lens[r]`` new tokens of every request (device int32 [max_requests]).
        A step that takes a request past ``max_len`` does not work out, whatever its last page has room for."""
        if self.max_len % self.page_size:          # else the table's width says it
            _vector(q_lens, "q_lens", _I32, self.max_requests, self.lens.get_device())
            q_lens = q_lens.masked_fill(q_lens > self.max_len - self.lens, -1)
        return page_plan(self.lens, q_lens, self.tables, self.free_pages, self.n_free, self.page_size, n_rows,
                         self.status)

    def commit(self, plan: PagePlan):
        """The planned tokens are in the cache: the step is over."""
        self.lens.copy_(plan.kv_lens)

    def release(self, done: torch.Tensor):
        """Frees the pages of the requests with ``done[r]`` (device bool [max_requests])."""
        page_release(done, self.tables, self.free_pages, self.n_free, self.status)
        self.lens.masked_fill_(done & (self.tables[:, 0] < 0), 0)       # a release that was refused leaves the pages

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
