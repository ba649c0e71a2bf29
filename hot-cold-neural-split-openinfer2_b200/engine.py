"""B200 drop-in for the FFN half of the reference's ``engine.py``.

* :class:`HotNeurons` -- one layer's hot FP8 neurons (the reference's hot file,
  splitter.py:221-226 / engine.py:251-264) re-laid out once at load into the
  kernel layout [n_hot][gate row | up row | down column] (12 KiB per neuron).
* :class:`FFNStack` -- L layers of SparseFFNLayer.forward (engine.py:292-312)
  with the predictor lookahead of DesdemonaEngine.forward (engine.py:421-438),
  run by one persistent cooperative kernel per token (``hc_ffn_stack``) plus
  the two predictor launches for layer 0's fetch set.
* :class:`BatchStack` -- the same L layers for a batch of tokens sharing one
  fetch set per layer (the union of the tokens' masks), every weight byte
  read once per 8 tokens (``hc_union_cold`` + ``hc_ffn_batch_layer``).
* :class:`SparseFFNLayer` -- the reference's per-layer module (same
  constructor) on the fused kernel.
* :func:`sparse_ffn` -- the reference's function signature (engine.py:173-209)
  for callers that already hold dense tensors.  It runs on CUDA tensors only.
"""
from __future__ import annotations

import ctypes
import math
import warnings
from pathlib import Path
from typing import Optional, Sequence

import numpy as np
import torch
import torch.distributed
import torch.nn as nn
import torch.nn.functional as F

import hc_native as N
import paged
from predictor import NeuronPredictor, PredictorRegistry, logit_threshold, unpack_mask
from splitter import HIDDEN_DIM, NEURON_RECORD_BYTES, ColdWeightStore, bits_to_words


# ─── Hot neurons ──────────────────────────────────────────────────────────────
class HotNeurons:
    """Hot FP8 neurons of one layer in the fused kernel's layout."""

    def __init__(self, neuron_ids: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                 scales: Optional[torch.Tensor] = None, device="cuda"):
        """gate/up: [n, H] float8_e4m3fn; down: [H, n] float8_e4m3fn (the
        reference's layouts); scales: optional fp32 [n, 3] per-neuron scales
        of (gate, up, down) -- absent means the reference's direct cast."""
        self.device = torch.device(device)
        self.ids = neuron_ids.to(torch.int64).cpu()
        n = int(self.ids.numel())
        self.n = n
        as_u8 = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.to(torch.float8_e4m3fn).view(torch.uint8)
        g, u, d = (as_u8(t.to(self.device)) for t in (gate, up, down))
        if g.shape != (n, HIDDEN_DIM) or u.shape != (n, HIDDEN_DIM) or d.shape != (HIDDEN_DIM, n):
            raise ValueError("hot tensors must be gate/up [n, H] and down [H, n]")
        self.packed = torch.stack([g, u, d.t()], dim=1).contiguous() if n else \
            torch.zeros(1, 3, HIDDEN_DIM, dtype=torch.uint8, device=self.device)
        self.scales = scales.to(self.device, torch.float32).contiguous() if scales is not None else None

    @classmethod
    def from_file(cls, path: str, device="cuda") -> "HotNeurons":
        """Load ``hot_weights/layer_XXX_expert_000.pt`` (splitter.py:221-226)."""
        w = torch.load(str(path), map_location="cpu")
        return cls(w["neuron_ids"], w["gate"], w["up"], w["down"], w.get("scales"), device)

    def decoded(self):
        """fp32 (gate [n,H], up [n,H], down [H,n]) with scales applied."""
        f = self.packed.view(torch.float8_e4m3fn).float()[: self.n]
        if self.scales is not None:
            f = f * self.scales[:, :, None]
        return f[:, 0], f[:, 1], f[:, 2].t()


# ─── Tensor parallelism over the neuron dimension ─────────────────────────────
def split_range(n: int, rank: int, size: int):
    """[lo, hi) of rank's share when n units are split over size ranks."""
    return n * rank // size, n * (rank + 1) // size


class _Share:
    """(rank, size) of a neuron split, for the share helpers."""

    def __init__(self, rank: int, size: int):
        self.rank, self.size = rank, size


class TPGroup:
    """The GPUs that share every layer's neurons, one process per GPU.

    Each rank allocates its exchange buffer (``hc_tp_alloc``), publishes its
    CUDA IPC handle through ``torch.distributed`` (any backend) and opens the
    other ranks' buffers; the fused stack kernel then adds every GPU's partial
    output of a layer by NVLink stores into those buffers.  Build one per
    process with the process group initialised and this rank's device
    current; call :meth:`close` before destroying the process group.
    """

    def __init__(self, group=None, device=None, nbytes: Optional[int] = None):
        """``nbytes``: size of each GPU's exchange buffer (default: the fused
        stack's, hc_tp_buffer_bytes)."""
        import ctypes
        import torch.distributed as dist
        self.size = dist.get_world_size(group)
        self.rank = dist.get_rank(group)
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        with torch.cuda.device(self.device):
            nbytes = int(N.lib.hc_tp_buffer_bytes(self.size)) if nbytes is None else int(nbytes)
            if nbytes <= 0:
                raise ValueError(f"tensor parallelism over {self.size} GPUs is not supported")
            buf = ctypes.c_void_p()
            N.check(N.lib.hc_tp_alloc(nbytes, ctypes.byref(buf)), "hc_tp_alloc")
            self._own = buf.value
            handle = (ctypes.c_uint8 * 64)()
            N.check(N.lib.hc_ipc_get_handle(ctypes.c_void_p(self._own), handle), "hc_ipc_get_handle")
            handles = [None] * self.size
            dist.all_gather_object(handles, bytes(handle), group=group)
            self._opened, ptrs = [], []
            for r, h in enumerate(handles):
                if r == self.rank:
                    ptrs.append(self._own)
                    continue
                hb = (ctypes.c_uint8 * 64).from_buffer_copy(h)
                peer = ctypes.c_void_p()
                N.check(N.lib.hc_ipc_open(hb, ctypes.byref(peer)), "hc_ipc_open")
                self._opened.append(peer.value)
                ptrs.append(peer.value)
            self.peer_buf = torch.tensor(ptrs, dtype=torch.int64, device=self.device)
        self.seq = 0            # layers exchanged so far through these buffers (the same on every rank)

    def close(self):
        for ptr in getattr(self, "_opened", []):
            N.lib.hc_ipc_close(ptr)
        self._opened = []
        if getattr(self, "_own", None):
            N.lib.hc_tp_free(self._own)
            self._own = None


# ─── Fused L-layer stack ──────────────────────────────────────────────────────
class FFNStack:
    """L layers of the hot/cold sparse FFN on one GPU, batch 1.

    forward(x) computes, for l = 0..L-1, x <- x + sparse_ffn(RMSNorm_l(x))
    with layer l's cold neurons = predictor_l(RMSNorm_l(x_{l-1})) & fetchable
    (x_{-1} = x_0: the engine's lookahead, engine.py:421-438).  A layer
    without a predictor fetches every cold neuron (engine.py:282-283).
    """

    def __init__(self, store: ColdWeightStore, hot: Sequence[HotNeurons], norms: Sequence[Optional[torch.Tensor]],
                 predictors: Sequence[Optional[NeuronPredictor]], activation: str = "silu",
                 act_on_both: bool = False, eps: float = 1e-5, threshold: float = 0.5,
                 layer_ids: Optional[Sequence[int]] = None, grid: int = 0, inter: Optional[int] = None,
                 tp: Optional[TPGroup] = None, wait_ns: int = 0):
        """With ``tp``, this GPU takes its share of every layer's neurons: hot
        neurons [r n_hot / N, (r+1) n_hot / N) of each layer's hot list and
        the cold ids of mask words [r W / N, (r+1) W / N); the output is
        the whole layer stack's, identical on every rank.  ``wait_ns``
        limits every bounded wait inside a launch (0 = the kernel's 2 s);
        an expired wait ends the launch with HC_ERR_TIMEOUT in the status.

        Over a store in pinned host memory (``source="pinned"``, the
        reference's cold tier outside the GPU, splitter.py:307-330) every
        layer fetches its predicted records over the bus into the store's
        device staging buffer right before it is computed, and the layers run
        one launch each (the next layer's set is still predicted inside the
        launch of the layer before it); only the hot rows, predictors and one
        section's worth of staging live in HBM."""
        self.store = store
        self.tp = tp
        self.pinned = getattr(store, "source", "device") == "pinned"
        if self.pinned and tp is not None and tp.size > 1:
            raise ValueError("a pinned cold store serves one GPU; tensor parallelism needs the store in HBM")
        self.wait_ns = int(wait_ns)
        self.device = store.device
        self.L = len(hot)
        self.layer_ids = list(layer_ids) if layer_ids is not None else list(range(self.L))
        self.inter = int(inter or store.I)
        if self.inter % 4:
            raise ValueError("the fused kernel needs intermediate_dim % 4 == 0")
        self.words = (self.inter + 31) // 32
        if tp is not None and tp.size > 1:
            hot = [self._hot_share(h, tp) for h in hot]
        self.hot = list(hot)
        self.norms = [n.to(self.device, torch.float32).contiguous() if n is not None else None for n in norms]
        self.predictors = list(predictors)
        for l, pr in enumerate(self.predictors[1:], start=1):
            # layers after the first are predicted inside the kernel (lookahead)
            if pr is not None and not (0 < pr.rank <= 96 and pr.rank % 8 == 0):
                raise ValueError(f"layer {l}: the fused kernel predicts with ranks that are multiples of 8 "
                                 f"up to 96 (got {pr.rank})")
        self.act = N.HC_ACT_RELU if activation == "relu" else N.HC_ACT_SILU
        self.act_on_both = bool(act_on_both)
        self.eps = float(eps)
        self.threshold = float(threshold)
        self.thr = logit_threshold(self.threshold)
        # fetchable cold ids: every hot id of the layer (not only this rank's share) is excluded
        self.fetch = torch.stack([store.fetch_bits(li, h.all_ids if hasattr(h, "all_ids") else h.ids, self.inter)
                                  for li, h in zip(self.layer_ids, self.hot)])
        if tp is not None and tp.size > 1:
            self.words_lo, hi = split_range(self.words, tp.rank, tp.size)
            self.words_n = hi - self.words_lo
        else:
            self.words_lo, self.words_n = 0, self.words
        descs, self._keep = [], []
        for l in range(self.L):
            li = self.layer_ids[l]
            p = self.predictors[l]
            wdt = p.down_t() if p is not None else None
            # a pinned store's records reach the kernel through the staging buffer only
            rec = store.staging() if self.pinned else store.section_records(li)
            self._keep += [rec, wdt]
            descs.append(N.LayerDesc(
                hot=N.ptr(self.hot[l].packed), hot_scale=N.ptr(self.hot[l].scales), norm_w=N.ptr(self.norms[l]),
                cold_records=N.ptr(rec), table=N.ptr(store.table[li]), fetch_bits=N.ptr(self.fetch[l]),
                pred_w_down_t=N.ptr(wdt), pred_w_up=N.ptr(p.up.weight.data) if p is not None else None,
                pred_b_up=N.ptr(p.up.bias.data) if p is not None else None,
                n_hot=self.hot[l].n, n_records=int(store.n_rec_host[li]), inter=self.inter,
                rank=p.rank if p is not None else 0))
        self.desc_dev = N.layer_desc_array(descs, self.device)
        self.grid = int(grid) if grid else int(N.lib.hc_ffn_stack_grid())
        if self.inter > 32768:
            raise ValueError("the fused kernel handles intermediate_dim <= 32768")
        if (self.words_n + self.grid - 1) // self.grid * 32 > 1024:
            raise ValueError(f"grid {self.grid} is too small for {self.inter} neurons per layer "
                             "(one CTA owns at most 1024 neuron ids)")
        self.ws = torch.zeros(int(N.lib.hc_ffn_stack_workspace_bytes(self.grid, self.inter)), dtype=torch.uint8,
                              device=self.device)
        self.masks = torch.zeros(self.L, self.words, dtype=torch.int32, device=self.device)
        self.status = N.new_status(self.device)
        self.x_out = torch.empty(HIDDEN_DIM, dtype=torch.float32, device=self.device)
        ones = torch.ones(self.inter, dtype=torch.bool)
        self._all_ones = bits_to_words(ones.numpy(), self.inter).to(self.device)

    def pred0_in_kernel(self) -> bool:
        """Layer 0's predictor runs inside the stack kernel (hc_ffn_stack with
        masks_given = 2) -- the kernel supports its rank."""
        p0 = self.predictors[0]
        return p0 is not None and 0 < p0.rank <= 96 and p0.rank % 8 == 0

    def first_mask(self, x: torch.Tensor):
        """Layer 0's predicted set from RMSNorm_0(x) (engine.py:422), on device
        (separate predictor launches; ``forward`` lets the stack kernel do it)."""
        p0 = self.predictors[0]
        if p0 is None:
            self.masks[0].copy_(self._all_ones)
        else:
            p0.predict_words(x.view(1, -1), self.threshold, norm_w=self.norms[0], eps=self.eps,
                             mask_out=self.masks[0:1])

    def launch(self, x: torch.Tensor, masks_given=False, x_hist: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, trace: Optional[torch.Tensor] = None,
               predict_last: bool = False, io_f16: bool = False) -> torch.Tensor:
        """One hc_ffn_stack launch.  ``masks_given``: False (row 0 of
        ``self.masks`` holds layer 0's set), True (every row given) or 2 (the
        kernel predicts layer 0 too).  ``predict_last``: the last layer is
        not computed, only its mask row predicted (from the input of the layer
        before it).  ``trace`` (int64 [L, grid, 40], device) (zeroed)
        receives per-CTA phase timestamps and waits (see include/hotcold.h).

        Over a pinned store a launch computes one layer (``L == 1``, or
        ``L == 2`` with ``predict_last``), whose set (mask row 0) is fetched
        into the staging buffer first."""
        if self.pinned:
            if self.L - (1 if predict_last else 0) != 1 or masks_given == 2:
                raise ValueError("over a pinned cold store a launch computes one layer whose set is given "
                                 "(forward() runs the layers one launch each)")
            self._stage(0)
        mg = 2 if masks_given == 2 else (1 if masks_given else 0)
        return self._launch_at(0, self.L, x, mg, x_hist, out, trace, predict_last, io_f16)

    def _stage(self, l: int):
        """Fetch layer l's records (mask row l & fetchable) into the staging buffer."""
        self.store.fetch_masked(self.layer_ids[l], self.masks[l], self.fetch[l], self.inter)

    def _launch_at(self, first: int, n: int, x: torch.Tensor, mg: int, x_hist, out, trace, predict_last: bool,
                   io_f16: bool) -> torch.Tensor:
        """hc_ffn_stack_tp over layers [first, first + n) of this stack."""
        out = self.x_out if out is None else out
        tp = None
        if self.tp is not None and self.tp.size > 1:
            tp = N.TPDesc(size=self.tp.size, rank=self.tp.rank, words_lo=self.words_lo, words_n=self.words_n,
                          peer_buf=N.ptr(self.tp.peer_buf), seq_base=self.tp.seq & 0xFFFFFFFF,
                          wait_ns=self.wait_ns)
            self.tp.seq += n - (1 if predict_last else 0)
        elif self.wait_ns or predict_last or io_f16:
            tp = N.TPDesc(size=1, rank=0, words_lo=0, words_n=self.words, peer_buf=None, seq_base=0,
                          wait_ns=self.wait_ns)
        if tp is not None:
            tp.predict_last = 1 if predict_last else 0
            tp.io_f16 = 1 if io_f16 else 0
        desc = N.ptr(self.desc_dev) + first * ctypes.sizeof(N.LayerDesc)
        N.check(N.lib.hc_ffn_stack_tp(desc, n, self.inter, N.ptr(x), N.ptr(self.masks[first]),
                                      mg, N.ptr(out), N.ptr(x_hist), self.eps, self.act,
                                      1 if self.act_on_both else 0, self.thr, self.grid, N.ptr(self.ws),
                                      N.ptr(self.status), N.ptr(trace),
                                      __import__("ctypes").byref(tp) if tp is not None else None,
                                      N.stream_handle()), "hc_ffn_stack")
        return out

    @staticmethod
    def _hot_share(h: "HotNeurons", tp: TPGroup) -> "HotNeurons":
        """This rank's slice of a layer's hot neurons (a view of the packed rows)."""
        lo, hi = split_range(h.n, tp.rank, tp.size)
        part = HotNeurons.__new__(HotNeurons)
        part.device = h.device
        part.all_ids = h.ids
        part.ids = h.ids[lo:hi]
        part.n = hi - lo
        part.packed = h.packed[lo:hi] if hi > lo else h.packed[:1]
        part.scales = h.scales[lo:hi].contiguous() if h.scales is not None and hi > lo else h.scales
        return part

    def trace_summary(self, trace: torch.Tensor, clock_ghz: float = 1.965) -> dict:
        """Mean / max over CTAs of each phase (us, or counts) from a trace;
        the subgroup-0 loop counters are SM cycles, converted at ``clock_ghz``."""
        t = trace.to(torch.float64).cpu()
        us = t / 1000.0
        out = {}

        def put(name, d):
            out[name] = (float(d.mean()), float(d.max()))

        sg_done = us[:, :, 4:8]
        put("phase0", us[:, :, 1] - us[:, :, 0])
        for k in range(4):
            put(f"subgroup{k}", us[:, :, 4 + k] - us[:, :, 1])
        put("subgroup_spread", sg_done.max(dim=2).values - sg_done.min(dim=2).values)
        put("y_sum", us[:, :, 9] - sg_done.max(dim=2).values)
        put("y_sum.decision", us[:, :, 38] - sg_done.max(dim=2).values)     # bias out, planner check, barrier
        put("y_sum.stage_add", us[:, :, 39] - us[:, :, 38])                 # two tree steps
        put("y_sum.final", us[:, :, 9] - us[:, :, 39])                      # last step, fence, barrier
        put("arrive", us[:, :, 8] - us[:, :, 9])
        put("arrive.bulk_reduce", us[:, :, 28] - us[:, :, 9])
        put("arrive.proxy_fence", us[:, :, 29] - us[:, :, 28])
        put("arrive.release", us[:, :, 8] - us[:, :, 29])
        if t.shape[0] > 1:          # layers with stamps (a traced slice may hold one)
            put("barrier_wait", us[1:, :, 0] - us[:-1, :, 8])
            put("layer", us[1:, :, 0] - us[:-1, :, 0])
            if not (self.tp is not None and self.tp.size > 1):
                # split of the barrier wait: the last CTA's arrival, its sighting, the next layer's input
                last = us[:-1, :, 8].max(dim=1).values[:, None]
                put("barrier.after_own_arrival_to_last", last - us[:-1, :, 8])
                put("barrier.last_arrival_to_seen", us[:-1, :, 32] - last)
                put("barrier.seen_to_layer_start", us[1:, :, 0] - us[:-1, :, 32])
        # layers after the first: the cold pool, its groups, then the hot groups
        # (layer 0: hot groups first); stamps 13/37 hot start/end, 11 pool, 12 cold end
        if t.shape[0] > 1:
            put("issue_wait_pool", us[1:, :, 11] - us[1:, :, 10])
            put("issue_cold", us[1:, :, 12] - us[1:, :, 11])
        put("issue_hot", us[:, :, 37] - us[:, :, 13])
        for name, ev in (("own_words_after_start", 21), ("planner_wake_after_start", 22),
                         ("plan_ready_after_start", 20)):
            stamped = t[:, :, ev] > 0                  # layers where the event happened
            if bool(stamped.any()):
                put(name, (us[:, :, ev] - us[:, :, 0])[stamped])
        cyc = t / (1000.0 * clock_ghz)          # subgroup-0 counters are SM cycles
        put("sg0_poll_wait", cyc[:, :, 16])
        put("sg0_cold_groups", cyc[:, :, 2])
        put("sg0_hot_groups", cyc[:, :, 3])
        put("sg0_other_groups", cyc[:, :, 23])
        put("sg0_group_barrier", cyc[:, :, 24])
        put("sg0_observe", cyc[:, :, 25])
        put("sg0_release", cyc[:, :, 26])
        put("sg0_total", cyc[:, :, 27])
        if self.tp is not None and self.tp.size > 1 and t.shape[2] > 36 and bool((t[:, :, 32] > 0).any()):
            # tensor parallel: local sum seen -> (CTA 0) its slice pushed -> every peer's words seen
            put("tp.local_seen_after_arrive", us[:, :, 32] - us[:, :, 8])
            put("tp.cta0_push", us[:, 0, 36] - us[:, 0, 32])
            put("tp.peers_seen_after_local", us[:-1, :, 35] - us[:-1, :, 32])
        put("issuer_slot_wait", us[:, :, 18])
        # the launch as a whole (layer 0's slot): CTA start -> layer 0 start, last layer's end -> CTA done
        put("launch.start_to_layer0", us[0, :, 0] - us[0, :, 33])
        put("launch.span", us[0, :, 34] - us[0, :, 33])
        put("dynamic_hot_claimed[n]", t[:, :, 15])
        put("cold_listed[n]", t[:, :, 17])
        put("cold_taken[n]", t[:, :, 30])
        put("groups[n]", t[:, :, 19])
        return out

    def forward(self, x: torch.Tensor, masks: Optional[torch.Tensor] = None, x_hist: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x: fp32 [H] on the device.  ``masks`` (int32 words [L, W]) forces
        the fetch set of every layer instead of running the predictors."""
        N.require_cuda(x)
        x = x.to(torch.float32).contiguous().view(-1)
        if self.pinned:
            return self._forward_pinned(x, masks, x_hist, out)
        if masks is not None:
            self.masks.copy_(masks)
            return self.launch(x, True, x_hist, out)
        if self.pred0_in_kernel():
            return self.launch(x, 2, x_hist, out)
        self.first_mask(x)
        return self.launch(x, False, x_hist, out)

    __call__ = forward

    def _forward_pinned(self, x: torch.Tensor, masks, x_hist, out) -> torch.Tensor:
        """forward() over a pinned store: per layer, fetch its records into
        the staging buffer, then one launch that computes it and (when the
        sets are not given) predicts the next layer's set from the same input
        -- the order of the whole-stack launch (engine.py:421-438)."""
        out = self.x_out if out is None else out
        if masks is not None:
            self.masks.copy_(masks)
        else:
            self.first_mask(x)
        if getattr(self, "_ping", None) is None:
            self._ping = torch.empty(2, HIDDEN_DIM, dtype=torch.float32, device=self.device)
        cur = x
        for l in range(self.L):
            if masks is None and l > 0 and self.predictors[l] is None:
                self.masks[l].copy_(self._all_ones)          # no predictor: every cold neuron
            self._stage(l)
            pair = masks is None and l + 1 < self.L and self.predictors[l + 1] is not None
            dst = out if l == self.L - 1 else self._ping[l % 2]
            self._launch_at(l, 2 if pair else 1, cur, 0, x_hist[l] if x_hist is not None else None, dst, None,
                            pair, False)
            cur = dst
        return out

    def decode_host(self, x_host: torch.Tensor, y_host: torch.Tensor) -> torch.Tensor:
        """Decode T tokens given in host memory: x_host [T, H] fp32 (pinned for
        an asynchronous copy) -> y_host [T, H].  One host-to-device copy of the
        inputs, T fused forwards, one device-to-host copy of the outputs, all
        on the current stream; returns without synchronising."""
        T = x_host.shape[0]
        if getattr(self, "_io_in", None) is None or self._io_in.shape[0] < T:
            self._io_in = torch.empty(T, HIDDEN_DIM, dtype=torch.float32, device=self.device)
            self._io_out = torch.empty(T, HIDDEN_DIM, dtype=torch.float32, device=self.device)
        xi, yo = self._io_in[:T], self._io_out[:T]
        xi.copy_(x_host, non_blocking=True)
        for t in range(T):
            self.forward(xi[t], out=yo[t])
        y_host.copy_(yo, non_blocking=True)
        return y_host

    def check(self):
        N.read_status(self.status, "hc_ffn_stack")
        if self.pinned:
            self.store.check()              # the staging copies

    def active_counts(self) -> torch.Tensor:
        """Active cold neurons per layer of the last forward (this GPU's share
        of the neuron ids under tensor parallelism)."""
        own = slice(self.words_lo, self.words_lo + self.words_n)
        m = (self.masks[:, own] & self.fetch[:, own]).to(torch.int64) & 0xFFFFFFFF
        return torch.stack([torch.tensor([bin(int(v)).count("1") for v in row.tolist()]).sum() for row in m.cpu()])


class BatchStack:
    """L layers of the hot/cold sparse FFN for a batch of B tokens on one GPU.

    forward(x [B, H]) computes, for l = 0..L-1, x_b <- x_b + sparse_ffn(
    RMSNorm_l(x_b)) for every token b, with one fetch set per layer and
    batch: the union over the batch's tokens of their active masks, & the
    fetchable cold ids.  The masks are either given ([L, B, W] int32 words,
    e.g. per-token Bernoulli draws) or the per-token predictions of each
    layer's predictor on RMSNorm_l(x_b); a layer without a predictor fetches
    every cold neuron (engine.py:282-283).  The reference's batched query
    (engine.py:277-279) asks the predictor once, on the batch mean of the
    normalised inputs; the union of per-token predictions contains every
    neuron a single token's own prediction selects.
    """

    def __init__(self, store: ColdWeightStore, hot: Sequence[HotNeurons], norms: Sequence[Optional[torch.Tensor]],
                 predictors: Optional[Sequence[Optional[NeuronPredictor]]] = None, activation: str = "silu",
                 act_on_both: bool = False, eps: float = 1e-5, threshold: float = 0.5,
                 layer_ids: Optional[Sequence[int]] = None, inter: Optional[int] = None, max_batch: int = 64,
                 dense_min_batch: int = 8, single_token_stack: bool = True, shard=None, group=None):
        """Batches of at least ``dense_min_batch`` tokens use the dense mode of
        hc_ffn_batch_layer: every record streamed, in storage order, from a
        packed copy of the layer made once here (hc_batch_pack, about the
        layer's own size again), and masked by the union -- their union covers
        most of each section, and whole contiguous blocks stream faster than
        per-record pieces.  A single token with given masks runs the fused
        batch-1 stack kernel (FFNStack) instead of the tensor-core kernels
        unless ``single_token_stack`` is False.

        ``shard=(rank, size)``: this GPU takes hot neurons [rank n_hot / size,
        (rank+1) n_hot / size) of each layer's hot list and the cold records
        with section indices in [rank n_rec / size, (rank+1) n_rec / size);
        each layer's partial output [B, 4096] is summed over the GPUs of
        ``group`` by one exchange kernel (hc_xchg_sum: NVLink stores into the
        peers' IPC-mapped buffers, bounded waits) that adds the sum into x, so
        every rank ends with the whole stack's output; a forward holds no
        library collective and a CUDA graph can capture it.  Sharded batches
        always stream the packed copy of the share (the union's flags
        select).  Build it on every rank with the process group initialised
        (the buffers' IPC handles are exchanged over ``group``) and call
        :meth:`close` before destroying the group.

        Over a store in pinned host memory each layer's union is fetched over
        the bus into the store's staging buffer before the layer runs (the
        gathered mode; no packed copies are made)."""
        self.store = store
        self.pinned = getattr(store, "source", "device") == "pinned"
        if self.pinned and shard is not None and int(shard[1]) > 1:
            raise ValueError("a pinned cold store serves one GPU; sharding needs the store in HBM")
        self.device = store.device
        self.L = len(hot)
        self.layer_ids = list(layer_ids) if layer_ids is not None else list(range(self.L))
        self.inter = int(inter or store.I)
        self.words = (self.inter + 31) // 32
        self.hot = list(hot)
        self.norms = [n.to(self.device, torch.float32).contiguous() if n is not None else None for n in norms]
        self.predictors = list(predictors) if predictors is not None else [None] * self.L
        self.activation = activation
        self.act = N.HC_ACT_RELU if activation == "relu" else N.HC_ACT_SILU
        self.act_on_both = bool(act_on_both)
        self.eps = float(eps)
        self.threshold = float(threshold)
        self.max_batch = int(max_batch)
        self._single_stack = None
        self.single_token_stack = bool(single_token_stack)
        self.shard = (0, 1) if shard is None else (int(shard[0]), int(shard[1]))
        self.group = group
        if not 0 <= self.shard[0] < self.shard[1]:
            raise ValueError(f"bad shard {shard}")
        self.fetch = torch.stack([store.fetch_bits(li, h.ids, self.inter) for li, h in zip(self.layer_ids, self.hot)])
        rank, size = self.shard
        if size > 1:
            self.hot = [FFNStack._hot_share(h, _Share(rank, size)) for h in self.hot]
        self.descs, self._keep, self.max_cold, self.rec_lo = [], [], [], []
        for l in range(self.L):
            li = self.layer_ids[l]
            rec = store.staging() if self.pinned else store.section_records(li)
            self._keep.append(rec)
            r0, r1 = split_range(int(store.n_rec_host[li]), rank, size)
            self.rec_lo.append(r0)
            self.max_cold.append(r1 - r0)
            self.descs.append(N.LayerDesc(
                hot=N.ptr(self.hot[l].packed), hot_scale=N.ptr(self.hot[l].scales), norm_w=N.ptr(self.norms[l]),
                cold_records=N.ptr(rec) + r0 * NEURON_RECORD_BYTES, table=N.ptr(store.table[li]),
                fetch_bits=N.ptr(self.fetch[l]), n_hot=self.hot[l].n, n_records=r1 - r0, inter=self.inter, rank=0))
        # the union (and its flags) always covers the whole section
        self.sec_records = [int(store.n_rec_host[li]) for li in self.layer_ids]
        max_neurons = max(h.n + c for h, c in zip(self.hot, self.max_cold))
        self.ws = torch.zeros(int(N.lib.hc_ffn_batch_workspace_bytes(max(max_neurons, 1))), dtype=torch.uint8,
                              device=self.device)
        self.rec = torch.zeros(self.L, max(max(self.sec_records), 1), dtype=torch.int32, device=self.device)
        self.count = torch.zeros(self.L, dtype=torch.int32, device=self.device)
        self.dense_min_batch = 1 if size > 1 else int(dense_min_batch)
        if self.pinned:
            self.dense_min_batch = self.max_batch + 1        # gathered mode only
        self.flag_stride = (max(max(self.sec_records), 1) + 15) // 16 * 16
        self.part = torch.zeros(self.max_batch, HIDDEN_DIM, dtype=torch.float32, device=self.device) \
            if size > 1 else None
        self.xg = None
        if size > 1:
            cap = self.max_batch * HIDDEN_DIM
            self.xg = TPGroup(group, self.device, nbytes=int(N.lib.hc_xchg_buffer_bytes(size, cap)))
            self.xg_cap = cap
            self._xdesc = N.TPDesc(size=size, rank=rank, words_lo=0, words_n=0, peer_buf=N.ptr(self.xg.peer_buf),
                                   seq_base=0, wait_ns=0)
        self.flags = torch.zeros(self.L, self.flag_stride, dtype=torch.uint8, device=self.device)
        # dense mode streams a packed copy of each layer (hc_batch_pack), built once here
        self.packed = [None] * self.L
        if self.dense_min_batch <= self.max_batch:
            s = N.stream_handle()
            for l in range(self.L):
                nbytes = int(N.lib.hc_batch_pack_bytes(self.hot[l].n, self.max_cold[l]))
                buf = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
                N.check(N.lib.hc_batch_pack(ctypes.byref(self.descs[l]), N.ptr(buf), s), "hc_batch_pack")
                self.packed[l] = buf
        self.pred_masks = torch.zeros(self.L, self.max_batch, self.words, dtype=torch.int32, device=self.device)
        self.status = N.new_status(self.device)
        self._all_ones = bits_to_words(torch.ones(self.inter, dtype=torch.bool).numpy(), self.inter).to(self.device)

    def _layer_masks(self, l: int, x: torch.Tensor) -> torch.Tensor:
        B = x.shape[0]
        out = self.pred_masks[l, :B]
        p = self.predictors[l]
        if p is None:
            out.copy_(self._all_ones.view(1, -1).expand(B, -1))
        else:
            p.predict_words(x, self.threshold, norm_w=self.norms[l], eps=self.eps, mask_out=out)
        return out

    def forward(self, x: torch.Tensor, masks: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                x_hist: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x: fp32 [B, H] on the device (B <= max_batch); returns the stack's
        output (``out`` if given, else a new tensor).  ``masks``: int32
        [L, B, W]; ``x_hist`` (optional [L, B, H]) receives every layer's output."""
        N.require_cuda(x)
        B = x.shape[0]
        if B < 1 or B > self.max_batch:
            raise ValueError(f"batch {B} outside [1, {self.max_batch}]")
        y = out if out is not None else torch.empty(B, HIDDEN_DIM, dtype=torch.float32, device=self.device)
        y.copy_(x.reshape(B, HIDDEN_DIM))
        if masks is not None:
            masks = masks.to(self.device, torch.int32).contiguous()
            if tuple(masks.shape) != (self.L, B, self.words):
                raise ValueError(f"masks must be [L={self.L}, B={B}, W={self.words}] int32 words")
        s = N.stream_handle()
        dense = B >= self.dense_min_batch
        flags = self.flags if dense else None
        if masks is not None and self._tables_contiguous():
            # every layer's fetch set is known up front: one launch for all layers
            t0 = self.store.table[self.layer_ids[0]]
            N.check(N.lib.hc_union_cold_layers(N.ptr(masks), self.L, masks.stride(0), B, masks.stride(1),
                                               self.inter, N.ptr(self.fetch), N.ptr(t0), N.ptr(self.rec),
                                               self.rec.stride(0), N.ptr(self.count), N.ptr(flags),
                                               self.flag_stride, s), "hc_union_cold_layers")
        if B == 1 and masks is not None and self.single_token_stack and self.shard[1] == 1 and self.inter % 4 == 0:
            # one token: the fused stack kernel (one persistent launch for every layer)
            st = self._single()
            st.forward(x.reshape(HIDDEN_DIM), masks=masks[:, 0, :], x_hist=x_hist[:, 0] if x_hist is not None else None,
                       out=y[0])
            if not self._tables_contiguous():
                for l in range(self.L):          # keep union_counts() / rec meaningful
                    m = masks[l]
                    N.check(N.lib.hc_union_cold_layers(N.ptr(m), 1, 0, B, m.stride(0), self.inter,
                                                       N.ptr(self.fetch[l]), N.ptr(self.store.table[self.layer_ids[l]]),
                                                       N.ptr(self.rec[l]), 0, N.ptr(self.count[l:l + 1]), None,
                                                       self.flag_stride, s), "hc_union_cold_layers")
            return y
        for l in range(self.L):
            if masks is None or not self._tables_contiguous():
                m = masks[l] if masks is not None else self._layer_masks(l, y)
                N.check(N.lib.hc_union_cold_layers(N.ptr(m), 1, 0, B, m.stride(0), self.inter, N.ptr(self.fetch[l]),
                                                   N.ptr(self.store.table[self.layer_ids[l]]), N.ptr(self.rec[l]),
                                                   0, N.ptr(self.count[l:l + 1]),
                                                   N.ptr(flags[l]) if dense else None, self.flag_stride, s),
                        "hc_union_cold_layers")
            if self.pinned:
                # the union's records over the bus into the staging buffer
                self.store.stage_records(self.layer_ids[l], self.rec[l, :self.sec_records[l]], self.store.staging(),
                                         self.count[l:l + 1])
            if self.part is None:
                N.check(N.lib.hc_ffn_batch_layer(ctypes.byref(self.descs[l]), N.ptr(self.packed[l]), N.ptr(y), B,
                                                 N.ptr(self.rec[l]),
                                                 N.ptr(self.count[l:l + 1]), self.max_cold[l],
                                                 N.ptr(flags[l]) if dense else None, self.eps, self.act,
                                                 1 if self.act_on_both else 0, N.ptr(self.ws), N.ptr(self.status), s),
                        "hc_ffn_batch_layer")
            else:
                # this GPU's share of the layer into part, then y += the sum of every GPU's part
                part = self.part[:B]
                part.zero_()
                N.check(N.lib.hc_ffn_batch_layer_partial(
                    ctypes.byref(self.descs[l]), N.ptr(self.packed[l]), N.ptr(y), B, N.ptr(self.rec[l]),
                    N.ptr(self.count[l:l + 1]), self.max_cold[l], N.ptr(flags[l]) + self.rec_lo[l], self.eps,
                    self.act, 1 if self.act_on_both else 0, N.ptr(self.ws), N.ptr(part), N.ptr(self.status), s),
                    "hc_ffn_batch_layer_partial")
                N.check(N.lib.hc_xchg_sum(N.ptr(part), B * HIDDEN_DIM, N.ptr(y), self.xg_cap,
                                          ctypes.byref(self._xdesc), N.ptr(self.status), s), "hc_xchg_sum")
            if x_hist is not None:
                x_hist[l].copy_(y)
        return y

    __call__ = forward

    def _single(self) -> "FFNStack":
        """The batch-1 stack over the same layers (built on first use)."""
        if self._single_stack is None:
            self._single_stack = FFNStack(self.store, self.hot, self.norms, [None] * self.L, self.activation,
                                          self.act_on_both, self.eps, self.threshold, layer_ids=self.layer_ids,
                                          inter=self.inter)
        return self._single_stack

    def _tables_contiguous(self) -> bool:
        """Layer ids consecutive, so table rows of layer l sit at table[first + l]."""
        ids = self.layer_ids
        return all(b == a + 1 for a, b in zip(ids, ids[1:]))

    def check(self):
        N.read_status(self.status, "hc_ffn_batch_layer")
        if self.pinned:
            self.store.check()              # the staging copies
        if self._single_stack is not None:
            self._single_stack.check()

    def close(self):
        """Release the exchange buffers of a sharded stack (before the process
        group is destroyed)."""
        if self.xg is not None:
            self.xg.close()
            self.xg = None

    def union_counts(self) -> torch.Tensor:
        """Cold records each layer fetched in the last forward."""
        return self.count.cpu()


# ─── Reference-compatible pieces ─────────────────────────────────────────────
def _gated_act(g, u, activation: str, act_on_both: bool):
    act = F.relu if activation == "relu" else F.silu
    return act(g) * act(u) if act_on_both else act(g) * u


def sparse_ffn(x, activation, act_on_both, gate_hot, up_hot, down_hot, gate_cold, up_cold, down_cold):
    """engine.py:173-209 for callers holding dense tensors (CUDA only).

    The hot half runs in x's dtype and the cold half in fp32, cast back, as
    the reference does.  The fused FP8/INT4 kernel path is :class:`FFNStack`
    / :class:`SparseFFNLayer`, which never materialises dense cold weights."""
    N.require_cuda(x)
    results = []
    if gate_hot is not None and gate_hot.shape[0] > 0:
        g = F.linear(x, gate_hot)
        u = F.linear(x, up_hot)
        results.append(F.linear(_gated_act(g, u, activation, act_on_both), down_hot))
    if gate_cold is not None and gate_cold.shape[0] > 0:
        xf = x.float()
        g = F.linear(xf, gate_cold)
        u = F.linear(xf, up_cold)
        results.append(F.linear(_gated_act(g, u, activation, act_on_both), down_cold).to(x.dtype))
    if not results:
        return torch.zeros_like(x)
    return sum(results)


class SparseFFNLayer(nn.Module):
    """The reference's SparseFFNLayer (engine.py:212-312) on the fused kernels.

    ``submit_cold_fetch`` returns the device mask words of the predicted set
    (no host sync, no thread pool).  ``forward`` runs RMSNorm + hot + cold +
    residual: one token row through the fused stack kernel (one layer), and
    B * T > 1 rows -- the reference's single sparse_ffn call over all rows
    with one fetch set (engine.py:292-312) -- through the batched tensor-core
    layer (hc_ffn_batch_layer), every weight byte read once per 64 rows."""

    _EID = 0

    def __init__(self, layer_idx: int, hot_dir: str, cold_store: ColdWeightStore,
                 predictor: Optional[PredictorRegistry], cfg: dict, device, executor=None,
                 ffn_norm_weight: Optional[torch.Tensor] = None):
        super().__init__()
        self.layer_idx = layer_idx
        self.cold_store = cold_store
        self.predictor = predictor
        self.device = torch.device(device)
        self.executor = executor
        self.activation = cfg.get("hidden_act", "silu")
        self.act_on_both = cfg.get("act_on_both", False)
        self.inter_dim = cfg["intermediate_dim"]
        self.eps = cfg["rms_norm_eps"]
        self.input_layernorm = nn.RMSNorm(cfg["hidden_dim"], eps=self.eps)
        if ffn_norm_weight is not None:
            self.input_layernorm.weight = nn.Parameter(ffn_norm_weight.to(self.device))
        self.input_layernorm.to(self.device)
        hot = hot_dir if isinstance(hot_dir, HotNeurons) else None
        p = None if hot is not None else Path(hot_dir) / f"layer_{layer_idx:03d}_expert_{self._EID:03d}.pt"
        if hot is not None:
            self.hot = hot
        elif p.exists():
            self.hot = HotNeurons.from_file(str(p), self.device)
        else:
            z8 = torch.zeros(0, HIDDEN_DIM, dtype=torch.float8_e4m3fn)
            self.hot = HotNeurons(torch.zeros(0, dtype=torch.int64), z8, z8, z8.t(), None, self.device)
        self._hot_id_set = set(self.hot.ids.tolist())
        self._pred = predictor.get(layer_idx, self._EID) if predictor is not None else None
        self._norm32 = self.input_layernorm.weight.detach().to(torch.float32).contiguous()
        self._stack = FFNStack(cold_store, [self.hot], [self._norm32], [self._pred], self.activation,
                               self.act_on_both, self.eps, layer_ids=[layer_idx], inter=self.inter_dim)
        self._batch: Optional[BatchStack] = None
        self._rows_in = self._rows_out = None

    def _query(self, x_normed: torch.Tensor) -> torch.Tensor:
        return x_normed[:, -1, :].mean(0, keepdim=True)          # engine.py:277

    def _mask_words(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Predicted-set words for input x [B, T, H] (not yet normalised)."""
        if self._pred is None:
            w = self._stack._all_ones.view(1, -1)
            return out.copy_(w) if out is not None else w.clone()
        if x.shape[0] == 1:
            row = x[0, -1:, :].to(torch.float32)
            return self._pred.predict_words(row, 0.5, norm_w=self._norm32, eps=self.eps, mask_out=out)
        q = self._query(self.normed32(x))
        return self._pred.predict_words(q, 0.5, mask_out=out)

    def normed32(self, x: torch.Tensor) -> torch.Tensor:
        """The layer's RMSNorm (post_attention_layernorm, engine.py:246-249) of
        x in fp32."""
        xf = x.to(torch.float32)
        return xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps) * self._norm32

    def _cold_ids_for(self, x_normed: torch.Tensor) -> list[int]:
        """engine.py:274-283: host list of the cold ids to fetch."""
        if self._pred is not None:
            mask = self.predictor.predict(self.layer_idx, self._EID, self._query(x_normed))
            ids = mask[0].nonzero(as_tuple=True)[0].tolist()
            return [i for i in ids if i not in self._hot_id_set]
        return [i for i in range(self.inter_dim) if i not in self._hot_id_set]

    def submit_cold_fetch(self, x: torch.Tensor, out: Optional[torch.Tensor] = None):
        """The lookahead prefetch (engine.py:285-290): device mask words."""
        return self._mask_words(x, out)

    def _batched(self, rows: int) -> BatchStack:
        if self._batch is None or self._batch.max_batch < rows:
            cap = max(64, 1 << (rows - 1).bit_length())
            self._batch = BatchStack(self.cold_store, [self.hot], [self._norm32], None, self.activation,
                                     self.act_on_both, self.eps, layer_ids=[self.layer_idx], inter=self.inter_dim,
                                     max_batch=cap, single_token_stack=False)
        return self._batch

    def forward_lookahead(self, x: torch.Tensor, words: torch.Tensor, nxt: "SparseFFNLayer",
                          next_words: torch.Tensor) -> torch.Tensor:
        """forward(x, words) for one token row that also predicts the next
        layer's fetch set from this x (its post-attention hidden state,
        engine.py:430-438) into ``next_words``, inside the same kernel
        launch.  ``words`` and ``next_words`` must be consecutive rows of one
        [L, W] int32 buffer."""
        pair = getattr(self, "_pair", None)
        if pair is None or pair[0] is not nxt:
            st = FFNStack(self.cold_store, [self.hot, nxt.hot], [self._norm32, nxt._norm32], [None, nxt._pred],
                          self.activation, self.act_on_both, self.eps,
                          layer_ids=[self.layer_idx, nxt.layer_idx], inter=self.inter_dim)
            pair = (nxt, st)
            self._pair = pair
        st = pair[1]
        base = words.untyped_storage().data_ptr()
        if next_words.untyped_storage().data_ptr() != base or \
                next_words.data_ptr() - words.data_ptr() != 4 * st.words:
            raise ValueError("words and next_words must be consecutive rows of one buffer")
        st.masks = words.view(-1).as_strided((2, st.words), (st.words, 1))
        B, T, H = x.shape
        if x.dtype == torch.float16:
            # fp16 hidden state in and out of the kernel (it computes in fp32)
            row = x.reshape(H).contiguous()
            out = torch.empty_like(row)
            st.launch(row, masks_given=False, out=out, predict_last=True, io_f16=True)
            return out.view(B, T, H)
        rows = x.reshape(B * T, H).to(torch.float32).contiguous()
        out = torch.empty_like(rows)
        st.launch(rows[0], masks_given=False, out=out[0], predict_last=True)
        return out.reshape(B, T, H).to(x.dtype)

    def forward(self, x: torch.Tensor, prefetch_future=None) -> torch.Tensor:
        B, T, H = x.shape
        words = prefetch_future if prefetch_future is not None else self._mask_words(x)
        rows = x.reshape(B * T, H).to(torch.float32).contiguous()
        n = rows.shape[0]
        if n == 1:
            self._stack.masks.copy_(words.view(1, -1))
            out = torch.empty_like(rows)
            self._stack.launch(rows[0], masks_given=True, out=out[0])
        else:
            # every row shares the one fetch set (engine.py:297-311)
            bst = self._batched(n)
            m = words.view(1, 1, -1).expand(1, n, -1)
            out = bst.forward(rows, masks=m)
        return out.reshape(B, T, H).to(x.dtype)

    def check(self):
        self._stack.check()
        if self._batch is not None:
            self._batch.check()
        if getattr(self, "_pair", None) is not None:
            self._pair[1].check()


# ─── Model shell (engine.py:61-158, :317-511) ─────────────────────────────────
# Attention, RoPE and sampling are torch code (they are not on the sparse-FFN
# path); the FFN half of every layer runs the kernels above.  The KV cache is
# preallocated once per sequence, so a decode step has static shapes and the
# whole step is captured in one CUDA graph.
def build_rope_cache(max_seq_len: int, head_dim: int, theta: float, device=None):
    """cos / sin tables [max_seq_len, head_dim // 2] in fp32 for rotary
    position embedding with base ``theta`` (engine.py:130-140)."""
    half = head_dim // 2
    # frequency i = theta^(-i / half), evaluated as 1 / theta^(i / half) in fp32
    inv = 1.0 / (float(theta) ** (torch.arange(half, device=device).float() / half))
    ang = torch.arange(max_seq_len, device=device).float()[:, None] * inv[None, :]
    return torch.cos(ang), torch.sin(ang)


def _rope_scaling(cfg: dict) -> Optional[dict]:
    """The configuration's ``rope_scaling`` as paged.rope_frequencies takes it: a stock entry that leaves the
    original length out means max_position_embeddings.  One of an unknown kind, or without a number that its kind
    needs, is left aside with a warning: the model then runs unscaled."""
    scaling = cfg.get("rope_scaling")
    if not scaling:
        return None
    kind = scaling.get("rope_type") or scaling.get("type") or "default"
    if kind == "default":
        return None
    if any(scaling.get(n) is None for n in paged.ROPE_SCALINGS.get(kind, (kind,))):
        warnings.warn(f"rope_scaling {scaling} is not known: positions are not scaled")
        return None
    original = scaling.get("original_max_position_embeddings") or cfg.get("max_position_embeddings")
    return {**scaling, "rope_type": kind, "original_max_position_embeddings": original}


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotary embedding of x [B, heads, T, D] (halves rotated as pairs,
    engine.py:143-158); cos / sin [T, D/2] are cast to x's dtype first."""
    d = x.shape[-1] // 2
    c = cos.to(x.dtype)[None, None]
    s = sin.to(x.dtype)[None, None]
    a, b = x[..., :d], x[..., d:]
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


class KVCache:
    """Preallocated key / value cache of every layer: [B, n_kv, capacity, D]
    fp16 per layer and tensor, filled up to ``length`` positions.  Indexing
    gives the reference's per-layer (k, v) pair (engine.py:111-115), views of
    the filled part."""

    def __init__(self, n_layers: int, batch: int, n_kv: int, capacity: int, head_dim: int, device,
                 dtype=torch.float16):
        self.k = torch.zeros(n_layers, batch, n_kv, capacity, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.capacity = capacity
        self.length = 0
        self.pos = torch.zeros(1, dtype=torch.int64, device=device)     # == length, on the device

    def __len__(self):
        return self.k.shape[0]

    def __getitem__(self, layer: int):
        return self.k[layer, :, :, :self.length], self.v[layer, :, :, :self.length]


class GroupedQueryAttention(nn.Module):
    """Grouped-query attention of one layer (engine.py:63-125): FP8-at-rest
    q/k/v/o weights computed in fp16, the layer's pre-norm, RoPE, causal
    softmax attention over the cache."""

    def __init__(self, layer_idx: int, weights: dict, cfg: dict, device="cuda", fp8_decode: bool = True):
        super().__init__()
        self.layer_idx = layer_idx
        self.n_q = cfg["num_attention_heads"]
        self.n_kv = cfg["num_key_value_heads"]
        self.hidden = cfg["hidden_dim"]
        self.head_dim = self.hidden // self.n_q
        pre = f"layer_{layer_idx:03d}."
        dev = torch.device(device)
        w16 = lambda n: weights[pre + n].to(dev).to(torch.float16)
        # q, k and v projections as one [H + 2 n_kv D, H] matrix: one GEMM instead of three
        self.qkv_weight = torch.cat([w16("q_proj"), w16("k_proj"), w16("v_proj")], dim=0).contiguous()
        self.o_weight = w16("o_proj").contiguous()
        # one-token steps read the FP8 bytes themselves (hc_fp8_gemv): half the weight traffic
        self.fp8_decode = bool(fp8_decode) and self.hidden == 4096 and self.n_q * self.head_dim == 4096
        if self.fp8_decode:
            w8 = lambda n: weights[pre + n].to(dev).to(torch.float8_e4m3fn).view(torch.uint8)
            self.qkv_w8 = torch.cat([w8("q_proj"), w8("k_proj"), w8("v_proj")], dim=0).contiguous()
            self.o_w8 = w8("o_proj").contiguous()
        # rotary layout of the configuration: part of the head, neighbouring pairs
        self.rotary_dim = int(self.head_dim * (cfg.get("partial_rotary_factor") or 1.0))
        self.rope_interleaved = bool(cfg.get("rope_interleaved", False))
        self.plain_rope = self.rotary_dim == self.head_dim and not self.rope_interleaved
        self.norm = nn.RMSNorm(self.hidden, eps=cfg["rms_norm_eps"]).to(dev)
        nw = weights.get(pre + "input_layernorm")
        if nw is not None:
            self.norm.weight = nn.Parameter(nw.to(dev).to(torch.float16))
        else:
            self.norm.to(torch.float16)
        # one-token steps as three kernels: RMSNorm + q/k/v GEMV, RoPE + cache write +
        # attention (hc_attn_decode), o GEMV + residual
        self.fused_decode = (self.fp8_decode and self.head_dim == 128 and self.n_q % self.n_kv == 0
                             and self.n_q // self.n_kv <= 8 and self.plain_rope)
        self.status = N.new_status(dev)

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cache: KVCache,
                start: Optional[int], pos: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [B, T, H] fp16.  ``start`` = the host's cache length (positions
        start.. start + T - 1), or None for a graph-captured decode step whose
        position is the device scalar ``pos`` (T = 1): the step then attends
        over the whole cache capacity with a mask past ``pos``."""
        B, T, H = x.shape
        D, nq, nkv = self.head_dim, self.n_q, self.n_kv
        one = self.fp8_decode and B * T == 1
        qkv = self._gemv(self.qkv_w8, self.norm(x)) if one else F.linear(self.norm(x), self.qkv_weight)
        if not self.plain_rope:          # rotated in place, among the rows of the projection
            rows = qkv.view(B * T, nq + 2 * nkv, D)
            at = torch.arange(T, device=x.device).repeat(B)
            paged.rope(rows[:, :nq], rows[:, nq:nq + nkv], cos, sin, at, interleaved=self.rope_interleaved,
                       q_out=rows[:, :nq], k_out=rows[:, nq:nq + nkv])
        q = qkv[..., :nq * D].view(B, T, nq, D).transpose(1, 2)
        k = qkv[..., nq * D:(nq + nkv) * D].view(B, T, nkv, D).transpose(1, 2)
        v = qkv[..., (nq + nkv) * D:].view(B, T, nkv, D).transpose(1, 2)
        if self.plain_rope:
            q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
        kc, vc = cache.k[self.layer_idx], cache.v[self.layer_idx]
        if start is not None:
            kc[:, :, start:start + T] = k
            vc[:, :, start:start + T] = v
            n = start + T
            keys, vals = kc[:, :, :n], vc[:, :, :n]
            if T > 1:                    # causal over the new positions (engine.py:121)
                i = torch.arange(T, device=x.device)[:, None] + start
                j = torch.arange(n, device=x.device)[None, :]
                out = F.scaled_dot_product_attention(q, keys, vals, attn_mask=j <= i, enable_gqa=True)
            else:
                out = self._attend_one(q, keys, vals, None)
        else:
            kc.index_copy_(2, pos, k)
            vc.index_copy_(2, pos, v)
            j = torch.arange(cache.capacity, device=x.device)
            out = self._attend_one(q, kc, vc, (j <= pos).view(1, 1, 1, -1))
        out = out.transpose(1, 2).reshape(B, T, nq * D)
        return self._gemv(self.o_w8, out) if one else F.linear(out, self.o_weight)

    def decode_residual(self, x: torch.Tensor, cos_t: torch.Tensor, sin_t: torch.Tensor, cache: KVCache,
                        pos: torch.Tensor) -> torch.Tensor:
        """x + attention(x) for one token x [1, 1, H] fp16 at the device
        position ``pos`` (its k / v are written into the cache there), in three
        launches: hc_fp8_gemv_ex (input_layernorm + q/k/v), hc_attn_decode
        (RoPE, cache write, grouped-query attention), hc_fp8_gemv_ex (o +
        residual).  ``cos_t`` / ``sin_t`` are the whole rotary tables."""
        xv = x.reshape(-1).contiguous()
        s = N.stream_handle()
        qkv = torch.empty(self.qkv_w8.shape[0], dtype=torch.float16, device=x.device)
        N.check(N.lib.hc_fp8_gemv_ex(N.ptr(self.qkv_w8), None, self.qkv_w8.shape[0], self.hidden, N.ptr(xv),
                                     N.ptr(self.norm.weight.data), float(self.norm.eps), None, N.ptr(qkv), s),
                "hc_fp8_gemv_ex")
        att = torch.empty(self.n_q * self.head_dim, dtype=torch.float16, device=x.device)
        kc, vc = cache.k[self.layer_idx], cache.v[self.layer_idx]
        N.check(N.lib.hc_attn_decode(N.ptr(qkv), N.ptr(cos_t), N.ptr(sin_t), N.ptr(pos), N.ptr(kc), N.ptr(vc),
                                     cache.capacity, self.n_q, self.n_kv, self.head_dim, N.ptr(att),
                                     N.ptr(self.status), s), "hc_attn_decode")
        y = torch.empty(1, 1, self.hidden, dtype=torch.float16, device=x.device)
        N.check(N.lib.hc_fp8_gemv_ex(N.ptr(self.o_w8), None, self.hidden, self.hidden, N.ptr(att), None, 0.0,
                                     N.ptr(xv), N.ptr(y), s), "hc_fp8_gemv_ex")
        return y

    def step_paged(self, x: torch.Tensor, cos_t: torch.Tensor, sin_t: torch.Tensor, cache: "paged.PagedKVCache",
                   plan: "paged.PagePlan", max_q: int) -> torch.Tensor:
        """x + attention(x) for the rows x [rows, H] fp16 of a planned step of many
        requests: their keys and values go into the paged 8-bit cache and every
        row attends over its request's pages (hc_rope_append, hc_paged_attn).
        ``cos_t`` / ``sin_t`` are the whole rotary tables."""
        n, D, nq, nkv = x.shape[0], self.head_dim, self.n_q, self.n_kv
        if self.fp8_decode and n == 1:
            qkv = self._gemv(self.qkv_w8, self.norm(x))
        else:
            qkv = F.linear(self.norm(x), self.qkv_weight)
        rows = qkv.view(n, nq + 2 * nkv, D)
        q = cache.rope_append(self.layer_idx, rows[:, :nq], rows[:, nq:nq + nkv], rows[:, nq + nkv:], cos_t, sin_t,
                              plan, interleaved=self.rope_interleaved)
        out = cache.attend(self.layer_idx, q, plan, max_q=max_q).view(n, nq * D)
        y = self._gemv(self.o_w8, out).view(n, -1) if self.fp8_decode and n == 1 else F.linear(out, self.o_weight)
        return x + y

    def _attend_one(self, q, keys, vals, mask):
        """Softmax attention of one query position per head, the query heads
        grouped onto their key-value head (head h reads kv head h // group,
        the reference's repeat_interleave, engine.py:117-121): two batched
        products and an fp32 softmax, with no expanded copy of the cache."""
        B, nq, _, D = q.shape
        g = nq // self.n_kv
        qg = q.reshape(B, self.n_kv, g, D)
        s = torch.matmul(qg, keys.transpose(-1, -2)).float() * (1.0 / math.sqrt(D))     # [B, nkv, g, S]
        if mask is not None:
            s = s.masked_fill(~mask, float("-inf"))
        p = torch.softmax(s, dim=-1).to(vals.dtype)
        return torch.matmul(p, vals).reshape(B, nq, 1, D)

    @staticmethod
    def _gemv(w8: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """y [1, 1, rows] = W x for one fp16 row x [1, 1, 4096], W e4m3 bytes [rows, 4096]."""
        xv = x.reshape(-1).contiguous()
        y = torch.empty(1, 1, w8.shape[0], dtype=torch.float16, device=x.device)
        N.check(N.lib.hc_fp8_gemv(N.ptr(w8), None, w8.shape[0], w8.shape[1], N.ptr(xv), N.ptr(y),
                                  N.stream_handle()), "hc_fp8_gemv")
        return y


def _sample(logits: torch.Tensor, temperature: float, top_p: float) -> torch.Tensor:
    """Greedy at temperature 0, else nucleus sampling (engine.py:493-511):
    keep the most probable tokens whose preceding cumulative mass is below
    top_p, renormalise, draw one."""
    if temperature == 0.0:
        return logits.argmax(dim=-1)
    probs = torch.softmax(logits / temperature, dim=-1)
    p_sorted, order = torch.sort(probs, dim=-1, descending=True)
    before = torch.cumsum(p_sorted, dim=-1) - p_sorted
    p_sorted = torch.where(before < top_p, p_sorted, torch.zeros_like(p_sorted))
    p_sorted = p_sorted / p_sorted.sum(dim=-1, keepdim=True)
    pick = torch.multinomial(p_sorted, num_samples=1)
    return order.gather(-1, pick).squeeze(-1)


class DesdemonaEngine(nn.Module):
    """The reference's inference engine (engine.py:317-488) with the sparse
    FFN on the B200 kernels.

    ``DesdemonaEngine(split_dir, predictor_dir, device, n_threads,
    max_seq_len)`` reads the same split artefacts (split_config.json,
    hot_weights/shared.pt, hot_weights/layer_XXX_expert_000.pt,
    cold_weights.bin + cold_index.npy) and the same predictor files.  The cold
    store is uploaded to HBM once; every layer's fetch set is predicted on the
    device (layer l+1's on layer l's post-attention hidden state, the
    reference's lookahead, engine.py:421-438) and never crosses to the host.
    ``generate`` prefills eagerly and replays one captured CUDA graph per
    decode step.  ``n_threads`` is accepted for signature compatibility (no
    host thread pool is needed).  ``cold_source="pinned"`` keeps
    cold_weights.bin in pinned host memory instead -- the reference's tiering
    (README.md:3-9, splitter.py:307-330): each layer's predicted records cross
    the bus into one shared staging buffer right before the layer runs."""

    def __init__(self, split_dir: Optional[str] = None, predictor_dir: Optional[str] = None, device: str = "cuda",
                 n_threads: int = 8, max_seq_len: int = 8192, *, cold_source: str = "device",
                 _parts: Optional[dict] = None):
        super().__init__()
        import json
        self.device = torch.device(device)
        self.n_threads = n_threads
        if _parts is None:
            with open(Path(split_dir) / "split_config.json") as f:
                self.cfg = json.load(f)
            if self.cfg.get("num_experts", 1) != 1:
                raise ValueError(f"split_dir contains a {self.cfg['num_experts']}-expert MoE split; "
                                 "this engine serves dense split-dense artifacts only.")
            shared = torch.load(str(Path(split_dir) / "hot_weights" / "shared.pt"), map_location="cpu")
            self.predictor = None
            if predictor_dir and Path(predictor_dir).exists():
                self.predictor = PredictorRegistry(predictor_dir, device=str(self.device))
            self.cold_store = ColdWeightStore(str(Path(split_dir) / "cold_weights.bin"),
                                              str(Path(split_dir) / "cold_index.npy"), self.cfg, device=self.device,
                                              source=cold_source)
            hots = [str(Path(split_dir) / "hot_weights")] * self.cfg["num_layers"]
        else:
            # in-memory artefacts (synthetic models): cfg, shared, cold_store, hot [HotNeurons], predictor
            self.cfg = _parts["cfg"]
            shared = _parts["shared"]
            self.predictor = _parts.get("predictor")
            self.cold_store = _parts["cold_store"]
            hots = _parts["hot"]
        cfg = self.cfg
        self.num_layers = cfg["num_layers"]
        H, vocab = cfg["hidden_dim"], cfg["vocab_size"]
        self.head_dim = H // cfg["num_attention_heads"]
        self.max_seq = min(max_seq_len, cfg.get("max_position_embeddings", max_seq_len))
        dev = self.device
        self.embed_tokens = nn.Embedding(vocab, H).to(dev)
        self.embed_tokens.weight = nn.Parameter(shared["embed_tokens"].to(dev).to(torch.float16), requires_grad=False)
        self.lm_head_weight = shared["lm_head"].to(dev).to(torch.float16)
        self.final_norm = nn.RMSNorm(H, eps=cfg["rms_norm_eps"]).to(dev)
        if "final_norm" in shared:
            self.final_norm.weight = nn.Parameter(shared["final_norm"].to(dev).to(torch.float16), requires_grad=False)
        else:
            self.final_norm.to(torch.float16)
        self.attention_layers = nn.ModuleList([GroupedQueryAttention(li, shared, cfg, dev)
                                               for li in range(self.num_layers)])
        self.ffn_layers = nn.ModuleList([
            SparseFFNLayer(li, hots[li], self.cold_store, self.predictor, cfg, dev, None,
                           ffn_norm_weight=shared.get(f"layer_{li:03d}.post_attention_layernorm"))
            for li in range(self.num_layers)])
        del shared
        self.requires_grad_(False)
        rotary, scaling = self.attention_layers[0].rotary_dim, _rope_scaling(cfg)
        if scaling or rotary != self.head_dim:
            self.cos_cache, self.sin_cache = paged.rope_tables(self.max_seq, rotary, cfg["rope_theta"], scaling, dev)
        else:
            self.cos_cache, self.sin_cache = build_rope_cache(self.max_seq, self.head_dim, cfg["rope_theta"], dev)
        W = (cfg["intermediate_dim"] + 31) // 32
        self._words = torch.zeros(self.num_layers, 1, W, dtype=torch.int32, device=dev)   # fetch sets in flight
        self.fused_lookahead = True
        self.fused_attention = True     # one-token steps: the three fused attention kernels
        self._graph = None
        self._graph_cache = None

    @classmethod
    def from_parts(cls, cfg: dict, shared: dict, cold_store: ColdWeightStore, hot: Sequence[HotNeurons],
                   predictor: Optional[PredictorRegistry] = None, device="cuda", max_seq_len: int = 8192):
        """An engine over in-memory artefacts (the split's contents without
        the files): ``shared`` has shared.pt's keys, ``hot`` one HotNeurons per
        layer."""
        return cls(None, None, device, max_seq_len=max_seq_len,
                   _parts={"cfg": cfg, "shared": shared, "cold_store": cold_store, "hot": list(hot),
                           "predictor": predictor})

    def new_cache(self, batch: int = 1, capacity: Optional[int] = None) -> KVCache:
        cap = min(capacity or self.max_seq, self.max_seq)
        return KVCache(self.num_layers, batch, self.cfg["num_key_value_heads"], cap, self.head_dim, self.device)

    def _layers(self, x: torch.Tensor, cos, sin, cache: KVCache, start: Optional[int], pos=None):
        """Attention + sparse FFN of every layer, with the fetch-set lookahead."""
        f = self.ffn_layers
        words = self._words
        one = x.shape[0] * x.shape[1] == 1 and self.fused_lookahead
        f[0].submit_cold_fetch(x, out=words[0])             # layer 0's set, on the embedding (engine.py:422)
        fused = x.shape[0] * x.shape[1] == 1 and self.fused_attention
        dpos = pos if pos is not None else cache.pos      # eager one-token steps: cache.pos == start
        for li in range(self.num_layers):
            att = self.attention_layers[li]
            if fused and att.fused_decode:
                x = att.decode_residual(x, self.cos_cache, self.sin_cache, cache, dpos)
            else:
                x = x + att(x, cos, sin, cache, start, pos)
            if li + 1 < self.num_layers:
                if one:
                    # one token: this layer's kernel also predicts the next layer's set
                    # from this post-attention state (engine.py:430-438)
                    x = f[li].forward_lookahead(x, words[li], f[li + 1], words[li + 1])
                    continue
                f[li + 1].submit_cold_fetch(x, out=words[li + 1])     # next layer's set on this state
            x = f[li](x, words[li])
        return x

    @torch.inference_mode()
    def forward(self, input_ids: torch.Tensor, kv_caches: Optional[KVCache] = None):
        """(logits [B, T, vocab], cache) for input_ids [B, T], continuing the
        cache's positions (engine.py:406-442).  A new cache holds up to
        max_seq_len positions."""
        B, T = input_ids.shape
        cache = kv_caches if kv_caches is not None else self.new_cache(B)
        start = cache.length
        if start + T > cache.capacity:
            raise ValueError(f"sequence of {start + T} positions exceeds the cache capacity {cache.capacity}")
        x = self.embed_tokens(input_ids.to(self.device))
        x = self._layers(x, self.cos_cache[start:start + T], self.sin_cache[start:start + T], cache, start)
        cache.length = start + T
        cache.pos.fill_(cache.length)
        logits = F.linear(self.final_norm(x), self.lm_head_weight)
        return logits, cache

    # -- decode step in one CUDA graph -------------------------------------
    def _decode_body(self, cache: KVCache):
        pos = cache.pos
        x = self.embed_tokens(self._tok.view(1, 1))
        cos = self.cos_cache.index_select(0, pos)
        sin = self.sin_cache.index_select(0, pos)
        x = self._layers(x, cos, sin, cache, None, pos)
        self._logits.copy_(F.linear(self.final_norm(x), self.lm_head_weight)[:, -1])
        pos.add_(1)

    def _capture(self, cache: KVCache):
        self._tok = torch.zeros(1, dtype=torch.int64, device=self.device)
        self._logits = torch.zeros(1, self.cfg["vocab_size"], dtype=torch.float16, device=self.device)
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream())
        saved = (cache.k.clone(), cache.v.clone(), cache.pos.clone())
        with torch.cuda.stream(s):
            self._decode_body(cache)                # warm-up outside capture (allocations, workspaces)
            torch.cuda.current_stream().synchronize()
            cache.k.copy_(saved[0])
            cache.v.copy_(saved[1])
            cache.pos.copy_(saved[2])
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                self._decode_body(cache)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        cache.k.copy_(saved[0])
        cache.v.copy_(saved[1])
        cache.pos.copy_(saved[2])
        self._graph, self._graph_cache = g, cache

    @torch.inference_mode()
    def decode_step(self, token: torch.Tensor, cache: KVCache) -> torch.Tensor:
        """Logits [1, vocab] of one new token (device int64 scalar) at the
        cache's next position, by one replay of the captured step."""
        if self._graph is None or self._graph_cache is not cache:
            self._capture(cache)
        self._tok.copy_(token.view(1))
        self._graph.replay()
        cache.length += 1
        return self._logits

    @torch.inference_mode()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int = 200, temperature: float = 0.7,
                 top_p: float = 0.9, eos_token_id=None, use_graph: bool = True) -> list[int]:
        """Generated token ids, prompt excluded, with the reference's stopping
        rule (engine.py:444-484): the first sampled EOS is kept and ends the
        sequence.  Tokens stay on the device until the end (one host read)."""
        if eos_token_id is None:
            eos = set()
        elif isinstance(eos_token_id, int):
            eos = {eos_token_id}
        else:
            eos = set(eos_token_id)
        if input_ids.dim() == 1:
            input_ids = input_ids.view(1, -1)
        if input_ids.shape[0] != 1:
            raise ValueError("generate decodes one sequence (batch 1), as the reference does")
        T = input_ids.shape[1]
        n_new = max(int(max_new_tokens), 1)
        cache = self.new_cache(1, T + n_new)
        logits, cache = self.forward(input_ids, cache)
        out = torch.empty(n_new, dtype=torch.int64, device=self.device)
        tok = _sample(logits[:, -1, :], temperature, top_p).view(1)
        out[0] = tok[0]
        count = 1
        while count < n_new:
            # the host looks at the tokens (for an EOS) only every 16 steps
            if eos and count % 16 == 0 and any(t in eos for t in out[:count].tolist()):
                break
            if use_graph:
                lg = self.decode_step(tok, cache)
            else:
                lg, cache = self.forward(tok.view(1, 1), cache)
                lg = lg[:, -1, :]
            tok = _sample(lg, temperature, top_p).view(1)
            out[count] = tok[0]
            count += 1
        ids = out[:count].tolist()
        if eos:
            for i, t in enumerate(ids):
                if t in eos:
                    return ids[:i + 1]
        return ids

    # -- many requests over the paged 8-bit cache ----------------------------
    def new_paged_cache(self, max_requests: int, n_pages: Optional[int] = None, page_size: int = 64,
                        max_len: Optional[int] = None) -> "paged.PagedKVCache":
        """A cache for up to ``max_requests`` requests of up to ``max_len``
        positions (default: the engine's limit) sharing ``n_pages`` pages
        (default: enough for all of them at full length)."""
        length = min(max_len or self.max_seq, self.max_seq)
        n = n_pages if n_pages is not None else max_requests * -(-length // page_size)
        return paged.PagedKVCache(self.num_layers, self.cfg["num_key_value_heads"], self.head_dim, n,
                                  page_size=page_size, max_requests=max_requests, max_len=length, device=self.device)

    @torch.inference_mode()
    def forward_paged(self, tokens: torch.Tensor, q_lens: Sequence[int], cache: "paged.PagedKVCache") -> torch.Tensor:
        """Logits [requests with new tokens, vocab] of every request's last row.

        ``q_lens[r]`` new tokens of request r follow its cached ones; ``tokens``
        [sum(q_lens)] holds them request after request.  All rows share one
        fetch set per layer, as a batch does in the reference (engine.py:277).
        A step that does not fit (too few free pages, a request past the
        cache's ``max_len``) raises ValueError and leaves the cache as it was."""
        q_lens = [int(n) for n in q_lens]
        rows = sum(q_lens)
        if len(q_lens) > cache.max_requests or tokens.dim() != 1 or tokens.shape[0] != rows or rows == 0 or \
                min(q_lens) < 0:
            raise ValueError("tokens must hold sum(q_lens) > 0 ids of at most max_requests requests")
        device_lens = torch.zeros(cache.max_requests, dtype=torch.int32)
        device_lens[:len(q_lens)] = torch.tensor(q_lens, dtype=torch.int32)
        # The host waits for the plan's outcome while the first fetch set is predicted: no layer runs on rows that
        # were not placed.
        seen = torch.empty(2, dtype=torch.int32, pin_memory=True)        # status before the plan, rows placed
        seen[:1].copy_(cache.status, non_blocking=True)
        plan = cache.plan(device_lens.to(self.device), rows)
        seen[1:].copy_(plan.cu_q[-1:], non_blocking=True)
        planned = torch.cuda.Event()
        planned.record(torch.cuda.current_stream(self.device))
        x = self.embed_tokens(tokens.to(self.device))
        f, words, max_q = self.ffn_layers, self._words, max(q_lens)
        f[0].submit_cold_fetch(x.view(rows, 1, -1), out=words[0])
        planned.synchronize()
        if int(seen[1]) != rows:         # nothing was taken, every row is padding
            cache.status.fill_(int(seen[0]))
            raise ValueError(f"the step's {rows} tokens do not fit the cache: {int(cache.n_free)} pages are free, "
                             f"requests hold up to {cache.max_len} positions")
        for li, att in enumerate(self.attention_layers):
            x = att.step_paged(x, self.cos_cache, self.sin_cache, cache, plan, max_q)
            if li + 1 < self.num_layers:
                f[li + 1].submit_cold_fetch(x.view(rows, 1, -1), out=words[li + 1])
            x = f[li](x.view(rows, 1, -1), words[li]).view(rows, -1)
        cache.commit(plan)
        last = [e - 1 for e, n in zip(np.cumsum(q_lens).tolist(), q_lens) if n]
        x = x[torch.tensor(last, device=self.device)]
        return F.linear(self.final_norm(x), self.lm_head_weight)

    @torch.inference_mode()
    def generate_batch(self, prompts: Sequence[torch.Tensor], max_new_tokens: int = 200, temperature: float = 0.7,
                       top_p: float = 0.9, eos_token_id=None, page_size: int = 64) -> list[list[int]]:
        """generate() for several prompts at once over one paged cache: the
        generated ids of each, prompt excluded, with generate()'s stopping rule.
        Finished requests give their pages back and leave the batch (the host
        looks at the tokens every 16 steps)."""
        eos = set() if eos_token_id is None else {eos_token_id} if isinstance(eos_token_id, int) else set(eos_token_id)
        prompts = [p.reshape(-1) for p in prompts]
        n_new = max(int(max_new_tokens), 1)
        lens = [p.shape[0] for p in prompts]
        if not prompts or min(lens) == 0 or max(lens) + n_new - 1 > self.max_seq:     # the last token is not cached
            raise ValueError(f"prompts must be non-empty and fit {self.max_seq} positions with the new tokens")
        pages = sum(-(-(n + n_new - 1) // page_size) for n in lens)
        cache = self.new_paged_cache(len(prompts), pages, page_size, max(lens) + n_new - 1)
        out = torch.empty(len(prompts), n_new, dtype=torch.int64, device=self.device)
        ids = [[] for _ in prompts]
        live = list(range(len(prompts)))
        logits = self.forward_paged(torch.cat([p.to(self.device) for p in prompts]), lens, cache)
        for step in range(n_new):
            out[live, step] = _sample(logits, temperature, top_p).view(-1)
            if step + 1 == n_new:
                break
            if eos and step % 16 == 15:
                made = out[:, :step + 1].tolist()
                ended = [r for r in live if any(t in eos for t in made[r])]
                for r in ended:
                    ids[r] = made[r]
                if ended:
                    done = torch.zeros(len(prompts), dtype=torch.bool)
                    done[ended] = True
                    cache.release(done.to(self.device))
                    live = [r for r in live if r not in ended]
                if not live:
                    break
            logits = self.forward_paged(out[live, step], [int(r in live) for r in range(len(prompts))], cache)
        cache.check()
        made = out.tolist()
        for r in range(len(prompts)):
            row = ids[r] or made[r]
            stop = next((i for i, t in enumerate(row) if t in eos), len(row) - 1)
            ids[r] = row[:stop + 1]
        return ids

    def check(self):
        for f in self.ffn_layers:
            f.check()
        for a in self.attention_layers:
            N.read_status(a.status, "hc_attn_decode")

    def close(self):
        self._graph = None
        self.cold_store.close()
