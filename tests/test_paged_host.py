"""The paged-cache operators' host side: refusals, struct layouts, tables (no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

FAKE = 1 << 20                    # an aligned address that no refused call dereferences


@pytest.fixture(scope="module")
def N():
    import hc_native
    return hc_native


def _pages(N, **kw):
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, n_pages=4, n_kv_heads=2, page_size=64, head_dim=128)
    d.update(kw)
    return N.KVPages(*[d[n] for n, _ in N.KVPages._fields_])


def _rope(N, **kw):
    d = dict(q=FAKE, k=FAKE, q_out=FAKE, k_out=FAKE, q_row=512, q_head=128, k_row=256, k_head=128, q_out_row=512,
             q_out_head=128, k_out_row=256, k_out_head=128, cos_t=FAKE, sin_t=FAKE, table_rows=8, positions=FAKE,
             n_rows=1, n_q_heads=4, n_kv_heads=2, head_dim=128, rotary_dim=128, interleaved=0, dtype=N.HC_F16)
    d.update(kw)
    return N.RopeArgs(*[d[n] for n, _ in N.RopeArgs._fields_])


def _attn(N, **kw):
    d = dict(q=FAKE, out=FAKE, lse=None, q_row=512, q_head=128, out_row=512, out_head=128, tables=FAKE,
             table_stride=8, table_width=8, cu_q=FAKE, kv_lens=FAKE, n_requests=1, n_rows=1, max_q=1, n_q_heads=4,
             scale=0.1, dtype=N.HC_F16)
    d.update(kw)
    return N.AttnArgs(*[d[n] for n, _ in N.AttnArgs._fields_])


def test_struct_layouts_match_the_header(N):
    assert ctypes.sizeof(N.KVPages) == 4 * 8 + 4 * 4
    assert ctypes.sizeof(N.RopeArgs) == 4 * 8 + 8 * 8 + 2 * 8 + 8 + 8 + 7 * 4 + 4
    assert N.RopeArgs.positions.offset == 120 and N.RopeArgs.dtype.offset == 152
    assert ctypes.sizeof(N.AttnArgs) == 3 * 8 + 4 * 8 + 8 + 8 + 8 + 2 * 8 + 6 * 4
    assert N.AttnArgs.cu_q.offset == 80 and N.AttnArgs.scale.offset == 112


def test_page_plan_and_release_refusals(N):
    def plan(**kw):
        d = dict(starts=FAKE, q=FAKE, n=1, tables=FAKE, stride=8, width=8, free=FAKE, n_pages=4, n_free=FAKE, page=16,
                 rows=4, cu=FAKE, kv=FAKE, pos=FAKE, slots=FAKE)
        d.update(kw)
        return N.lib.hc_page_plan(d["starts"], d["q"], d["n"], d["tables"], d["stride"], d["width"], d["free"],
                                  d["n_pages"], d["n_free"], d["page"], d["rows"], d["cu"], d["kv"], d["pos"],
                                  d["slots"], None, None)
    for bad in ({"starts": None}, {"q": None}, {"tables": None}, {"free": None}, {"n_free": None}, {"cu": None},
                {"kv": None}, {"pos": None}, {"slots": None}, {"n": 0}, {"n": -1}, {"width": 0}, {"stride": 7},
                {"n_pages": 0}, {"page": 0}, {"rows": -1}, {"width": 1 << 28, "stride": 1 << 28}):
        assert plan(**bad) == N.HC_ERR_ARG, bad
    assert plan(n=2049) == N.HC_ERR_UNSUPPORTED

    def release(done=FAKE, n=1, tables=FAKE, stride=8, width=8, free=FAKE, n_pages=4, n_free=FAKE):
        return N.lib.hc_page_release(done, n, tables, stride, width, free, n_pages, n_free, None, None)
    for bad in ({"done": None}, {"n": 0}, {"tables": None}, {"stride": 4}, {"width": 0}, {"free": None},
                {"n_pages": 0}, {"n_free": None}):
        assert release(**bad) == N.HC_ERR_ARG, bad
    assert release(n=2049) == N.HC_ERR_UNSUPPORTED


def test_rope_and_append_refusals(N):
    def rope(**kw):
        return N.lib.hc_rope(ctypes.byref(_rope(N, **kw)), None, None)
    for bad in ({"q": None}, {"k": None}, {"q_out": None}, {"k_out": None}, {"cos_t": None}, {"sin_t": None},
                {"positions": None}, {"n_rows": -1}, {"n_q_heads": 0}, {"n_kv_heads": 0}, {"head_dim": 0},
                {"rotary_dim": 0}, {"rotary_dim": 63}, {"rotary_dim": 130}, {"table_rows": 0}, {"dtype": N.HC_F32},
                {"interleaved": 2}, {"q": FAKE + 1}, {"cos_t": FAKE + 2}, {"positions": FAKE + 4}):
        assert rope(**bad) == N.HC_ERR_ARG, bad
    assert N.lib.hc_rope(None, None, None) == N.HC_ERR_ARG
    assert rope(n_rows=0) == N.HC_OK                      # nothing to do

    def append(cache=None, k=FAKE, v=FAKE, slots=FAKE, rows=1, dtype=N.HC_F16):
        c = _pages(N, **(cache or {}))
        return N.lib.hc_kv_append(ctypes.byref(c), k, 256, 128, v, 256, 128, slots, rows, dtype, None, None)
    for bad in ({"k": None}, {"v": None}, {"slots": None}, {"rows": -1}, {"dtype": N.HC_F32}, {"k": FAKE + 1},
                {"cache": {"k": None}}, {"cache": {"v_scale": None}}, {"cache": {"n_pages": 0}},
                {"cache": {"n_kv_heads": 0}}, {"cache": {"k": FAKE + 8}}):
        assert append(**bad) == N.HC_ERR_ARG, bad
    for bad in ({"cache": {"page_size": 48}}, {"cache": {"page_size": 8}}, {"cache": {"head_dim": 96}}):
        assert append(**bad) == N.HC_ERR_UNSUPPORTED, bad
    assert append(rows=0) == N.HC_OK

    def both(cache=None, v=FAKE, slots=FAKE, **kw):
        c = _pages(N, **(cache or {}))
        return N.lib.hc_rope_append(ctypes.byref(_rope(N, **kw)), ctypes.byref(c), v, 256, 128, slots, None, None)
    assert both(n_kv_heads=4) == N.HC_ERR_ARG              # not the cache's heads
    assert both(head_dim=64, rotary_dim=64) == N.HC_ERR_ARG
    assert both(v=None) == N.HC_ERR_ARG and both(slots=None) == N.HC_ERR_ARG
    assert both(k_out=None, n_rows=0) == N.HC_OK           # the keys go into the cache


def test_paged_attention_refusals(N):
    def attn(cache=None, ws=FAKE, size=1 << 30, **kw):
        c = _pages(N, **(cache or {}))
        return N.lib.hc_paged_attn(ctypes.byref(_attn(N, **kw)), ctypes.byref(c), ws, size, None, None)
    for bad in ({"q": None}, {"out": None}, {"tables": None}, {"cu_q": None}, {"kv_lens": None}, {"n_requests": 0},
                {"n_rows": -1}, {"max_q": -1}, {"n_q_heads": 3}, {"n_q_heads": 0}, {"table_width": 0},
                {"table_stride": 4}, {"dtype": N.HC_F32}, {"q": FAKE + 1}, {"ws": None}, {"ws": FAKE + 8},
                {"size": 64}, {"cache": {"k": FAKE + 4}}, {"cache": {"n_pages": 0}}, {"cache": {"k_scale": None}}):
        assert attn(**bad) == N.HC_ERR_ARG, bad
    for bad in ({"cache": {"page_size": 24}}, {"cache": {"head_dim": 256}}, {"n_q_heads": 34}, {"n_requests": 2049}):
        assert attn(**bad) == N.HC_ERR_UNSUPPORTED, bad
    assert attn(n_rows=0, ws=None) == N.HC_OK
    assert N.lib.hc_paged_attn_workspace_bytes(0, 1, 4, 2, 128) == -1
    assert N.lib.hc_paged_attn_workspace_bytes(1, 1, 4, 2, 96) == -1
    assert N.lib.hc_paged_attn_workspace_bytes(1, 1, 4, 2, 128) > 0


def test_python_refusals():
    import paged
    with pytest.raises(RuntimeError):                      # no CPU fallback
        paged.page_plan(*[torch.zeros(1, dtype=torch.int32)] * 2, torch.zeros(1, 4, dtype=torch.int32),
                        torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 16, 4)
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        paged.rope(x, x, torch.zeros(4, 32), torch.zeros(4, 32), torch.zeros(1, dtype=torch.int64))
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.uint8)
    with pytest.raises(RuntimeError):
        paged.kv_append(x, x, torch.zeros(1, dtype=torch.int64), pages, pages, torch.zeros(2, 2), torch.zeros(2, 2))
    with pytest.raises(ValueError):
        paged.rope_frequencies(63, 10000.0)
    with pytest.raises(ValueError):
        paged.rope_frequencies(64, 10000.0, {"rope_type": "unheard of", "factor": 2.0,
                                             "original_max_position_embeddings": 64})
    with pytest.raises(ValueError):
        paged.rope_frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 2.0})


def test_rope_frequencies_by_kind():
    import paged
    d, theta = 128, 500000.0
    plain = np.array([theta ** (-2 * i / d) for i in range(d // 2)])
    f, a = paged.rope_frequencies(d, theta)
    assert a == 1.0 and np.allclose(f.numpy(), plain, rtol=1e-14)
    f, a = paged.rope_frequencies(d, theta, {"type": "linear", "factor": 4.0})
    assert a == 1.0 and np.allclose(f.numpy(), plain / 4, rtol=1e-14)
    # the base is raised only beyond the original length
    dyn = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 1000}
    assert np.allclose(paged.rope_frequencies(d, theta, dyn, 500)[0].numpy(), plain, rtol=1e-12)
    base = theta * (2 * 4000 / 1000 - 1) ** (d / (d - 2))
    assert np.allclose(paged.rope_frequencies(d, theta, dyn, 4000)[0].numpy(),
                       [base ** (-2 * i / d) for i in range(d // 2)], rtol=1e-12)
    # by wavelength: short ones kept, long ones divided, a ramp between
    ll = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    f = paged.rope_frequencies(d, theta, ll)[0].numpy()
    for i, w in enumerate(2 * math.pi / plain):
        if w < 8192 / 4:
            want = plain[i]
        elif w > 8192:
            want = plain[i] / 8
        else:
            s = (8192 / w - 1) / 3
            want = (1 - s) * plain[i] / 8 + s * plain[i]
        assert abs(f[i] - want) < 1e-13 * want
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    f, a = paged.rope_frequencies(d, theta, yarn)
    turns = 4096 * plain / (2 * math.pi)
    assert abs(a - (0.1 * math.log(4) + 1)) < 1e-12
    f = f.numpy()
    assert np.allclose(f[turns > 40], plain[turns > 40]) and np.allclose(f[turns < 0.5], plain[turns < 0.5] / 4)
    assert (np.diff(f / plain) <= 1e-15).all()
    # the tables' angles are 64-bit ones: the fastest pair at a far position
    cos, sin = paged.rope_tables(131072, 8, theta)
    assert cos.dtype == torch.float32
    assert abs(float(cos[131071, 0]) - math.cos(131071.0)) < 2 ** -24
    assert abs(float(sin[131071, 0]) - math.sin(131071.0)) < 2 ** -24


def test_oracle_e4m3_against_torch():
    from oracle import paged_oracle as O
    every = torch.arange(256, dtype=torch.uint8)
    ours, theirs = O.e4m3_decode(every.numpy()), every.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ours, theirs, equal_nan=True)
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(0)) * s for s in (0.003, 0.1, 5.0, 120.0)])
    mid = torch.tensor((O.POSITIVE[1:] + O.POSITIVE[:-1]) / 2, dtype=torch.float32)     # ties
    x = torch.cat([x.clamp(-448, 448), mid, -mid])
    assert np.array_equal(O.e4m3_encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert O.page_scale(448.0) == 1.0 and O.page_scale(448.0001) == 2.0 and O.page_scale(0.0) == 2.0 ** -40


def test_yarn_attention_factor_and_ramp():
    import paged
    y = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "mscale": 1.0}
    t = 0.1 * math.log(40) + 1
    assert abs(paged.rope_frequencies(64, 1e4, y)[1] - t) < 1e-12
    y["mscale_all_dim"] = 0.707
    assert abs(paged.rope_frequencies(64, 1e4, y)[1] - t / (0.0707 * math.log(40) + 1)) < 1e-12
    assert paged.rope_frequencies(64, 1e4, dict(y, mscale_all_dim=1.0))[1] == 1.0
    assert paged.rope_frequencies(64, 1e4, dict(y, attention_factor=1.5))[1] == 1.5
    # without rounding of the ramp's ends: the pair that turns 32 times is kept, the one that turns once divided
    f, _ = paged.rope_frequencies(64, 1e4, dict(y, truncate=False))
    freq = np.array([1e4 ** (-i / 32) for i in range(32)])
    end = [32 * math.log(4096 / (n * 2 * math.pi)) / math.log(1e4) for n in (32, 1)]
    ramp = np.clip((np.arange(32) - end[0]) / (end[1] - end[0]), 0, 1)
    assert np.allclose(f.numpy(), freq * (1 - ramp) + freq / 40 * ramp, rtol=1e-12)


def test_paged_refusals_of_scales_and_sizes(N):
    import paged
    c = _pages(N)
    for scale in (float("nan"), float("inf"), -float("inf")):
        assert N.lib.hc_paged_attn(ctypes.byref(_attn(N, scale=scale)), ctypes.byref(c), FAKE, 1 << 30, None,
                                   None) == N.HC_ERR_ARG
    assert N.lib.hc_paged_attn(ctypes.byref(_attn(N, n_rows=(1 << 29) + 1)), ctypes.byref(c), FAKE, 1 << 30, None,
                               None) == N.HC_ERR_UNSUPPORTED
    with pytest.raises(ValueError):
        paged.rope_frequencies(2, 1e4, {"rope_type": "dynamic", "factor": 2.0,
                                        "original_max_position_embeddings": 64}, 128)
    for bad in ({"page_size": 24}, {"max_requests": 2049}, {"max_len": 0}):
        with pytest.raises(ValueError):
            paged.PagedKVCache(1, 1, 64, 4, device="cpu", **bad)
    with pytest.raises(ValueError):
        paged.PagedKVCache(1, 1, 96, 4, device="cpu")
