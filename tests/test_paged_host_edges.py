"""Host side of the paged serving path at the edges of what it takes (no GPU)."""
import warnings

import pytest


def test_stock_rope_scaling_entries():
    """What model configurations hold builds an engine: an original length that is left out is the configuration's
    own, a kind that is not known is left aside and said so."""
    import engine
    import paged
    base = {"max_position_embeddings": 4096, "rope_theta": 10000.0}

    def read(scaling):
        return engine._rope_scaling({**base, "rope_scaling": scaling})
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for none in (None, {}, {"rope_type": "default"}, {"type": "default", "factor": 2.0}, {"rope_type": None}):
            assert read(none) is None
        assert engine._rope_scaling(base) is None
        for stock in ({"type": "dynamic", "factor": 2.0}, {"type": "yarn", "factor": 4.0},
                      {"rope_type": "linear", "type": "linear", "factor": 2.0},
                      {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0}):
            got = read(stock)
            assert got["original_max_position_embeddings"] == 4096
            freq, _ = paged.rope_frequencies(128, 10000.0, got, 8192)
            apart, _ = paged.rope_frequencies(128, 10000.0, {**stock, "original_max_position_embeddings": 4096}, 8192)
            plain, _ = paged.rope_frequencies(128, 10000.0)
            assert (freq == apart).all() and not (freq == plain).all()
        given = read({"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024})
        assert given["original_max_position_embeddings"] == 1024
    for odd in ({"type": "longrope", "long_factor": [1.0], "short_factor": [1.0]}, {"rope_type": "yarn"},
                {"type": "linear", "factor": None}, {"rope_type": "llama3", "factor": 8.0}):
        with pytest.warns(UserWarning, match="not scaled"):
            assert read(odd) is None


def test_split_config_carries_the_rotary_layout():
    """A model's scaling, partial head and pair layout reach the engine; a plain one is written as before."""
    from types import SimpleNamespace as C

    import engine
    import splitter
    llama = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 8192}
    for plain in (C(rope_theta=500000.0), C(rope_theta=500000.0, rope_scaling=None),
                  C(rope_parameters={"rope_theta": 500000.0, "rope_type": "default"}),
                  C(rope_theta=500000.0, partial_rotary_factor=1.0, rope_interleaved=False)):
        assert splitter._rotary_config(plain) == {"rope_theta": 500000.0}
    assert splitter._rotary_config(C()) == {"rope_theta": 10000.0}
    got = splitter._rotary_config(C(rope_theta=500000.0, rope_scaling=llama))
    assert got == {"rope_theta": 500000.0, "rope_scaling": llama}
    got = splitter._rotary_config(C(rope_parameters={**llama, "rope_theta": 500000.0, "partial_rotary_factor": 0.5}))
    assert got["rope_theta"] == 500000.0 and got["partial_rotary_factor"] == 0.5
    assert engine._rope_scaling({**got, "max_position_embeddings": 131072})["factor"] == 8.0
    got = splitter._rotary_config(C(rope_theta=1e4, partial_rotary_factor=0.25, rope_interleaved=True))
    assert got == {"rope_theta": 1e4, "partial_rotary_factor": 0.25, "rope_interleaved": True}


def test_row_counts_past_the_index_range_are_refused():
    """Row indices are 32-bit and step past the last row by a grid's width."""
    import ctypes

    import hc_native as N
    from test_paged_host import FAKE, _pages, _rope
    for rows, pages in (((1 << 30) + 1, {}), ((1 << 31) - 1, {}), ((1 << 31) - 32, {"head_dim": 64})):
        assert N.lib.hc_page_plan(FAKE, FAKE, 1, FAKE, 8, 8, FAKE, 4, FAKE, 16, rows, FAKE, FAKE, FAKE, FAKE, None,
                                  None) == N.HC_ERR_UNSUPPORTED
        c = ctypes.byref(_pages(N, **pages))
        a = _rope(N, n_rows=rows, head_dim=pages.get("head_dim", 128), rotary_dim=64)
        assert N.lib.hc_rope(ctypes.byref(a), None, None) == N.HC_ERR_UNSUPPORTED
        assert N.lib.hc_kv_append(c, FAKE, 0, 128, FAKE, 0, 128, FAKE, rows, N.HC_F16, None,
                                  None) == N.HC_ERR_UNSUPPORTED
        assert N.lib.hc_rope_append(ctypes.byref(a), c, FAKE, 0, 128, FAKE, None, None) == N.HC_ERR_UNSUPPORTED


def test_misaligned_addresses_are_refused():
    """Every pointer that a kernel reads or writes through, by the size of what it points to."""
    import ctypes

    import hc_native as N
    from test_paged_host import FAKE, _attn, _pages, _rope
    plan = dict(starts=4, q=4, tables=4, free=4, n_free=4, cu=4, kv=4, pos=8, slots=8, status=4)
    for name, size in plan.items():
        p = {n: FAKE + (size // 2 if n == name else 0) for n in plan}
        assert N.lib.hc_page_plan(p["starts"], p["q"], 1, p["tables"], 8, 8, p["free"], 4, p["n_free"], 16, 4, p["cu"],
                                  p["kv"], p["pos"], p["slots"], p["status"], None) == N.HC_ERR_ARG, name
    for bad in ({"tables"}, {"free"}, {"n_free"}, {"status"}):
        p = {n: FAKE + 2 * (n in bad) for n in ("tables", "free", "n_free", "status")}
        assert N.lib.hc_page_release(FAKE, 1, p["tables"], 8, 8, p["free"], 4, p["n_free"], p["status"],
                                     None) == N.HC_ERR_ARG, bad
    c = ctypes.byref(_pages(N))
    for kw, status in (({"cu_q": FAKE + 2}, None), ({"kv_lens": FAKE + 1}, None), ({"lse": FAKE + 2}, None),
                       ({"tables": FAKE + 2}, None), ({}, FAKE + 2)):
        assert N.lib.hc_paged_attn(ctypes.byref(_attn(N, **kw)), c, FAKE, 1 << 30, status, None) == N.HC_ERR_ARG, kw
    a = ctypes.byref(_rope(N))
    assert N.lib.hc_rope(a, FAKE + 2, None) == N.HC_ERR_ARG
    assert N.lib.hc_kv_append(c, FAKE, 256, 128, FAKE, 256, 128, FAKE, 1, N.HC_F16, FAKE + 1, None) == N.HC_ERR_ARG
    assert N.lib.hc_rope_append(a, c, FAKE, 256, 128, FAKE, FAKE + 2, None) == N.HC_ERR_ARG
