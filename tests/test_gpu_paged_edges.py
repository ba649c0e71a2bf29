"""The paged-cache operators where values, lengths or tables are at the edge of what they take.

Oracle and helpers are those of test_gpu_paged.py; tolerances are derived at each test.
"""
import math

import numpy as np
import pytest
import torch

import test_gpu_paged as T
from test_gpu_paged import (HALF_STEP, N, P, _angles, _cache, _check_append, _check_attention, _filled, _gen, _i32,
                            _i64, _np, _step)

pytestmark = pytest.mark.gpu


# ─── attention: weights far below the largest ─────────────────────────────────
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,nats", [(1, 128, 17.0), (1, 64, 17.6), (3, 128, 17.6), (1, 128, 20.0),
                                           (40, 128, 17.0), (40, 64, 17.6), (40, 128, 20.0)])
def test_paged_attention_behind_a_sink(P, rows, dim, nats, dtype):
    """One key of value 0 takes nearly all of the weight; 20,000 equal keys of value 1 share the rest.

    With the sink at exponent d = nats log2(e), a weight beside it is rounded by max(2^-11, 2^(d - 36)) of itself
    (weights are at least 2^(11 - d), f16's step at the bottom is 2^-24), all of them alike.  Sums of 20,000 keys in
    fp32, 16 at a time, in the product and in the denominator, each step off by at most 2^-23: 2 * 1251 * 2^-23.
    The scores, exponentials and the reciprocal: 2^-14, as in test_gpu_paged.py.  Then the output's half step, half of
    f16's last step included."""
    page, nkv, nq, n = 64, 1, 4, 20001
    g = _gen(dim)
    tables, cu, kv, n_pages = _step([(n + rows - 1, rows)], page, g)
    kp = torch.zeros(n_pages, nkv, page, dim, dtype=torch.uint8, device="cuda")
    vp = torch.full_like(kp, 0x38)                                     # 1.0
    ks, vs = torch.ones(n_pages, nkv, device="cuda"), torch.ones(n_pages, nkv, device="cuda")
    first = int(tables[0, 0])
    kp[first, 0, 0, 0], vp[first, 0, 0] = 0x38, 0
    q = torch.zeros(rows, nq, dim, device="cuda", dtype=dtype)
    q[:, :, 0] = 1.0
    out = P.paged_attention(q, kp, vp, ks, vs, tables, cu, kv, max_q=rows, scale=nats).double()
    scale = float(np.float32(nats))
    seen = torch.arange(n - 1, n - 1 + rows, dtype=torch.float64, device="cuda")        # keys beside the sink
    want = (seen * math.exp(-scale) / (1 + seen * math.exp(-scale)))[:, None, None]
    d = scale / math.log(2)
    rel = max(2.0 ** -11, 2.0 ** (d - 36)) + 2 * 1251 * 2.0 ** -23 + 2.0 ** -14
    tol = want * (rel + HALF_STEP[dtype]) * 1.01 + 2.0 ** -25
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / want).max().item()


@pytest.mark.parametrize("nq,nkv,dim,page,dtype", [(8, 2, 128, 64, torch.float16), (4, 1, 64, 16, torch.bfloat16)])
@pytest.mark.parametrize("spans", [[(700, 1), (3000, 2)], [(500, 200), (2500, 40)]])
@pytest.mark.parametrize("way", [1, -1])
def test_paged_attention_scores_that_climb(P, spans, nq, nkv, dim, page, dtype, way):
    """The largest score moves on with the keys (the reference is raised again and again, outputs and sums with it),
    or stays behind at the first ones."""
    g = _gen(nq + page)
    tables, cu, kv, n_pages = _step(spans, page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    kp, _, ks, _ = cache
    e4m3 = kp.view(torch.float8_e4m3fn)
    for r, (n, _) in enumerate(spans):
        pos = torch.arange(-(-n // page) * page, device="cuda").view(-1, page)
        rise = (pos if way > 0 else n - pos).float() * (40.0 / n)       # score in nats that dimension 0 adds
        ids = tables[r, :-(-n // page)].long()
        ks[ids] = 1.0
        x = torch.randn(len(ids), nkv, page, dim, generator=g, device="cuda")
        x[..., 0] = rise[:, None]
        e4m3[ids] = x.to(torch.float8_e4m3fn)
    q = torch.randn(int(cu[-1]), nq, dim, generator=g, device="cuda") * 0.5
    q[..., 0] = dim ** 0.5
    q = q.to(dtype)
    lse = torch.empty(q.shape[:2], device="cuda")
    for m in (1, max(n for _, n in spans)):
        out = P.paged_attention(q, *cache, tables, cu, kv, max_q=m, lse=lse)
        _check_attention(out, lse, q, cache, tables, cu, kv)


# ─── keys that are not finite, or that the rotation makes so ──────────────────
def _edge_rows(rows, heads, dim, dtype, g):
    """Rows of ordinary values with infinities, NaN and pairs whose sums pass the type (and, in bf16, fp32)."""
    x = torch.randn(rows, heads, dim, generator=g, device="cuda")
    big = 65504.0 if dtype is torch.float16 else 3.3e38
    inf = float("inf")
    at = torch.randint(0, dim, (rows, heads, 2), generator=g, device="cuda")
    what = torch.tensor([inf, -inf, float("nan"), big, -big, 1.0], device="cuda")
    pick = what[torch.randint(0, 6, (rows, heads, 2), generator=g, device="cuda")]
    x.scatter_(2, at, pick)
    x[1::4] = big                            # every pair of the row at the top: a c - b s and a s + b c
    x[3::4, :, ::2] = -big
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,rotary,interleaved", [
    (24, 128, 128, False), (24, 64, 32, True), (24, 64, 18, False), (1100, 128, 128, False), (1100, 64, 64, True),
    (1100, 128, 30, True),
])
def test_keys_that_are_not_finite(P, N, rows, dim, rotary, interleaved, dtype):
    """The rotation of infinities and of sums that overflow is the definition's (in 64 bits, rounded to fp32 and to
    the type), and the cache holds them saturated at 448 times the scale, NaN as 0."""
    nq, nkv, page = 4, 2, 64
    g = _gen(rows + rotary)
    cos, sin = _angles(P, 3000, rotary)
    pos = torch.arange(rows, device="cuda")              # position 0 among them: sin is 0, and 0 times infinity NaN
    k = _edge_rows(rows, nkv, dim, dtype, g)
    v = torch.randn(rows, nkv, dim, generator=g, device="cuda").to(dtype)
    q = torch.randn(rows, nq, dim, generator=g, device="cuda").to(dtype)
    with np.errstate(invalid="ignore"):
        want = T.O.rotate(k.double().cpu().numpy(), cos.double().cpu().numpy(), sin.double().cpu().numpy(),
                          pos.tolist(), interleaved)
    want = torch.from_numpy(want).float().to(dtype)
    assert want.isinf().any() and want.isnan().any() and want[1::4].isinf().any()
    got = P.rope(q, k, cos, sin, pos, interleaved=interleaved)[1].cpu()
    lost = want.isnan()
    assert torch.equal(got.isnan(), lost) and torch.equal(got.masked_fill(lost, 0), want.masked_fill(lost, 0))
    n_pages = -(-rows // page)
    cache = _cache(n_pages, nkv, page, dim, seed=3)
    before = _np(*cache)
    st = N.new_status("cuda")
    P.rope_append(q, k, v, cos, sin, pos, pos, *cache, interleaved=interleaved, status=st)
    assert int(st) == N.HC_ERR_RANGE
    _check_append(cache, before, want.cuda(), v, pos)


# ─── the cache object ─────────────────────────────────────────────────────────
@pytest.mark.parametrize("max_len,page", [(20, 16), (1, 16), (127, 64), (64, 64)])
def test_paged_cache_holds_max_len_positions(P, N, max_len, page):
    """Not as many as its last page has room for: tables of angles end there."""
    c = P.PagedKVCache(1, 1, 64, 8, page_size=page, max_requests=2, max_len=max_len)
    plan = c.plan(_i32([max_len, 0]), max_len)
    assert plan.positions.tolist() == list(range(max_len)) and plan.kv_lens.tolist() == [max_len, 0]
    c.commit(plan)
    c.check()
    free = int(c.n_free)
    for q_lens in ([1, 0], [0, max_len + 1], [2 ** 31 - 1, 0]):
        plan = c.plan(_i32(q_lens), max_len + 1)
        assert (plan.slots == -1).all() and int(c.n_free) == free and plan.kv_lens.tolist() == [max_len, 0]
        with pytest.raises(N.HotColdError):
            c.check()
        c.status.zero_()
    plan = c.plan(_i32([0, max_len]), max_len + 1)                    # the other request has its room still
    assert plan.kv_lens.tolist() == [max_len, max_len]
    c.check()
    with pytest.raises(ValueError):
        c.plan(_i32([1]), 1)


# ─── page release ─────────────────────────────────────────────────────────────
@pytest.mark.parametrize("row", [
    [3, -1, -1, 7, -1], [3, -1, 5, -1, -1, -1], [1, 2, 3, 4, -1, 5, 6, -1], [-1, -1, -1, -1, 8],
    [-1, 3, -1, -1, -1, -1, -1, -1, -1], list(range(1, 34)) + [-1] * 40 + [40] + [-1] * 30,
])
def test_page_release_of_a_row_with_any_hole(P, N, row):
    tables = _i32([row, [0] + [-1] * (len(row) - 1)])
    free, n_free, st = _i32([9] + [-1] * 99), _i32([1]), N.new_status("cuda")
    before = tables.clone()
    P.page_release(torch.tensor([True, True], device="cuda"), tables, free, n_free, st)
    assert int(st) == N.HC_ERR_RANGE and int(n_free) == 1 and torch.equal(tables, before)
    assert free.tolist() == [9] + [-1] * 99
    # a request that goes on may hold what it likes
    st.zero_()
    P.page_release(torch.tensor([False, True], device="cuda"), tables, free, n_free, st)
    N.read_status(st, "page_release")
    assert int(n_free) == 2 and free[:2].tolist() == [9, 0] and torch.equal(tables[0], before[0])


@pytest.mark.parametrize("requests,width,every", [(2048, 70, 1), (2047, 33, 3), (1025, 5, 2), (40, 300, 1), (3, 9000, 1),
                                                  (1, 1, 1), (33, 64, 5)])
def test_page_release_of_many_requests_and_wide_tables(P, N, requests, width, every):
    rng = np.random.default_rng(requests)
    held = rng.integers(0, width + 1, requests)
    held[0] = width
    order = rng.permutation(int(held.sum()) + 7).astype(np.int32)
    wide = np.full((requests, width + 3), 5, np.int32)                 # what lies past a row's width is not the table's
    wide[:, :width] = -1
    at = np.concatenate([[0], np.cumsum(held)])
    for r in range(requests):
        wide[r, :held[r]] = order[at[r]:at[r + 1]]
    free = np.full(len(order), -1, np.int32)
    free[:7] = order[at[-1]:]
    done = np.arange(requests) % every == 0
    dt, dfree, dn, st = torch.tensor(wide).cuda(), torch.tensor(free).cuda(), _i32([7]), N.new_status("cuda")
    P.page_release(torch.tensor(done).cuda(), dt[:, :width], dfree, dn, st)
    N.read_status(st, "page_release")
    back = np.concatenate([wide[r, :held[r]] for r in range(requests) if done[r]])
    free[7:7 + len(back)] = back
    wide[done, :width] = -1
    assert int(dn) == 7 + len(back)
    assert np.array_equal(dfree.cpu().numpy(), free) and np.array_equal(dt.cpu().numpy(), wide)


def test_paged_cache_release_that_is_refused_keeps_the_lengths(P, N):
    c = P.PagedKVCache(1, 1, 64, 8, page_size=16, max_requests=3, max_len=64)
    c.commit(c.plan(_i32([40, 5, 0]), 45))
    page = int(c.tables[0, 1])
    c.tables[0, 1] = -1
    c.release(torch.ones(3, dtype=torch.bool, device="cuda"))
    with pytest.raises(N.HotColdError):
        c.check()
    assert c.lens.tolist() == [40, 5, 0] and int(c.n_free) == 4
    c.status.zero_()
    c.tables[0, 1] = page
    c.release(torch.tensor([True, False, True], device="cuda"))
    c.check()
    assert c.lens.tolist() == [0, 5, 0] and int(c.n_free) == 7


# ─── offsets that claim more rows than there are ──────────────────────────────
@pytest.mark.parametrize("requests", [4, 40, 300])
def test_paged_prompt_attention_serves_no_more_rows_than_there_are(P, N, requests):
    """Two requests of 60 of 100 rows each, the offsets going back between them: both tiles fit the launch, and still
    neither is served; in order, they are."""
    page, nq, nkv, dim = 64, 8, 2, 64
    g = _gen(requests)
    tables, _, _, n_pages = _step([(300, 0)], page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    tables, kv = tables.expand(requests, -1).contiguous(), _i32([300] * requests)
    q = torch.randn(100, nq, dim, generator=g, device="cuda").half()
    out, st = torch.full_like(q, 9.0), N.new_status("cuda")
    P.paged_attention(q, *cache, tables, _i32([0, 60, 0, 60] + [60] * (requests - 3)), kv, max_q=100, out=out, status=st)
    assert int(st) == N.HC_ERR_RANGE and (out == 9).all()
    st.zero_()
    cu = _i32([0, 60, 60, 100] + [100] * (requests - 3))
    P.paged_attention(q, *cache, tables, cu, kv, max_q=100, out=out, status=st)
    N.read_status(st, "paged_attention")
    _check_attention(out, None, q, cache, tables[:3], cu[:4], kv[:3])
    # offsets that end in zeros go back, but claim no row twice: the requests before them are served
    st.zero_()
    out.fill_(9.0)
    P.paged_attention(q, *cache, tables, _i32([0, 60, 60, 100] + [0] * (requests - 3)), kv, max_q=100, out=out,
                      status=st)
    assert (int(st) == N.HC_ERR_RANGE) == (requests > 3)
    _check_attention(out, None, q, cache, tables[:3], cu[:4], kv[:3])


@pytest.mark.parametrize("rows", [1, 1100])
def test_kv_append_flags_values_past_the_largest_scale(P, N, rows):
    """448 * 2^40 is held; the next bf16 value saturates, and that is reported like an infinity."""
    top = 448.0 * 2.0 ** 40
    x = torch.randn(rows, 1, 64, device="cuda", generator=_gen(rows)).bfloat16()
    x[rows // 2, 0, 5] = top
    slots = torch.arange(rows, device="cuda")
    for value, flagged in ((top, 0), (-top, 0), (450.0 * 2.0 ** 40, N.HC_ERR_RANGE), (-3e38, N.HC_ERR_RANGE)):
        k = x.clone()
        k[rows // 2, 0, 5] = value
        cache = _cache(18, 1, 64, 64, seed=1)
        before, st = _np(*cache), N.new_status("cuda")
        P.kv_append(x, k, slots, *cache, status=st)
        assert int(st) == flagged
        _check_append(cache, before, x, k, slots)
        assert k[rows // 2, 0, 5].item() == value or value == -3e38
