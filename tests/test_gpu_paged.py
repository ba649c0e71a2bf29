"""GPU parity of the paged-cache operators against their plain 64-bit forms (oracle/paged_oracle.py).

Tolerances.  Integers and cache bytes are equal.  A rotated query is one fp32
fma of an fp32 product, rounded: 2^-23 (|a c| + |b s|) and half a step of its
type.  Attention: weights rounded to f16 (2^-11 each, and 2^-25 below f16's
normal range, where a weight of 1 goes with at most 448 times the largest value
scale), the output's half step, and 2^-14 of the weighted |v| for the fp32
scores, exponentials and sums (a score of magnitude 30 is off by at most 30 *
2^-20 relative to its weight).
"""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def P():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import paged
    return paged


@pytest.fixture(scope="module")
def N():
    import hc_native
    return hc_native


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ─── page plan ────────────────────────────────────────────────────────────────
def _pool(starts, page, width, n_pages, seed):
    """Tables that hold every request's cached tokens, and the stack of the other pages."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(n_pages)
    tables = np.full((len(starts), width), -1)
    at = 0
    for r, s in enumerate(starts):
        n = -(-s // page)
        tables[r, :n] = order[at:at + n]
        at += n
    free = np.full(n_pages, -1)
    free[:n_pages - at] = order[at:]
    return tables, free, n_pages - at


@pytest.mark.parametrize("starts,q_lens,page,width,pad", [
    ([0], [1], 16, 1, 0),
    ([0, 0], [0, 0], 64, 2, 3),
    ([15, 16, 17, 0, 63], [1, 1, 1, 0, 2], 16, 5, 0),
    ([0, 100, 5], [700, 0, 33], 128, 9, 40),
    ([3, 0, 129, 64], [61, 64, 127, 1], 64, 4, 1),
    ([7] * 33, [1] * 33, 32, 3, 31),
    (list(range(0, 2048)), [1 + (i * 7) % 5 for i in range(2048)], 16, 140, 100),
    ([0, 2000, 31], [5000, 1, 3000], 16, 330, 17),
])
def test_page_plan(P, N, starts, q_lens, page, width, pad):
    n_pages = sum(-(-(s + q) // page) for s, q in zip(starts, q_lens)) + 5
    tables, free, n_free = _pool(starts, page, width, n_pages, len(starts))
    rows = sum(q_lens) + pad
    cu, kv, pos, slot, t2, nf = O.plan(starts, q_lens, tables, free, n_free, page, rows)
    dt, dfree, dn, st = _i32(tables), _i32(free), _i32([n_free]), N.new_status("cuda")
    for _ in range(2):                       # planned again, the step takes nothing more
        plan = P.page_plan(_i32(starts), _i32(q_lens), dt, dfree, dn, page, rows, st)
        N.read_status(st, "page_plan")
        assert np.array_equal(plan.cu_q.cpu().numpy(), cu)
        assert np.array_equal(plan.kv_lens.cpu().numpy(), kv)
        assert np.array_equal(plan.positions.cpu().numpy(), pos)
        assert np.array_equal(plan.slots.cpu().numpy(), slot)
        assert np.array_equal(dt.cpu().numpy(), t2) and int(dn) == nf
    assert np.array_equal(dfree.cpu().numpy(), free)


@pytest.mark.parametrize("case", ["pages", "rows", "width", "negative q", "negative start", "free count"])
def test_page_plan_that_does_not_work_out(P, N, case):
    starts, q_lens, page, rows, width = [10, 0, 20], [30, 5, 1], 16, 40, 4
    tables, free, n_free = _pool(starts, page, width, 12, 1)
    if case == "pages":
        n_free = 2                           # three are needed
    if case == "rows":
        rows = 35
    if case == "width":
        q_lens = [30, 5, 45]
        rows = 80
    if case == "negative q":
        q_lens = [30, -1, 1]
    if case == "negative start":
        starts = [10, -3, 20]
    if case == "free count":
        n_free = 13
    dt, dn, st = _i32(tables), _i32([n_free]), N.new_status("cuda")
    plan = P.page_plan(_i32(starts), _i32(q_lens), dt, _i32(free), dn, page, rows, st)
    assert int(st) == N.HC_ERR_RANGE
    assert int(dn) == n_free and np.array_equal(dt.cpu().numpy(), tables)
    assert not plan.cu_q.any() and plan.kv_lens.tolist() == starts
    assert (plan.positions == -1).all() and (plan.slots == -1).all()


def test_page_plan_flags_stray_pages(P, N):
    dt, st = _i32([[9, -1], [0, -1]]), N.new_status("cuda")         # page 9 of 4
    plan = P.page_plan(_i32([3, 3]), _i32([1, 1]), dt, _i32([1, 2, 3, 0]), _i32([3]), 16, 2, st)
    assert int(st) == N.HC_ERR_RANGE and plan.slots.tolist() == [-1, 3] and plan.positions.tolist() == [3, 3]


def test_page_release(P, N):
    tables, free, n_free = _pool([70, 0, 33, 16, 90], 16, 6, 20, 3)
    dt, dfree, dn, st = _i32(tables), _i32(free), _i32([n_free]), N.new_status("cuda")
    done = torch.tensor([True, True, False, True, False], device="cuda")
    P.page_release(done, dt, dfree, dn, st)
    N.read_status(st, "page_release")
    back = [p for r in (0, 1, 3) for p in tables[r] if p >= 0]
    assert int(dn) == n_free + len(back)
    assert dfree[:n_free].tolist() == free[:n_free].tolist()
    assert dfree[n_free:n_free + len(back)].tolist() == back
    want = tables.copy()
    want[[0, 1, 3]] = -1
    assert np.array_equal(dt.cpu().numpy(), want)
    P.page_release(done, dt, dfree, dn, st)                          # nothing left there
    N.read_status(st, "page_release")
    assert int(dn) == n_free + len(back)
    # more pages than the pool has: refused whole
    dn2 = _i32([18])
    P.page_release(torch.ones(5, dtype=torch.bool, device="cuda"), dt, dfree, dn2, st)
    assert int(st) == N.HC_ERR_RANGE and int(dn2) == 18 and np.array_equal(dt.cpu().numpy(), want)


# ─── rotary positions ─────────────────────────────────────────────────────────
def _angles(P, rows, rotary):
    return P.rope_tables(rows, rotary, 500000.0, device="cuda")


def _check_rope(q_out, k_out, q, k, cos, sin, positions, interleaved):
    c, s = cos.double().cpu().numpy(), sin.double().cpu().numpy()
    pos = positions.cpu().numpy()
    want_k = O.rotate(k.double().cpu().numpy(), c, s, pos, interleaved)
    assert torch.equal(k_out.cpu(), torch.from_numpy(want_k).float().to(k.dtype))
    qd = q.double().cpu().numpy()
    want = O.rotate(qd, c, s, pos, interleaved)
    size = O.rotate(np.abs(qd), np.abs(c), -np.abs(s), pos, interleaved)      # |a c| + |b s| of the first, bounds both
    size = np.maximum(size, O.rotate(np.abs(qd), np.abs(c), np.abs(s), pos, interleaved))
    tol = 2.0 ** -23 * np.abs(size) + HALF_STEP[q.dtype] * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -25
    assert (np.abs(q_out.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,nq,nkv,dim,rotary,interleaved", [
    (1, 32, 8, 128, 128, False), (1, 1, 1, 64, 64, True), (7, 4, 2, 128, 64, True), (5, 7, 1, 64, 32, False),
    (3, 2, 2, 128, 96, False), (3, 2, 1, 64, 2, True), (9, 3, 1, 128, 18, False), (2, 2, 2, 80, 80, True),
    (300, 8, 2, 64, 64, False),
])
def test_rope(P, N, rows, nq, nkv, dim, rotary, interleaved, dtype):
    g = _gen(rows + dim + rotary)
    far = 131072 if rotary <= 32 else 5000
    cos, sin = _angles(P, far, rotary)
    qkv = torch.randn(rows, nq + 2 * nkv, dim, generator=g, device="cuda").to(dtype)
    q, k = qkv[:, :nq], qkv[:, nq:nq + nkv]
    positions = torch.randint(0, far, (rows,), generator=g, device="cuda")
    positions[0] = far - 1
    st = N.new_status("cuda")
    q_out, k_out = P.rope(q, k, cos, sin, positions, interleaved=interleaved, status=st)
    _check_rope(q_out, k_out, q, k, cos, sin, positions, interleaved)
    # in place, among the rows of the projection, and into a transposed layout
    both = qkv.clone()
    P.rope(both[:, :nq], both[:, nq:nq + nkv], cos, sin, positions, interleaved=interleaved, status=st,
           q_out=both[:, :nq], k_out=both[:, nq:nq + nkv])
    assert torch.equal(both[:, :nq], q_out) and torch.equal(both[:, nq:nq + nkv], k_out)
    assert torch.equal(both[:, nq + nkv:], qkv[:, nq + nkv:])
    turned = torch.empty(nq, rows, dim, dtype=dtype, device="cuda").transpose(0, 1)
    P.rope(q, k, cos, sin, positions, interleaved=interleaved, status=st, q_out=turned)
    assert torch.equal(turned, q_out)
    N.read_status(st, "rope")


def test_rope_any_alignment_padding_and_far_positions(P, N):
    g = _gen(5)
    cos, sin = _angles(P, 64, 64)
    flat = torch.randn(4 * (6 * 64 + 3) + 1, generator=g, device="cuda").half()
    x = flat[1:].view(4, 6 * 64 + 3)[:, 1:1 + 6 * 64].unflatten(1, (6, 64))       # odd base and row stride
    q, k = x[:, :4], x[:, 4:]
    positions = _i64([63, -1, 64, 5])                                             # padding, outside, inside
    st = N.new_status("cuda")
    q_out, k_out = torch.full((4, 4, 64), 7.0, device="cuda").half(), torch.full((4, 2, 64), 7.0, device="cuda").half()
    P.rope(q, k, cos, sin, positions, q_out=q_out, k_out=k_out, status=st)
    assert int(st) == N.HC_ERR_RANGE
    assert (q_out[1:3] == 7).all() and (k_out[1:3] == 7).all()
    at = [0, 3]
    _check_rope(q_out[at], k_out[at], q[at], k[at], cos, sin, positions[at], False)
    # the same rows aligned give the same bits
    qa, ka = P.rope(q[at].contiguous(), k[at].contiguous(), cos, sin, positions[at])
    assert torch.equal(qa, q_out[at]) and torch.equal(ka, k_out[at])
    e = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    assert P.rope(e, e, cos, sin, _i64([]))[0].shape == (0, 2, 64)


def test_rope_refuses(P):
    cos, sin = _angles(P, 8, 64)
    x = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    pos = _i64([0, 1])
    for bad in (dict(q=x.float()), dict(k=x[:1]), dict(k=x.bfloat16()), dict(q=x[..., :32]), dict(q=x[0]),
                dict(cos=cos.double()), dict(sin=sin[:4]), dict(positions=pos.int()), dict(positions=pos[:1]),
                dict(q_out=x[:1]), dict(q=x.transpose(1, 2)), dict(cos=cos.cpu())):
        a = dict(q=x, k=x, cos=cos, sin=sin, positions=pos)
        a.update(bad)
        with pytest.raises((ValueError, RuntimeError)):
            P.rope(**a)


# ─── the cache's write ────────────────────────────────────────────────────────
def _cache(n_pages, nkv, page, dim, seed=None):
    kp = torch.zeros(n_pages, nkv, page, dim, dtype=torch.uint8, device="cuda")
    ks = torch.zeros(n_pages, nkv, device="cuda")
    vp, vs = kp.clone(), ks.clone()
    if seed is not None:                 # whatever an earlier use of the pages left there
        g = _gen(seed)
        for p in (kp, vp):
            p.copy_(torch.randint(0, 256, p.shape, generator=g, device="cuda", dtype=torch.uint8))
            p[(p & 127) == 127] = 1
        for s in (ks, vs):
            s.copy_(2.0 ** torch.randint(-9, 3, s.shape, generator=g, device="cuda").float())
    return kp, vp, ks, vs


def _np(*ts):
    return [t.cpu().numpy() for t in ts]


def _check_append(cache, before, k, v, slots, rows=None):
    sl = slots.cpu().numpy()
    for which, x in ((0, k), (1, v)):
        want, scale = O.append(before[which], before[2 + which], x.double().cpu().numpy(), sl)
        got = cache[which].cpu().numpy()
        assert np.array_equal(cache[2 + which].cpu().numpy(), scale.astype(np.float32))
        assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,dim,nkv,spans", [
    (16, 64, 1, [(0, 1)]), (16, 128, 8, [(0, 16), (5, 3), (15, 2)]), (32, 128, 3, [(31, 70), (0, 33)]),
    (64, 128, 2, [(63, 1), (64, 1), (65, 1), (10, 200)]), (128, 64, 5, [(0, 128), (127, 130), (1, 17)]),
    (64, 64, 8, [(i, 1) for i in range(40)]), (16, 128, 2, [(3, 900)]), (128, 128, 1, [(100, 1200), (0, 40)]),
])
def test_kv_append(P, N, page, dim, nkv, spans, dtype):
    width = max(-(-(s + n) // page) for s, n in spans)
    n_pages = width * len(spans) + 1
    g = _gen(page + dim + len(spans))
    order = torch.randperm(n_pages, generator=g, device="cuda")
    slots = []
    for r, (s, n) in enumerate(spans):
        pos = torch.arange(s, s + n, device="cuda")
        slots.append(order[r * width + pos // page] * page + pos % page)
    slots = torch.cat(slots)
    rows = slots.numel()
    cache = _cache(n_pages, nkv, page, dim, seed=rows)
    before = _np(*cache)
    qkv = torch.randn(rows, 3 * nkv, dim, generator=g, device="cuda")
    qkv *= 10.0 ** torch.randint(-3, 3, (rows, 1, 1), generator=g, device="cuda")     # some raise their page's scale
    qkv = qkv.to(dtype)
    k, v = qkv[:, nkv:2 * nkv], qkv[:, 2 * nkv:]
    st = N.new_status("cuda")
    P.kv_append(k, v, slots, *cache, status=st)
    N.read_status(st, "kv_append")
    _check_append(cache, before, k, v, slots)
    # written again (a step that is replayed), the cache stays as it is
    once = [t.clone() for t in cache]
    P.kv_append(k, v, slots, *cache, status=st)
    assert all(torch.equal(a, b) for a, b in zip(once, cache))


def test_kv_append_token_by_token_and_restarted_page(P, N):
    """Tokens one call at a time: the scale follows the largest value so far, and
    a page that is used anew forgets its old scale."""
    cache = _cache(3, 2, 16, 64, seed=3)
    g = _gen(4)
    k, v = (torch.randn(20, 2, 64, generator=g, device="cuda").half() * 0.01 for _ in range(2))
    k[5] *= 300
    v[11] *= 9000
    slots = torch.cat([torch.arange(32, 48), torch.arange(0, 4)]).cuda()
    for t in range(20):
        before = _np(*cache)
        P.kv_append(k[t:t + 1], v[t:t + 1], slots[t:t + 1], *cache)
        _check_append(cache, before, k[t:t + 1], v[t:t + 1], slots[t:t + 1])
    before = _np(*cache)
    P.kv_append(k[:2], v[:2], slots[:2], *cache)
    _check_append(cache, before, k[:2], v[:2], slots[:2])
    assert (cache[2][2] < 2.0 ** -10).all()


def test_kv_append_values_at_the_edges(P, N):
    """Zeros, subnormals, the largest value of a type, scales at a power's border, infinities and NaN."""
    cache = _cache(8, 1, 16, 64, seed=9)
    x = torch.zeros(7, 1, 64, device="cuda")
    x[1, 0, 0] = 448.0                       # exactly scale 1
    x[1, 0, 1:5] = torch.tensor([2.0 ** -9, 2.0 ** -10, 2.0 ** -10 * 1.5, -2.0 ** -10])     # subnormals and a tie
    x[2, 0, 3] = 450.0                       # just past it: scale 2
    x[3, 0, 0] = 6e-8
    x[4, 0, :3] = torch.tensor([float("inf"), 3.0, float("-inf")])
    x[5, 0, :2] = torch.tensor([float("nan"), -2.0])
    x[6, 0, 7] = 65504.0
    x = x.half()
    slots = _i64([i * 16 for i in range(7)])
    st = N.new_status("cuda")
    before = _np(*cache)
    P.kv_append(x[:4], x[:4], slots[:4], *cache, status=st)
    N.read_status(st, "kv_append")
    P.kv_append(x[6:], x[6:], slots[6:], *cache, status=st)
    N.read_status(st, "kv_append")
    P.kv_append(x[4:6], x[4:6], slots[4:6], *cache, status=st)
    assert int(st) == N.HC_ERR_RANGE         # reported, and nothing of it in the cache
    _check_append(cache, before, x, x, slots)
    assert (cache[2][:7, 0].tolist() == [2.0 ** -40, 1.0, 2.0, 2.0 ** -32, 2.0 ** -7, 2.0 ** -7, 2.0 ** 8])
    assert not cache[0].view(torch.float8_e4m3fn)[:7, :, :1].float().isnan().any()
    big = torch.full((1, 1, 64), 3e38, device="cuda").bfloat16()
    P.kv_append(big, big, _i64([112]), *cache)
    assert cache[2][7, 0] == 2.0 ** 40 and (cache[0][7, 0, 0] == 126).all()


def test_kv_append_padding_and_bad_slots(P, N):
    cache = _cache(4, 2, 16, 128, seed=1)
    before = [t.clone() for t in cache]
    x = torch.randn(6, 2, 128, device="cuda").half()
    st = N.new_status("cuda")
    P.kv_append(x, x, _i64([-1] * 6), *cache, status=st)
    N.read_status(st, "kv_append")
    P.kv_append(x, x, _i64([64, 1 << 40, -5, -1, 63 + (1 << 32), 64]), *cache, status=st)
    assert int(st) == N.HC_ERR_RANGE
    assert all(torch.equal(a, b) for a, b in zip(before, cache))
    # rows of one page that do not follow one another: the first run is written, the rest left out
    st.zero_()
    P.kv_append(x, x, _i64([16, 17, 17, 20, -1, 33]), *cache, status=st)
    assert int(st) == N.HC_ERR_RANGE
    b = _np(*before)
    _check_append(cache, b, x, x, _i64([16, 17, -1, -1, -1, 33]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,rotary,interleaved,page,aligned", [
    (128, 128, False, 64, True), (128, 64, True, 16, True), (64, 64, False, 128, True), (64, 18, False, 32, True),
    (128, 128, False, 32, False), (64, 30, True, 16, False),
])
def test_rope_append_is_rope_then_append(P, N, dim, rotary, interleaved, page, aligned, dtype):
    nq, nkv = 6, 3
    g = _gen(dim + rotary)
    spans = [(0, 5), (page - 1, 2), (3, 300), (17, 1)]
    pos = torch.cat([torch.arange(s, s + n, device="cuda") for s, n in spans] + [_i64([-1, -1])])
    slots = torch.cat([torch.arange(s, s + n, device="cuda") + 512 * r for r, (s, n) in enumerate(spans)]
                      + [_i64([-1, -1])])
    rows = pos.numel()
    cos, sin = _angles(P, 400, rotary)
    wide = torch.randn(rows, (nq + 2 * nkv) * dim + 3, generator=g, device="cuda").to(dtype)
    qkv = wide[:, :-3].contiguous() if aligned else wide[:, 1:-2]
    qkv = qkv.unflatten(1, (nq + 2 * nkv, dim))
    q, k, v = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    a, b = _cache(2048 // page, nkv, page, dim, seed=2), _cache(2048 // page, nkv, page, dim, seed=2)
    st = N.new_status("cuda")
    q1 = torch.full((rows, nq, dim), 3.0, device="cuda").to(dtype)
    k1, q2 = torch.full((rows, nkv, dim), 3.0, device="cuda").to(dtype), q1.clone()
    P.rope(q, k, cos, sin, pos, interleaved=interleaved, q_out=q1, k_out=k1, status=st)
    P.kv_append(k1, v, slots, *a, status=st)
    P.rope_append(q, k, v, cos, sin, pos, slots, *b, interleaved=interleaved, q_out=q2, status=st)
    N.read_status(st, "rope_append")
    assert torch.equal(q1, q2) and (q2[-2:] == 3).all()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # a row without a position in the tables is not written
    pos[2] = 400
    before = [t.clone() for t in b]
    P.rope_append(q, k, v, cos, sin, pos, slots, *b, interleaved=interleaved, q_out=q2, status=st)
    assert int(st) == N.HC_ERR_RANGE
    p0 = 0
    assert torch.equal(b[0][p0, :, 2], before[0][p0, :, 2]) and torch.equal(q2[2], q1[2])


# ─── attention ────────────────────────────────────────────────────────────────
def _filled(n_pages, nkv, page, dim, g, spread=0):
    def one(mean):
        x = torch.randn(n_pages, nkv, page, dim, generator=g, device="cuda") + mean
        s = 2.0 ** torch.randint(-7 - spread, -6 + spread, (n_pages, nkv), generator=g, device="cuda").float()
        return (x / 2.0 ** -7).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s
    kp, ks = one(0.0)
    vp, vs = one(0.3)
    return kp, vp, ks, vs


def _step(spans, page, g, spare=2):
    """tables, cu_q, kv_lens of requests given as (kv_len, q_len)."""
    width = max(1, max(-(-kv // page) for kv, _ in spans)) + 1
    n_pages = sum(-(-kv // page) for kv, _ in spans) + spare
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    tables = torch.full((len(spans), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, (kv, _) in enumerate(spans):
        n = -(-kv // page)
        tables[r, :n] = order[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum([q for _, q in spans])])
    return tables, _i32(cu.tolist()), _i32([kv for kv, _ in spans]), n_pages


def _check_attention(out, lse, q, cache, tables, cu, kv, scale=None):
    arrays = _np(*cache)
    qd, tb, cn, kn = q.double().cpu().numpy(), tables.cpu().numpy(), cu.cpu().numpy(), kv.cpu().numpy()
    want, want_lse = O.attention(qd, *arrays, tb, cn, kn, scale)
    size, _ = O.attention(qd, arrays[0], arrays[1] & 127, arrays[2], arrays[3], tb, cn, kn, scale)    # of |v|
    rows = int(cn[-1])
    used = [p for r in range(len(kn)) for p in tb[r, :-(-kn[r] // cache[0].shape[2])]]
    vs_max = float(arrays[3][used].max()) if used else 0.0
    tol = (HALF_STEP[q.dtype] * np.abs(want) * 1.001 + (2.0 ** -11 + 2.0 ** -14) * size
           + 2.0 ** -25 * (kn.max() * 448 * vs_max + 1))
    got = out.double().cpu().numpy()[:rows]
    bad = np.abs(got - want[:rows]) > tol[:rows]
    assert not np.isnan(got).any() and not bad.any(), np.abs(got - want[:rows])[bad].max()
    if lse is not None:
        l = lse.double().cpu().numpy()[:rows]
        fin = np.isfinite(want_lse[:rows])
        assert np.array_equal(fin, np.isfinite(l)) and (l[~fin] == -np.inf).all()
        assert (np.abs(l[fin] - want_lse[:rows][fin]) <= 2.0 ** -14 + 2.0 ** -20 * np.abs(want_lse[:rows][fin])).all()


SPANS = {
    "one key": [(1, 1)],
    "one token": [(513, 1)],
    "decode": [(1, 1), (15, 1), (16, 1), (17, 1), (64, 1), (65, 1), (300, 1), (127, 1), (128, 1)],
    "no keys and short": [(0, 0), (0, 2), (1, 3), (33, 0), (7, 7), (5, 9)],
    "few tokens": [(40, 2), (129, 5), (3, 3), (260, 4)],
    "prompts": [(70, 70), (200, 33), (129, 129), (40, 1)],
}


@pytest.mark.parametrize("spans", list(SPANS))
@pytest.mark.parametrize("nq,nkv,dim,page,dtype", [
    (32, 8, 128, 64, torch.float16), (8, 8, 64, 16, torch.bfloat16), (7, 1, 128, 32, torch.bfloat16),
    (16, 1, 64, 128, torch.float16), (10, 2, 128, 16, torch.float16), (16, 2, 64, 64, torch.bfloat16),
])
def test_paged_attention(P, N, spans, nq, nkv, dim, page, dtype):
    spans = SPANS[spans]
    g = _gen(nq * dim + page + len(spans))
    tables, cu, kv, n_pages = _step(spans, page, g)
    cache = _filled(n_pages, nkv, page, dim, g, spread=2)
    rows = int(cu[-1]) + 3
    q = torch.randn(rows, nq, dim, generator=g, device="cuda").to(dtype)
    out = torch.full_like(q, 9.0)
    lse = torch.full((rows, nq), 9.0, device="cuda")
    st = N.new_status("cuda")
    max_q = max(n for _, n in spans)
    P.paged_attention(q, *cache, tables, cu, kv, max_q=max_q, out=out, lse=lse, status=st)
    N.read_status(st, "paged_attention")
    assert (out[-3:] == 9).all() and (lse[-3:] == 9).all()            # rows behind the last request
    _check_attention(out, lse, q, cache, tables, cu, kv)
    # max_q only chooses kernels
    for other in (1, 4096):
        o2 = P.paged_attention(q, *cache, tables, cu, kv, max_q=other)
        _check_attention(o2, None, q, cache, tables, cu, kv)
    # the same call gives the same bits
    o3 = torch.full_like(q, 9.0)
    P.paged_attention(q, *cache, tables, cu, kv, max_q=max_q, out=o3)
    assert torch.equal(o3, out)


@pytest.mark.parametrize("nq,nkv,dim,spans", [(8, 2, 128, [(20000, 1)]), (4, 4, 64, [(9000, 1), (30, 1), (17001, 2)]),
                                              (16, 1, 128, [(12345, 1)])])
def test_paged_attention_long_contexts_are_split(P, N, nq, nkv, dim, spans):
    page, g = 64, _gen(dim + nq)
    tables, cu, kv, n_pages = _step(spans, page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    q = torch.randn(int(cu[-1]), nq, dim, generator=g, device="cuda").half()
    lse = torch.empty(q.shape[:2], device="cuda")
    out = P.paged_attention(q, *cache, tables, cu, kv, max_q=2, lse=lse)
    _check_attention(out, lse, q, cache, tables, cu, kv)


@pytest.mark.parametrize("nq,nkv,dim,page,dtype,spans", [
    (8, 2, 128, 64, torch.float16, [(9000, 40)]), (8, 1, 64, 128, torch.bfloat16, [(5000, 64), (3, 20), (4097, 9)]),
    (4, 1, 128, 16, torch.bfloat16, [(2600, 300), (1500, 1), (1, 1)]), (4, 2, 64, 32, torch.float16, [(1030, 1030)]),
])
def test_paged_attention_rows_over_long_contexts_are_cut(P, N, nq, nkv, dim, page, dtype, spans):
    """Few tiles of many rows over long contexts: their keys are cut into pieces that are joined;
    rows near the diagonal see part of the last piece only."""
    g = _gen(dim + nq + page)
    tables, cu, kv, n_pages = _step(spans, page, g)
    cache = _filled(n_pages, nkv, page, dim, g, spread=1)
    rows = int(cu[-1])
    q = torch.randn(rows + 2, nq, dim, generator=g, device="cuda").to(dtype)
    out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
    st = N.new_status("cuda")
    P.paged_attention(q, *cache, tables, cu, kv, max_q=max(n for _, n in spans), out=out, lse=lse, status=st)
    N.read_status(st, "paged_attention")
    assert (out[rows:] == 9).all() and (lse[rows:] == 9).all()
    _check_attention(out, lse, q, cache, tables, cu, kv)
    wide = torch.zeros(rows + 2, nq, dim + 1, device="cuda").to(dtype)[:, :, 1:]              # outputs at odd addresses
    P.paged_attention(q, *cache, tables, cu, kv, max_q=max(n for _, n in spans), out=wide)
    assert torch.equal(wide[:rows], out[:rows])


def test_paged_attention_strides_scale_and_large_queries(P, N):
    page, nq, nkv, dim = 32, 8, 4, 64
    g = _gen(11)
    tables, cu, kv, n_pages = _step([(100, 1), (35, 3)], page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    wide = torch.randn(4, nq * dim + 5, generator=g, device="cuda").half()
    q = wide[:, 3:3 + nq * dim].unflatten(1, (nq, dim))                # rows at odd addresses
    out = torch.empty(4, nq * dim + 1, device="cuda").half()[:, 1:].unflatten(1, (nq, dim))
    P.paged_attention(q, *cache, tables, cu, kv, max_q=3, scale=0.03, out=out)
    _check_attention(out, None, q, cache, tables, cu, kv, scale=0.03)
    heads_first = torch.empty(nq, 4, dim, device="cuda").half().transpose(0, 1)
    P.paged_attention(q, *cache, tables, cu, kv, max_q=3, scale=0.03, out=heads_first)
    assert torch.equal(heads_first, out)
    wide_t = torch.full((2, 64), -1, dtype=torch.int32, device="cuda")
    wide_t[:, :tables.shape[1]] = tables
    o2 = P.paged_attention(q, *cache, wide_t[:, :tables.shape[1]], cu, kv, max_q=3, scale=0.03)
    assert torch.equal(o2, out)
    # bf16 reaches past f16's range at both ends
    for size in (1e8, 1e-12):
        qb = (q.float() * size).bfloat16()
        out = P.paged_attention(qb, *cache, tables, cu, kv, max_q=3, scale=0.1 / size)
        _check_attention(out, None, qb, cache, tables, cu, kv, scale=0.1 / size)


def test_paged_attention_ignores_what_lies_behind(P, N):
    """NaN bytes behind a request's length, in its own last page and in pages of the table that
    no position reaches, and NaN scales of other pages."""
    page, nq, nkv, dim = 64, 8, 2, 128
    g = _gen(21)
    spans = [(70, 1), (64, 2), (1, 1), (100, 40)]
    tables, cu, kv, n_pages = _step(spans, page, g, spare=6)
    cache = _filled(n_pages, nkv, page, dim, g)
    q = torch.randn(int(cu[-1]), nq, dim, generator=g, device="cuda").half()
    want = {m: P.paged_attention(q, *cache, tables, cu, kv, max_q=m) for m in (1, 40)}
    kp, vp, ks, vs = cache
    used = set()
    for r, (n, _) in enumerate(spans):
        for j in range(-(-n // page)):
            p = int(tables[r, j])
            used.add(p)
            kp[p, :, max(0, n - j * page):] = 127
            vp[p, :, max(0, n - j * page):] = 255
    for p in range(n_pages):
        if p not in used:
            kp[p], vp[p], ks[p], vs[p] = 127, 127, float("nan"), float("inf")
    spare = [p for p in range(n_pages) if p not in used]
    for r in range(len(spans)):
        tables[r, -1] = spare[0]
    for m in (1, 40):
        assert torch.equal(P.paged_attention(q, *cache, tables, cu, kv, max_q=m), want[m])


def test_paged_attention_flags_what_is_outside(P, N):
    page, nq, nkv, dim = 16, 4, 2, 64
    g = _gen(31)
    tables, cu, kv, n_pages = _step([(40, 1), (20, 1), (33, 1)], page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    q = torch.randn(3, nq, dim, generator=g, device="cuda").half()
    st = N.new_status("cuda")
    good = P.paged_attention(q, *cache, tables, cu, kv, max_q=1, status=st)
    N.read_status(st, "paged_attention")
    for value in (-1, n_pages, 1 << 30):
        bad = tables.clone()
        bad[1, 1] = value                                              # a page of request 1
        for m in (1, 64):
            st.zero_()
            out = P.paged_attention(q, *cache, bad, cu, kv, max_q=m, status=st)
            assert int(st) == N.HC_ERR_RANGE
            alone = P.paged_attention(q, *cache, tables, cu, kv, max_q=m)
            assert torch.equal(out[[0, 2]], alone[[0, 2]]) and not out.isnan().any()
    # lengths past the table, rows past the array, offsets that go back: those requests are left out
    for change in (dict(kv=_i32([40, 1000, 33])), dict(kv=_i32([40, -1, 33])), dict(cu=_i32([0, 1, 9, 3])),
                   dict(cu=_i32([0, 1, 0, 0]))):
        for m in (1, 64):
            st.zero_()
            out = torch.full_like(q, 5.0)
            a = dict(cu=cu, kv=kv)
            a.update(change)
            P.paged_attention(q, *cache, tables, a["cu"], a["kv"], max_q=m, out=out, status=st)
            assert int(st) == N.HC_ERR_RANGE
            # to the formula's tolerance, not bit for bit: without request 1 the keys are cut into
            # other shares, and fp32 partial sums joined in another order round differently
            _check_attention(out[:1], None, q[:1], cache, tables[:1], cu[:2], kv[:1])
    assert torch.equal(good, P.paged_attention(q, *cache, tables, cu, kv, max_q=1))


def test_cache_past_32_bits(P, N):
    """Pages whose byte offsets pass 2^32."""
    nkv, page, dim, n_pages = 8, 128, 128, 33500
    cache = [torch.empty(n_pages, nkv, page, dim, dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache += [torch.zeros(n_pages, nkv, device="cuda") for _ in range(2)]
    last = [n_pages - 1, 32768, n_pages - 2]
    g = _gen(41)
    n = 300
    k, v = (torch.randn(n, nkv, dim, generator=g, device="cuda").half() for _ in range(2))
    pos = torch.arange(n, device="cuda")
    slots = _i64(last)[pos // page] * page + pos % page
    small = [t[last].clone() for t in cache]
    P.kv_append(k, v, slots, *cache)
    P.kv_append(k, v, pos, *small)
    for a, b in zip(cache, small):
        if a.dim() == 2:
            assert torch.equal(a[last], b)
        else:
            assert torch.equal(a[last].transpose(1, 2).reshape(-1, nkv, dim)[:n],
                               b.transpose(1, 2).reshape(-1, nkv, dim)[:n])
    q = torch.randn(40, 16, dim, generator=g, device="cuda").half()
    for rows in (1, 40):
        cu, kv = _i32([0, rows]), _i32([n])
        far = P.paged_attention(q[:rows], *cache, _i32([last]), cu, kv, max_q=rows)
        near = P.paged_attention(q[:rows], *small, _i32([[0, 1, 2]]), cu, kv, max_q=rows)
        assert torch.equal(far, near)


# ─── a step as it is used ─────────────────────────────────────────────────────
def test_serving_steps_in_a_graph_on_another_stream(P, N):
    """Prompts, then decode steps replayed from one captured graph on a side stream, a request
    that ends and its pages' next owner: plan, rope + append, attention, against the plain forms."""
    page, nq, nkv, dim, n_pages, width = 16, 8, 2, 64, 40, 12
    cos, sin = _angles(P, 400, 32)
    cache = _cache(n_pages, nkv, page, dim, seed=6)
    tables = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    free, n_free = torch.arange(n_pages, dtype=torch.int32, device="cuda"), _i32([n_pages])
    lens, q_lens = _i32([0, 0, 0]), _i32([0, 0, 0])
    st = N.new_status("cuda")
    g = _gen(51)
    rows = 64
    qkv = torch.zeros(rows, nq + 2 * nkv, dim, dtype=torch.float16, device="cuda")

    def step(max_q):
        plan = P.page_plan(lens, q_lens, tables, free, n_free, page, rows, st)
        q = torch.zeros(rows, nq, dim, dtype=torch.float16, device="cuda")
        P.rope_append(qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:], cos, sin, plan.positions, plan.slots,
                      *cache, q_out=q, status=st)
        out = torch.zeros_like(q)
        P.paged_attention(q, *cache, tables, plan.cu_q, plan.kv_lens, max_q=max_q, out=out, status=st)
        lens.copy_(plan.kv_lens)
        return plan, q, out

    def fresh():
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))

    def check(before, t0, nf0, l0, plan, q, out):
        cu, kv, pos, slot, t2, nf = O.plan(l0.tolist(), q_lens.tolist(), t0, free.cpu().numpy(), nf0, page, rows)
        assert np.array_equal(plan.slots.cpu().numpy(), slot) and np.array_equal(tables.cpu().numpy(), t2)
        assert int(n_free) == nf
        k = O.rotate(qkv[:, nq:nq + nkv].double().cpu().numpy(), cos.double().cpu().numpy(),
                     sin.double().cpu().numpy(), pos, False)
        k16 = torch.from_numpy(k).float().half()
        _check_append(cache, before, k16, qkv[:, nq + nkv:], plan.slots)
        _check_attention(out, None, q, cache, tables, plan.cu_q, plan.kv_lens)

    def run(max_q=None, graph=None, res=None):
        fresh()
        before, t0, nf0, l0 = _np(*cache), tables.cpu().numpy(), int(n_free), lens.cpu().numpy()
        if graph is None:
            res = step(max_q)
        else:
            graph.replay()
        torch.cuda.synchronize()
        N.read_status(st, "step")
        check(before, t0, nf0, l0, *res)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q_lens.copy_(_i32([20, 0, 33]))
        run(33)                                            # prompts; request 1 sits out
        q_lens.copy_(_i32([1, 17, 1]))
        run(17)
        q_lens.copy_(_i32([1, 1, 1]))
        run(1)
        state = [t.clone() for t in (*cache, tables, n_free, lens)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = step(1)
        for t, s in zip((*cache, tables, n_free, lens), state):
            t.copy_(s)
        for _ in range(20):
            run(graph=graph, res=res)
        P.page_release(torch.tensor([False, True, False], device="cuda"), tables, free, n_free, st)
        lens[1] = 0
        q_lens.copy_(_i32([1, 30, 0]))
        run(30)                                            # the freed pages' next owner
        q_lens.copy_(_i32([1, 1, 1]))
        for _ in range(3):
            run(graph=graph, res=res)
    torch.cuda.current_stream().wait_stream(side)


# ─── sizes at which a call takes another way ──────────────────────────────────
@pytest.mark.parametrize("rows_each,requests,page,dim,nkv", [
    (1, 1100, 16, 128, 2), (1, 600, 64, 64, 1), (3, 400, 32, 128, 1), (1, 20, 128, 128, 5), (17, 70, 16, 64, 3),
])
def test_kv_append_many_short_runs(P, N, rows_each, requests, page, dim, nkv):
    """A decode step of many requests: every run enters a page that holds tokens already, or begins one."""
    g = _gen(rows_each + requests)
    n_pages = requests * 2 + 3
    at = torch.randint(0, page, (requests, 1), generator=g, device="cuda") + torch.arange(rows_each, device="cuda")
    order = torch.randperm(n_pages, generator=g, device="cuda")[:2 * requests].view(requests, 2)
    slots = (order.gather(1, at // page) * page + at % page).view(-1)
    slots[rows_each * 5:rows_each * 6] = -1
    cache = _cache(n_pages, nkv, page, dim, seed=requests)
    before = _np(*cache)
    kv = torch.randn(slots.numel(), 2 * nkv, dim, generator=g, device="cuda")
    kv = (kv * 10.0 ** torch.randint(-3, 3, (slots.numel(), 1, 1), generator=g, device="cuda")).half()
    st = N.new_status("cuda")
    P.kv_append(kv[:, :nkv], kv[:, nkv:], slots, *cache, status=st)
    N.read_status(st, "kv_append")
    _check_append(cache, before, kv[:, :nkv], kv[:, nkv:], slots)


@pytest.mark.parametrize("lens,page", [((500,), 32), ((1023, 0), 64), ((700, 324), 16), ((1, 1500, 800), 128),
                                       ((33,) * 40, 64)])
@pytest.mark.parametrize("dim,rotary,interleaved,aligned", [(128, 128, False, True), (128, 64, True, True),
                                                            (64, 64, False, True), (64, 22, False, False)])
def test_rope_append_of_prompts_is_rope_then_append(P, N, lens, page, dim, rotary, interleaved, aligned):
    nq, nkv, g = 4, 2, _gen(sum(lens) + dim)
    spans = [((7 * r) % 50, n) for r, n in enumerate(lens)]
    pos = torch.cat([torch.arange(s, s + n, device="cuda") for s, n in spans] + [_i64([-1] * 3)])
    wide = -(-max(s + n for s, n in spans) // page) * page
    slots = torch.cat([torch.arange(s, s + n, device="cuda") + wide * r for r, (s, n) in enumerate(spans)]
                      + [_i64([-1] * 3)])
    rows = pos.numel()
    cos, sin = _angles(P, 1600, rotary)
    qkv = torch.randn(rows, (nq + 2 * nkv) * dim + 1, generator=g, device="cuda").half()
    qkv = (qkv[:, :-1].contiguous() if aligned else qkv[:, 1:]).unflatten(1, (nq + 2 * nkv, dim))
    q, k, v = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    n_pages = len(lens) * wide // page
    a, b = _cache(n_pages, nkv, page, dim, seed=2), _cache(n_pages, nkv, page, dim, seed=2)
    st = N.new_status("cuda")
    before = _np(*a)
    k1 = torch.zeros_like(k, memory_format=torch.contiguous_format)
    q1, _ = P.rope(q, k, cos, sin, pos, interleaved=interleaved, k_out=k1, status=st)
    P.kv_append(k1, v, slots, *a, status=st)
    _check_append(a, before, k1, v, slots)
    q2 = torch.full_like(q1, 3.0)
    P.rope_append(q, k, v, cos, sin, pos, slots, *b, interleaved=interleaved, q_out=q2, status=st)
    N.read_status(st, "rope_append")
    assert torch.equal(q1[:-3], q2[:-3]) and (q2[-3:] == 3).all()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("requests", [33, 257, 2048])
def test_paged_attention_many_requests(P, N, requests):
    """More requests than a kernel keeps the lengths of; some without keys, some with many rows."""
    page, nq, nkv, dim = 16, 8, 2, 64
    g = _gen(requests)
    spans = [(1 + (13 * r) % 40, (1 + r % 3) if r % 7 else 0) for r in range(requests)]
    spans = [(max(kv, n), n) for kv, n in spans]
    spans[requests // 2] = (90, 70)                  # several tiles
    spans[-1] = (50, 9)
    spans[3] = (0, 0)
    tables, cu, kv, n_pages = _step(spans, page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    rows = int(cu[-1])
    q = torch.randn(rows + 1, nq, dim, generator=g, device="cuda").half()
    st = N.new_status("cuda")
    for max_q in (1, 70):
        out, lse = torch.full_like(q, 9.0), torch.full((rows + 1, nq), 9.0, device="cuda")
        P.paged_attention(q, *cache, tables, cu, kv, max_q=max_q, out=out, lse=lse, status=st)
        N.read_status(st, "paged_attention")
        assert (out[rows] == 9).all()
        _check_attention(out, lse, q, cache, tables, cu, kv)


@pytest.mark.parametrize("spans", [[(300, 1), (5, 1), (9000, 1)], [(300, 200), (40, 1)], [(6000, 50)]])
def test_paged_attention_over_its_queries_and_any_scale(P, N, spans):
    page, nq, nkv, dim = 64, 8, 2, 128
    g = _gen(len(spans))
    tables, cu, kv, n_pages = _step(spans, page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    q = torch.randn(int(cu[-1]), nq, dim, generator=g, device="cuda").half()
    m = max(n for _, n in spans)
    want = P.paged_attention(q, *cache, tables, cu, kv, max_q=m)
    inplace = q.clone()
    assert P.paged_attention(inplace, *cache, tables, cu, kv, max_q=m, out=inplace) is inplace
    assert torch.equal(inplace, want)
    for scale in (0.0, -0.07):                       # the mean of the values; signs turned
        out = P.paged_attention(q, *cache, tables, cu, kv, max_q=m, scale=scale)
        _check_attention(out, None, q, cache, tables, cu, kv, scale=scale)
    with pytest.raises(N.HotColdError):
        P.paged_attention(q, *cache, tables, cu, kv, max_q=m, scale=float("nan"))


def test_two_graphs_replayed_beside_each_other(P, N):
    """Two captured calls hold a workspace each: they may run at once."""
    page, nq, nkv, dim = 64, 8, 2, 128
    g = _gen(77)
    sides = []
    for spans in ([(7000, 1), (300, 1)], [(5000, 40), (9000, 1)]):
        tables, cu, kv, n_pages = _step(spans, page, g)
        cache = _filled(n_pages, nkv, page, dim, g)
        q = torch.randn(int(cu[-1]), nq, dim, generator=g, device="cuda").half()
        m = max(n for _, n in spans)
        want = P.paged_attention(q, *cache, tables, cu, kv, max_q=m)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = P.paged_attention(q, *cache, tables, cu, kv, max_q=m)
        sides.append((stream, graph, out, want, (q, cache, tables, cu, kv)))
    for _ in range(30):
        for stream, graph, *_ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, want, _ in sides:
        assert torch.equal(out, want)


def test_paged_cache_object(P, N):
    """plan, append, attend, commit, release and check as methods, over two layers of one table."""
    c = P.PagedKVCache(2, 2, 64, 7, page_size=16, max_requests=3, max_len=64)
    assert len(c) == 2 and c.tables.shape == (3, 4) and [t.shape[0] for t in c[1]] == [7] * 4
    g = _gen(5)
    q_lens = _i32([20, 0, 30])
    plan = c.plan(q_lens, 52)
    kv = torch.randn(2, 2, 52, 2, 64, generator=g, device="cuda").half()
    q = torch.randn(52, 4, 64, generator=g, device="cuda").half()
    for layer in range(2):
        before = _np(*c[layer])
        c.append(layer, kv[layer, 0], kv[layer, 1], plan)
        _check_append(c[layer], before, kv[layer, 0], kv[layer, 1], plan.slots)
        out = torch.zeros_like(q)
        c.attend(layer, q, plan, max_q=30, out=out)
        _check_attention(out, None, q, c[layer], c.tables, plan.cu_q, plan.kv_lens)
    c.commit(plan)
    c.check()
    assert c.lens.tolist() == [20, 0, 30] and int(c.n_free) == 3
    c.release(torch.tensor([False, False, True], device="cuda"))
    assert c.lens.tolist() == [20, 0, 0] and int(c.n_free) == 5 and (c.tables[2] == -1).all()
    plan = c.plan(_i32([0, 0, 64]), 64)
    assert int(c.n_free) == 1
    c.check()
    plan = c.plan(_i32([0, 40, 64]), 104)            # more pages than are left: nothing is taken
    assert int(c.n_free) == 1 and (plan.slots == -1).all()
    with pytest.raises(N.HotColdError):
        c.check()


@pytest.mark.parametrize("kv_len", [300, 6000])
def test_paged_attention_offsets_that_go_back_and_forth(P, N, kv_len):
    """Every other request claims the same rows: more tiles than the rows allow."""
    page, nq, nkv, dim, n = 64, 8, 2, 64, 60
    g = _gen(kv_len)
    tables, _, _, n_pages = _step([(kv_len, 0)], page, g)
    cache = _filled(n_pages, nkv, page, dim, g)
    q = torch.randn(100, nq, dim, generator=g, device="cuda").half()
    out, st = torch.full((101, nq, dim), 9.0, device="cuda").half(), N.new_status("cuda")
    cu = _i32([0, 100] * (n // 2) + [0])
    P.paged_attention(q, *cache, tables.expand(n, -1).contiguous(), cu, _i32([kv_len] * n), max_q=100, out=out[:100],
                      status=st)
    assert int(st) == N.HC_ERR_RANGE and (out[100] == 9).all()
    good, st = _i32([0, 100]), N.new_status("cuda")        # the next call is none the worse
    lens = _i32([kv_len])
    got = P.paged_attention(q, *cache, tables, good, lens, max_q=100, status=st)
    N.read_status(st, "paged_attention")
    _check_attention(got, None, q, cache, tables, good, lens)


@pytest.mark.parametrize("row", [[3, -1, 5, 7], [3, 4, 9, -1], [3, -7, 5, 6]])
def test_page_release_of_a_row_with_a_hole_or_a_stray_page(P, N, row):
    tables, free, n_free, st = _i32([row, [1, 2, -1, -1]]), _i32([0] + [-1] * 8), _i32([1]), N.new_status("cuda")
    before = tables.clone()
    P.page_release(torch.tensor([True, True], device="cuda"), tables, free, n_free, st)
    assert int(st) == N.HC_ERR_RANGE and int(n_free) == 1 and torch.equal(tables, before)
    assert free.tolist() == [0] + [-1] * 8
