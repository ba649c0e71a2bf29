"""The engine's paged steps that do not fit, and what generate_batch answers, checked from outside."""
import pytest
import torch

from test_gpu_paged_engine import LOGIT_TOL, VOCAB, _Plain, _rel, make

pytestmark = pytest.mark.gpu


def _tokens(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


def test_forward_paged_refuses_a_step_without_pages(make):
    """Pages run out in the middle of a run: the step raises and takes nothing, and after a release it runs as if it
    had not been tried."""
    eng = make()
    page = 16
    cache, twin = (eng.new_paged_cache(2, n_pages=4, page_size=page, max_len=200) for _ in range(2))
    a, b, c = _tokens(40, 1), _tokens(20, 2), _tokens(9, 3)
    first = eng.forward_paged(a, [40, 0], cache)                       # 3 of 4 pages
    assert _rel(first, eng.forward_paged(a, [40, 0], twin)) < LOGIT_TOL
    state = [t.clone() for t in (cache.lens, cache.tables, cache.n_free, cache.k, cache.v, cache.k_scale)]
    for _ in range(2):
        with pytest.raises(ValueError, match="fit"):
            eng.forward_paged(b, [0, 20], cache)
    with pytest.raises(ValueError, match="fit"):
        eng.forward_paged(torch.cat([c, b]), [9, 20], cache)           # neither request, though one would fit
    now = (cache.lens, cache.tables, cache.n_free, cache.k, cache.v, cache.k_scale)
    assert all(torch.equal(x, y) for x, y in zip(state, now))
    cache.check()                                                      # reported by the exception already
    assert _rel(eng.forward_paged(c, [9, 0], cache), eng.forward_paged(c, [9, 0], twin)) < LOGIT_TOL
    done = torch.tensor([True, False], device="cuda")
    cache.release(done)
    twin.release(done)
    assert _rel(eng.forward_paged(b, [0, 20], cache), eng.forward_paged(b, [0, 20], twin)) < LOGIT_TOL
    cache.check()
    eng.check()
    # an error that was there before the refused step is still reported
    cache.status.fill_(4)
    with pytest.raises(ValueError, match="fit"):
        eng.forward_paged(_tokens(60, 4), [60, 0], cache)
    assert int(cache.status) == 4
    # a request that outgrows its table row
    small = eng.new_paged_cache(1, n_pages=20, page_size=page, max_len=32)
    eng.forward_paged(_tokens(32, 5), [32], small)
    with pytest.raises(ValueError, match="fit"):
        eng.forward_paged(_tokens(1, 6), [1], small)
    assert small.lens.tolist() == [32]


def test_forward_paged_refuses_positions_past_max_len(make):
    """max_len is not a multiple of the page: the rest of the last page is not for use."""
    eng = make()
    cache = eng.new_paged_cache(2, page_size=16, max_len=20)
    eng.forward_paged(_tokens(19, 1), [19], cache)
    with pytest.raises(ValueError, match="20 positions"):
        eng.forward_paged(_tokens(2, 2), [2], cache)
    eng.forward_paged(_tokens(1, 3), [1], cache)
    with pytest.raises(ValueError, match="20 positions"):
        eng.forward_paged(_tokens(1, 4), [1], cache)
    assert cache.lens.tolist() == [20, 0]
    cache.check()


def test_engine_builds_with_stock_rope_scaling(make):
    plain = make().cos_cache
    for stock, same in (({"type": "yarn", "factor": 4.0}, False), ({"type": "dynamic", "factor": 2.0}, True),
                        ({"rope_type": "default"}, True)):       # dynamic: the engine ends at the original length
        got = make(rope_scaling=stock).cos_cache
        assert ((got - plain).abs().max() < 1e-3) == same          # fp32 angles against 64-bit ones
    with pytest.warns(UserWarning, match="not scaled"):
        eng = make(rope_scaling={"type": "longrope", "factor": 4.0}, partial_rotary_factor=None)
    assert torch.equal(eng.cos_cache, plain)


def test_split_to_engine_keeps_the_rotary_layout(tmp_path):
    """From a model's configuration through split_dense to the engine's tables."""
    import json
    import os
    import sys

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    sys.path.insert(0, os.path.join(os.path.dirname(__file__), "golden"))
    import engine
    import paged
    import splitter
    import stub_models
    model = stub_models.engine_stub_model()
    model.config.rope_scaling = {"rope_type": "linear", "factor": 4.0}
    model.config.partial_rotary_factor = 0.5
    profile = tmp_path / "profile.json"
    profile.write_text(json.dumps(stub_models.engine_stub_profile()))
    splitter.split_dense(model, str(profile), str(tmp_path / "split"), hot_count=16)
    eng = engine.DesdemonaEngine(str(tmp_path / "split"), max_seq_len=64)
    cos, sin = paged.rope_tables(64, 64, 10000.0, {"rope_type": "linear", "factor": 4.0}, device="cuda")
    assert torch.equal(eng.cos_cache, cos) and torch.equal(eng.sin_cache, sin)
    assert len(eng.generate_batch([_tokens(5, 1) % 64, _tokens(9, 2) % 64], 4, temperature=0.0)[1]) == 4


def _follows(eng, prompt, made):
    """Every token that was made has the plain model's largest logit to the engine's tolerance: an element is off by
    at most the norm's bound, its own logit and the largest one."""
    ids = torch.cat([prompt, torch.tensor(made, device="cuda")])[:-1]
    page = 16
    cache, plain = eng.new_paged_cache(1, page_size=page), _Plain(eng, 512 // page, page)
    with torch.inference_mode():
        plan = cache.plan(torch.tensor([len(ids)], dtype=torch.int32, device="cuda"), len(ids))
        logits = plain.step(ids, plan, cache.tables.cpu().numpy())[len(prompt) - 1:].double()
    short = logits.max(-1).values - logits.gather(1, torch.tensor(made, device="cuda")[:, None])[:, 0]
    return bool((short <= 2 * LOGIT_TOL * logits.norm(dim=-1)).all())


def test_generate_batch_follows_the_plain_model(make):
    """Greedy tokens of three prompts against the plain model, and again with an end token that takes one request out
    in the middle, whose pages the others then grow into."""
    eng = make()
    prompts = [_tokens(n, n) for n in (5, 70, 33)]
    full = eng.generate_batch(prompts, 40, temperature=0.0, page_size=16)
    assert [len(r) for r in full] == [40] * 3
    for p, r in zip(prompts, full):
        assert _follows(eng, p, r)
    assert not _follows(eng, prompts[0], full[1])            # the check tells requests apart
    # an end token that one request makes among its first 15 and the others never do
    picks = [(r, t) for r in range(3) for t in full[r][:15] if all(t not in full[o] for o in range(3) if o != r)]
    assert picks
    for r, eos in (picks[0], picks[-1]):
        cut = eng.generate_batch(prompts, 40, temperature=0.0, eos_token_id=[eos, VOCAB + 1], page_size=16)
        for i, (p, row) in enumerate(zip(prompts, cut)):
            assert _follows(eng, p, row)
            assert (row.index(eos) == len(row) - 1) if eos in row else len(row) == 40
        assert cut[r][-1] == eos and len(cut[r]) <= 40
    eng.check()


def test_generate_batch_of_one_is_the_step_by_step_loop(make):
    eng = make()
    prompt = _tokens(20, 9)
    cache, tok, want = eng.new_paged_cache(1, page_size=32, max_len=60), prompt, []
    for _ in range(24):
        tok = eng.forward_paged(tok, [len(tok)], cache).argmax(-1)
        want.append(int(tok))
    got = eng.generate_batch([prompt], 24, temperature=0.0, page_size=32)[0]
    assert len(got) == 24 and _follows(eng, prompt, got) and _follows(eng, prompt, want)
    cache.check()


def test_generate_batch_up_to_the_last_position(make):
    """As generate(): the last token that is made takes no position."""
    eng = make()
    prompt = _tokens(500, 3)
    one = eng.generate(prompt, 13, temperature=0.0)
    got = eng.generate_batch([prompt, prompt[:16]], 13, temperature=0.0, page_size=16)
    assert [len(r) for r in (one, *got)] == [13] * 3
    with pytest.raises(ValueError):
        eng.generate_batch([prompt], 14, temperature=0.0)
    eng.check()
