"""The engine over the paged 8-bit cache, and configurations with other rotary layouts.

The model's plain form runs the engine's own norms, projections and FFN layers
and computes the attention in 64 bits from the definitions (rotation, e4m3 pages,
causal softmax; oracle/paged_oracle.py).  Logits agree to 2e-2, the tolerance of
the engine's other tests: fp16 projections and an FFN whose sums run in another
order.  Without predictors every record is fetched, so that tolerance is not
crossed by a fetch set that another rounding decided.
"""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
LOGIT_TOL = 2e-2
L, H, VOCAB, NQ, NKV, INTER = 2, 4096, 256, 32, 8, 1024


@pytest.fixture(scope="module")
def make():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import engine
    import hc_synth
    syn = hc_synth.make_stack(n_layers=L, inter=INTER, hot_frac=0.2, rank=64, activation="silu", act_on_both=False,
                              seed=7)
    g = torch.Generator(device="cuda").manual_seed(8)
    shared = {}
    for li in range(L):
        for name, rows in (("q_proj", H), ("k_proj", NKV * 128), ("v_proj", NKV * 128), ("o_proj", H)):
            shared[f"layer_{li:03d}.{name}"] = (torch.randn(rows, H, generator=g, device="cuda") * 0.02).to(
                torch.float8_e4m3fn)
        shared[f"layer_{li:03d}.input_layernorm"] = (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).half()
        shared[f"layer_{li:03d}.post_attention_layernorm"] = syn.norms[li].half()
    shared["embed_tokens"] = torch.randn(VOCAB, H, generator=g, device="cuda").half()
    shared["lm_head"] = (torch.randn(VOCAB, H, generator=g, device="cuda") * 0.02).half()
    base = {"hidden_dim": H, "intermediate_dim": INTER, "num_layers": L, "vocab_size": VOCAB,
            "num_attention_heads": NQ, "num_key_value_heads": NKV, "rope_theta": 500000.0, "rms_norm_eps": 1e-5,
            "hidden_act": "silu", "act_on_both": False, "max_position_embeddings": 512, "num_experts": 1}

    def build(**extra):
        return engine.DesdemonaEngine.from_parts({**base, **extra}, dict(shared), syn.store, syn.hot, None,
                                                 device="cuda", max_seq_len=512)
    return build


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


class _Plain:
    """The engine's steps with the attention in 64 bits over its own copy of the pages."""

    def __init__(self, eng, n_pages, page):
        self.eng, self.page = eng, page
        self.pages = [[np.zeros((n_pages, NKV, page, 128), np.uint8) for _ in range(2)] for _ in range(L)]
        self.scales = [[np.zeros((n_pages, NKV)) for _ in range(2)] for _ in range(L)]

    def step(self, tokens, plan, tables):
        e = self.eng
        pos, slots = plan.positions.cpu().numpy(), plan.slots.cpu().numpy()
        cos, sin = e.cos_cache.double().cpu().numpy(), e.sin_cache.double().cpu().numpy()
        x = e.embed_tokens(tokens)
        rows = x.shape[0]
        words = [f._mask_words(x.view(rows, 1, -1)) for f in e.ffn_layers]
        for li, att in enumerate(e.attention_layers):
            qkv = torch.nn.functional.linear(att.norm(x), att.qkv_weight).view(rows, NQ + 2 * NKV, 128)
            q, k, v = (t.double().cpu().numpy() for t in (qkv[:, :NQ], qkv[:, NQ:NQ + NKV], qkv[:, NQ + NKV:]))
            q = O.rotate(q, cos, sin, pos, att.rope_interleaved).astype(np.float16).astype(np.float64)
            k = O.rotate(k, cos, sin, pos, att.rope_interleaved).astype(np.float16).astype(np.float64)
            for i, t in enumerate((k, v)):
                self.pages[li][i], self.scales[li][i] = O.append(self.pages[li][i], self.scales[li][i], t, slots)
            out, _ = O.attention(q, *self.pages[li], *self.scales[li], tables, plan.cu_q.cpu().numpy(),
                                 plan.kv_lens.cpu().numpy())
            out = torch.from_numpy(out.reshape(rows, -1)).cuda().half()
            x = x + torch.nn.functional.linear(out, att.o_weight)
            x = e.ffn_layers[li](x.view(rows, 1, -1), words[li]).view(rows, -1)
        return torch.nn.functional.linear(e.final_norm(x), e.lm_head_weight)


@pytest.mark.parametrize("extra", [
    {}, {"rope_interleaved": True, "partial_rotary_factor": 0.5},
    {"rope_scaling": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 128}},
])
def test_forward_paged_matches_the_plain_model(make, extra):
    eng = make(**extra)
    page = 16
    cache = eng.new_paged_cache(3, n_pages=24, page_size=page, max_len=200)
    plain = _Plain(eng, 24, page)
    gen = torch.Generator().manual_seed(2)
    # prompts, a step in which one request waits, single tokens
    for q_lens in ([21, 0, 40], [1, 17, 1], [1, 1, 1], [0, 1, 0]):
        tokens = torch.randint(0, VOCAB, (sum(q_lens),), generator=gen).cuda()
        with torch.inference_mode():
            starts = cache.lens.clone()
            plan = cache.plan(torch.tensor(q_lens, dtype=torch.int32, device="cuda"), len(tokens))
            want = plain.step(tokens, plan, cache.tables.cpu().numpy())
        got = eng.forward_paged(tokens, q_lens, cache)            # plans the same step again
        assert torch.equal(cache.lens, starts + torch.tensor(q_lens, dtype=torch.int32, device="cuda"))
        last = [int(c) - 1 for c, n in zip(plan.cu_q[1:], q_lens) if n]
        assert got.shape == (len(last), VOCAB)
        for a, b in zip(got, want[last]):
            assert _rel(a, b) < LOGIT_TOL
    cache.check()
    eng.check()


def test_other_rotary_layouts_on_the_contiguous_cache(make):
    """Part of the head and neighbouring pairs on the one-request path: prompt and tokens against fp32 torch."""
    eng = make(rope_interleaved=True, partial_rotary_factor=0.25)
    assert not any(a.fused_decode for a in eng.attention_layers)
    att = eng.attention_layers[0]
    cache = eng.new_cache(1, 64)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(1, 20, H, generator=gen, device="cuda").half()
    with torch.inference_mode():
        got = att(x, eng.cos_cache[:20], eng.sin_cache[:20], cache, 0)
        qkv = torch.nn.functional.linear(att.norm(x), att.qkv_weight).view(20, NQ + 2 * NKV, 128)
        c, s = eng.cos_cache.cpu().numpy(), eng.sin_cache.cpu().numpy()
        assert c.shape[1] == 16
        q, k = (torch.from_numpy(O.rotate(t.double().cpu().numpy(), c, s, range(20), True)).cuda()
                for t in (qkv[:, :NQ], qkv[:, NQ:NQ + NKV]))
        k, v = (t.repeat_interleave(NQ // NKV, 1) for t in (k, qkv[:, NQ + NKV:].double()))
        sc = torch.einsum("qhd,khd->hqk", q, k) / 128 ** 0.5
        sc = sc.masked_fill(torch.ones(20, 20, device="cuda").triu(1).bool(), float("-inf"))
        out = torch.einsum("hqk,khd->qhd", sc.softmax(-1), v).reshape(20, -1)
        want = out @ att.o_weight.double().T
    # fp16 q, k, v, weights and output: each rounds by 2^-11; 5e-3 leaves room for the half-precision products' sums
    assert _rel(got[0], want) < 5e-3
    toks = eng.generate(torch.randint(0, VOCAB, (1, 9), generator=torch.Generator().manual_seed(4)).cuda(), 6, 0.0)
    eager = eng.generate(torch.randint(0, VOCAB, (1, 9), generator=torch.Generator().manual_seed(4)).cuda(), 6, 0.0,
                         use_graph=False)
    assert len(toks) == 6 and toks == eager


def test_generate_batch(make):
    eng = make()
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, VOCAB, (n,), generator=gen).cuda() for n in (5, 70, 33)]
    a = eng.generate_batch(prompts, 20, temperature=0.0, page_size=16)
    assert [len(r) for r in a] == [20, 20, 20] and all(0 <= t < VOCAB for r in a for t in r)
    assert a == eng.generate_batch(prompts, 20, temperature=0.0, page_size=16)
    # an end token: kept, and nothing after it
    eos = a[1][17]
    b = eng.generate_batch(prompts, 20, temperature=0.0, eos_token_id=eos, page_size=16)
    for full, cut in zip(a, b):
        n = full.index(eos) + 1 if eos in full[:16] else len(cut)
        assert cut == full[:n] or (eos in cut and cut.index(eos) == len(cut) - 1)
    for bad in ([], [prompts[0], prompts[0][:0]], [torch.zeros(500, dtype=torch.int64)]):
        with pytest.raises(ValueError):
            eng.generate_batch(bad, 20)
    with pytest.raises(ValueError):
        eng.forward_paged(prompts[0], [4], eng.new_paged_cache(1, 4))
