"""The decode step over quantised caches and with sampled tokens: DecodeState(kv_bits=, sampler=) and generate().

The caches that a state starts from are compared bit for bit with kv_quantize of the prefill's rows; its logits with
those of a twin whose attention is computed in float64 over the caches' values and rounded to bf16 once, within the
2e-2 (relative L2, and absolute relative to max(1, |ref|)) that several bf16 layers make of differing roundings;
replays of the captured step with the eager step bit for bit."""
import pytest
import torch

from tests.attn_util import assert_close_grad, to_np
from tests.test_inference_gpu import _model, _prompts, _Streamer, _Tok
from tests.test_kvquant_gpu import clone_cache, values_of

pytestmark = pytest.mark.gpu


def _prefill(m, headroom, steps, prune=False):
    from tokengate_amd import inference as I
    split = [I.split_state_span(p) for p in _prompts([600, 333, 70], [(20, 500), (0, 300), (5, 60)], 5)]
    return m.prefill(split, [64, 1000, 7], prune_below_gate=prune, decode_headroom=steps + 1 if headroom else 0)


def _attention64(qkv, rope, lw, shape, cache, kv_start, kv_used, max_k, scale, workspace, bias_raw=None, q_head_scale=None,
                 q_row_scale=None, out=None):
    """decode_attention_quant with its attention in float64."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    pos = torch.zeros(qkv.shape[0], dtype=torch.int64, device=qkv.device)
    k1, v1 = (torch.zeros(qkv.shape[0], shape.n_kv_heads, 128, dtype=torch.bfloat16, device=qkv.device) for _ in range(2))
    # the rotary table as the angles of one position each (the kernel of the prefill rotates by pos * inv_freq)
    q = torch.empty(qkv.shape[0], shape.n_heads, 128, dtype=torch.bfloat16, device=qkv.device)
    for b in range(qkv.shape[0]):
        ang = torch.atan2(rope[b, :, 1].double(), rope[b, :, 0].double()).float()
        q[b] = dec.qk_norm_rope(qkv[b:b + 1].clone(), pos[:1] + 1, lw, shape, ang, k1[b:b + 1], v1[b:b + 1], q_head_scale,
                                q_row_scale[b:b + 1] if q_row_scale is not None else None)[0]
    Q.kv_quantize(k1, v1, cache, dst_rows=kv_start + kv_used - 1)
    k, v = (t.to(qkv.device) for t in values_of(cache))
    g = shape.n_heads // shape.n_kv_heads
    for b in range(qkv.shape[0]):
        s, n = int(kv_start[b]), int(kv_used[b])
        kk, vv = (t[s:s + n].repeat_interleave(g, 1).transpose(0, 1) for t in (k, v))
        z = (kk * q[b].double()[:, None]).sum(-1)
        if bias_raw is not None:
            z = z + bias_raw[b, :, :n].double()
        out[b] = (torch.softmax(z * scale, -1)[..., None] * vv).sum(1).bfloat16()
    return out


@pytest.mark.parametrize("bits,headroom,prune,ssmax", [(4, False, False, False), (4, True, True, True), (8, True, False, True),
                                                       (8, False, True, False)])
def test_decode_over_quantised_caches(cuda, monkeypatch, bits, headroom, prune, ssmax):
    from tokengate_amd import decode as D
    from tokengate_amd import kvquant as Q
    m = _model(cuda, ssmax=ssmax)
    steps = 3
    pfs = [_prefill(m, headroom, steps, prune) for _ in range(2)]
    st = D.DecodeState(m.weights, m.gate, m.gate_layer, pfs[0], steps + 1, prune, kv_bits=bits)
    for l, kv in enumerate(st.kv):
        pf, g = pfs[0], 0 if l <= m.gate_layer else 1
        cu = pf.cu_kept if prune or g else pf.cu_prompt
        gap = pf.decode_headroom
        for b in range(3):
            n, s = cu[b + 1] - cu[b], st.groups[g].seg[b]
            src = slice(cu[b] + b * gap, cu[b] + b * gap + n)
            one = Q.QuantKV.alloc(n, kv.n_kv_heads, bits, cuda)
            Q.kv_quantize(pf.kv[l].k[src], pf.kv[l].v[src], one)
            assert torch.equal(kv.k[:, s:s + n], one.k) and torch.equal(kv.v_meta[:, s:s + n], one.v_meta)
            assert torch.equal(kv.v[:, s:s + n], one.v) and torch.equal(kv.k_meta[:, s:s + n], one.k_meta)
            assert not bool(kv.k[:, s + n:s + n + steps + 1].any())
    twin = D.DecodeState(m.weights, m.gate, m.gate_layer, pfs[1], steps + 1, prune, kv_bits=bits)
    cur = pfs[0].first_tokens
    for i in range(steps):
        nxt = st.step(cur)
        with monkeypatch.context() as mp:
            mp.setattr(D, "decode_attention_quant", _attention64)
            twin.step(cur)
        torch.cuda.synchronize()
        for b in range(3):
            assert_close_grad(f"seq {b} step {i}", to_np(st.last_logits[b].float().cpu()), to_np(twin.last_logits[b].float().cpu()),
                              rel_l2=2e-2)
        assert torch.equal(nxt, st.last_logits.argmax(1))
        cur = nxt


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_graph_replays_match_eager(cuda, bits):
    """Quantised caches and sampled tokens in the captured step: every replay equals the eager step, with eager work
    between the replays."""
    from tokengate_amd import decode as D
    m = _model(cuda, seed=6, ssmax=True)
    steps = 6
    pfs = [_prefill(m, True, steps) for _ in range(2)]
    sam = [D.TokenSampler(D.Sampling([0.8, 0.0, 1.2], [0, 5, 40], [0.9, 1.0, 0.95], 0.01, seed=3), 3, m.config.vocab, steps + 1, cuda)
           for _ in range(2)]
    eager = D.DecodeState(m.weights, m.gate, m.gate_layer, pfs[0], steps + 1, kv_bits=bits, sampler=sam[0])
    graph = D.DecodeState(m.weights, m.gate, m.gate_layer, pfs[1], steps + 1, graph=True, kv_bits=bits, sampler=sam[1])
    ce = cg = pfs[0].first_tokens
    for i in range(steps):
        ce, cg = eager.step(ce), graph.step(cg)
        junk = torch.randn(1 << 20, device=cuda).sum()
        torch.cuda.synchronize()
        assert torch.equal(ce, cg) and torch.equal(eager.last_logits, graph.last_logits), i
        assert torch.equal(eager.last_logprobs, graph.last_logprobs) and bool(torch.isfinite(junk))
        assert int(ce[1]) == int(eager.last_logits[1].argmax())
    with pytest.raises(RuntimeError, match="random numbers"):
        eager.step(ce)


def test_generate_with_sampling_and_quantised_caches(cuda):
    from tokengate_amd import inference as I
    m = _model(cuda, seed=4)
    prompts = _prompts([400, 250], [(10, 380), (5, 240)], 9)
    kw = dict(max_new_tokens=6, max_kept_prefill_tokens=[50, 10_000])
    greedy = m.generate(prompts, None, **kw)
    assert greedy.logprobs is None
    one = m.generate(prompts, None, temperature=0.9, top_k=1, **kw)
    assert one.token_ids == greedy.token_ids and all(abs(p) < 1e-6 for row in one.logprobs for p in row)
    a = m.generate(prompts, None, temperature=1.5, top_p=0.98, seed=11, **kw)
    b = m.generate(prompts, None, temperature=1.5, top_p=0.98, seed=11, **kw)
    c = m.generate(prompts, None, temperature=1.5, top_p=0.98, seed=12, **kw)
    assert a.token_ids == b.token_ids and a.logprobs == b.logprobs and a.token_ids != c.token_ids
    assert all(len(t) == 6 and len(p) == 6 and all(x <= 0 for x in p) for t, p in zip(a.token_ids, a.logprobs))
    mixed = m.generate(prompts, None, temperature=[0.0, 1.5], seed=11, **kw)
    assert mixed.token_ids[0] == greedy.token_ids[0]
    for bits in (8, 4):
        q = m.generate(prompts, None, kv_bits=bits, **kw)
        assert all(len(t) == 6 for t in q.token_ids) and [t[0] for t in q.token_ids] == [t[0] for t in greedy.token_ids]
        assert q.n_kept == greedy.n_kept and q.kept_pos == greedy.kept_pos
    # the first EOS ends a row, its log probability included
    eos = a.token_ids[0][2]
    streamer = _Streamer()
    out = m.generate(prompts, _Tok(eos), temperature=1.5, top_p=0.98, seed=11, streamer=streamer, kv_bits=16, **kw)
    n = a.token_ids[0].index(eos) + 1
    assert out.token_ids[0] == a.token_ids[0][:n] and out.logprobs[0] == a.logprobs[0][:n] and streamer.ended
    for bad in (dict(kv_bits=2), dict(temperature=-1.0), dict(top_p=1.5, temperature=1.0), dict(temperature=[1.0])):
        with pytest.raises(ValueError):
            m.generate(prompts, None, **bad, **kw)


def test_release_and_refusals(cuda):
    from tokengate_amd import decode as D
    m = _model(cuda, seed=4)
    pf = _prefill(m, False, 3)
    with pytest.raises(ValueError, match="kv_bits"):
        D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, kv_bits=5)
    few = D.TokenSampler(D.Sampling(), 3, m.config.vocab, 2, cuda)
    with pytest.raises(ValueError, match="random numbers"):
        D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, sampler=few)
    st = D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, kv_bits=4, release_kv=True)
    assert all(kv is None for kv in pf.kv)
    first = clone_cache(st.kv[0])
    st.step(pf.first_tokens)
    torch.cuda.synchronize()
    for b, s in enumerate(st.groups[0].seg):               # one row after each sequence, and nothing else, has changed
        n = st.groups[0].n0[b]
        assert torch.equal(st.kv[0].k[:, s:s + n], first.k[:, s:s + n]) and bool(st.kv[0].k[:, s + n].any())
        assert not bool(st.kv[0].k[:, s + n + 1:s + n + 4].any())


@pytest.mark.parametrize("draws,steps", [(4, 3), (5, 4), (9, 4)])
def test_steps_that_a_sampler_allows(cuda, draws, steps):
    """A state takes max_steps steps, one less than its sampler has random numbers for (the first are the first token's), and
    max_new_tokens at most; each with its own."""
    from tokengate_amd import decode as D
    m = _model(cuda, seed=4)
    pf = _prefill(m, False, 4)
    sam = D.TokenSampler(D.Sampling(1.3, seed=5), 3, m.config.vocab, draws, cuda)
    st = D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, kv_bits=8, sampler=sam)
    assert st.max_steps == steps
    sam.set_step(0)
    cur, _ = sam(pf.logits.float())
    for i in range(steps):
        cur = st.step(cur)
        assert torch.equal(sam.u, sam.draws[i + 1])
        assert torch.equal(cur, sam(st.last_logits)[0])
    with pytest.raises(RuntimeError, match="random numbers" if draws == 4 else "full"):
        st.step(cur)
    assert D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, kv_bits=8).max_steps == 4


def test_samplers_of_another_batch(cuda):
    """A sampler for other sequences or fewer tokens than the state's is refused before anything is appended."""
    from tokengate_amd import decode as D
    m = _model(cuda, seed=4)
    pf = _prefill(m, False, 4)
    for b, vocab in ((2, m.config.vocab), (4, m.config.vocab), (3, m.config.vocab - 1)):
        sam = D.TokenSampler(D.Sampling(), b, vocab, 6, cuda)
        with pytest.raises(ValueError, match="sampler is for"):
            D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, sampler=sam)
    D.DecodeState(m.weights, m.gate, m.gate_layer, pf, 4, sampler=D.TokenSampler(D.Sampling(), 3, m.config.vocab, 6, cuda))


@pytest.mark.parametrize("B,bits", [(3, 4), (8, 16), (11, 8), (11, 16)])
def test_long_vocabularies_and_batches(cuda, B, bits):
    """A vocabulary whose sampling takes two launches and a workspace, inside the captured step, and batches of more rows than
    the fused projections take: every replay equals the eager step, and every token is what the definition draws from
    the step's logits."""
    import numpy as np
    from tests.test_inference_gpu import SMALL
    from tests.test_sample_gpu import reference
    from tokengate_amd import decode as D
    from tokengate_amd import decoder as dec
    from tokengate_amd import inference as I
    m = I.load_model("random:9", gate_layer=1, device=cuda, shape=dec.DecoderShape(**dict(SMALL, vocab=20480)))
    lens = [70 + 41 * b for b in range(B)]
    split = [I.split_state_span(p) for p in _prompts(lens, [(5, n - 10) for n in lens], 6)]
    steps = 4
    pfs = [m.prefill(split, [40] * B, decode_headroom=steps + 1) for _ in range(2)]
    kind = [b % 4 for b in range(B)]
    s = D.Sampling([0.0 if k == 0 else 0.7 + 0.1 * k for k in kind], [20 if k == 1 else 0 for k in kind],
                   [0.9 if k == 2 else 1.0 for k in kind], [0.02 if k == 3 else 0.0 for k in kind], seed=4)
    sam = [D.TokenSampler(s, B, 20480, steps + 1, cuda) for _ in range(2)]
    eager = D.DecodeState(m.weights, m.gate, m.gate_layer, pfs[0], steps, kv_bits=bits, sampler=sam[0])
    graph = D.DecodeState(m.weights, m.gate, m.gate_layer, pfs[1], steps, graph=True, kv_bits=bits, sampler=sam[1])
    ce = cg = pfs[0].first_tokens
    near = 0
    for i in range(steps):
        ce, cg = eager.step(ce), graph.step(cg)
        junk = torch.randn(1 << 20, device=cuda).sum()
        torch.cuda.synchronize()
        assert torch.equal(ce, cg) and torch.equal(eager.last_logits, graph.last_logits), i
        assert torch.equal(eager.last_logprobs, graph.last_logprobs) and bool(torch.isfinite(junk))
        for b in range(B):
            t, k, p, mp = (float(np.float32(v[b])) for v in (s.temperature, s.top_k, s.top_p, s.min_p))
            tok, lp, border = reference(eager.last_logits[b].cpu().numpy(), float(sam[0].u[b]), t, int(k), p, mp)
            near += border
            if not border:
                assert int(ce[b]) == tok and abs(float(eager.last_logprobs[b]) - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -34
    assert near <= 1


def test_generate_with_a_padded_vocabulary(cuda):
    """A head of more rows than the configuration's vocabulary (padded ones): sampling is over the head's."""
    import dataclasses
    from tests.test_inference_gpu import SMALL
    from tokengate_amd import decoder as dec
    from tokengate_amd import inference as I
    m = I.load_model("random:9", gate_layer=1, device=cuda, shape=dec.DecoderShape(**dict(SMALL, vocab=20480)))
    prompts = _prompts([90, 120], [(5, 80), (10, 100)], 3)
    want = m.generate(prompts, None, max_new_tokens=4, temperature=1.2, seed=2)
    m.weights.shape = dataclasses.replace(m.config, vocab=2000)
    got = m.generate(prompts, None, max_new_tokens=4, temperature=1.2, seed=2)
    assert got.token_ids == want.token_ids and got.logprobs == want.logprobs
