"""The paged operators as a program uses them: prompts taken in chunks and decoded, prefixes shared by several sequences, captured
steps, other streams, caches past 4 GiB, and the gated prefill and decode over pages (prefill_batch(page_rows=),
DecodeState, generate(page_rows=)).  Tolerances as in test_paged_gpu; where several bf16 layers lie between, 2e-2 relative L2 as
for the other caches."""
import pytest
import torch

from paged_util import BF, D, attend, cache_of, keys_of, near, normal, shape_of, table_of, weights
from tests.attn_util import assert_close_grad, to_np
from tests.test_inference_gpu import _model, _prompts

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("page,layout", [(16, "heads"), (64, "rows"), (256, "both")])
def test_chunks_then_decode(page, layout):
    """Three sequences, each prompt in chunks of its own, then single tokens: every output against float64 attention over rows
    that qk_norm_rope made of the whole."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    g = _gen(1)
    H, Hkv, total = 16, 8, [300, 77, 130]
    shape, lw = shape_of(H, Hkv), weights(g)
    inv = dec.rope_inv_freq(shape, DEV)
    qkv = [normal(g, n, (H + 2 * Hkv) * D) for n in total]
    whole = []
    for b, n in enumerate(total):
        k, v = (torch.empty(n, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        q = dec.qk_norm_rope(qkv[b].clone(), torch.arange(n, device=DEV) + 5 * b, lw, shape, inv, k, v).clone()
        whole.append((q, k, v))
    table, n_pages = table_of(g, total, page)
    cache = cache_of(g, n_pages, Hkv, page, layout, fill=float("nan"))
    done = [0, 0, 0]

    def check(out, new):
        at = 0
        for b, m in enumerate(new):
            q, k, v = whole[b]
            n = done[b]
            if m:
                ref, mass = attend(q[n - m:n], k[:n].double(), v[:n].double(), torch.ones(n, dtype=torch.bool, device=DEV), SCALE,
                                   causal_from=n - m)
                near(out[at:at + m], ref, mass, BF, (b, n))
            at += m

    for new in ([128, 1, 40], [0, 60, 30], [150, 0, 50]):
        rows = torch.cat([qkv[b][done[b]:done[b] + m] for b, m in enumerate(new)])
        pos = torch.cat([torch.arange(done[b], done[b] + m, device=DEV) + 5 * b for b, m in enumerate(new)])
        done = [x + m for x, m in zip(done, new)]
        cu = _i32([0, new[0], new[0] + new[1], sum(new)])
        slots, rope = P.paged_begin(pos, inv, cu, _i32(done), table, cache)
        q = P.paged_append(rows, rope, lw, shape, cache, slots)
        check(P.paged_attention(q, cache, table, cu, _i32(done), max(new), 300, SCALE), new)
    ws = P.paged_decode_attention_workspace(3, shape, 300, DEV)
    pos = torch.tensor([done[b] + 5 * b for b in range(3)], device=DEV)
    used = _i32(done)
    for _ in range(5):
        rows = torch.stack([qkv[b][done[b]] for b in range(3)])
        done = [x + 1 for x in done]
        rope, _ = dec.decode_begin(pos, inv, used)
        check(P.paged_decode_attention(rows, rope, lw, shape, cache, table, used, 300, SCALE, ws), [1, 1, 1])
    for b, n in enumerate(done):
        k, v, _ = keys_of(cache, table, b, n)
        assert torch.equal(k.to(torch.bfloat16), whole[b][1][:n]) and torch.equal(v.to(torch.bfloat16), whole[b][2][:n])


def test_shared_prefix():
    """Five sequences that begin with the same two pages and go on in their own."""
    from tokengate_amd import paged as P
    g = _gen(2)
    H, Hkv, page, used = 16, 8, 32, [65, 70, 90, 66, 100]
    shape, lw = shape_of(H, Hkv), weights(g)
    cache = cache_of(g, 14, Hkv, page)
    table = torch.full((5, 4), -1, dtype=torch.int32, device=DEV)
    table[:, 0], table[:, 1] = 9, 2
    own = iter([0, 1, 3, 4, 5, 6, 7, 8])
    for b, n in enumerate(used):
        for j in range(2, (n + page - 1) // page):
            table[b, j] = next(own)
    qkv = normal(g, 5, (H + 2 * Hkv) * D)
    rope = torch.rand(5, 64, 2, generator=g, device=DEV) * 2 - 1
    before = cache.k[[9, 2]].clone()
    out = P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32(used), 128, SCALE,
                                   P.paged_decode_attention_workspace(5, shape, 128, DEV))
    assert torch.equal(cache.k[[9, 2]], before)
    q = P.paged_append(qkv, rope, lw, shape, cache_of(g, 14, Hkv, page), _i32([-1] * 5))
    for b, n in enumerate(used):
        ref, mass = attend(q[b:b + 1], *keys_of(cache, table, b, n), SCALE)
        near(out[b:b + 1], ref, mass, BF * BF, b)


def test_captured_steps():
    """A prompt chunk and decode steps in captured graphs, replayed with eager work in between and with counters that move on the
    device; two graphs with a workspace each."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    g = _gen(3)
    H, Hkv, page, used0 = 16, 8, 16, [700, 1, 250]
    shape, lw = shape_of(H, Hkv), weights(g)
    inv = dec.rope_inv_freq(shape, DEV)
    table, n = table_of(g, [x + 8 for x in used0], page)
    base = cache_of(g, n, Hkv, page)
    rows = normal(g, 3, (H + 2 * Hkv) * D)
    cu = _i32([0, 1, 2, 3])

    def make():
        cache = P.PagedKV(base.k.clone(), base.v.clone())
        return cache, torch.tensor([700, 3, 260], device=DEV), _i32(used0), P.paged_decode_attention_workspace(3, shape, 720, DEV)

    def step(cache, pos, used, ws):
        rope, _ = dec.decode_begin(pos, inv, used)
        out = P.paged_decode_attention(rows, rope, lw, shape, cache, table, used, 720, SCALE, ws)
        slots, rope2 = P.paged_begin(pos, inv, cu, used, table, cache)
        q = P.paged_append(rows, rope2, lw, shape, cache, slots)      # the same keys again, a position on
        return out, P.paged_attention(q, cache, table, cu, used, 1, 720, SCALE)

    eager, graphs = make(), [make() for _ in range(2)]
    first = [step(*s) for s in (eager, *graphs)]
    assert all(torch.equal(x, y) for f in first[1:] for x, y in zip(first[0], f))
    torch.cuda.synchronize()
    captured = []
    for s in graphs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            captured.append((gr, step(*s)))
    for i in range(4):
        want = step(*eager)
        torch.randn(1000, 1000, device=DEV).sum()
        for gr, out in captured:
            gr.replay()
        torch.cuda.synchronize()
        for _, out in captured:
            assert all(torch.equal(x, y) for x, y in zip(out, want)), i
    for s in graphs:
        assert torch.equal(s[0].k, eager[0].k) and torch.equal(s[0].v, eager[0].v)


def test_two_streams():
    """Calls that overlap on two streams, with a workspace each."""
    from tokengate_amd import paged as P
    g = _gen(4)
    H, Hkv, page, used = 16, 2, 64, [9000, 400]
    shape, lw = shape_of(H, Hkv), weights(g)
    table, n = table_of(g, used, page)
    caches = [cache_of(g, n, Hkv, page) for _ in range(2)]
    qkv = normal(g, 2, (H + 2 * Hkv) * D)
    rope = torch.rand(2, 64, 2, generator=g, device=DEV)
    u = _i32(used)
    ws = [P.paged_decode_attention_workspace(2, shape, 9000, DEV) for _ in range(2)]
    call = lambda i: P.paged_decode_attention(qkv, rope, lw, shape, caches[i], table, u, 9000, SCALE, ws[i])
    want = [call(i).clone() for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


def test_workspace_serves_smaller_calls():
    from tokengate_amd import paged as P
    g = _gen(5)
    H, Hkv, page = 16, 8, 16
    shape, lw = shape_of(H, Hkv), weights(g)
    ws = P.paged_decode_attention_workspace(20, shape, 20000, DEV)
    for B, n in ((20, 300), (1, 20000), (3, 5000), (20, 700)):
        used = [n] * B
        table, n_pages = table_of(g, used, page)
        cache = cache_of(g, n_pages, Hkv, page)
        qkv, rope = normal(g, B, (H + 2 * Hkv) * D), torch.rand(B, 64, 2, generator=g, device=DEV)
        call = lambda w: P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32(used), n, SCALE, w)
        assert torch.equal(call(ws), call(P.paged_decode_attention_workspace(B, shape, n, DEV)))
    with pytest.raises(RuntimeError, match="workspace"):
        call(torch.zeros(16, dtype=torch.uint8, device=DEV))


def test_cache_past_4_gib():
    """Pages whose offsets pass 32 bits, in elements too."""
    from tokengate_amd import paged as P
    g = _gen(6)
    H, Hkv, page, n_pages = 16, 8, 64, 34000                      # 65536 elements a page: 2.2e9
    shape, lw = shape_of(H, Hkv), weights(g)
    cache = P.PagedKV.alloc(n_pages, Hkv, page, DEV)
    used, ids = [150, 70], [[n_pages - 1, 3, n_pages - 2], [n_pages - 3, 33000, -1]]
    table = _i32(ids)
    for i in {x for row in ids for x in row if x >= 0}:
        cache.k[i], cache.v[i] = normal(g, Hkv, page, D), normal(g, Hkv, page, D)
    qkv, rope = normal(g, 2, (H + 2 * Hkv) * D), torch.rand(2, 64, 2, generator=g, device=DEV)
    out = P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32(used), 192, SCALE,
                                   P.paged_decode_attention_workspace(2, shape, 192, DEV))
    slots = _i32([(n_pages - 2) * page + 149 - 128, 33000 * page + 69 - 64])
    assert torch.equal(cache.v[slots.long() // page, :, slots.long() % page].flatten(1), qkv[:, (H + Hkv) * D:])
    q = P.paged_append(qkv, rope, lw, shape, cache, slots)
    two = P.paged_attention(q, cache, table, _i32([0, 1, 2]), _i32(used), 1, 192, SCALE)
    for b, n in enumerate(used):
        ref, mass = attend(q[b:b + 1], *keys_of(cache, table, b, n), SCALE)
        near(out[b:b + 1], ref, mass, BF * BF, b)
        near(two[b:b + 1], ref, mass, BF, b)


# ---- the gated prefill and decode over pages -----------------------------------------------------------------------

def _prefill(m, steps, page_rows):
    from tokengate_amd import inference as I
    split = [I.split_state_span(p) for p in _prompts([600, 333, 70], [(20, 500), (0, 300), (5, 60)], 5)]
    return m.prefill(split, [64, 1000, 7], decode_headroom=steps, page_rows=page_rows)


@pytest.mark.parametrize("page,ssmax", [(16, False), (64, True)])
def test_prefill_and_decode(cuda, page, ssmax):
    from tokengate_amd import decode as D_
    m = _model(cuda, ssmax=ssmax)
    steps = 4
    one, two = _prefill(m, steps, 0), _prefill(m, steps, page)
    assert one.n_kept == two.n_kept and torch.equal(one.kept_positions, two.kept_positions)
    for l, c in enumerate(two.kv):                               # the rows that the first layer makes are the same bits
        pg = two.pages_below if l <= m.gate_layer else two.pages_above
        cu, gap = one.cu_prompt if l <= m.gate_layer else one.cu_kept, one.decode_headroom
        for b in range(3):
            n = cu[b + 1] - cu[b]
            k, v, there = keys_of(c, pg.table, b, n)
            rows = slice(cu[b] + b * gap, cu[b] + b * gap + n)
            assert bool(there.all())
            if l == 0:
                assert torch.equal(k.to(torch.bfloat16), one.kv[l].k[rows]) and torch.equal(v.to(torch.bfloat16), one.kv[l].v[rows])
            else:
                assert_close_grad(f"layer {l} seq {b}", to_np(k.float().cpu()), to_np(one.kv[l].k[rows].float().cpu()), rel_l2=2e-2)
    for b in range(3):
        assert_close_grad(f"seq {b}", to_np(two.logits[b].float().cpu()), to_np(one.logits[b].float().cpu()), rel_l2=2e-2)
    three = _prefill(m, steps, page)
    a = D_.DecodeState(m.weights, m.gate, m.gate_layer, one, steps)
    b_ = D_.DecodeState(m.weights, m.gate, m.gate_layer, two, steps)
    c = D_.DecodeState(m.weights, m.gate, m.gate_layer, three, steps, graph=True)
    cur = one.first_tokens
    for i in range(steps):
        nxt = a.step(cur)
        b_.step(cur)
        c.step(cur)
        for s in range(3):
            assert_close_grad(f"seq {s} step {i}", to_np(b_.last_logits[s].float().cpu()), to_np(a.last_logits[s].float().cpu()),
                              rel_l2=2e-2)
        assert torch.equal(b_.last_logits, c.last_logits)
        cur = nxt
    for x, y in zip(two.kv, three.kv):
        assert all(torch.equal(keys_of(x, two.pages_above.table if l else two.pages_below.table, 0, 8)[l],
                               keys_of(y, three.pages_above.table if l else three.pages_below.table, 0, 8)[l]) for l in range(2))
    with pytest.raises(RuntimeError, match="caches are full"):
        b_.step(cur)


@pytest.mark.parametrize("page", [16, 64])
def test_decode_appends_alike(cuda, page):
    """Every key and value of every layer, the appended ones too, after decode steps taken eagerly and replayed; and what the steps
    appended has replaced what the pages held."""
    from tokengate_amd import decode as D_
    m = _model(cuda)
    steps = 4
    pfs = [_prefill(m, steps, page) for _ in range(2)]
    tables = [(pf.pages_below if l <= m.gate_layer else pf.pages_above).table for pf in pfs for l in range(len(pf.kv))]
    lengths = [[cu[b + 1] - cu[b] for b in range(3)] for cu in (pfs[0].cu_prompt, pfs[0].cu_kept)]
    layers = len(pfs[0].kv)

    def rows(i, l, b, n):
        k, v, there = keys_of(pfs[i].kv[l], tables[i * layers + l], b, n)
        assert bool(there.all())
        return k, v

    for i in range(2):
        for l in range(layers):                                  # no number where the steps are to write
            table, c = tables[i * layers + l], pfs[i].kv[l]
            for b in range(3):
                n = lengths[l > m.gate_layer][b]
                for j in range(n, n + steps):
                    c.k[table[b, j // page], :, j % page] = float("nan")
                    c.v[table[b, j // page], :, j % page] = float("nan")
    states = [D_.DecodeState(m.weights, m.gate, m.gate_layer, pf, steps, graph=g) for pf, g in zip(pfs, (False, True))]
    cur = pfs[0].first_tokens
    for _ in range(steps):
        nxt = [s.step(cur) for s in states]
        assert torch.equal(states[0].last_logits, states[1].last_logits)
        cur = nxt[0]
    for l in range(layers):
        for b in range(3):
            n = lengths[l > m.gate_layer][b] + steps
            for x, y in zip(rows(0, l, b, n), rows(1, l, b, n)):
                assert bool(x.isfinite().all()) and torch.equal(x, y), (l, b)


def test_generate(cuda):
    m = _model(cuda)
    prompts = _prompts([300, 90], [(10, 250), (0, 60)], 7)
    one = m.generate(prompts, max_new_tokens=6, max_kept_prefill_tokens=50)
    two = m.generate(prompts, max_new_tokens=6, max_kept_prefill_tokens=50, page_rows=32)
    assert two.n_kept == one.n_kept and two.kept_pos == one.kept_pos and len(two.token_ids) == 2
    again = m.generate(prompts, max_new_tokens=6, max_kept_prefill_tokens=50, page_rows=32)
    assert again.token_ids == two.token_ids
    drawn = m.generate(prompts, max_new_tokens=4, max_kept_prefill_tokens=50, page_rows=16, temperature=0.8, seed=3)
    assert all(len(t) == len(p) for t, p in zip(drawn.token_ids, drawn.logprobs))


def test_refusals(cuda):
    from tokengate_amd import decode as D_
    m = _model(cuda)
    with pytest.raises(ValueError, match="power of two"):
        _prefill(m, 2, 24)
    with pytest.raises(ValueError, match="kv_bits 16"):
        m.generate(_prompts([30], [(2, 20)], 1), kv_bits=4, page_rows=16)
    with pytest.raises(ValueError, match="prune_below_gate"):
        m.generate(_prompts([30], [(2, 20)], 1), prune_below_gate=True, page_rows=16)
    pf = _prefill(m, 2, 16)
    with pytest.raises(ValueError, match="fewer new tokens"):
        D_.DecodeState(m.weights, m.gate, m.gate_layer, pf, 3)
    with pytest.raises(ValueError, match="kv_bits 16"):
        D_.DecodeState(m.weights, m.gate, m.gate_layer, pf, 2, kv_bits=8)
