"""The paged KV cache: paged_begin, paged_append, paged_attention and paged_decode_attention against float64, and against the
operators over contiguous caches.  Tolerances: an output is rounded to bf16 (2^-8 of it); paged_attention's weights p are
bf16, p (1 + d) with |d| <= 2^-8, and as their sum is of the same numbers the output moves by sum p d (v - out), at most 2^-8
(sum p |v| + |out|); paged_decode_attention's weights are two bf16 numbers, 2^-16; logits from fp32 sums move a weight by
their own error, 2^-12 here."""
import math
import sys

import pytest
import torch

from paged_util import BF, D, attend, cache_of, keys_of, near, normal, shape_of, slots_of, table_of, weights

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rope(pos):
    from tokengate_amd import decoder as dec
    inv = dec.rope_inv_freq(shape_of(1, 1), DEV).double()
    a = pos.double()[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _rows64(qkv, H, Hkv, lw, rope, eps):
    """(q, k, v) rows in float64, before their rounding."""
    x = qkv[:, :(H + 2 * Hkv) * D].double().unflatten(1, (H + 2 * Hkv, D))

    def turn(y, w):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
        c, s = rope[:, None, :, 0].double(), rope[:, None, :, 1].double()
        a, b = y[..., :64], y[..., 64:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    return turn(x[:, :H], lw.q_norm), turn(x[:, H:H + Hkv], lw.k_norm), x[:, H + Hkv:]


# ---- begin and append ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("page,new,used", [(16, [1], [1]), (16, [5, 0, 17, 1], [5, 3, 40, 16]), (64, [130, 1], [130, 65]),
                                           (256, [3] * 70, list(range(3, 73)))])
def test_begin(page, new, used):
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    g = _gen(1)
    table, n = table_of(g, [u + 1 for u in used], page)
    cache = cache_of(g, n, 1, page)
    if len(used) > 1:
        table[1, 0] = n + 7                                      # names no page
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    T = cu[-1] + 3                                               # rows behind the last sequence
    pos = torch.randint(0, 200000, (T,), generator=g, device=DEV)
    inv = dec.rope_inv_freq(shape_of(1, 1), DEV)
    slots, rope = P.paged_begin(pos, inv, _i32(cu), _i32(used), table, cache)
    ref = []
    for b, x in enumerate(new):
        for i in range(x):
            key = used[b] - x + i
            p = int(table[b, key // page]) if key >= 0 else -1
            ref.append(p * page + key % page if 0 <= p < n else -1)
    assert slots.tolist() == ref + [-1] * 3
    p1 = pos.clone()
    again, _ = dec.decode_begin(p1, inv)
    assert torch.equal(rope, again)


def test_begin_without_room():
    """More new rows than keys, and keys past the table's columns: no slot."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    g = _gen(2)
    cache = cache_of(g, 4, 1, 16)
    table = _i32([[2], [3]])
    pos = torch.arange(8, device=DEV)
    slots, _ = P.paged_begin(pos, dec.rope_inv_freq(shape_of(1, 1), DEV), _i32([0, 4, 8]), _i32([2, 18]), table, cache)
    assert slots.tolist() == [-1, -1, 32, 33, 48 + 14, 48 + 15, -1, -1]


@pytest.mark.parametrize("T,H,Hkv,page,layout,scaled,in_place", [
    (1, 16, 8, 16, "heads", False, False), (7, 16, 8, 16, "rows", True, False), (130, 5, 5, 64, "both", True, True),
    (65, 12, 4, 32, "heads", False, True), (33, 3, 1, 16, "heads", True, False), (1000, 16, 2, 256, "rows", False, False),
    (9, 32, 8, 64, "heads", True, False)])
def test_append(T, H, Hkv, page, layout, scaled, in_place):
    from tokengate_amd import paged as P
    g = _gen(T)
    shape, lw = shape_of(H, Hkv), weights(g)
    table, n = table_of(g, [T + 11], page)
    cache = cache_of(g, n, Hkv, page, layout)
    slots = slots_of(table, page, [(0, 11 + t) for t in range(T)])
    if T > 4:
        slots[3], slots[4] = -1, n * page                        # outside the cache: queries only
    wide = normal(g, T, (H + 2 * Hkv) * D + 24)
    qkv = wide[:, :(H + 2 * Hkv) * D] if T % 2 else wide[:, 8:8 + (H + 2 * Hkv) * D]
    rope = _rope(torch.randint(0, 40000, (T,), generator=g, device=DEV))
    qs = 0.5 + torch.rand(H, generator=g, device=DEV) if scaled else None
    rs = torch.rand(T, generator=g, device=DEV) if scaled else None
    q64, k64, v64 = _rows64(qkv, H, Hkv, lw, rope, shape.rms_eps)
    k0, v0, w0 = cache.k.clone(), cache.v.clone(), wide.clone()
    out = qkv[:, :H * D].unflatten(1, (H, D)) if in_place else None
    q = P.paged_append(qkv, rope, lw, shape, cache, slots, qs, rs, out=out)
    assert not in_place or q.data_ptr() == qkv.data_ptr()
    tol = 1e-5                                                   # fp32 sums, a rotation's two products
    big = lambda x: x.abs() + x.roll(64, -1).abs()
    f = torch.ones(T, H, device=DEV, dtype=torch.float64)
    if scaled:
        f = (qs[None] * rs[:, None]).to(torch.bfloat16).double()
    ref = q64 * f[..., None]
    rounds = 2 if scaled else 1                                  # the rotated query, and its product with the scale
    assert bool(((q.double() - ref).abs() <= rounds * (BF * (1 + BF)) * ref.abs() + tol * big(ref)).all())
    seen = torch.zeros(n, page, dtype=torch.bool, device=DEV)
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < n * page:
            continue
        at = (s // page, slice(None), s % page)
        seen[s // page, s % page] = True
        assert torch.equal(cache.v[at], v64[t].to(torch.bfloat16))
        assert bool(((cache.k[at].double() - k64[t]).abs() <= BF * k64[t].abs() + tol * big(k64[t])).all())
    free = ~seen[:, None, :, None]
    assert torch.equal(torch.where(free, cache.k, 0), torch.where(free, k0, 0))     # other rows as they were
    assert torch.equal(torch.where(free, cache.v, 0), torch.where(free, v0, 0))
    if not in_place:
        assert torch.equal(wide, w0)


def test_append_equals_contiguous():
    """The bits of qk_norm_rope, at far positions too, with paged_begin's table."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    g = _gen(5)
    H, Hkv, page, new, used = 16, 8, 64, [70, 1, 200], [100, 1, 1000]
    shape, lw, T = shape_of(H, Hkv), weights(g), 271
    table, n = table_of(g, used, page)
    cache = cache_of(g, n, Hkv, page)
    qkv = normal(g, T, (H + 2 * Hkv) * D)
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=DEV)
    inv = dec.rope_inv_freq(shape, DEV)
    qs, rs = torch.rand(H, generator=g, device=DEV), torch.rand(T, generator=g, device=DEV)
    slots, rope = P.paged_begin(pos, inv, _i32([0, 70, 71, 271]), _i32(used), table, cache)
    q = P.paged_append(qkv, rope, lw, shape, cache, slots, qs, rs)
    k, v = torch.empty(T, Hkv, D, dtype=torch.bfloat16, device=DEV), torch.empty(T, Hkv, D, dtype=torch.bfloat16, device=DEV)
    q1 = dec.qk_norm_rope(qkv.clone(), pos, lw, shape, inv, k, v, qs, rs)
    assert torch.equal(q, q1)
    at = slots.long()
    assert torch.equal(cache.k[at // page, :, at % page], k) and torch.equal(cache.v[at // page, :, at % page], v)


# ---- attention of several rows --------------------------------------------------------------------------------------

def _attention(new, used, H, Hkv, page, layout="heads", bias=None, seed=0, max_q=None, max_k=None, prepare=None, fill=None,
               average=()):
    """average: heads of which only that the output is an average of the values is checked."""
    from tokengate_amd import paged as P
    g = _gen(seed)
    table, n = table_of(g, used, page)
    cache = cache_of(g, n, Hkv, page, layout)
    if fill is not None:                                         # whatever no key of the sequences holds
        held = torch.zeros(n, page, dtype=torch.bool, device=DEV)
        for b, u in enumerate(used):
            at = slots_of(table, page, [(b, j) for j in range(u)]).long()
            held[at // page, at % page] = True
        for t in (cache.k, cache.v):
            t.copy_(torch.where(held[:, None, :, None], t, torch.full_like(t, fill)))
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    max_q, max_k = max_q or max(new), max_k or max(used)
    q = normal(g, cu[-1] + 2, H, D)
    bias = bias(g, len(used), H, max_k + 3) if bias else None
    if prepare:
        prepare(cache, table, bias)
    out = torch.full_like(q, 7.0)
    got = P.paged_attention(q, cache, table, _i32(cu), _i32(used), max_q, max_k, SCALE, bias, out=out)
    assert got is out and bool((out[cu[-1]:] == 7.0).all())      # rows of no sequence as they were
    for b, (m, u) in enumerate(zip(new, used)):
        if not m:
            continue
        k, v, there = keys_of(cache, table, b, u)
        ref, mass = attend(q[cu[b]:cu[b + 1]], k, v, there, SCALE, None if bias is None else bias[b, :, :u], u - m)
        for h in average:
            x, y = out[cu[b]:cu[b + 1], h].double(), v[:, h // (H // Hkv)]
            assert bool((x <= y.amax(0) + BF * y.abs().amax(0)).all()) and bool((x >= y.amin(0) - BF * y.abs().amax(0)).all())
        rest = [h for h in range(H) if h not in average]
        near(out[cu[b]:cu[b + 1], rest], ref[:, rest], mass[:, rest], BF, (b, m, u))
    return q, cache, table, out


def _normal_bias(g, B, H, n):
    return 4 * torch.randn(B, H, n, generator=g, device=DEV)


@pytest.mark.parametrize("new,used,H,Hkv,page,layout,bias", [
    ([1], [1], 16, 8, 16, "heads", False), ([2], [2], 16, 8, 16, "heads", True),
    ([17, 3, 64], [33, 3, 65], 16, 8, 16, "rows", True), ([65], [130], 5, 5, 32, "both", False),
    ([128, 1, 129], [128, 300, 1025], 12, 4, 64, "heads", True), ([33], [4100], 16, 8, 64, "heads", False),
    ([16], [9000], 16, 2, 128, "rows", True), ([300, 0, 7], [300, 9, 700], 16, 8, 256, "heads", False),
    ([513], [1500], 8, 8, 16, "heads", True), ([40] * 30, [90] * 30, 16, 8, 16, "heads", False),
    ([700, 350, 90, 64], [1000, 351, 800, 64], 7, 1, 64, "heads", True)])
def test_attention(new, used, H, Hkv, page, layout, bias):
    _attention(new, used, H, Hkv, page, layout, _normal_bias if bias else None, seed=sum(new) + H)


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("page,bias", [(16, False), (64, True), (16, True)])
def test_attention_whatever_unused_rows_hold(fill, page, bias):
    """Rows behind a sequence's last key, and pages of no sequence."""
    _attention([5, 70], [5, 777], 16, 8, page, bias=_normal_bias if bias else None, fill=fill)


@pytest.mark.parametrize("new,used,H,Hkv,page,bias", [
    ([1 + b % 23 for b in range(70)], [40 + 3 * b for b in range(70)], 16, 8, 16, True),
    ([3] * 66, [1900 + b for b in range(66)], 4, 2, 64, True), ([b % 3 for b in range(300)], [b % 3 + b for b in range(300)], 5, 5, 32, False),
    ([129] * 65, [700] * 65, 4, 4, 16, False)])
def test_attention_of_many_sequences(new, used, H, Hkv, page, bias):
    """More sequences than lanes; every sequence has keys of no page."""
    def prepare(cache, table, _):
        table[:, 1] = cache.n_pages
    _attention(new, used, H, Hkv, page, bias=_normal_bias if bias else None, seed=len(new), prepare=prepare)


@pytest.mark.parametrize("page,missing,masked", [(16, False, False), (64, True, False), (32, True, True), (128, False, True)])
def test_attention_of_long_caches(page, missing, masked):
    """Few rows over many keys, cut into chunks, some of them without a key that is seen."""
    def bias(g, B, H, n):
        x = _normal_bias(g, B, H, n)
        if masked:
            x[:, 1, 64:] = -math.inf
            x[3, 2] = -math.inf
            x[4, 3, ::2] = torch.finfo(torch.float32).min
        return x

    def prepare(cache, table, _):
        if missing:
            table[1, 3:], table[2, :40 * 16 // page], table[5, ::3] = -1, 2 ** 31 - 1, -7
    used = [6000, 5999, 4100, 33, 5000, 3001, 128, 20]
    _, _, _, out = _attention([20, 1, 33, 33, 7, 0, 40, 20], used, 8, 4, page, bias=bias, prepare=prepare)
    if masked:
        assert bool((out[54:87, 2] == 0).all())


def test_attention_past_the_last_level_cache():
    """Long prompt parts of sequences whose keys outgrow it."""
    _attention([1100, 1030], [40000, 38001], 4, 4, 64, bias=_normal_bias)


def test_attention_sizes_at_their_ends():
    """A max_q far past every segment, a max_k of 0, one page table and one bias for all sequences."""
    from tokengate_amd import paged as P
    g = _gen(11)
    H, Hkv, page, new, n = 8, 4, 32, [5, 40, 1], 70
    table, n_pages = table_of(g, [n], page)
    cache = cache_of(g, n_pages, Hkv, page)
    q, cu, used = normal(g, 46, H, D), _i32([0, 5, 45, 46]), _i32([n] * 3)
    bias = _normal_bias(g, 1, 1, n)
    tables, biases = table.expand(3, -1), bias.expand(3, H, n)
    a = P.paged_attention(q, cache, tables, cu, used, 40, n, SCALE, biases)
    b = P.paged_attention(q, cache, tables, cu, used, 2 ** 31 - 1, n, SCALE, biases)
    assert torch.equal(a, b)
    k, v, there = keys_of(cache, table, 0, n)
    for b, m in enumerate(new):
        rows = slice(int(cu[b]), int(cu[b]) + m)
        near(a[rows], *attend(q[rows], k, v, there, SCALE, bias[0].expand(H, n), n - m), BF)
    assert bool((P.paged_attention(q, cache, tables, cu, used, 40, 0, SCALE) == 0).all())
    assert P.paged_attention(q, cache, tables[:0], cu[:1], used[:0], 40, n, SCALE).shape == q.shape
    assert P.paged_attention(q[:0], cache, tables, cu, used, 40, n, SCALE).shape == (0, H, D)


@pytest.mark.parametrize("max_q", [2 ** 31, 2 ** 32 + 3, 2 ** 40])
def test_attention_max_q_past_32_bits(max_q):
    """Any max_q past the rows is their count."""
    from tokengate_amd import paged as P
    g = _gen(14)
    H, Hkv, page = 8, 4, 32
    table, n_pages = table_of(g, [90, 33], page)
    cache = cache_of(g, n_pages, Hkv, page)
    q, cu, used = normal(g, 45, H, D), _i32([0, 40, 45]), _i32([90, 33])
    a = P.paged_attention(q, cache, table, cu, used, 40, 90, SCALE, out=torch.full_like(q, 7.0))
    assert torch.equal(a, P.paged_attention(q, cache, table, cu, used, max_q, 90, SCALE, out=torch.full_like(q, 7.0)))


def test_attention_more_queries_than_keys():
    """The first queries see no key: zeros."""
    _, _, _, out = _attention([20, 9], [6, 0], 16, 8, 16)
    assert bool((out[:14] == 0).all()) and bool((out[20:29] == 0).all()) and not bool((out[14:20] == 0).all())


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("bias", [False, True])
def test_attention_missing_pages(page, bias):
    """Entries that name no page hide their keys."""
    def prepare(cache, table, _):
        table[0, 1], table[0, 4], table[1, 0] = -1, cache.n_pages, -5
    _, _, _, out = _attention([30, 4, 100], [300, 15, 400], 16, 8, page, bias=_normal_bias if bias else None, prepare=prepare)
    assert bool((out[30:34] == 0).all())


@pytest.mark.parametrize("H,Hkv", [(16, 8), (5, 5), (12, 4)])
@pytest.mark.parametrize("fill", [None, float("nan"), float("-inf")])
def test_attention_hidden_by_bias(H, Hkv, fill):
    """-inf hides a key from the head whatever its rows hold; a head that sees nothing gives zeros."""
    used, new, page = [200, 140], [70, 33], 16

    def bias(g, B, H_, n):
        x = _normal_bias(g, B, H_, n)
        x[:, :, 5:30] = -math.inf
        x[0, 0] = -math.inf
        x[1, :, ::3] = -math.inf
        return x

    def prepare(cache, table, b):
        if fill is None:
            return
        for s, u in enumerate(used):                             # keys that no head sees
            dead = (b[s, :, :u] == -math.inf).all(0).nonzero().flatten().tolist()
            at = slots_of(table, page, [(s, j) for j in dead]).long()
            cache.k[at // page, :, at % page] = fill
            cache.v[at // page, :, at % page] = fill

    _, _, _, out = _attention(new, used, H, Hkv, page, bias=bias, prepare=prepare)
    assert bool((out[:70, 0] == 0).all())


@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30, -1e9])
def test_attention_masks_of_large_numbers(low):
    """A finite mask: nothing beside visible keys; alone, all keys weigh alike as their logits are the mask's.  Near 1e9
    fp32 numbers are 64 apart, and a logit is four sums, each off by up to 32: with the scale 11.3 in the exponent, so that the weights
    of a head that sees nothing else are not determined, but for being positive."""
    def bias(g, B, H, n):
        x = torch.zeros(B, H, n, device=DEV)
        x[:, ::2, 10:90] = low
        x[:, 1] = low
        return x
    average = [1] if low == -1e9 else []
    _attention([1], [150], 16, 8, 16, bias=bias, average=average)
    _attention([40], [150], 16, 8, 64, bias=bias, average=average)


@pytest.mark.parametrize("scale", [0.7, 1.0, 1.5])
@pytest.mark.parametrize("new,used", [([1], [150]), ([40], [150]), ([200, 30, 5], [300, 250, 777]), ([20, 3], [6000, 20]), ([33], [9000])])
def test_attention_masks_past_the_range_when_scaled(monkeypatch, new, used, scale):
    """The lowest float times a scale of log2(e) of its own passes fp32's range: a row that sees nothing else still has the
    average of its values."""
    def bias(g, B, H, n):
        x = torch.zeros(B, H, n, device=DEV)
        x[:, ::2, 10:90] = torch.finfo(torch.float32).min
        x[:, 1] = torch.finfo(torch.float32).min
        x[0, 3, ::2], x[0, 3, 1::2] = -math.inf, torch.finfo(torch.float32).min
        return x
    monkeypatch.setattr(sys.modules[__name__], "SCALE", scale)
    _attention(new, used, 8, 4, 64, bias=bias)
    _attention(new, used, 5, 5, 16, bias=bias)


@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30, -3e9, -math.inf])
@pytest.mark.parametrize("new,used", [([40], [300]), ([200, 30, 5], [300, 250, 777])])
def test_attention_masks_of_the_first_keys(low, new, used):
    """Left padding: whole tiles of masked keys, and rows that see no other, before the ones that count.  (-3e9: a
    maximum past 2^28.)"""
    def bias(g, B, H, n):
        x = _normal_bias(g, B, H, n)
        x[:, ::3, :200] = low
        return x
    # a row that sees masked keys alone has their average, by weights that fp32 logits near 3e9 do not give
    _attention(new, used, 6, 3, 64, bias=bias, average=[0, 3] if low == -3e9 else [])


@pytest.mark.parametrize("new,used", [([50], [300]), ([300, 20], [300, 450]), ([17], [5000])])
@pytest.mark.parametrize("H,Hkv", [(8, 4), (5, 5), (6, 2)])
def test_attention_hidden_from_some_heads(new, used, H, Hkv):
    """Keys hidden from some heads, with rows that are no numbers: the others' outputs are no numbers where they see one, and
    these heads' are as if the rows were not there."""
    from tokengate_amd import paged as P
    g, page = _gen(21), 64
    table, n = table_of(g, used, page)
    cache = cache_of(g, n, Hkv, page)
    bias = _normal_bias(g, len(used), H, max(used))
    bad = [3, 70, 71, 200]
    for b in range(len(used)):
        bias[b, ::2, bad] = -math.inf
        at = slots_of(table, page, [(b, j) for j in bad]).long()
        cache.k[at[:2] // page, :, at[:2] % page] = math.nan
        cache.v[at[2:] // page, :, at[2:] % page] = math.inf
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    q = normal(g, cu[-1], H, D)
    out = P.paged_attention(q, cache, table, _i32(cu), _i32(used), max(new), max(used), SCALE, bias)
    seen = list(range(0, H, 2))
    clean = P.PagedKV(*(torch.where(t.isfinite(), t, torch.zeros_like(t)) for t in (cache.k, cache.v)))
    for b, (m, u) in enumerate(zip(new, used)):
        rows = slice(cu[b], cu[b] + m)
        ref, mass = attend(q[rows], *keys_of(clean, table, b, u), SCALE, bias[b, :, :u], u - m)
        near(out[rows][:, seen], ref[:, seen], mass[:, seen], BF, b)
        if H > 1:
            assert not bool(out[cu[b] + m - 1, 1].isfinite().all())


def test_attention_near_contiguous():
    """varlen_kv_attention's outputs: both are within the tolerance of float64 (their key groups and chunks, and so the order
    of their sums, may differ)."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    g = _gen(3)
    H, Hkv, page, new, used = 16, 8, 16, [200, 1300, 33], [900, 1300, 80]
    table, n = table_of(g, used, page)
    cache = cache_of(g, n, Hkv, page)
    cu = _i32([0, 200, 1500, 1533])
    start = _i32([0, 900, 2200])
    k, v = torch.empty(2280, Hkv, D, dtype=torch.bfloat16, device=DEV), torch.empty(2280, Hkv, D, dtype=torch.bfloat16, device=DEV)
    for b, u in enumerate(used):
        s = int(start[b])
        k[s:s + u], v[s:s + u] = (t.to(torch.bfloat16) for t in keys_of(cache, table, b, u)[:2])
    q = normal(g, 1533, H, D)
    for bias in (None, _normal_bias(g, 3, H, 1300)):
        got = P.paged_attention(q, cache, table, cu, _i32(used), 1300, 1300, SCALE, bias)
        two = dec.varlen_kv_attention(q, k, v, cu, start, _i32(used), 1300, 1300, SCALE, bias)
        for b, (m, u) in enumerate(zip(new, used)):
            rows = slice(int(cu[b]), int(cu[b]) + m)
            ref, mass = attend(q[rows], *keys_of(cache, table, b, u), SCALE, None if bias is None else bias[b, :, :u], u - m)
            near(got[rows], ref, mass, BF)
            near(two[rows], ref, mass, BF)


# ---- one new token per sequence ---------------------------------------------------------------------------------------

def _decode(used, H, Hkv, page, layout="heads", bias=None, scaled=False, seed=0, max_k=None, prepare=None, fill=None, ws=None,
            calls=1):
    from tokengate_amd import paged as P
    g = _gen(seed)
    shape, lw, B = shape_of(H, Hkv), weights(g), len(used)
    table, n = table_of(g, used, page)
    cache = cache_of(g, n, Hkv, page, layout)
    if fill is not None:
        held = torch.zeros(n, page, dtype=torch.bool, device=DEV)
        for b, u in enumerate(used):
            at = slots_of(table, page, [(b, j) for j in range(u - 1)]).long()
            held[at // page, at % page] = True
        for t in (cache.k, cache.v):
            t.copy_(torch.where(held[:, None, :, None], t, torch.full_like(t, fill)))
    max_k = max_k or max(max(used), 1)
    qkv = normal(g, B, (H + 2 * Hkv) * D + 8)[:, :(H + 2 * Hkv) * D]
    rope = _rope(_i32(used) + 9)
    qs = 0.5 + torch.rand(H, generator=g, device=DEV) if scaled else None
    rs = 0.5 + 0.5 * torch.rand(B, generator=g, device=DEV) if scaled else None
    bias = bias(g, B, H, max_k + 3) if bias else None
    if prepare:
        prepare(cache, table, bias)
    k0, v0 = cache.k.clone(), cache.v.clone()
    ws = P.paged_decode_attention_workspace(B, shape, max_k, DEV) if ws is None else ws
    outs = [P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32(used), max_k, SCALE, ws, bias, qs, rs)
            for _ in range(calls)]
    # the appended rows are paged_append's, bit for bit, and no other row has changed
    q = torch.empty(B, H, D, dtype=torch.bfloat16, device=DEV)
    ref = P.PagedKV(k0, v0)
    slots = []
    for b, u in enumerate(used):
        u = min(u, max_k)
        p = int(table[b, (u - 1) // page]) if u > 0 else -1
        slots.append(p * page + (u - 1) % page if 0 <= p < n else -1)
    P.paged_append(qkv, rope, lw, shape, ref, _i32(slots), qs, rs, out=q)
    bits = lambda t: t.contiguous().view(torch.int16)
    assert torch.equal(bits(cache.k), bits(ref.k)) and torch.equal(bits(cache.v), bits(ref.v))
    for b, u in enumerate(used):
        u = min(u, max_k)
        if u <= 0:
            assert all(bool((o[b] == 0).all()) for o in outs)
            continue
        k, v, there = keys_of(cache, table, b, u)
        want, mass = attend(q[b:b + 1], k, v, there, SCALE, None if bias is None else bias[b, :, :u])
        for o in outs:
            near(o[b:b + 1], want, mass, BF * BF, (b, u))
    assert all(torch.equal(o, outs[0]) for o in outs)
    return outs[0]


@pytest.mark.parametrize("used,H,Hkv,page,layout,bias,scaled", [
    ([1], 16, 8, 16, "heads", True, False), ([2, 1, 3, 0], 16, 8, 16, "rows", True, True),
    ([16, 17, 18, 15], 5, 5, 16, "both", False, False), ([33, 32, 31], 12, 4, 32, "heads", True, False),
    ([65, 64, 129, 128, 127], 16, 2, 64, "heads", False, True), ([300], 16, 8, 16, "heads", False, False),
    ([2321], 16, 8, 64, "heads", True, True), ([1000, 4], 16, 1, 256, "rows", True, False),
    ([777, 0, 900], 20, 1, 16, "heads", True, True), ([500, 90], 28, 4, 64, "rows", False, False),
    ([5000, 300, 1], 6, 2, 128, "heads", True, True), ([4097] * 9, 32, 8, 16, "heads", False, False),
    (list(range(1, 90)), 4, 4, 16, "heads", True, False), ([20000, 3], 16, 8, 64, "rows", False, False)])
def test_decode(used, H, Hkv, page, layout, bias, scaled):
    _decode(used, H, Hkv, page, layout, _normal_bias if bias else None, scaled, seed=sum(used) + H, calls=2)


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("H,Hkv,bias", [(16, 8, False), (16, 8, True), (16, 1, True), (3, 3, True)])
def test_decode_whatever_unused_rows_hold(fill, H, Hkv, bias):
    _decode([1, 40, 333], H, Hkv, 16, bias=_normal_bias if bias else None, fill=fill)


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("bias", [False, True])
def test_decode_missing_pages(page, bias):
    """Entries that name no page hide their keys, the new one among them (nothing is then appended)."""
    def prepare(cache, table, _):
        table[0, 1], table[0, 3], table[1, 0] = -1, cache.n_pages, -5
        table[2, 99 // page] = -1
    out = _decode([300, 15, 100], 16, 8, page, bias=_normal_bias if bias else None, prepare=prepare)
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("H,Hkv", [(16, 8), (5, 5), (12, 4), (16, 2), (16, 1)])
@pytest.mark.parametrize("fill", [None, float("nan"), float("inf")])
def test_decode_hidden_by_bias(H, Hkv, fill):
    """-inf hides a key from its head whatever its rows hold, also where another head sees the key's neighbours."""
    used, page = [200, 140, 60], 16

    def bias(g, B, H_, n):
        x = _normal_bias(g, B, H_, n)
        x[:, :, 5:30] = -math.inf
        x[0, 0] = -math.inf
        x[1, :, ::3] = -math.inf
        x[2, :, 59] = -math.inf                                  # the new key
        return x

    def prepare(cache, table, b):
        for s, u in enumerate(used):
            dead = (b[s, :, :u] == -math.inf).all(0).nonzero().flatten().tolist()
            at = slots_of(table, page, [(s, j) for j in dead]).long()
            if fill is not None:
                cache.k[at // page, :, at % page] = fill
                cache.v[at // page, :, at % page] = fill

    out = _decode(used, H, Hkv, page, bias=bias, prepare=prepare)
    assert bool((out[0, 0] == 0).all())


def test_decode_hidden_from_one_head():
    """A row of NaN that one head of a group hides and the other sees: that one's output alone is NaN."""
    from tokengate_amd import paged as P
    g = _gen(8)
    H, Hkv, page, used = 4, 2, 16, 100
    shape, lw = shape_of(H, Hkv), weights(g)
    table, n = table_of(g, [used], page)
    cache = cache_of(g, n, Hkv, page)
    at = int(slots_of(table, page, [(0, 37)])[0])
    cache.v[at // page, 0, at % page] = math.nan
    bias = torch.zeros(1, H, used, device=DEV)
    bias[0, 1, 37] = -math.inf
    out = P.paged_decode_attention(normal(g, 1, (H + 2 * Hkv) * D), _rope(_i32([100])), lw, shape, cache, table, _i32([used]), used,
                                   SCALE, P.paged_decode_attention_workspace(1, shape, used, DEV), bias)
    assert bool(out[0, 0].isnan().all()) and bool(out[0, 1:].isfinite().all())


@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30])
def test_decode_masks_of_large_numbers(low):
    def bias(g, B, H, n):
        x = torch.zeros(B, H, n, device=DEV)
        x[:, ::2, 10:90] = low
        x[:, 1] = low
        return x
    _decode([150, 15], 16, 8, 16, bias=bias)


@pytest.mark.parametrize("scale", [0.7, 1.0, 1.5])
@pytest.mark.parametrize("H,Hkv", [(16, 8), (5, 5), (16, 1)])
def test_decode_masks_past_the_range_when_scaled(monkeypatch, H, Hkv, scale):
    def bias(g, B, H, n):
        x = torch.zeros(B, H, n, device=DEV)
        x[:, ::2, 10:90] = torch.finfo(torch.float32).min
        x[:, 1] = torch.finfo(torch.float32).min
        x[0, 3, ::2], x[0, 3, 1::2] = -math.inf, torch.finfo(torch.float32).min
        return x
    monkeypatch.setattr(sys.modules[__name__], "SCALE", scale)
    _decode([150, 15, 6000, 1], H, Hkv, 16, bias=bias)


@pytest.mark.parametrize("H,Hkv", [(16, 8), (16, 1)])
def test_decode_large_values(H, Hkv):
    """Values near the largest float: no sum passes fp32's range."""
    def prepare(cache, table, _):
        cache.v.mul_(3e38 / 8)
        cache.v.clamp_(-3e38, 3e38)
    _decode([3000, 40], H, Hkv, 64, prepare=prepare)


def test_decode_more_keys_than_max():
    """kv_used past max_k: the first max_k keys, of which the last is the new one."""
    _decode([100, 70], 16, 8, 16, bias=_normal_bias, max_k=64)


def test_decode_of_very_many_sequences():
    """More units than the workspace has counters: none is cut, and the others' rows stay as they were."""
    from tokengate_amd import paged as P
    H, Hkv, page, B = 16, 8, 16, 2100
    g = _gen(12)
    shape, lw = shape_of(H, Hkv), weights(g)
    used = [b % 5 for b in range(B)]
    used[7] = 3000
    table, n = table_of(g, [max(u, 1) if u < 99 else u for u in used], page)
    cache = cache_of(g, n, Hkv, page)
    qkv, rope = normal(g, B, (H + 2 * Hkv) * D), torch.rand(B, 64, 2, generator=g, device=DEV)
    ws = P.paged_decode_attention_workspace(B, shape, 3000, DEV)
    out = P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32(used), 3000, SCALE, ws)
    assert not bool(ws[:1 << 16].any())
    few = list(range(40)) + list(range(B - 40, B))
    q = P.paged_append(qkv, rope, lw, shape, cache, torch.full((B,), -1, dtype=torch.int32, device=DEV))
    for b in few:
        if used[b] == 0:
            assert bool((out[b] == 0).all())
            continue
        near(out[b:b + 1], *attend(q[b:b + 1], *keys_of(cache, table, b, used[b]), SCALE), BF * BF, b)
    few = _i32(few).long()                                       # the workspace serves a cut launch of fewer
    a = P.paged_decode_attention(qkv[few], rope[few], lw, shape, cache, table[few], _i32(used)[few], 3000, SCALE, ws)
    two = P.paged_decode_attention_workspace(80, shape, 3000, DEV)
    assert torch.equal(a, P.paged_decode_attention(qkv[few], rope[few], lw, shape, cache, table[few], _i32(used)[few], 3000, SCALE, two))


def test_decode_without_keys():
    from tokengate_amd import paged as P
    g = _gen(13)
    H, Hkv, page = 16, 8, 16
    shape, lw = shape_of(H, Hkv), weights(g)
    cache = cache_of(g, 4, Hkv, page)
    k0 = cache.k.clone()
    qkv, rope = normal(g, 3, (H + 2 * Hkv) * D), torch.rand(3, 64, 2, generator=g, device=DEV)
    ws = P.paged_decode_attention_workspace(3, shape, 0, DEV)
    table = torch.zeros(3, 1, dtype=torch.int32, device=DEV)
    assert bool((P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32([0, 0, 0]), 16, SCALE, ws) == 0).all())
    assert bool((P.paged_decode_attention(qkv, rope, lw, shape, cache, table, _i32([1, 2, 3]), 0, SCALE, ws) == 0).all())
    assert P.paged_decode_attention(qkv[:0], rope, lw, shape, cache, table, _i32([]), 16, SCALE, ws).shape == (0, H, D)
    assert torch.equal(cache.k, k0)
