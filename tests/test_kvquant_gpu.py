"""KV caches of 4 and 8 bits: kv_quantize, kv_dequantize and decode_attention_quant.

Quantising and reading back are compared bit for bit with the definition evaluated on the CPU (fp32 division and
rounding there are IEEE's, as the kernel's are; code times step is exact in fp32, so one addition rounds).

Attention is compared with float64 over the values s c + m that the cache holds.  With P the weights and z the
logits, the kernel may be off by (a rounding to bf16, of 8 significant bits, by 2^-8 relative)
  * the weights' rounding before the value product, to two bf16 numbers, 2^-16 each, where a value counts by its code's
    part s c (the least values' part is summed in fp32): 2^-16 sum P s c; at 4 bits codes are held as 128 + c here too,
    taken off at the end, and the sums of 128 + L times a step are good to 2^-18;
  * the logits' fp32 sums: a group's 32 products of a bf16 query value and a code are summed from -128 sum q on (at 4
    bits codes are held as 128 + c), at most 2^-20 (128 + L) sum |q| a group (16 roundings), so
    dz = scale max_j sum_g s_jg 2^-20 (128 + L) sum_{d in g} |q_d| + 2^-20 max |z|, and 2 dz sum P |v|;
  * the output's rounding to bf16: 2^-8 |out|; and 2^-18 sum P |v| for the fp32 sums of the values.
(The kernel's weights have 24 bits and its codes are 16 + c, the offset taken off every 32 keys: these bounds are those of
16 bits and of 128 + c taken off at the end, which it stays well below; the tests of keys that cancel hold it to its own.)
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def ref_quantize(x, bits):
    """(codes by element (..., 128), s (..., 4), m (..., 4)) of bf16 values on the CPU, fp32 operations."""
    L = torch.tensor(float((1 << bits) - 1))
    x = x.cpu().float().unflatten(-1, (4, 32))
    m, top = x.amin(-1), x.amax(-1)
    span = top - m
    s = (span / L.expand_as(span)).bfloat16().float()
    s = torch.where(s < 2.0 ** -100, torch.zeros_like(s), s)
    c = ((x - m[..., None]) / torch.where(s > 0, s, torch.full_like(s, float("inf")))[..., None]).round()
    c = c.clamp(0, float(L))
    bad = ~torch.isfinite(span)
    c[bad] = 0
    s[bad] = m[bad] = float("nan")
    return c.flatten(-2).to(torch.uint8), s, m


def codes_of(cache, t):
    """Element codes (Hkv, rows, 128) of a cache's code tensor, on the CPU."""
    w = t.cpu().unflatten(-1, (16, cache.bits))
    if cache.bits == 4:
        w = torch.stack([w & 15, w >> 4], -1).flatten(-2)
    return w.transpose(-1, -2).flatten(-2)


def values_of(cache, dtype=torch.float64):
    """(k, v) (rows, Hkv, 128) that the cache stands for."""
    out = []
    for t, meta in ((cache.k, cache.k_meta), (cache.v, cache.v_meta)):
        sm = meta.cpu().to(dtype)
        c = codes_of(cache, t).to(dtype).unflatten(-1, (4, 32))
        out.append((c * sm[..., :1] + sm[..., 1:]).flatten(-2).transpose(0, 1))
    return out


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b, 7.0))


def check_quantized(cache, k, v, rows):
    for name, x in (("k", k), ("v", v)):
        c, s, m = ref_quantize(x.transpose(0, 1), cache.bits)
        sm = getattr(cache, name + "_meta").cpu()[:, rows]
        assert same(sm[..., 0].float(), s) and same(sm[..., 1].float(), m), name
        assert torch.equal(codes_of(cache, getattr(cache, name))[:, rows], c), name


def rand_rows(dev, n, hkv, seed, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(std * torch.randn(n, hkv, 128, generator=g, device=dev)).bfloat16() for _ in range(2)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,hkv", [(1, 8), (15, 1), (17, 5), (1000, 2), (4099, 8)])
def test_quantize_and_read_back(cuda, bits, n, hkv):
    from tokengate_amd import kvquant as Q
    k, v = rand_rows(cuda, n, hkv, n + bits)
    cache = Q.QuantKV.alloc(n, hkv, bits, cuda)
    Q.kv_quantize(k, v, cache)
    back = Q.kv_dequantize(cache)
    torch.cuda.synchronize()
    check_quantized(cache, k, v, slice(None))
    for got, want in zip(back, values_of(cache, torch.float32)):
        assert torch.equal(got.cpu(), want.bfloat16())
    # half a step of the group, and the step's rounding to bf16 (2^-8 of L steps) at the largest code
    for got, x, meta in zip(values_of(cache), (k, v), (cache.k_meta, cache.v_meta)):
        s = meta[..., 0].double().cpu().transpose(0, 1).repeat_interleave(32, -1)
        assert bool(((got - x.cpu().double()).abs() <= s * (0.5 + (2 ** bits - 1) * 2.0 ** -8)).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_odd_groups(cuda, bits):
    """Constants, zeros of both signs, steps below the least, quotients half way between two codes, large values, and
    groups that hold a NaN, an infinity or a range past fp32."""
    from tokengate_amd import kvquant as Q
    L = 2 ** bits - 1
    x = torch.randn(12, 4, 32, generator=torch.Generator().manual_seed(3))
    x[0] = 1.5
    x[1] = 0.0
    x[1, 1] = -0.0
    x[1, 2, ::2] = -0.0
    x[2] *= 2.0 ** -110
    x[3, 0], x[3, 1] = x[3, 0] * 2.0 ** -95, x[3, 1] * 2.0 ** -126
    x[4, 0] = torch.arange(32) * 0.5                     # step 15.5 / 15 or / 255
    x[4, 1] = torch.arange(32).clamp(max=30) * (L / 30)
    x[4, 2] = torch.tensor([0.0, float(L)] + [0.5 + i % L for i in range(30)])      # step 1: ties
    x[5] = 1000 + x[5]
    x[6] = x[6] * 1e38 / 4
    x[7, 1, 5] = float("nan")
    x[8, 2, 31] = float("inf")
    x[9, 3, 0] = -float("inf")
    x[10, 0, 0], x[10, 0, 1] = 3e38, -3e38
    x[11, 0, 3], x[11, 0, 4] = float("inf"), -float("inf")
    k = x.flatten(1)[:, None].bfloat16().to(cuda)
    v = k.flip(0).contiguous()
    cache = Q.QuantKV.alloc(12, 1, bits, cuda)
    Q.kv_quantize(k, v, cache)
    back = Q.kv_dequantize(cache)
    torch.cuda.synchronize()
    check_quantized(cache, k, v, slice(None))
    for got, want in zip(back, values_of(cache, torch.float32)):
        assert same(got.cpu().float(), want.bfloat16().float())
    assert bool(back[0][7, 0, 32:64].isnan().all()) and bool(torch.isfinite(back[0][7, 0, 64:]).all())
    assert torch.equal(back[0][0], k[0])


@pytest.mark.parametrize("bits", [4, 8])
def test_row_maps_strides_and_untouched_rows(cuda, bits):
    """Strided sources, source and target maps, entries outside that are skipped, rows that no entry names, a slice of
    a longer cache, and reading back in another order with repeated and outside entries."""
    from tokengate_amd import kvquant as Q
    n, hkv = 37, 3
    wide = torch.randn(n, 5 * hkv, 128, generator=torch.Generator(device=cuda).manual_seed(5), device=cuda).bfloat16()
    k, v = wide[:, hkv:2 * hkv], wide[:, 3 * hkv + 1:4 * hkv + 1]
    whole = Q.QuantKV.alloc(90, hkv, bits, cuda)
    for t in (whole.k, whole.v):
        t.fill_(0xA5)
    for t in (whole.k_meta, whole.v_meta):
        t.fill_(3.0)
    cut = slice(20, 80)
    cache = Q.QuantKV(bits, whole.k[:, cut], whole.k_meta[:, cut], whole.v[:, cut], whole.v_meta[:, cut])
    src = torch.tensor([5, 36, 0, 37, -1, 7, 8], dtype=torch.int32, device=cuda)      # 37 and -1 are outside
    dst = torch.tensor([59, 3, 60, 4, 5, -3, 0], dtype=torch.int32, device=cuda)      # 60 and -3 are outside
    Q.kv_quantize(k, v, cache, dst_rows=dst, src_rows=src)
    rows = torch.tensor([3, 59, 3, 60, -1, 0, 0], dtype=torch.int32, device=cuda)
    out = tuple(torch.full((9, 2 * hkv, 128), 9.0, dtype=torch.bfloat16, device=cuda)[:, ::2] for _ in range(2))
    Q.kv_dequantize(cache, rows=rows, out=out)
    torch.cuda.synchronize()
    check_quantized(cache, k[[5, 36, 8]], v[[5, 36, 8]], [59, 3, 0])
    rest = [r for r in range(90) if r not in (79, 23, 20)]
    for t, m in ((whole.k, whole.k_meta), (whole.v, whole.v_meta)):
        assert bool((t[:, rest] == 0xA5).all()) and bool((m[:, rest] == 3.0).all())
    for got, want in zip(out, values_of(cache, torch.float32)):
        want = want.bfloat16()
        assert torch.equal(got[:7].cpu(), torch.stack([want[3], want[59], want[3], 0 * want[3], 0 * want[3], want[0], want[0]]))
        assert bool((got[7:] == 9.0).all())


def attn_case(dev, used, gap, H, Hkv, bits, seed, bias, scaled):
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    g = torch.Generator(device=dev).manual_seed(seed)
    B, D = len(used), 128
    shape = dec.DecoderShape(n_layers=1, n_heads=H, n_kv_heads=Hkv, d_model=H * D)
    bf = lambda *s, std=1.0, mean=0.0: (mean + std * torch.randn(*s, generator=g, device=dev)).bfloat16()
    lw = dec.LayerWeights(None, None, bf(D, std=0.3, mean=1.0), bf(D, std=0.3, mean=1.0), None, None, None, None)
    start, r = [], 3
    for n in used:
        start.append(r)
        r += n + gap
    cache = Q.QuantKV.alloc(r, Hkv, bits, dev)
    Q.kv_quantize(bf(r, Hkv, D), bf(r, Hkv, D), cache)
    qkv = bf(B, (H + 2 * Hkv) * D)
    pos = torch.tensor([n + 7 for n in used], device=dev)
    max_k = max(used) + gap
    bias = 3 * torch.randn(B, H, max_k + 5, generator=g, device=dev) if bias else None
    qs = 0.5 + torch.rand(H, generator=g, device=dev) if scaled else None
    rs = torch.rand(B, generator=g, device=dev) if scaled else None
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    return dict(shape=shape, lw=lw, qkv=qkv, pos=pos, inv=dec.rope_inv_freq(shape, dev), cache=cache, start=i32(start),
                used=i32(used), max_k=max_k, bias=bias, qs=qs, rs=rs)


def clone_cache(c):
    from tokengate_amd import kvquant as Q
    return Q.QuantKV(c.bits, c.k.clone(), c.k_meta.clone(), c.v.clone(), c.v_meta.clone())


def run_attn(c, cache, ws, **kw):
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    rope, _ = dec.decode_begin(c["pos"].clone(), c["inv"])
    return Q.decode_attention_quant(c["qkv"], rope, c["lw"], c["shape"], cache, c["start"], c["used"], c["max_k"], SCALE,
                                    ws, c["bias"], c["qs"], c["rs"], **kw)


def check_attn(c, out, cache, skip=()):
    """out and the appended rows against float64 over what the cache held before (c["cache"])."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    shape, old, bits = c["shape"], c["cache"], c["cache"].bits
    B, Hkv, group = c["qkv"].shape[0], shape.n_kv_heads, shape.n_heads // shape.n_kv_heads
    k1, v1 = (torch.zeros(B, Hkv, 128, dtype=torch.bfloat16, device=out.device) for _ in range(2))
    q = dec.qk_norm_rope(c["qkv"].clone(), c["pos"], c["lw"], shape, c["inv"], k1, v1, c["qs"], c["rs"])
    want = clone_cache(old)
    Q.kv_quantize(k1, v1, want, dst_rows=c["start"] + c["used"] - 1)
    for a, b in ((cache.k, want.k), (cache.v, want.v), (cache.k_meta, want.k_meta), (cache.v_meta, want.v_meta)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), "cache after the append"
    kk, vv = (t.to(out.device) for t in values_of(want))
    ks, vm = want.k_meta[..., 0].double(), want.v_meta[..., 1].double().repeat_interleave(32, -1)
    vs = want.v_meta[..., 0].double().repeat_interleave(32, -1)
    L = 2 ** bits - 1
    for b in range(B):
        s, n = int(c["start"][b]), int(c["used"][b])
        for h in range(shape.n_heads):
            if (b, h) in skip:
                continue
            kh = h // group
            qd = q[b, h].double()
            k, v = kk[s:s + n, kh], vv[s:s + n, kh]
            z = k @ qd
            if c["bias"] is not None:
                z = z + c["bias"][b, h, :n].double()
            z = z * SCALE
            p = torch.softmax(z, 0)
            ref, mass = p @ v, p @ v.abs()
            coded = p @ (v - vm[kh, s:s + n])
            steps = p @ vs[kh, s:s + n]
            dz = SCALE * 2.0 ** -20 * (128 + L) * float((ks[kh, s:s + n] * qd.abs().view(4, 32).sum(1)).sum(1).max()) \
                + 2.0 ** -20 * float(z[torch.isfinite(z)].abs().max())
            tol = 2.0 ** -16 * coded + 2.0 ** -18 * (128 + L) * steps + 2.0 ** -8 * ref.abs() + (2 * dz + 2.0 ** -18) * mass + 1e-30
            err = (out[b, h].double() - ref).abs()
            assert bool((err <= tol).all()), (b, h, float((err / tol).max()))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("used,gap,H,Hkv,bias,scaled", [
    ([1], 0, 16, 8, True, False),                       # the new key alone
    ([2, 1, 3], 900, 16, 8, True, True),                # far fewer keys than the capacity
    ([64], 0, 16, 8, False, False), ([65], 0, 16, 8, False, False), ([129, 128, 127, 63], 1, 16, 8, True, False),
    ([2321], 1023, 16, 8, True, True), ([32769], 7, 16, 8, False, False),
    ([700, 5000, 33, 1600, 64, 63, 2, 9000], 5, 16, 8, True, True),
    ([1300, 40], 3, 5, 5, True, False), ([900, 17], 0, 16, 2, True, True), ([450] * 40, 2, 12, 4, True, False),
    ([333, 70], 3, 14, 2, False, True), ([500], 0, 4, 1, False, False)])
def test_decode_attention_quant(cuda, bits, used, gap, H, Hkv, bias, scaled):
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, used, gap, H, Hkv, bits, 11 + sum(used), bias, scaled)
    ws = Q.decode_attention_quant_workspace(len(used), c["shape"], c["max_k"], cuda)
    outs = []
    for _ in range(3):                                  # the workspace's counters are zero again after each
        cache = clone_cache(c["cache"])
        outs.append(run_attn(c, cache, ws))
    torch.cuda.synchronize()
    check_attn(c, outs[0], cache)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_shared_workspace(cuda):
    """Launches of different batch sizes, head counts, bits and key counts share one workspace."""
    from tokengate_amd import kvquant as Q
    sizes = [([3000] * 4, 16, 8, 4), ([2500] * 12, 16, 8, 8), ([900] * 40, 12, 4, 4), ([20000], 16, 8, 8), ([700] * 30, 16, 2, 4)]
    cases = [attn_case(cuda, used, 3, H, Hkv, bits, 40 + len(used), True, False) for used, H, Hkv, bits in sizes]
    ws = max((Q.decode_attention_quant_workspace(len(c["used"]), c["shape"], c["max_k"], cuda) for c in cases),
             key=lambda t: t.numel())
    for i in (0, 1, 2, 0, 4, 3, 1, 2, 4):
        cache = clone_cache(cases[i]["cache"])
        out = torch.full((len(sizes[i][0]), sizes[i][1], 128), float("nan"), dtype=torch.bfloat16, device=cuda)
        run_attn(cases[i], cache, ws, out=out)
        torch.cuda.synchronize()
        check_attn(cases[i], out, cache)


@pytest.mark.parametrize("bits", [4, 8])
def test_hidden_rows(cuda, bits):
    """A bias of -inf hides a row, also one that holds NaN; a head that sees no row gets zeros; the lowest finite
    bias is a bias like any other (all rows at it: all alike, as no product survives the addition)."""
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, [300, 41], 2000, 16, 8, bits, 5, True, False)
    kb, cache = c["bias"], c["cache"]
    kb[:, 3] = -float("inf")
    kb[:, 3, 17] = 0.5
    kb[1, 6] = -float("inf")
    kb[0, 9] = torch.finfo(torch.float32).min
    kb[0, 10, 100:] = torch.finfo(torch.float32).min
    s0 = int(c["start"][0])
    for h in range(16):                                 # rows 200 .. 204 of sequence 0 hold NaN, and no head sees them
        kb[0, h, 200:205] = -float("inf")
    cache.k_meta[:, s0 + 200:s0 + 205] = float("nan")
    cache.v_meta[:, s0 + 200:s0 + 205] = float("nan")
    cache.v_meta[:, s0 + 202, 1] = float("inf")
    ws = Q.decode_attention_quant_workspace(2, c["shape"], c["max_k"], cuda)
    got = clone_cache(cache)
    out = run_attn(c, got, ws)
    torch.cuda.synchronize()
    k, v = values_of(got)
    for b in range(2):
        one = v[int(c["start"][b]) + 17, 1]
        m = got.v_meta[1, int(c["start"][b]) + 17, :, 1].double().cpu().repeat_interleave(32)
        # a weight of 1: its rounding to bf16 times the step
        assert bool(((out[b, 3].double().cpu() - one).abs() <= 2.0 ** -8 * (one - m) + 2.0 ** -8 * one.abs() + 1e-6).all())
    assert bool((out[1, 6] == 0).all())
    assert bool(torch.isfinite(out).all())
    rows = [r for r in range(300) if not 200 <= r < 205]
    mean = v[s0:s0 + 300, 4][rows]
    assert bool(((out[0, 9].double().cpu() - mean.mean(0)).abs() <= 2.0 ** -8 * mean.abs().mean(0) * 2 + 2.0 ** -8 * mean.mean(0).abs() + 1e-3).all())
    # the rest, with the hidden rows' NaN replaced
    cache.k_meta[:, s0 + 200:s0 + 205] = 0.0
    cache.v_meta[:, s0 + 200:s0 + 205] = 0.0
    for t in (got.k_meta, got.v_meta):
        t[:, s0 + 200:s0 + 205] = 0.0
    check_attn(c, out, got, skip={(1, 6), (0, 9)})


def test_nan_rows_that_are_seen(cuda):
    """A key that holds NaN makes its heads' outputs NaN, a value that holds one the group's."""
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, [150], 0, 16, 8, 4, 6, False, False)
    s0 = int(c["start"][0])
    c["cache"].k_meta[2, s0 + 70, 1] = float("nan")
    c["cache"].v_meta[5, s0 + 3, 2] = float("nan")
    ws = Q.decode_attention_quant_workspace(1, c["shape"], c["max_k"], cuda)
    out = run_attn(c, clone_cache(c["cache"]), ws)
    torch.cuda.synchronize()
    bad = torch.isnan(out[0].cpu())
    want = torch.zeros(16, 128, dtype=torch.bool)
    want[4:6] = True
    want[10:12, 64:96] = True
    assert torch.equal(bad, want)


def test_rows_outside_the_cache(cuda):
    """Sequences whose rows are not all in the cache, or without rows, append nothing and get zeros; a count past
    max_k counts as max_k."""
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, [50, 60, 70, 80], 0, 16, 8, 4, 8, False, False)
    rows = c["cache"].rows
    c["start"][0] = rows - 49                           # one row past the end
    c["used"][1] = 0
    c["start"][2] = -1
    c["used"][3] = 90
    ws = Q.decode_attention_quant_workspace(4, c["shape"], c["max_k"], cuda)
    cache = clone_cache(c["cache"])
    out = run_attn(c, cache, ws)
    torch.cuda.synchronize()
    assert bool((out[:3] == 0).all())
    one = dict(c, qkv=c["qkv"][3:].contiguous(), pos=c["pos"][3:].contiguous(), start=c["start"][3:].contiguous(),
               used=c["used"][3:].contiguous().fill_(80))
    check_attn(one, out[3:], cache)


def test_long_cache(cuda):
    """Rows whose byte offsets pass 2^31 and 2^32, from a sequence's start there."""
    from tokengate_amd import kvquant as Q
    rows, hkv = 9_000_000, 8                             # codes: 4.6 GB
    c = attn_case(cuda, [700], 0, 16, hkv, 4, 9, False, False)
    long = Q.QuantKV.alloc(rows, hkv, 4, cuda)
    at = rows - 700 - 3
    for a, b in ((long.k, c["cache"].k), (long.v, c["cache"].v), (long.k_meta, c["cache"].k_meta), (long.v_meta, c["cache"].v_meta)):
        a[:, at:at + 703] = b
    ws = Q.decode_attention_quant_workspace(1, c["shape"], c["max_k"], cuda)
    small = clone_cache(c["cache"])
    want = run_attn(c, small, ws)
    c["start"] += at
    out = run_attn(c, long, ws)
    r = torch.arange(at, at + 703, dtype=torch.int32, device=cuda)
    got, back = Q.kv_dequantize(long, rows=r), Q.kv_dequantize(small)
    k, v = rand_rows(cuda, 5, hkv, 2)
    Q.kv_quantize(k, v, long, dst_rows=r[-5:].contiguous())
    Q.kv_quantize(k, v, small, dst_rows=torch.arange(698, 703, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(got, back))
    assert torch.equal(long.k[:, -5:], small.k[:, -5:]) and torch.equal(long.v_meta[:, -5:], small.v_meta[:, -5:])


def test_side_stream_and_graph(cuda):
    """Quantise, attend and read back on a side stream, and captured and replayed with other inputs."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, [1500, 200], 4, 16, 8, 4, 21, True, True)
    ws = Q.decode_attention_quant_workspace(2, c["shape"], c["max_k"], cuda)
    rope, _ = dec.decode_begin(c["pos"].clone(), c["inv"])
    new = c["start"] + c["used"] - 1
    k, v = rand_rows(cuda, 2, 8, 77)

    def step(cache):
        Q.kv_quantize(k, v, cache, dst_rows=new)
        out = Q.decode_attention_quant(c["qkv"], rope, c["lw"], c["shape"], cache, c["start"], c["used"], c["max_k"], SCALE,
                                       ws, c["bias"], c["qs"], c["rs"])
        return out, Q.kv_dequantize(cache, rows=new)

    eager = clone_cache(c["cache"])
    want, rows = step(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, rows2 = step(clone_cache(c["cache"]))
    side.synchronize()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(rows, rows2))
    cache = clone_cache(c["cache"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, read = step(cache)
    for i in range(3):
        c["qkv"].copy_(torch.randn(c["qkv"].shape, generator=torch.Generator(device=cuda).manual_seed(i), device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        ref = clone_cache(c["cache"])
        w, r = step(ref)
        torch.cuda.synchronize()
        assert torch.equal(out, w) and all(torch.equal(a, b) for a, b in zip(read, r)), i


def test_read_back_for_other_query_counts(cuda):
    """The bridge to varlen_kv_attention: several query rows over rows read back, against float64 over the bf16
    values (weights and output 2^-8 each)."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    k, v = rand_rows(cuda, 200, 8, 31)
    cache = Q.QuantKV.alloc(200, 8, 4, cuda)
    Q.kv_quantize(k, v, cache)
    kk, vv = Q.kv_dequantize(cache)
    q = rand_rows(cuda, 5, 16, 32)[0]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)
    out = dec.varlen_kv_attention(q, kk, vv, i32(0, 5), i32(0), i32(200), 5, 200, SCALE)
    torch.cuda.synchronize()
    for i in range(5):
        n = 196 + i
        a, b = kk[:n].double().repeat_interleave(2, 1), vv[:n].double().repeat_interleave(2, 1)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[i].double(), a) * SCALE, -1)
        ref, mass = torch.einsum("hn,nhd->hd", p, b), torch.einsum("hn,nhd->hd", p, b.abs())
        assert bool(((out[i].double() - ref).abs() <= 2.0 ** -8 * mass + 2.0 ** -8 * ref.abs() + 2e-5).all())


@pytest.mark.parametrize("used,H,Hkv,checked", [
    ([100 + 37 * i for i in range(130)], 8, 8, 7),          # more sequences than a wave has lanes; two rounds
    ([300 + 997 * i % 5000 for i in range(70)], 16, 8, 5),  # a cut that is corrected
    ([1 + 61 * i % 700 for i in range(2100)], 8, 8, 400),   # more units than counters: nothing is cut
    ([0, 5, 0, 3000, 1], 16, 8, 1)])                        # sequences of no key among others
def test_many_ragged_sequences(cuda, used, H, Hkv, checked):
    """Cuts of every kind: all sequences in one launch, and every `checked`-th one in a launch of its own, which cuts
    them in another way and is compared in float64.  Both are off by half a step of bf16, 2^-8 of an element, for the
    last rounding and by less than 2^-8 of the head's largest for everything else."""
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, used, 2, H, Hkv, 4, 77 + len(used), False, False)
    ws = Q.decode_attention_quant_workspace(len(used), c["shape"], c["max_k"], cuda)
    cache = clone_cache(c["cache"])
    for _ in range(2):
        out = run_attn(c, cache, ws)
    torch.cuda.synchronize()
    B = len(used)
    some = [b for b in range(0, B, checked) if used[b] > 0]
    part = dict(c, qkv=c["qkv"][some], pos=c["pos"][some], start=c["start"][some], used=c["used"][some])
    alone = clone_cache(c["cache"])
    got = run_attn(part, alone, ws)
    torch.cuda.synchronize()
    check_attn(part, got, alone)
    a, b = got.float(), out[some].float()
    assert bool(((a - b).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -7 * a.abs().amax(-1, keepdim=True)).all())
    assert all(bool((out[i] == 0).all()) for i in range(B) if used[i] == 0)


def test_strides_of_single_rows(cuda):
    """A dimension of one entry may have any stride; head-major and padded outputs."""
    from tokengate_amd import kvquant as Q
    g = torch.Generator(device=cuda).manual_seed(5)
    k, v = (torch.randn(6, 3, 128, generator=g, device=cuda).bfloat16() for _ in range(2))
    c = Q.QuantKV.alloc(6, 3, 8, cuda)
    Q.kv_quantize(k, v, c)
    want = Q.kv_dequantize(c)
    heads = tuple(torch.empty(3, 6, 128, dtype=torch.bfloat16, device=cuda).transpose(0, 1) for _ in range(2))
    wide = tuple(torch.empty(6, 4, 136, dtype=torch.bfloat16, device=cuda)[:, 1:, :128] for _ in range(2))
    for out in (heads, wide):
        got = Q.kv_dequantize(c, out=out)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = Q.QuantKV.alloc(1, 3, 8, cuda)
    odd = lambda t: t[:1].contiguous().as_strided((1, 3, 128), (3, 128, 1))
    Q.kv_quantize(odd(k), odd(v), one)
    got = Q.kv_dequantize(one, out=tuple(odd(torch.empty_like(t)) for t in (k, v)))
    assert all(torch.equal(a, b[:1]) for a, b in zip(got, want))
    # a decode step of one sequence whose row has a stride of nothing
    case = attn_case(cuda, [70], 1, 16, 8, 4, 9, False, False)
    ws = Q.decode_attention_quant_workspace(1, case["shape"], case["max_k"], cuda)
    a = run_attn(case, clone_cache(case["cache"]), ws)
    row = case["qkv"][0].clone()
    b = run_attn(dict(case, qkv=row.as_strided((1, row.numel()), (3, 1))), clone_cache(case["cache"]), ws)
    assert torch.equal(a, b)


def mirrored_case(dev, used, H, Hkv, bits, seed, bias_std):
    """A case whose cached keys come in pairs 2 i, 2 i + 1 of the same key and bias and of values s c - s L / 2 of opposite
    signs, with a new value of 0: every output is 0 exactly.  (s = 1; L / 2 is a bf16 number.)"""
    c = attn_case(dev, used, 1, H, Hkv, bits, seed, True, False)
    assert all(n % 2 == 1 for n in used)
    cache, g = c["cache"], torch.Generator(device=dev).manual_seed(seed)
    L = 2 ** bits - 1
    cache.v.copy_(torch.randint(256, cache.v.shape, generator=g, device=dev, dtype=torch.uint8))
    cache.v_meta[..., 0] = 1.0
    cache.v_meta[..., 1] = -L / 2
    c["bias"] = torch.empty(c["bias"].shape, device=dev).normal_(generator=g).mul_(bias_std)
    c["qkv"][:, (H + Hkv) * 128:] = 0.0
    for b, n in enumerate(used):
        s = int(c["start"][b])
        for t in (cache.k, cache.k_meta, cache.v):
            t[:, s + 1:s + n - 1:2] = t[:, s:s + n - 2:2]
        cache.v[:, s + 1:s + n - 1:2] ^= 255                # every code c to L - c
        c["bias"][b, :, 1:n - 1:2] = c["bias"][b, :, 0:n - 2:2]
    return c


@pytest.mark.parametrize("bits", [4, 8])
def test_long_sequences_whose_values_cancel(cuda, bits):
    """16384 keys in pairs.  A block of 32 keys goes through two instructions, of 32 additions each, that round at sizes of
    at most O = 16 + (L + 1) / 2 + 16 + L times the block's weights, and the sum before a block is next to nothing: as
    independent roundings of 2^-24 of that at most, the outputs' errors have a root mean square below
    2^-24 sqrt(64 blocks) O 32 max P.  (An offset that is carried from block to block is rounded at the size of all
    the blocks' weights.)"""
    from tokengate_amd import kvquant as Q
    n, B = 16385, 32
    c = mirrored_case(cuda, [n] * B, 16, 8, bits, 4, 0.3)
    c["qkv"][:, :16 * 128] *= 0.01
    c["lw"].q_norm.mul_(0.01)                              # (logits from the bias: weights within a factor of ten)
    ws = Q.decode_attention_quant_workspace(B, c["shape"], c["max_k"], cuda)
    out = run_attn(c, clone_cache(c["cache"]), ws).double()
    L = 2 ** bits - 1
    z = c["bias"][..., :n - 1].double() * SCALE
    most = float(torch.softmax(z, -1).max()) * 1.5          # (the products' part of z is below 0.2)
    tol = 2.0 ** -24 * (64 * n / 32) ** 0.5 * (32 + (L + 1) / 2 + L) * 32 * most
    rms = float(out.square().mean().sqrt())
    assert rms <= tol, (rms, tol)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (16, 8), (16, 2), (12, 4)])
def test_weights_of_two_keys_that_cancel(cuda, bits, H, Hkv):
    """Two keys of opposite values, one of the largest logit whose value is 0, and the new one: the outputs, 0, are off by
    the rounding of the two's weight w times L.  In 24 bits that is less than the sums' roundings: two products and their
    offsets, at sizes of at most 2 (16 + (L + 1) / 2) w or 16 + L + as much, four of them of 2^-24; and as much again for
    the weights' smaller parts, the least values' sum and the merge.  (A weight of 16 bits is off by up to 2^-17, times L.)"""
    from tokengate_amd import kvquant as Q
    used = [4] * 12
    c = mirrored_case(cuda, [3] * 12, H, Hkv, bits, 3, 1.0)
    c["used"] += 1                                          # (a free row after each)
    c["qkv"][:, :H * 128] *= 0.01
    c["lw"].q_norm.mul_(0.01)
    for b, s in enumerate(c["start"].tolist()):
        for t in (c["cache"].v, c["cache"].v_meta):
            t[:, s + 2] = 0                                 # the third key's value
        c["bias"][b, :, 0] = 20 * torch.rand(H, generator=torch.Generator().manual_seed(b)).to(cuda)
        c["bias"][b, :, 1] = c["bias"][b, :, 0]
        c["bias"][b, :, 2] = 20.0
        c["bias"][b, :, 3] = 0.0
    ws = Q.decode_attention_quant_workspace(len(used), c["shape"], c["max_k"], cuda)
    out = run_attn(c, clone_cache(c["cache"]), ws).double().abs()
    w = torch.softmax(c["bias"][..., :4].double() * SCALE, -1)[..., 0]      # (products of q and k are below 0.02)
    L = 2 ** bits - 1
    tol = 1.05 * w[..., None] * 2 * 4 * 2.0 ** -24 * (2 * (16 + (L + 1) / 2) + 16 + L)
    assert bool((out <= tol).all()), float((out / tol).max())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (16, 8), (16, 2)])
def test_values_near_the_largest_float(cuda, bits, H, Hkv):
    """Value groups whose values and steps reach up to fp32's largest, some keys or all of them, in one group or all, with
    the largest logits late: the weighted means are finite, as in float64."""
    from tokengate_amd import kvquant as Q
    used = [5, 300, 700, 1500, 64]
    c = attn_case(cuda, used, 3, H, Hkv, bits, 91, True, False)
    c["bias"] += torch.linspace(0, 200, c["bias"].shape[-1], device=cuda)    # (logits rise by up to 18)
    s = c["start"].tolist()
    g = torch.Generator(device=cuda).manual_seed(1)
    v = torch.randn(c["cache"].rows, Hkv, 4, 32, generator=g, device=cuda)
    big = torch.rand(v.shape, generator=g, device=cuda) * 2 - 1
    v[s[0]:s[0] + 4] = 1.6e38 * big[s[0]:s[0] + 4]
    v[s[1]:s[1] + 300, :, 1] = 1.6e38 * big[s[1]:s[1] + 300, :, 1]           # one group of every key
    v[s[2] + 650] = 1.6e38 * big[s[2] + 650]                                 # one key late in its sequence
    v[s[3]:s[3] + 1500] = 3e36 * big[s[3]:s[3] + 1500]
    v[s[3]:s[3] + 1500, :, 2] = 3.2e38 - 1e37 * big[s[3]:s[3] + 1500, :, 2].abs()   # all near the largest, of one sign
    v[s[4] + 10] = 3.3e38
    Q.kv_quantize(v.flatten(2).bfloat16(), v.flatten(2).bfloat16(), c["cache"])
    k = torch.randn(v.flatten(2).shape, generator=g, device=cuda).bfloat16()
    keys = Q.QuantKV.alloc(c["cache"].rows, Hkv, bits, cuda)
    Q.kv_quantize(k, k, keys)
    c["cache"].k.copy_(keys.k)
    c["cache"].k_meta.copy_(keys.k_meta)
    ws = Q.decode_attention_quant_workspace(len(used), c["shape"], c["max_k"], cuda)
    cache = clone_cache(c["cache"])
    out = run_attn(c, cache, ws)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all())
    check_attn(c, out, cache)


@pytest.mark.parametrize("bits", [4, 8])
def test_interleaved_outputs(cuda, bits):
    """Rows to read back into whose heads lie among those of other tensors, to the last element that may be written."""
    from tokengate_amd import kvquant as Q
    n, hkv = 6, 4
    k, v = rand_rows(cuda, n, hkv, 12)
    c = Q.QuantKV.alloc(n, hkv, bits, cuda)
    Q.kv_quantize(k, v, c)
    want = Q.kv_dequantize(c)

    def check(view):
        """view: of a flat buffer, (n, hkv, 128); the rest of the buffer is left as it was."""
        flat = [torch.full((16 * n * hkv * 128,), 9.0, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
        got = Q.kv_dequantize(c, out=tuple(view(f) for f in flat))
        for f, g, w in zip(flat, got, want):
            assert torch.equal(g, w)
            g.fill_(9.0)
            assert bool((f == 9.0).all())
    check(lambda f: f[:n * (2 * hkv - 1) * 128].view(n, 2 * hkv - 1, 128)[:, ::2])            # every second head
    check(lambda f: f[:hkv * (2 * n - 1) * 128].view(hkv, 2 * n - 1, 128)[:, ::2].transpose(0, 1))   # every second row of a head
    check(lambda f: f.as_strided((n, hkv, 128), (3 * 128, 19 * 128, 1)))                      # rows of one head among another's
    check(lambda f: f.as_strided((n, hkv, 128), (9 * 128, 2 * 128, 1)))
    check(lambda f: f.as_strided((n, hkv, 128), (5 * 128, 7 * 128, 1)))                       # neither within the other


@pytest.mark.parametrize("bits", [4, 8])
def test_sources_of_any_strides(cuda, bits):
    """One row for every head (a head stride of 0), one for every place (a row stride of 0), heads that overlap."""
    from tokengate_amd import kvquant as Q
    k, v = rand_rows(cuda, 7, 1, 8)
    flat = torch.randn(4096, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).bfloat16()
    for a, b in ((k.expand(7, 5, 128), v.expand(7, 5, 128)), (k[:1].expand(7, 5, 128), v[:1].expand(7, 5, 128)),
                 (flat.as_strided((7, 5, 128), (256, 64, 1)), flat.as_strided((7, 5, 128), (8, 16, 1)))):
        c, d = (Q.QuantKV.alloc(7, 5, bits, cuda) for _ in range(2))
        Q.kv_quantize(a, b, c)
        Q.kv_quantize(a.contiguous(), b.contiguous(), d)
        assert torch.equal(c.k, d.k) and torch.equal(c.v, d.v)
        assert torch.equal(c.k_meta, d.k_meta) and torch.equal(c.v_meta, d.v_meta) and bool(c.k.any())


@pytest.mark.parametrize("bits", [4, 8])
def test_groups_of_many_binary_orders(cuda, bits):
    """Groups whose least value and values differ by many binary orders, so that x - m has up to 24 bits or is rounded,
    bit for bit."""
    from tokengate_amd import kvquant as Q
    g = torch.Generator().manual_seed(9)
    n = 4096
    x = torch.randn(n, 4, 32, generator=g) * 2.0 ** torch.randint(-24, 3, (n, 4, 32), generator=g)
    x[:, 0] = x[:, 0].abs()
    x[:, 1, 0] = -(1 + 2.0 ** -7) * 2.0 ** -16          # a least value far below the others' last bit
    x[:, 1, 1:] = x[:, 1, 1:].abs() + 0.5
    x[:, 2] = 1.0 + x[:, 2].abs() * 2.0 ** -6
    x[0, 3] = torch.tensor([1.0, -(1 + 2.0 ** -7) * 2.0 ** -16] * 16)
    k = x.flatten(1)[:, None].bfloat16().to(cuda)
    v = (k.float() * 2.0 ** 60).bfloat16()
    cache = Q.QuantKV.alloc(n, 1, bits, cuda)
    Q.kv_quantize(k, v, cache)
    torch.cuda.synchronize()
    check_quantized(cache, k, v, slice(None))


@pytest.mark.parametrize("bits,used,H,Hkv", [(4, [1 + 61 * i % 700 for i in range(2100)], 8, 8),   # nothing is cut
                                             (8, [100 + 37 * i for i in range(130)], 8, 8),        # two rounds
                                             (8, [300 + 997 * i % 5000 for i in range(70)], 12, 4)])
def test_rows_that_a_large_launch_appends(cuda, bits, used, H, Hkv):
    """Every sequence's new row as kv_quantize has it, every other row as it was, and outputs of sequences all over the
    batch in float64."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    c = attn_case(cuda, used, 2, H, Hkv, bits, 5 + len(used), True, True)
    B = len(used)
    ws = Q.decode_attention_quant_workspace(B, c["shape"], c["max_k"], cuda)
    cache, want = clone_cache(c["cache"]), clone_cache(c["cache"])
    out = run_attn(c, cache, ws)
    k1, v1 = (torch.empty(B, Hkv, 128, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    dec.qk_norm_rope(c["qkv"].clone(), c["pos"], c["lw"], c["shape"], c["inv"], k1, v1, c["qs"], c["rs"])
    Q.kv_quantize(k1, v1, want, dst_rows=c["start"] + c["used"] - 1)
    torch.cuda.synchronize()
    for a, b in ((cache.k, want.k), (cache.v, want.v), (cache.k_meta, want.k_meta), (cache.v_meta, want.v_meta)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    some = list(range(0, B, max(1, B // 30)))
    rows = lambda t: t[some].contiguous()
    part = dict(c, qkv=rows(c["qkv"]), pos=rows(c["pos"]), start=rows(c["start"]), used=rows(c["used"]), bias=rows(c["bias"]),
                rs=rows(c["rs"]))
    view = clone_cache(c["cache"])                      # (check_attn appends only these sequences' rows)
    new = (part["start"] + part["used"] - 1).long()
    for a, b in ((view.k, cache.k), (view.v, cache.v), (view.k_meta, cache.k_meta), (view.v_meta, cache.v_meta)):
        a[:, new] = b[:, new]
    check_attn(part, rows(out), view)
