"""The operators of a decode step over a quantised KV cache, as cases that can be timed and compared.

Kinds of case (the `kind` of each dict):

  roundtrip  kv_quantize and kv_dequantize: the K and V rows of a layer are quantised into its cache and read
             back as bf16.
  attention  decode_attention_quant: one token for every sequence, from the raw q|k|v projection rows to the
             attention output over a cache of 4 or 8 bits, the new rows quantised on the way in; the appended
             rows are read back.
  sample     sample_rows: the next token of every row of logits with temperature, top-k, top-p and min-p, from
             given random numbers, and its log probability.

The quantised form of a K or V row of one head (128 bf16 values): groups g = 0 .. 3 of 32 consecutive values,
each with its least value m and a step s = bf16((max - m) / L), L = 15 or 255, both bf16; a value is held as the
whole number c nearest to (x - m) / s in 0 .. L and stands for s c + m.  (Steps under 2^-100 are held as 0; a group
whose max - m is not finite reads back as NaN.)

The plain forms are elementary torch operations in 32 bits (sums of probabilities in 64); `exact` is in float64.
"""
import math

import torch

own = False

D = 128                      # head dim
GROUP = 32                   # values that share a step and a least value
EPS = 1e-6
SCALE = D ** -0.5
VOCAB = 151936
DEVICE = "cuda"


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # the rows of one decode step of eight sequences
        dict(name="roundtrip_8_4bit", kind="roundtrip", rows=8, kv_heads=8, bits=4, gap=False, strided=False),
        # one layer of a 4k prompt, straight from the projection's rows
        dict(name="roundtrip_4096_8bit", kind="roundtrip", rows=4096, kv_heads=8, bits=8, gap=False, strided=True),
        # one layer of five packed prompts, into a cache with room after each
        dict(name="roundtrip_98765_4bit", kind="roundtrip", rows=98765, kv_heads=8, bits=4, gap=True, strided=False),
        # a short chat prompt: launch, row stage and merge count
        dict(name="attention_b1_300_4bit", kind="attention", seqs=1, max_k=300, ragged=False, heads=16, kv_heads=8,
             bits=4, bias=False, scaled=False),
        # the pruned cache of a 32k prompt (K = 2000) with its gate bias and query scales
        dict(name="attention_b1_2320_4bit", kind="attention", seqs=1, max_k=2320, ragged=False, heads=16, kv_heads=8,
             bits=4, bias=True, scaled=True),
        # a layer below the gate: the whole 32k prompt
        dict(name="attention_b1_32769_4bit", kind="attention", seqs=1, max_k=32769, ragged=False, heads=16, kv_heads=8,
             bits=4, bias=False, scaled=False),
        # a served batch with gate bias, 8 bits
        dict(name="attention_b64_4099_8bit", kind="attention", seqs=64, max_k=4099, ragged=True, heads=16, kv_heads=8,
             bits=8, bias=True, scaled=False),
        # eight prompts of 16k to 128k
        dict(name="attention_b8_131072_4bit", kind="attention", seqs=8, max_k=131072, ragged=True, heads=16,
             kv_heads=8, bits=4, bias=False, scaled=False),
        # one chat turn with the usual settings
        dict(name="sample_b1_k20", kind="sample", rows=1, vocab=VOCAB, temperature=0.7, top_k=20, top_p=0.8, min_p=0.0,
             mixed=False),
        # nucleus sampling without top-k
        dict(name="sample_b8_p95", kind="sample", rows=8, vocab=VOCAB, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0,
             mixed=False),
        # the whole distribution (training rollouts)
        dict(name="sample_b4_plain", kind="sample", rows=4, vocab=VOCAB, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             mixed=False),
        # a served batch whose rows have settings of their own
        dict(name="sample_b64_mixed", kind="sample", rows=64, vocab=VOCAB, temperature=1.0, top_k=50, top_p=0.9,
             min_p=0.05, mixed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["roundtrip", "attention", "attention", "sample"])
    if kind == "roundtrip":
        return dict(kind=kind, rows=_log_int(rng, 1, 98000), kv_heads=rng.choice([1, 2, 4, 5, 8]), bits=rng.choice([4, 8]),
                    gap=rng.random() < 0.5, strided=rng.random() < 0.5)
    if kind == "attention":
        seqs = _log_int(rng, 1, 64)
        heads, kv_heads = rng.choice([(16, 8), (16, 8), (12, 4), (16, 2), (8, 8), (5, 5)])
        return dict(kind=kind, seqs=seqs, max_k=_log_int(rng, 1, min(131072, 400000 // seqs)), ragged=rng.random() < 0.6,
                    heads=heads, kv_heads=kv_heads, bits=rng.choice([4, 4, 8]), bias=rng.random() < 0.5,
                    scaled=rng.random() < 0.5)
    return dict(kind=kind, rows=_log_int(rng, 1, 64), vocab=rng.choice([VOCAB, _log_int(rng, 500, VOCAB)]),
                temperature=round(rng.uniform(0.3, 1.6), 2), top_k=rng.choice([0, 0, 1, 20, 50, 1000, 20000]),
                top_p=rng.choice([1.0, 0.5, 0.8, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                mixed=rng.random() < 0.4)


# ---- inputs ------------------------------------------------------------------------------------

def _lengths(case, g):
    """Keys of every sequence, the new one included."""
    n, m = case["seqs"], case["max_k"]
    if not case["ragged"]:
        return [m] * n
    u = torch.rand(n, generator=g, device=DEVICE).cpu().tolist()
    lens = [max(1, min(m, round(m * (0.125 + 0.875 * x)))) for x in u]
    lens[n // 2] = m
    return lens


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*size, std=1.0, mean=0.0):
        return torch.randn(*size, generator=g, device=DEVICE).mul_(std).add_(mean).to(torch.bfloat16)

    s = dict(case)
    if case["kind"] == "roundtrip":
        n, hkv = case["rows"], case["kv_heads"]
        if case["strided"]:      # k and v inside projection rows [q | k | v] with as many query heads
            row = normal(n, 3 * hkv * D)
            s["src_k"] = row[:, hkv * D:2 * hkv * D].unflatten(1, (hkv, D))
            s["src_v"] = row[:, 2 * hkv * D:].unflatten(1, (hkv, D))
        else:
            s["src_k"], s["src_v"] = normal(n, hkv, D), normal(n, hkv, D)
        rows, s["map"] = n, None
        if case["gap"]:          # five sequences, seven free rows after each
            cut = [n * i // 5 for i in range(6)]
            s["map"] = torch.cat([torch.arange(cut[i], cut[i + 1], dtype=torch.int32) + 7 * i for i in range(5)]).to(DEVICE)
            rows = n + 35
        s["cache"] = _empty_cache(rows, hkv, case["bits"])
        return s
    if case["kind"] == "attention":
        b, h, hkv = case["seqs"], case["heads"], case["kv_heads"]
        lens = _lengths(case, g)
        start, rows = [], 0
        for n in lens:           # room for 16 more rows after each sequence
            start.append(rows)
            rows += n + 16
        chunk = max(1, (1 << 27) // (hkv * D))
        cache = _empty_cache(rows, hkv, case["bits"])
        for name in ("k", "v"):
            for r in range(0, rows, chunk):
                m = min(chunk, rows - r)
                c, t = _quantise(torch.randn(hkv, m, D, generator=g, device=DEVICE), case["bits"])
                cache[name][:, r:r + m] = c
                cache[name + "_meta"][:, r:r + m] = t
        s["cache"] = cache
        s["qkv"] = normal(b, (h + 2 * hkv) * D)
        s["q_norm"], s["k_norm"] = normal(D, std=0.1, mean=1.0), normal(D, std=0.1, mean=1.0)
        used = torch.tensor(lens, device=DEVICE)
        inv = 1e6 ** (-torch.arange(0, D, 2, device=DEVICE, dtype=torch.float64) / D)
        angle = (used + 9).double()[:, None] * inv
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        s["start"] = torch.tensor(start, dtype=torch.int32, device=DEVICE)
        s["used"] = used.to(torch.int32)
        s["new_rows"] = s["start"] + s["used"] - 1
        s["limit"] = max(lens) + 16
        s["bias"] = torch.randn(b, h, s["limit"], generator=g, device=DEVICE).mul_(4.0) if case["bias"] else None
        s["q_head"] = 0.7 + 0.6 * torch.rand(h, generator=g, device=DEVICE) if case["scaled"] else None
        s["q_row"] = 0.6 + 0.4 * torch.rand(b, generator=g, device=DEVICE) if case["scaled"] else None
        return s
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, generator=g, device=DEVICE).mul_(2.0)
    peaks = torch.randint(v, (n, 24), generator=g, device=DEVICE)
    x.scatter_add_(1, peaks, 3.0 + 9.0 * torch.rand(n, 24, generator=g, device=DEVICE))
    s["logits"] = x.to(torch.bfloat16).float()      # the LM head's values are bf16
    s["u"] = torch.rand(n, generator=g, device=DEVICE)
    t, k, p, m = (torch.full((n,), case[f], device=DEVICE, dtype=d) for f, d in
                  (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32),
                   ("min_p", torch.float32)))
    if case["mixed"]:            # rows of other requests: greedy, without top-k, without top-p
        kind = torch.randint(4, (n,), generator=g, device=DEVICE)
        t = torch.where(kind == 0, torch.zeros_like(t), t)
        k = torch.where(kind == 1, torch.zeros_like(k), k)
        p = torch.where(kind == 2, torch.ones_like(p), p)
        m = torch.where(kind == 3, torch.zeros_like(m), m)
    s.update(temperature=t, top_k=k, top_p=p, min_p=m)
    return s


def _empty_cache(rows, kv_heads, bits):
    """Codes (kv_heads, rows, 16 bits) bytes and (step, least value) of each group, for K and V."""
    out = {}
    for name in ("k", "v"):
        out[name] = torch.zeros(kv_heads, rows, 16 * bits, dtype=torch.uint8, device=DEVICE)
        out[name + "_meta"] = torch.zeros(kv_heads, rows, D // GROUP, 2, dtype=torch.bfloat16, device=DEVICE)
    return out


# ---- the plain forms ---------------------------------------------------------------------------

def _quantise(x, bits):
    """(codes, meta) of bf16 values x (..., 128).  Word w (of 4 bytes, at 8 bits of 8) holds the elements 16 e + w."""
    top = (1 << bits) - 1
    x = x.to(torch.bfloat16).float().unflatten(-1, (D // GROUP, GROUP))
    least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = most - least
    step = (span / torch.full_like(span, top)).to(torch.bfloat16).float()      # (a tensor: quotients, no reciprocals)
    step = torch.where(step < 2.0 ** -100, torch.zeros_like(step), step)
    c = ((x - least) / torch.where(step > 0, step, torch.full_like(step, math.inf))).round().clamp(0, top)
    fine = torch.isfinite(span)
    c = torch.where(fine, c, torch.zeros_like(c)).to(torch.uint8).flatten(-2)
    meta = torch.where(fine, torch.cat([step, least], -1), torch.full_like(span, float("nan"))).to(torch.bfloat16)
    e = c.unflatten(-1, (8, 16)).transpose(-1, -2)              # (..., word, e)
    if bits == 4:
        e = e[..., 0::2] | (e[..., 1::2] << 4)
    return e.flatten(-2), meta


def _values(codes, meta, bits):
    """fp32 values that the codes (..., 16 bits) stand for."""
    e = codes.unflatten(-1, (16, bits))
    if bits == 4:
        e = torch.stack([e & 15, e >> 4], -1).flatten(-2)
    c = e.transpose(-1, -2).flatten(-2).float().unflatten(-1, (D // GROUP, GROUP))
    m = meta.float()
    return (c * m[..., :1] + m[..., 1:]).flatten(-2)


def _bf16(x):
    return x.to(torch.bfloat16).to(x.dtype)


def _norm_rope(x, weight, rope):
    """RMSNorm of head rows x (B, heads, 128) and rotation of the halves; bf16 values."""
    y = weight.float() * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS))
    cos, sin = (t.repeat(1, 2)[:, None] for t in rope.unbind(-1))
    half = torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1)
    return _bf16(y * cos + half * sin)


def _plain_attention(s):
    b, h, hkv, bits, n = s["seqs"], s["heads"], s["kv_heads"], s["bits"], s["max_k"]
    row = s["qkv"].float().unflatten(1, (h + 2 * hkv, D))
    q = _norm_rope(row[:, :h], s["q_norm"], s["rope"])
    if s["scaled"]:
        q = _bf16(q * _bf16(s["q_row"][:, None] * s["q_head"])[..., None])
    cache, new = s["cache"], s["new_rows"].long()
    back = {}
    for name, x in (("k", _norm_rope(row[:, h:h + hkv], s["k_norm"], s["rope"])), ("v", row[:, h + hkv:])):
        codes, meta = _quantise(x.transpose(0, 1), bits)
        cache[name][:, new] = codes
        cache[name + "_meta"][:, new] = meta
        back[name] = _values(codes, meta, bits).transpose(0, 1).to(torch.bfloat16).contiguous()
    at = torch.arange(n, device=DEVICE)
    there = at < s["used"][:, None]                              # (B, n)
    rows = (s["start"][:, None] + torch.where(there, at, torch.zeros_like(at))).long()
    k, v = (_values(cache[x][:, rows], cache[x + "_meta"][:, rows], bits).transpose(0, 1) for x in ("k", "v"))
    z = torch.matmul(q.view(b, hkv, h // hkv, D), k.transpose(-1, -2).contiguous()).view(b, h, n)
    if s["bias"] is not None:
        z = z + s["bias"][..., :n]
    z = torch.where(there[:, None], z * SCALE, torch.full_like(z, -math.inf))
    top = z.amax(-1, keepdim=True)
    p = torch.where(z == -math.inf, torch.zeros_like(z), torch.exp(z - top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p.view(b, hkv, h // hkv, n), v).view(b, h, D).to(torch.bfloat16)
    return {"out": out, "k": back["k"], "v": back["v"]}


def _plain_sample(s):
    x = s["logits"]
    v = x.shape[1]
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    val = val.double()
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((val - val[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    at = torch.arange(v, device=x.device)
    k = s["top_k"].long()[:, None]
    w = torch.where((at < torch.where((k <= 0) | (k > v), torch.full_like(k, v), k)), w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    p = s["top_p"].double()[:, None]
    w = torch.where((p >= 1) | (before < p * w.sum(1, keepdim=True)) | (at == 0), w, torch.zeros_like(w))
    w = torch.where((w >= s["min_p"].double()[:, None]) | (at == 0), w, torch.zeros_like(w))
    w = torch.where(greedy & (at > 0), torch.zeros_like(w), w)
    cum, total = w.cumsum(1), w.sum(1, keepdim=True)
    over = cum > s["u"].double()[:, None] * total
    place = torch.where(over.any(1), over.int().argmax(1), (w > 0).sum(1) - 1)[:, None]
    return {"token": idx.gather(1, place)[:, 0], "logprob": (w.gather(1, place) / total).log()[:, 0].float()}


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "roundtrip":
        rows = slice(0, s["rows"]) if s["map"] is None else s["map"].long()
        back = []
        for name in ("k", "v"):
            codes, meta = _quantise(s["src_" + name].transpose(0, 1), s["bits"])
            s["cache"][name][:, rows], s["cache"][name + "_meta"][:, rows] = codes, meta
            got = _values(s["cache"][name][:, rows], s["cache"][name + "_meta"][:, rows], s["bits"])
            back.append(got.transpose(0, 1).to(torch.bfloat16).contiguous())
        return back
    return _plain_attention(s) if s["kind"] == "attention" else _plain_sample(s)


def _run_own(s):
    from tokengate_amd import decoder, kvquant
    if s["kind"] == "sample":
        if "workspace" not in s:         # kept with the logits' buffer, as a decode loop does
            s["workspace"] = decoder.sample_rows_workspace(*s["logits"].shape, s["logits"].device)
        token, logprob = decoder.sample_rows(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                                             workspace=s["workspace"], logprob=True)
        return {"token": token, "logprob": logprob}
    if "quant" not in s:                 # the cache's handle
        c = s["cache"]
        s["quant"] = kvquant.QuantKV(s["bits"], c["k"], c["k_meta"], c["v"], c["v_meta"])
    if s["kind"] == "roundtrip":
        kvquant.kv_quantize(s["src_k"], s["src_v"], s["quant"], dst_rows=s["map"])
        return list(kvquant.kv_dequantize(s["quant"], rows=s["map"], n_rows=s["rows"]))
    if "workspace" not in s:             # a decode loop's weights, shape and workspace
        s["shape"] = decoder.DecoderShape(n_layers=1, n_heads=s["heads"], n_kv_heads=s["kv_heads"], rms_eps=EPS)
        s["weights"] = decoder.LayerWeights(None, None, s["q_norm"], s["k_norm"], None, None, None, None)
        s["workspace"] = kvquant.decode_attention_quant_workspace(s["seqs"], s["shape"], s["limit"], s["qkv"].device)
    out = kvquant.decode_attention_quant(s["qkv"], s["rope"], s["weights"], s["shape"], s["quant"], s["start"], s["used"],
                                         s["limit"], SCALE, s["workspace"], s["bias"], s["q_head"], s["q_row"])
    k, v = kvquant.kv_dequantize(s["quant"], rows=s["new_rows"], n_rows=s["seqs"])
    return {"out": out, "k": k, "v": v}


def work(case):
    if case["kind"] == "roundtrip":
        held = 2 * case["rows"] * case["kv_heads"] * (16 * case["bits"] + 16)
        return {"bytes": 2 * held + 2 * 2 * case["rows"] * case["kv_heads"] * D * 2, "flops": 0}
    if case["kind"] == "attention":
        keys = case["max_k"] * (1 + (case["seqs"] - 1) * (0.5625 if case["ragged"] else 1.0))   # (expected)
        held = 2 * (16 * case["bits"] + 16) * case["kv_heads"]
        rows = case["seqs"] * (case["heads"] * 2 * 2 + case["kv_heads"] * 2 * 4) * D
        return {"bytes": keys * (held + (4 * case["heads"] if case["bias"] else 0)) + rows,
                "flops": 4.0 * D * case["heads"] * keys}
    return {"bytes": case["rows"] * (4.0 * case["vocab"] + 32), "flops": 0}


# ---- the definition in float64 -----------------------------------------------------------------

def _exact_group(x, bits):
    """The values that a row of bf16 values (..., 128) is held as."""
    L = 2 ** bits - 1
    out = torch.empty_like(x)
    for g in range(4):
        part = x[..., 32 * g:32 * g + 32]
        lo, hi = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        s = ((hi - lo) / L).to(torch.bfloat16).double()
        s = torch.where(s < 2.0 ** -100, torch.zeros_like(s), s)
        c = torch.clamp(torch.round((part - lo) / torch.where(s > 0, s, torch.ones_like(s))), 0, L)
        out[..., 32 * g:32 * g + 32] = lo + s * c
    return out


def _exact_read(codes, meta, bits):
    """float64 values of codes (heads, n, 16 bits): element 16 e + w is nibble (byte) e of word (pair of words) w."""
    heads, n, _ = codes.shape
    out = torch.empty(heads, n, D, dtype=torch.float64, device=codes.device)
    for e in range(8):
        c = (codes[:, :, e // 2::4] >> (4 * (e % 2))) & 15 if bits == 4 else codes[:, :, e::8]
        s, m = meta[:, :, e // 2, 0].double()[..., None], meta[:, :, e // 2, 1].double()[..., None]
        out[:, :, 16 * e:16 * e + 16] = c.double() * s + m
    return out


def _exact_head(x, w, rope):
    """x (heads, 128) of one token."""
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
    a, b = y[:, :64], y[:, 64:]
    c, s = rope[:, 0].double(), rope[:, 1].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(torch.bfloat16).double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "roundtrip":
        return [_exact_group(s[x].double(), case["bits"]) for x in ("src_k", "src_v")]
    if case["kind"] == "attention":
        h, hkv = case["heads"], case["kv_heads"]
        outs, ks, vs = [], [], []
        for b in range(case["seqs"]):
            row = s["qkv"][b].double().view(h + 2 * hkv, D)
            q = _exact_head(row[:h], s["q_norm"], s["rope"][b])
            if case["scaled"]:
                f = (s["q_row"][b] * s["q_head"]).to(torch.bfloat16).double()      # the scale is a bf16 number
                q = (q * f[:, None]).to(torch.bfloat16).double()
            k1 = _exact_group(_exact_head(row[h:h + hkv], s["k_norm"], s["rope"][b]), case["bits"])
            v1 = _exact_group(row[h + hkv:], case["bits"])
            r0, n = int(s["start"][b]), int(s["used"][b])
            c = s["cache"]
            k = _exact_read(c["k"][:, r0:r0 + n], c["k_meta"][:, r0:r0 + n], case["bits"])
            v = _exact_read(c["v"][:, r0:r0 + n], c["v_meta"][:, r0:r0 + n], case["bits"])
            k[:, n - 1], v[:, n - 1] = k1, v1
            out = torch.empty(h, D, dtype=torch.float64, device=DEVICE)
            for i in range(h):
                z = k[i // (h // hkv)] @ q[i]
                if s["bias"] is not None:
                    z = z + s["bias"][b, i, :n].double()
                out[i] = torch.softmax(z / math.sqrt(D), 0) @ v[i // (h // hkv)]
            outs.append(out)
            ks.append(k1)
            vs.append(v1)
        return {"out": torch.stack(outs), "k": torch.stack(ks), "v": torch.stack(vs)}
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    t, k, p, m, u = (s[f].double().cpu().numpy() for f in ("temperature", "top_k", "top_p", "min_p", "u"))
    token, logprob = [], []
    for b in range(x.shape[0]):
        order = np.lexsort((np.arange(x.shape[1]), -x[b]))
        if t[b] <= 0:
            token.append(int(order[0]))
            logprob.append(0.0)
            continue
        if 0 < k[b] < len(order):
            order = order[:int(k[b])]
        w = np.exp((x[b, order] - x[b, order[0]]) / t[b])
        if p[b] < 1:
            keep = max(1, int(np.searchsorted(np.cumsum(w), p[b] * w.sum())) + 1)
            order, w = order[:keep], w[:keep]
        keep = max(1, int((w >= m[b]).sum()))
        order, w = order[:keep], w[:keep]
        i = min(keep - 1, int(np.searchsorted(np.cumsum(w), u[b] * w.sum(), side="right")))
        token.append(int(order[i]))
        logprob.append(math.log(w[i] / w.sum()))
    return {"token": torch.tensor(token, device=DEVICE), "logprob": torch.tensor(logprob, dtype=torch.float64)}
