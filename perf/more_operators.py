"""The operators of a paged KV cache, as cases that can be timed and compared.

Kinds of case (the `kind` of each dict):

  append     paged_append: q/k RMSNorm and rotary embedding of raw q|k|v projection rows, the queries to rows of
             their own, the keys and values into the pages that the rows' slots name.
  attention  paged_attention: causal attention of several query rows per sequence (a prompt, or a part of one whose
             beginning is in the cache) over pages named by a table.
  decode     paged_decode_attention: one new token per sequence, from the raw q|k|v projection row to the attention
             output, its key and value appended to the sequence's last page.

The cache: k and v of logical shape (pages, KV heads, page rows, 128), bf16; key j of sequence b is row j % page of
page table[b, j // page].  The logit of a query and a key is scale * (q . k + bias[b, head, key]).

The plain forms are elementary torch operations in 32 bits; `exact` is in float64.
"""
import math

import torch

own = False

D = 128                      # head dim
EPS = 1e-6
SCALE = D ** -0.5
DEVICE = "cuda"


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one token of each of eight sequences
        dict(name="append_8", kind="append", rows=8, seqs=8, heads=16, kv_heads=8, page=16, scaled=False, token_major=False),
        # five prompts of about a thousand tokens, kept rows of a pruned prompt with query scales
        dict(name="append_4099", kind="append", rows=4099, seqs=5, heads=16, kv_heads=8, page=64, scaled=True,
             token_major=False),
        # one layer of a 32k prompt
        dict(name="append_32768", kind="append", rows=32768, seqs=1, heads=16, kv_heads=8, page=64, scaled=False,
             token_major=False),
        # a question of 33 tokens after a cached article
        dict(name="attention_b1_33_32769", kind="attention", seqs=1, max_q=33, max_k=32769, ragged=False, heads=16,
             kv_heads=8, page=64, bias=False, token_major=False),
        # the kept rows of a pruned prompt with their gate bias
        dict(name="attention_b1_2320_2320", kind="attention", seqs=1, max_q=2320, max_k=2320, ragged=False, heads=16,
             kv_heads=8, page=64, bias=True, token_major=False),
        # the next prompt chunks of a served batch, small pages
        dict(name="attention_b12_700_4099", kind="attention", seqs=12, max_q=700, max_k=4099, ragged=True, heads=16,
             kv_heads=8, page=16, bias=False, token_major=True),
        # the last chunk of a 32k prompt
        dict(name="attention_b1_8192_32768", kind="attention", seqs=1, max_q=8192, max_k=32768, ragged=False, heads=16,
             kv_heads=8, page=64, bias=False, token_major=False),
        # a short chat prompt: launch, row stage and merge count
        dict(name="decode_b1_300", kind="decode", seqs=1, max_k=300, ragged=False, heads=16, kv_heads=8, page=16,
             bias=False, scaled=False, token_major=False),
        # the pruned cache of a 32k prompt (K = 2000) with its gate bias and query scales
        dict(name="decode_b1_2320", kind="decode", seqs=1, max_k=2320, ragged=False, heads=16, kv_heads=8, page=64,
             bias=True, scaled=True, token_major=False),
        # a layer below the gate: the whole 32k prompt
        dict(name="decode_b1_32769", kind="decode", seqs=1, max_k=32769, ragged=False, heads=16, kv_heads=8, page=64,
             bias=False, scaled=False, token_major=False),
        # a served batch with gate bias, small pages
        dict(name="decode_b64_4099", kind="decode", seqs=64, max_k=4099, ragged=True, heads=16, kv_heads=8, page=16,
             bias=True, scaled=False, token_major=True),
        # eight prompts of 16k to 128k
        dict(name="decode_b8_131072", kind="decode", seqs=8, max_k=131072, ragged=True, heads=16, kv_heads=8, page=64,
             bias=False, scaled=False, token_major=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "decode", "decode"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (12, 4), (16, 2), (8, 8), (5, 5), (16, 1)])
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, page=rng.choice([16, 32, 64, 64, 128, 256]),
                token_major=rng.random() < 0.4)
    if kind == "append":
        rows = _log_int(rng, 1, 32000)
        return dict(case, rows=rows, seqs=_log_int(rng, 1, min(rows, 64)), scaled=rng.random() < 0.5)
    if kind == "attention":
        seqs = _log_int(rng, 1, 24)
        max_k = _log_int(rng, 2, min(32768, 100000 // seqs))
        return dict(case, seqs=seqs, max_k=max_k, max_q=_log_int(rng, 2, min(max_k, 8192 // seqs)), ragged=rng.random() < 0.6,
                    bias=rng.random() < 0.5)
    seqs = _log_int(rng, 1, 64)
    return dict(case, seqs=seqs, max_k=_log_int(rng, 1, min(131072, 400000 // seqs)), ragged=rng.random() < 0.6,
                bias=rng.random() < 0.5, scaled=rng.random() < 0.5)


def _spread(n, most, ragged):
    """Lengths of n sequences of up to `most`, an eighth of it to all of it."""
    if not ragged:
        return [most] * n
    return [most] + [max(1, round(most * (0.125 + 0.875 * ((i * 0.6180339887) % 1.0)))) for i in range(1, n)]


def _lengths(case):
    """(new rows, keys with the new ones) of every sequence."""
    n = case["seqs"]
    if case["kind"] == "append":
        cut = [case["rows"] * i // n for i in range(n + 1)]
        new = [cut[i + 1] - cut[i] for i in range(n)]
        return new, [x + 37 for x in new]
    keys = _spread(n, case["max_k"], case["ragged"])
    if case["kind"] == "decode":
        return [1] * n, keys
    new = _spread(n, case["max_q"], case["ragged"])
    return [min(x, y) for x, y in zip(new[:1] + new[:0:-1], keys)], keys


# ---- inputs ------------------------------------------------------------------------------------

def _rotation(positions):
    """(cos, sin) (n, 64, 2) of the positions' angles."""
    inv = 1e6 ** (-torch.arange(0, D, 2, device=DEVICE, dtype=torch.float64) / D)
    angle = positions.double()[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*size, std=1.0, mean=0.0):
        return torch.randn(*size, generator=g, device=DEVICE).mul_(std).add_(mean).to(torch.bfloat16)

    s = dict(case)
    n, h, hkv, page = case["seqs"], case["heads"], case["kv_heads"], case["page"]
    new, keys = _lengths(case)
    order = torch.randperm(n, generator=g, device=DEVICE).cpu().tolist()
    new, keys = [new[i] for i in order], [keys[i] for i in order]
    # the pages of every sequence, anywhere in a pool that holds a few more; entries past a sequence's pages name none
    need = [(x + page - 1) // page for x in keys]
    pool = sum(need) + 5
    where = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((n, max(need) + 1), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b in range(n):
        table[b, :need[b]] = where[at:at + need[b]]
        at += need[b]
    s["table"], s["pool"] = table, pool
    for name in ("k", "v"):
        size = (pool, page, hkv, D) if case["token_major"] else (pool, hkv, page, D)
        x = torch.randn(size, generator=g, device=DEVICE, dtype=torch.bfloat16)
        s[name] = x.transpose(1, 2) if case["token_major"] else x
    s["used"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE)
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
    if case["kind"] == "attention":
        s["q"] = normal(cu[-1], h, D)
    else:
        s["qkv"] = normal(cu[-1], (h + 2 * hkv) * D)
        s["q_norm"], s["k_norm"] = normal(D, std=0.1, mean=1.0), normal(D, std=0.1, mean=1.0)
        key = torch.cat([torch.arange(k - q, k) for q, k in zip(new, keys)]).to(DEVICE)      # of every row
        seq = torch.repeat_interleave(torch.arange(n), torch.tensor(new)).to(DEVICE)
        s["rope"] = _rotation(key + 9)
        s["slots"] = table[seq, key // page] * page + (key % page).to(torch.int32)
        s["q_head"] = 0.7 + 0.6 * torch.rand(h, generator=g, device=DEVICE) if case["scaled"] else None
        s["q_row"] = 0.6 + 0.4 * torch.rand(cu[-1], generator=g, device=DEVICE) if case["scaled"] else None
    if case["kind"] != "append":
        s["bias"] = torch.randn(n, h, case["max_k"], generator=g, device=DEVICE).mul_(4.0) if case["bias"] else None
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _norm_rope(x, weight, rope):
    """RMSNorm of head rows x (rows, heads, 128) and rotation of the halves; bf16 values."""
    y = weight.float() * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS))
    cos, sin = (t.repeat(1, 2)[:, None] for t in rope.unbind(-1))
    half = torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1)
    return (y * cos + half * sin).to(torch.bfloat16)


def _plain_append(s):
    """The queries (rows, heads, 128); keys and values go to their slots."""
    h, hkv, page = s["heads"], s["kv_heads"], s["page"]
    row = s["qkv"].unflatten(1, (h + 2 * hkv, D))
    q = _norm_rope(row[:, :h].float(), s["q_norm"], s["rope"])
    if s["scaled"]:
        factor = (s["q_row"][:, None] * s["q_head"]).to(torch.bfloat16).float()
        q = (q.float() * factor[..., None]).to(torch.bfloat16)
    at, off = (s["slots"] // page).long(), (s["slots"] % page).long()
    s["k"][at, :, off] = _norm_rope(row[:, h:h + hkv].float(), s["k_norm"], s["rope"])
    s["v"][at, :, off] = row[:, h + hkv:]
    return q


def _plain_attention(s, q):
    """out (rows, heads, 128) of the query rows q: the rows of a sequence are its last keys' queries."""
    n, h, hkv, page, most = s["seqs"], s["heads"], s["kv_heads"], s["page"], s["max_k"]
    pages = s["table"][:, :(most + page - 1) // page].long().clamp(min=0)
    k, v = (s[x][pages].float().transpose(1, 2).reshape(n, hkv, -1, D)[:, :, :most] for x in ("k", "v"))
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    rows = s.get("max_q", 1)
    i = torch.arange(rows, device=DEVICE)
    there = i < new[:, None]                                                   # (n, rows)
    src = (s["cu"][:-1, None] + torch.minimum(i, (new - 1)[:, None])).long()
    qs = q[src].float().transpose(1, 2).reshape(n, hkv, h // hkv * rows, D)
    z = torch.matmul(qs, k.transpose(-1, -2).contiguous()).view(n, h, rows, most)
    if s["bias"] is not None:
        z += s["bias"][:, :, None]
    last = s["used"].long()[:, None] - new[:, None] + i                        # each row's own key
    seen = torch.arange(most, device=DEVICE) <= last[..., None]
    z = torch.where(seen[:, None], z * SCALE, -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hkv, h // hkv * rows, most), v.contiguous()).view(n, h, rows, D)
    return out.transpose(1, 2)[there].to(torch.bfloat16)


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "attention":
        return _plain_attention(s, s["q"])
    q = _plain_append(s)
    out = q if s["kind"] == "append" else _plain_attention(s, q)
    return {"out": out, "k": s["k"], "v": s["v"]}


def _run_own(s):
    from tokengate_amd import decoder, paged
    if "cache" not in s:                 # a serving loop's cache, weights, shape and workspace
        s["cache"] = paged.PagedKV(s["k"], s["v"])
        s["shape"] = decoder.DecoderShape(n_layers=1, n_heads=s["heads"], n_kv_heads=s["kv_heads"], rms_eps=EPS)
        if s["kind"] != "attention":
            s["weights"] = decoder.LayerWeights(None, None, s["q_norm"], s["k_norm"], None, None, None, None)
        if s["kind"] == "decode":
            s["workspace"] = paged.paged_decode_attention_workspace(s["seqs"], s["shape"], s["max_k"], s["qkv"].device)
    if s["kind"] == "append":
        out = paged.paged_append(s["qkv"], s["rope"], s["weights"], s["shape"], s["cache"], s["slots"], s["q_head"],
                                 s["q_row"])
    elif s["kind"] == "attention":
        return paged.paged_attention(s["q"], s["cache"], s["table"], s["cu"], s["used"], s["max_q"], s["max_k"], SCALE,
                                     s["bias"])
    else:
        out = paged.paged_decode_attention(s["qkv"], s["rope"], s["weights"], s["shape"], s["cache"], s["table"], s["used"],
                                           s["max_k"], SCALE, s["workspace"], s["bias"], s["q_head"], s["q_row"])
    return {"out": out, "k": s["k"], "v": s["v"]}


def work(case):
    new, keys = _lengths(case)
    h, hkv = case["heads"], case["kv_heads"]
    rows = sum(new)
    if case["kind"] == "append":
        return {"bytes": rows * (2 * (h + 2 * hkv) * D * 2 + D * 4 + 4), "flops": 0}
    held = sum(keys) * (hkv * D * 2 * 2 + (4 * h if case["bias"] else 0))
    io = rows * h * D * 2 * 2 + (rows * hkv * D * 2 * 4 if case["kind"] == "decode" else 0)
    pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(new, keys))
    return {"bytes": held + io, "flops": 4.0 * D * h * pairs}


# ---- the definition in float64 -----------------------------------------------------------------

def _exact_head(x, w, rope):
    """x (rows, heads, 128) in float64, before any rounding."""
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
    a, b = y[..., :64], y[..., 64:]
    c, t = rope[:, None, :, 0].double(), rope[:, None, :, 1].double()
    return torch.cat([a * c - b * t, b * c + a * t], -1)


def _exact_rows(s):
    """(queries, keys, values) of the new rows; what the definition rounds on the way is rounded."""
    h, hkv = s["heads"], s["kv_heads"]
    row = s["qkv"].double().view(-1, h + 2 * hkv, D)
    q = _exact_head(row[:, :h], s["q_norm"], s["rope"])
    if s["scaled"]:
        f = (s["q_row"][:, None] * s["q_head"]).to(torch.bfloat16).double()          # the scale is a bf16 number
        q = q.to(torch.bfloat16).double() * f[..., None]
    return q, _exact_head(row[:, h:h + hkv], s["k_norm"], s["rope"]).to(torch.bfloat16), row[:, h + hkv:].to(torch.bfloat16)


def exact(case, seed):
    s = prepare(case, seed)
    h, hkv, page = case["heads"], case["kv_heads"], case["page"]
    if case["kind"] == "attention":
        q = s["q"].double()
    else:
        q, k_new, v_new = _exact_rows(s)
        for i, slot in enumerate(s["slots"].tolist()):
            s["k"][slot // page, :, slot % page] = k_new[i]
            s["v"][slot // page, :, slot % page] = v_new[i]
        if case["kind"] == "append":
            return {"out": q, "k": s["k"], "v": s["v"]}
        q = q.to(torch.bfloat16).double()
    cu, used = s["cu"].tolist(), s["used"].tolist()
    out = torch.empty(cu[-1], h, D, dtype=torch.float64, device=DEVICE)
    for b in range(case["seqs"]):
        m, n = cu[b + 1] - cu[b], used[b]
        ids = s["table"][b, :(n + page - 1) // page].long()
        for j in range(h):
            k, v = (s[x][ids, j // (h // hkv)].reshape(-1, D)[:n].double() for x in ("k", "v"))
            z = q[cu[b]:cu[b + 1], j] @ k.t()
            if s["bias"] is not None:
                z = z + s["bias"][b, j, :n].double()
            z.masked_fill_(torch.ones(m, n, dtype=torch.bool, device=DEVICE).triu(n - m + 1), -math.inf)
            out[cu[b]:cu[b + 1], j] = torch.softmax(z / math.sqrt(D), -1) @ v
    return out if case["kind"] == "attention" else {"out": out, "k": s["k"], "v": s["v"]}
