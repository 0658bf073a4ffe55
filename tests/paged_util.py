"""Inputs and float64 references of the paged KV cache's tests."""
import torch

D = 128
BF = 2.0 ** -8                   # half a step of bf16, relative
LOGITS = 2.0 ** -12              # fp32 dot products of 128 terms and exponents of logits under 64 or so


def shape_of(H, Hkv):
    from tokengate_amd import decoder as dec
    return dec.DecoderShape(n_layers=1, n_heads=H, n_kv_heads=Hkv, d_model=H * D)


def normal(g, *size, std=1.0, mean=0.0):
    return (mean + std * torch.randn(*size, generator=g, device=g.device)).to(torch.bfloat16)


def weights(g):
    from tokengate_amd import decoder as dec
    return dec.LayerWeights(None, None, normal(g, D, std=0.3, mean=1.0), normal(g, D, std=0.3, mean=1.0), None, None, None, None)


def cache_of(g, n_pages, Hkv, page, layout="heads", fill=None):
    """A cache of normal values (or of `fill`): heads: rows of a head contiguous; rows: (pages, rows, heads, 128);
    both: K and V in one tensor, with unused elements behind each row."""
    from tokengate_amd import paged as P

    def values(*size):
        return normal(g, *size) if fill is None else torch.full(size, fill, dtype=torch.bfloat16, device=g.device)

    if layout == "heads":
        return P.PagedKV(values(n_pages, Hkv, page, D), values(n_pages, Hkv, page, D))
    if layout == "rows":
        return P.PagedKV(values(n_pages, page, Hkv, D).transpose(1, 2), values(n_pages, page, Hkv, D).transpose(1, 2))
    x = values(n_pages, page, 2, Hkv, D + 8)
    return P.PagedKV(x[:, :, 0, :, :D].transpose(1, 2), x[:, :, 1, :, :D].transpose(1, 2))


def table_of(g, used, page, extra=2, spare=3):
    """(page table, pages of the cache): every sequence's pages anywhere in the cache; entries past them -1."""
    need = [(n + page - 1) // page for n in used]
    n = sum(need) + spare
    where = torch.randperm(n, generator=g, device=g.device).to(torch.int32)
    table = torch.full((len(used), max(need) + extra), -1, dtype=torch.int32, device=g.device)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = where[at:at + m]
        at += m
    return table, n


def slots_of(table, page, keys):
    """Slot of key keys[t][1] of sequence keys[t][0]."""
    t = table.cpu().tolist()
    return torch.tensor([t[b][j // page] * page + j % page for b, j in keys], dtype=torch.int32, device=table.device)


def keys_of(cache, table, b, n):
    """(k, v, there) of keys 0 .. n - 1 of sequence b in float64: (n, Hkv, 128) and which have a page."""
    page = cache.page_rows
    ids = table[b, :(n + page - 1) // page].long()
    there = ((ids >= 0) & (ids < cache.n_pages)).repeat_interleave(page)[:n]
    k, v = (t[ids.clamp(0, cache.n_pages - 1)].transpose(1, 2).flatten(0, 1)[:n].double() for t in (cache.k, cache.v))
    return k, v, there


def attend(q, k, v, there, scale, bias=None, causal_from=None):
    """(out, sum of p |v|) in float64 of queries q (m, H, 128) over keys (n, Hkv, 128): query i sees keys up to causal_from + i
    (None: all); bias (H, n).  What is hidden may hold anything; rows that see nothing: 0."""
    m, H, _ = q.shape
    n, Hkv, _ = k.shape
    out = torch.zeros(m, H, D, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    if n == 0:
        return out, mass
    seen = there[None].expand(m, n)
    if causal_from is not None:
        seen = seen & (torch.arange(n, device=q.device)[None] <= causal_from + torch.arange(m, device=q.device)[:, None])
    for h in range(H):
        g = h // (H // Hkv)
        ok = seen if bias is None else seen & (bias[h] != -torch.inf)[None]
        any_key = ok.any(0)
        kk = torch.where(any_key[:, None], k[:, g], torch.zeros_like(k[:, g]))
        vv = torch.where(any_key[:, None], v[:, g], torch.zeros_like(v[:, g]))
        z = q[:, h].double() @ kk.t()
        if bias is not None:
            z = (z + torch.where(any_key, bias[h].double(), torch.zeros_like(bias[h].double()))[None])
        z = torch.where(ok, z * scale, -torch.inf)
        p = torch.where(ok, torch.exp(z - z.amax(-1, keepdim=True)), torch.zeros_like(z))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        out[:, h], mass[:, h] = p @ vv, p @ vv.abs()
    return out, mass


def near(got, ref, mass, weight, what=""):
    """|got - ref| within the weights' rounding (`weight`, of the sum of p |v - out|), the output's, and fp32 sums'."""
    assert torch.isfinite(got).all(), what
    err = (got.double() - ref).abs()
    ok = err <= (weight + LOGITS) * (mass + ref.abs()) + BF * ref.abs()
    assert bool(ok.all()), (what, float((err - BF * ref.abs()).max()), float((err / (mass + 1e-30)).max()))
