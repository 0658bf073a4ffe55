"""A KV cache in pages: rows appended with their rotation, attention of prompt chunks and of single tokens over it.

    cache = PagedKV.alloc(n_pages, n_kv_heads, page_rows=64, device="cuda")     # one layer's
    slots, rope = paged_begin(positions, inv_freq, cu_q, kv_used, page_table, cache)   # once per step, for all layers
    q = paged_append(qkv, rope, layer_weights, shape, cache, slots)
    out = paged_attention(q, cache, page_table, cu_q, kv_used, max_q, max_k, scale)
    out = paged_decode_attention(qkv, rope, ...)          # one new token per sequence, append and attention in one launch

Key j of sequence b is row j % page_rows of page page_table[b, j // page_rows] (int32).  An entry outside the cache's pages
names none: its keys weigh nothing, and nothing is written to them.  Sequences may share pages (a prompt's prefix) that
none of them appends to; which pages are free is the caller's to keep.  bf16, head_dim 128.
"""
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from tokengate_amd import _lib
from tokengate_amd.decoder import DecoderShape, LayerWeights, PageGeo, h2d

HEAD_DIM = 128
_I32, _F32, _BF16, _U8 = torch.int32, torch.float32, torch.bfloat16, torch.uint8
_NO_BIAS = (None, 0, 0)


def _apart(t: torch.Tensor) -> bool:
    """Whether rows of 128 values (the last dimension) do not overlap: every stride is past what the smaller ones span."""
    apart = HEAD_DIM
    for stride, size in sorted((stride, size) for stride, size in zip(t.stride()[:-1], t.shape) if size > 1):
        if stride < apart:
            return False
        apart = size * stride
    return True


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """(page, head, row) strides.  A dimension of one entry may have any stride."""
    if not _apart(t):
        raise RuntimeError("PagedKV: rows overlap")
    ps, hs, rs, _ = t.stride()
    return ps if t.shape[0] > 1 else 0, hs if t.shape[1] > 1 else 0, rs


@dataclass(frozen=True)
class PagedKV:
    """One layer's pages: k and v (pages, KV heads, page rows, 128) bf16, values contiguous, other strides any multiples of
    8 (a view of (pages, rows, heads, 128), or of a tensor that holds both, will do); page rows a power of two from 16 to
    65536.  k and v share no memory.  The fields of a cache are not replaced; a copy has the copied tensors."""
    k: torch.Tensor
    v: torch.Tensor

    def __post_init__(self):
        k, v = self.k, self.v
        for t in (k, v):
            if t.dtype is not torch.bfloat16 or t.dim() != 4 or t.shape[3] != HEAD_DIM or t.stride(3) != 1:
                raise RuntimeError("PagedKV: k and v must be bf16 (pages, KV heads, page rows, 128), values contiguous")
        n, hkv, rows, _ = k.shape
        if v.shape != k.shape or v.device != k.device:
            raise RuntimeError("PagedKV: k and v must have one shape and device")
        if n < 1 or not 1 <= hkv <= 256:
            raise RuntimeError("PagedKV: at least one page, 1 to 256 KV heads")
        if rows < 16 or rows > 65536 or rows & (rows - 1):
            raise RuntimeError(f"PagedKV: page rows must be a power of two from 16 to 65536 (got {rows})")
        if n * rows >= 2 ** 31:
            raise RuntimeError("PagedKV: less than 2^31 rows")
        if any(x % 8 for t in (k, v) for x in t.stride()[:3]) or any(t.data_ptr() % 16 for t in (k, v)):
            raise RuntimeError("PagedKV: strides must be multiples of 8 elements, tensors 16-byte aligned")
        if k.data_ptr() == v.data_ptr():
            raise RuntimeError("PagedKV: k and v share memory")
        self.__dict__.update(n_pages=n, n_kv_heads=hkv, page_rows=rows, device_index=k.get_device(),
                             _args=(k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), n, rows))

    def __setstate__(self, state):               # copies and unpickled caches: of the tensors that they got
        self.__dict__.update(state)
        self.__post_init__()

    @staticmethod
    def alloc(n_pages: int, n_kv_heads: int, page_rows: int, device) -> "PagedKV":
        """Pages whose rows of one head are contiguous; what they hold is not initialised."""
        size = (n_pages, n_kv_heads, page_rows, HEAD_DIM)
        return PagedKV(torch.empty(size, dtype=torch.bfloat16, device=device),
                       torch.empty(size, dtype=torch.bfloat16, device=device))

    @property
    def nbytes(self) -> int:
        return 2 * self.k.numel() * 2


def _ints(what: str, name: str, t: torch.Tensor, n: int, dev: int) -> int:
    if t.dtype is not torch.int32 or not t.is_contiguous() or t.numel() < n or t.get_device() != dev:
        raise RuntimeError(f"{what}: {name} must be contiguous int32 of at least {n} entries, on the cache's device")
    return t.data_ptr()


def _max_k(what: str, max_k: int) -> int:
    n = int(max_k)                               # (the call takes 32 bits: a larger number would be cut)
    if not 0 <= n < 1 << 24:
        raise RuntimeError(f"{what}: max_k must be in 0..2^24 - 1 (got {max_k})")
    return n


def _table(what: str, t: torch.Tensor, n_seqs: int, max_k: int, page_rows: int, dev: int) -> tuple:
    """(pointer, stride, columns) of a page table."""
    if t.dtype is not _I32 or t.dim() != 2 or t.get_device() != dev:
        raise RuntimeError(f"{what}: page_table must be int32 (sequences, pages), rows contiguous, on the cache's device")
    (rows, cols), (rs, cs) = t.shape, t.stride()
    if rows < n_seqs or cols < 1 or (cs != 1 and cols > 1):
        raise RuntimeError(f"{what}: page_table must be int32 (sequences, pages), rows contiguous, on the cache's device")
    if cols * page_rows < max_k:
        raise RuntimeError(f"{what}: page_table's columns hold fewer than max_k keys")
    return t.data_ptr(), rs if rows > 1 else cols, cols


def _floats(what: str, name: str, t: Optional[torch.Tensor], n: int, dev: int):
    if t is None:
        return None
    if t.dtype is not torch.float32 or not t.is_contiguous() or t.numel() < n or t.get_device() != dev:
        raise RuntimeError(f"{what}: {name} must be contiguous fp32 of at least {n} entries, on the cache's device")
    return t.data_ptr()


def _bias(what: str, t: Optional[torch.Tensor], n_seqs: int, n_heads: int, max_k: int, dev: int) -> tuple:
    if t is None:
        return None, 0, 0
    if t.dtype is not torch.float32 or t.dim() != 3 or t.get_device() != dev or t.shape[0] != n_seqs or t.shape[1] != n_heads \
            or t.shape[2] < max_k or (t.stride(2) != 1 and t.shape[2] > 1):
        raise RuntimeError(f"{what}: bias must be fp32 (sequences, heads, >= max_k), key axis contiguous, on the cache's device")
    return t.data_ptr(), t.stride(0) if n_seqs > 1 else 0, t.stride(1) if n_heads > 1 else 0


def _qkv(what: str, qkv: torch.Tensor, shape: DecoderShape, cache: PagedKV) -> int:
    width = (shape.n_heads + 2 * shape.n_kv_heads) * HEAD_DIM
    if qkv.dtype is not _BF16 or qkv.dim() != 2 or qkv.shape[1] < width or qkv.stride(1) != 1:
        raise RuntimeError(f"{what}: qkv must be bf16 rows of every head's q, k and v")
    if cache.n_kv_heads != shape.n_kv_heads or cache.device_index != qkv.get_device() or shape.head_dim != HEAD_DIM:
        raise RuntimeError(f"{what}: the cache has other KV heads or is on another device")
    return qkv.stride(0) if qkv.shape[0] > 1 else width


def _weights(what: str, lw: LayerWeights, dev: int) -> None:
    for t in (lw.q_norm, lw.k_norm):
        if t.dtype is not _BF16 or not t.is_contiguous() or t.numel() != HEAD_DIM or t.get_device() != dev:
            raise RuntimeError(f"{what}: norm weights must be contiguous bf16 (128,) on the cache's device")


def paged_begin(positions: torch.Tensor, inv_freq: torch.Tensor, cu_q: torch.Tensor, kv_used: torch.Tensor,
                page_table: torch.Tensor, cache: PagedKV) -> Tuple[torch.Tensor, torch.Tensor]:
    """Starts a step of packed rows at positions (T,) int64 (tg_paged_begin): (slots (T,) int32, rope (T, 64, 2) fp32) for
    paged_append.  Row t of sequence b (cu_q[b] <= t < cu_q[b + 1]) is one of the sequence's last keys, of kv_used[b] with these;
    rows of no sequence or page get slot -1."""
    dev, T, n = cache.device_index, positions.numel(), cu_q.numel() - 1
    if positions.dtype is not torch.int64 or not positions.is_contiguous() or positions.get_device() != dev:
        raise RuntimeError("paged_begin: positions must be contiguous int64 on the cache's device")
    if n < 1:
        raise RuntimeError("paged_begin: cu_q needs an entry per sequence and one more")
    if inv_freq.numel() != HEAD_DIM // 2:
        raise RuntimeError("paged_begin: inv_freq must be 64 frequencies")
    args = (_floats("paged_begin", "inv_freq", inv_freq, 64, dev), _ints("paged_begin", "cu_q", cu_q, n + 1, dev),
            _ints("paged_begin", "kv_used", kv_used, n, dev), n,
            *_table("paged_begin", page_table, n, 0, cache.page_rows, dev))
    slots = torch.empty(T, dtype=torch.int32, device=positions.device)
    rope = torch.empty(T, HEAD_DIM // 2, 2, dtype=torch.float32, device=positions.device)
    if T:
        _lib.call_on(dev, "tg_paged_begin", positions.data_ptr(), T, *args, cache.n_pages, cache.page_rows, slots.data_ptr(),
                     rope.data_ptr())
    return slots, rope


def paged_append(qkv: torch.Tensor, rope: torch.Tensor, lw: LayerWeights, shape: DecoderShape, cache: PagedKV,
                 slots: torch.Tensor, q_head_scale: Optional[torch.Tensor] = None,
                 q_row_scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decoder.qk_norm_rope into pages (tg_paged_append; the same bits): normalises and rotates the raw q|k|v projection
    rows qkv (T, >= (H + 2 Hkv) 128) with the rotary table rope (T, 64, 2) and writes k and v to the cache rows slots (T,)
    int32 = page * page_rows + row; a slot outside the cache writes none.  Returns the queries (T, H, 128): out, by
    default a new tensor; out may be qkv's own query columns (qkv[:, :H * 128].unflatten(1, (H, 128)): in place).  No two
    rows may name one slot."""
    H, dev = shape.n_heads, cache.device_index
    rs = _qkv("paged_append", qkv, shape, cache)
    T = qkv.shape[0]
    qw, kw = lw.q_norm, lw.k_norm
    if not (slots.dtype is _I32 and slots.numel() >= T and slots.is_contiguous() and slots.get_device() == dev
            and rope.dtype is _F32 and rope.numel() >= T * HEAD_DIM and rope.is_contiguous() and rope.get_device() == dev
            and qw.dtype is _BF16 and kw.dtype is _BF16 and qw.numel() == HEAD_DIM and kw.numel() == HEAD_DIM
            and qw.is_contiguous() and kw.is_contiguous() and qw.get_device() == dev and kw.get_device() == dev):
        _ints("paged_append", "slots", slots, T, dev)
        _floats("paged_append", "rope", rope, T * HEAD_DIM, dev)
        _weights("paged_append", lw, dev)
    qh = None if q_head_scale is None else _floats("paged_append", "q_head_scale", q_head_scale, H, dev)
    qr = None if q_row_scale is None else _floats("paged_append", "q_row_scale", q_row_scale, T, dev)
    if out is None:
        out = torch.empty((T, H, HEAD_DIM), dtype=_BF16, device=qkv.device)
        ors, ohs = H * HEAD_DIM, HEAD_DIM
    else:
        if out.dtype is not _BF16 or tuple(out.shape) != (T, H, HEAD_DIM) or out.stride(2) != 1 or out.get_device() != dev:
            raise RuntimeError("paged_append: out must be bf16 (rows, H, 128), values contiguous, on the cache's device")
        if not _apart(out):
            raise RuntimeError("paged_append: rows of out overlap")
        ors, ohs = out.stride(0) if T > 1 else 0, out.stride(1) if H > 1 else HEAD_DIM
    if T:
        _lib.call_on(dev, "tg_paged_append", qkv.data_ptr(), rs, rope.data_ptr(), T, H, shape.n_kv_heads, HEAD_DIM, qw.data_ptr(),
                     kw.data_ptr(), shape.rms_eps, qh, qr, out.data_ptr(), ors, ohs, slots.data_ptr(), *cache._args)
    return out


def paged_attention(q: torch.Tensor, cache: PagedKV, page_table: torch.Tensor, cu_q: torch.Tensor, kv_used: torch.Tensor,
                    max_q: int, max_k: int, scale: float, bias_raw: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decoder.varlen_kv_attention over pages (tg_paged_attention): causal attention of every packed query segment cu_q[b]
    .. cu_q[b + 1] - 1 of q (T, H, 128), at most max_q rows (any number past T is T), over keys 0 .. kv_used[b] - 1 of its
    sequence (at most max_k), the last query with the last key.  bias_raw (nseq, H, >= max_k) fp32 in raw-score units; -inf
    hides a key from a head whatever its row holds; rows of keys that only come after a query have to be finite.  Rows that
    see no key get zeros, rows of no segment keep what out holds."""
    what, dev, n = "paged_attention", cache.device_index, cu_q.numel() - 1
    if q.dtype is not torch.bfloat16 or q.dim() != 3 or q.shape[2] != HEAD_DIM or q.stride(2) != 1 or q.get_device() != dev:
        raise RuntimeError("paged_attention: q must be bf16 (rows, H, 128), values contiguous, on the cache's device")
    T, H, _ = q.shape
    Hkv = cache.n_kv_heads
    if H < 1 or H % Hkv:
        raise RuntimeError(f"paged_attention: {H} query heads are not a multiple of the cache's {Hkv}")
    if n < 0:
        raise RuntimeError("paged_attention: cu_q needs an entry per sequence and one more")
    if out is None:
        out = torch.empty((T, H, HEAD_DIM), dtype=torch.bfloat16, device=q.device)
    elif out.dtype is not torch.bfloat16 or out.shape != q.shape or out.stride(2) != 1 or out.get_device() != dev:
        raise RuntimeError("paged_attention: out must be bf16 like q, values contiguous, on the cache's device")
    elif not _apart(out):
        raise RuntimeError("paged_attention: rows of out overlap")
    cu = _ints(what, "cu_q", cu_q, n + 1, dev)
    used = _ints(what, "kv_used", kv_used, n, dev)
    max_k, max_q = _max_k(what, max_k), min(int(max_q), T)
    if max_q < 0:
        raise RuntimeError(f"{what}: max_q must not be negative (got {max_q})")
    bias = _bias(what, bias_raw, n, H, max_k, dev)
    if n == 0 or T == 0:
        return out
    table = _table(what, page_table, n, max_k, cache.page_rows, dev)
    # (the size is of the current device's launch plan, as everything of the call)
    ws, ws_ptr, ws_bytes = _lib.fwd_workspace("tg_paged_attention_workspace_size", q.device, n, max_q, max_k, T, H, Hkv)
    _lib.call_on(dev, "tg_paged_attention", q.data_ptr(), q.stride(0) if T > 1 else H * HEAD_DIM,
                 q.stride(1) if H > 1 else HEAD_DIM, *cache._args, *table, cu, used, n, max_q, max_k, T, H, Hkv,
                 HEAD_DIM, *bias, float(scale), out.data_ptr(), out.stride(0) if T > 1 else H * HEAD_DIM,
                 out.stride(1) if H > 1 else HEAD_DIM, ws_ptr, ws_bytes)
    return out


def paged_decode_attention_workspace(n_seqs: int, shape: DecoderShape, max_k: int, device) -> torch.Tensor:
    """Zeroed workspace for paged_decode_attention calls of up to n_seqs sequences and max_k keys (its counters stay zero
    between calls), for one stream: calls that may overlap need one each."""
    n = int(_lib.load().tg_paged_decode_attention_workspace_size(n_seqs, shape.n_heads, shape.n_kv_heads,
                                                                 _max_k("paged_decode_attention_workspace", max_k)))
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def paged_decode_attention(qkv: torch.Tensor, rope: torch.Tensor, lw: LayerWeights, shape: DecoderShape, cache: PagedKV,
                           page_table: torch.Tensor, kv_used: torch.Tensor, max_k: int, scale: float,
                           workspace: torch.Tensor, bias_raw: Optional[torch.Tensor] = None,
                           q_head_scale: Optional[torch.Tensor] = None, q_row_scale: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decoder.decode_attention over pages in one launch (tg_paged_decode_attention): the new key and value of sequence b
    become key kv_used[b] - 1, and its query attends over keys 0 .. kv_used[b] - 1 (at most max_k); bias_raw (nseq, H,
    >= max_k) as decode_attention, -inf hides a key whatever its row holds.  A sequence of kv_used 0 (a free place of a
    padded batch) appends nothing and gets zeros.  No sequence may append a row that another one reads or appends."""
    dev, H, Hkv = cache.device_index, shape.n_heads, shape.n_kv_heads
    rs = _qkv("paged_decode_attention", qkv, shape, cache)
    B = qkv.shape[0]
    qw, kw = lw.q_norm, lw.k_norm
    # one test for what nearly every call passes; what does not pass it is looked at again for its message
    if not (kv_used.dtype is _I32 and kv_used.numel() >= B and kv_used.is_contiguous() and kv_used.get_device() == dev
            and rope.dtype is _F32 and rope.numel() >= B * HEAD_DIM and rope.is_contiguous() and rope.get_device() == dev
            and qw.dtype is _BF16 and kw.dtype is _BF16 and qw.numel() == HEAD_DIM and kw.numel() == HEAD_DIM
            and qw.is_contiguous() and kw.is_contiguous() and qw.get_device() == dev and kw.get_device() == dev
            and workspace.dtype is _U8 and workspace.is_contiguous() and workspace.get_device() == dev):
        _ints("paged_decode_attention", "kv_used", kv_used, B, dev)
        _floats("paged_decode_attention", "rope", rope, B * HEAD_DIM, dev)
        _weights("paged_decode_attention", lw, dev)
        raise RuntimeError("paged_decode_attention: workspace must be contiguous bytes on the cache's device")
    qh = None if q_head_scale is None else _floats("paged_decode_attention", "q_head_scale", q_head_scale, H, dev)
    qr = None if q_row_scale is None else _floats("paged_decode_attention", "q_row_scale", q_row_scale, B, dev)
    max_k = _max_k("paged_decode_attention", max_k)
    bias = _NO_BIAS if bias_raw is None else _bias("paged_decode_attention", bias_raw, B, H, max_k, dev)
    if out is None:
        out = torch.empty((B, H, HEAD_DIM), dtype=_BF16, device=qkv.device)
        ors = H * HEAD_DIM
    else:
        if out.dtype is not _BF16 or tuple(out.shape) != (B, H, HEAD_DIM) or out.stride(2) != 1 \
                or (H > 1 and out.stride(1) != HEAD_DIM) or out.get_device() != dev:
            raise RuntimeError("paged_decode_attention: out must be bf16 (B, H, 128) rows on the cache's device")
        ors = out.stride(0) if B > 1 else H * HEAD_DIM
    if B == 0:
        return out
    table = _table("paged_decode_attention", page_table, B, max_k, cache.page_rows, dev)
    _lib.call_on(dev, "tg_paged_decode_attention", qkv.data_ptr(), rs, rope.data_ptr(), B, H, Hkv, HEAD_DIM, qw.data_ptr(),
                 kw.data_ptr(), shape.rms_eps, qh, qr, *cache._args, *table, kv_used.data_ptr(), max_k, *bias, float(scale),
                 out.data_ptr(), ors, workspace.data_ptr(), workspace.numel())
    return out


def page_tables(lengths: List[int], room: int, page_rows: int, device) -> Tuple[torch.Tensor, int]:
    """(page table, pages) of sequences of these lengths with room for `room` more keys each, one after the other."""
    need = [(n + room + page_rows - 1) // page_rows for n in lengths]
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(first, first + n, dtype=torch.int32)
        first += n
    return h2d(table, device), max(first, 1)


def prompt_pages(cu: List[int], cu_dev: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, shape: DecoderShape,
                 layers: int, room: int, page_rows: int) -> Tuple[PageGeo, List[PagedKV]]:
    """Paged caches for `layers` layers of packed prompts cu[b] .. cu[b + 1] - 1 at these positions, with room for `room` more
    keys each: the geometry for decoder.run_layers, and the caches."""
    dev = positions.device
    lens = [cu[b + 1] - cu[b] for b in range(len(cu) - 1)]
    table, n_pages = page_tables(lens, room, page_rows, dev)
    caches = [PagedKV.alloc(n_pages, shape.n_kv_heads, page_rows, dev) for _ in range(layers)]
    used = h2d(torch.tensor(lens, dtype=torch.int32), dev)
    slots, rope = paged_begin(positions, inv_freq, cu_dev, used, table, caches[0])
    return PageGeo(table, used, max(lens), slots, rope), caches
