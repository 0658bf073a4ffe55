"""KV caches of 4 and 8 bits: quantised as they are written, read back, and attended over in a decode step.

    cache = QuantKV.alloc(rows, n_kv_heads, bits=4, device="cuda")
    kv_quantize(kv.k, kv.v, cache, dst_rows=rows)         # bf16 rows (a prefill's LayerKV) into cache rows
    k, v = kv_dequantize(cache, rows=rows)                # bf16 again, e.g. for varlen_kv_attention
    out = decode_attention_quant(qkv, rope, ...)          # decoder.decode_attention over the quantised cache

A row of one head (128 bf16 values) is four groups of 32 consecutive values.  Each group has its least
value m and a step s = bf16((max - m) / L), L = 15 at 4 bits and 255 at 8, both bf16; a value x is held as
the whole number c = round((x - m) / s) in 0 .. L and stands for s c + m.  A group whose max - m is not
finite (a NaN or an infinity among its values) reads back as NaN; steps under 2^-100 are held as 0.  A row
of one head takes 80 bytes at 4 bits and 144 at 8, against 256 in bf16.
"""
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from tokengate_amd import _lib
from tokengate_amd.decoder import DecoderShape, LayerWeights

HEAD_DIM = 128
GROUPS = 4


@dataclass(frozen=True)
class QuantKV:
    """One layer's cache: codes (Hkv, rows, 16 * bits) uint8 and meta (Hkv, rows, 4, 2) bf16 = (s, m) of each
    group, for K and for V.  Element 16 e + w of a row is nibble (byte) e of its word (pair of words) w.  The
    rows of a head are contiguous; the heads may be further apart (a slice of rows of a longer cache).  The fields of
    a cache are not replaced (dataclasses.replace makes another one); a copy has the copied tensors."""
    bits: int
    k: torch.Tensor
    k_meta: torch.Tensor
    v: torch.Tensor
    v_meta: torch.Tensor

    def __post_init__(self):
        if self.bits not in (4, 8):
            raise RuntimeError(f"QuantKV: 4 or 8 bits (got {self.bits})")
        hkv, rows = self.k.shape[:2]
        n = 16 * self.bits
        for t in (self.k, self.v):
            if t.dtype != torch.uint8 or tuple(t.shape) != (hkv, rows, n) or t.stride()[1:] != (n, 1):
                raise RuntimeError(f"QuantKV: codes must be uint8 (heads, rows, {n}) with contiguous rows")
        for t in (self.k_meta, self.v_meta):
            if t.dtype != torch.bfloat16 or tuple(t.shape) != (hkv, rows, GROUPS, 2) or t.stride()[1:] != (8, 2, 1):
                raise RuntimeError("QuantKV: meta must be bf16 (heads, rows, 4, 2) with contiguous rows")
        head_rows = self.k.stride(0) // n if hkv > 1 else rows
        if hkv > 1 and (any(t.stride(0) != head_rows * n for t in (self.k, self.v))
                        or any(t.stride(0) != head_rows * 8 for t in (self.k_meta, self.v_meta))):
            raise RuntimeError("QuantKV: codes and meta must have the same rows between heads")
        if len({t.device for t in (self.k, self.v, self.k_meta, self.v_meta)}) != 1:
            raise RuntimeError("QuantKV: tensors on different devices")
        self.__dict__.update(rows=rows, n_kv_heads=hkv, head_rows=head_rows, device_index=self.k.get_device())

    def __setstate__(self, state):               # copies and unpickled caches: of the tensors that they got
        self.__dict__.update(state)
        self.__post_init__()

    @property
    def _args(self) -> tuple:
        """What every call passes on."""
        return (self.k.data_ptr(), self.k_meta.data_ptr(), self.v.data_ptr(), self.v_meta.data_ptr(), self.rows,
                self.head_rows)

    @staticmethod
    def alloc(rows: int, n_kv_heads: int, bits: int, device) -> "QuantKV":
        """A cache of `rows` rows; rows that were never written read back as 0."""
        if bits not in (4, 8):
            raise RuntimeError(f"QuantKV: 4 or 8 bits (got {bits})")
        c = [torch.zeros(n_kv_heads, rows, 16 * bits, dtype=torch.uint8, device=device) for _ in range(2)]
        m = [torch.zeros(n_kv_heads, rows, GROUPS, 2, dtype=torch.bfloat16, device=device) for _ in range(2)]
        return QuantKV(bits, c[0], m[0], c[1], m[1])

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.k_meta, self.v, self.v_meta))


def _row_map(what: str, t: Optional[torch.Tensor], n: int, cache: QuantKV):
    if t is None:
        return None
    if t.dtype is not torch.int32 or not t.is_contiguous() or t.numel() < n or t.get_device() != cache.device_index:
        raise RuntimeError(f"{what}: row maps must be contiguous int32 on the cache's device, an entry per row")
    return t.data_ptr()


def _bf16_rows(what: str, t: torch.Tensor, cache: QuantKV):
    """(pointer, row stride, head stride) and the rows of k or v."""
    if t.dtype is torch.bfloat16 and t.dim() == 3 and t.get_device() == cache.device_index:
        n, hkv, d = t.shape
        rs, hs, es = t.stride()
        if hkv == cache.n_kv_heads and d == HEAD_DIM and es == 1:
            return (t.data_ptr(), rs if n > 1 else hkv * HEAD_DIM, hs if hkv > 1 else HEAD_DIM), n
    raise RuntimeError(f"{what}: k and v must be bf16 (rows, {cache.n_kv_heads}, 128) on the cache's device, values "
                       "contiguous")


def kv_quantize(k: torch.Tensor, v: torch.Tensor, cache: QuantKV, dst_rows: Optional[torch.Tensor] = None,
                src_rows: Optional[torch.Tensor] = None, n_rows: Optional[int] = None) -> None:
    """Quantises K / V rows (rows, Hkv, 128) bf16, any row and head strides (multiples of 8), into the cache in one
    launch (tg_kv_quantize): source row src_rows[t] (int32; default t) to cache row dst_rows[t] (int32; default
    t), t < n_rows (default: an entry of the maps, else every source row).  Entries outside the source or the cache
    are skipped; cache rows that no entry names keep what they hold; two entries may not name the same cache row."""
    k_args, n = _bf16_rows("kv_quantize", k, cache)
    v_args, n_v = _bf16_rows("kv_quantize", v, cache)
    if n != n_v:
        raise RuntimeError("kv_quantize: k and v must have the same rows")
    if n_rows is None:
        n_rows = src_rows.numel() if src_rows is not None else dst_rows.numel() if dst_rows is not None else n
    src = _row_map("kv_quantize", src_rows, n_rows, cache)
    dst = _row_map("kv_quantize", dst_rows, n_rows, cache)
    if n_rows == 0:
        return
    _lib.call_on(cache.device_index, "tg_kv_quantize", *k_args, *v_args, n, src, dst, n_rows, cache.n_kv_heads,
                 HEAD_DIM, cache.bits, *cache._args)


def kv_dequantize(cache: QuantKV, rows: Optional[torch.Tensor] = None, n_rows: Optional[int] = None,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) (n_rows, Hkv, 128) bf16 of the cache rows rows[t] (int32; default t) in one launch
    (tg_kv_dequantize): bf16(s c + m).  n_rows defaults to an entry of the map, else every row; an entry outside
    the cache reads as 0.  out: two bf16 tensors to write to (at least n_rows rows, none of which overlap)."""
    if n_rows is None:
        n_rows = rows.numel() if rows is not None else cache.rows
    ptr = _row_map("kv_dequantize", rows, n_rows, cache)
    if out is None:
        shape, dev, stride = (n_rows, cache.n_kv_heads, HEAD_DIM), cache.k.device, cache.n_kv_heads * HEAD_DIM
        k, v = (torch.empty(shape, dtype=torch.bfloat16, device=dev), torch.empty(shape, dtype=torch.bfloat16, device=dev))
        k_args, v_args = (k.data_ptr(), stride, HEAD_DIM), (v.data_ptr(), stride, HEAD_DIM)
    else:
        k, v = out
        k_args, n = _bf16_rows("kv_dequantize", k, cache)
        v_args, n_v = _bf16_rows("kv_dequantize", v, cache)
        if n < n_rows or n_v < n_rows:
            raise RuntimeError("kv_dequantize: out holds fewer rows than are read")
    if n_rows == 0:
        return k, v
    _lib.call_on(cache.device_index, "tg_kv_dequantize", *cache._args, cache.n_kv_heads, HEAD_DIM, cache.bits, ptr,
                 n_rows, *k_args, *v_args)
    return k, v


def decode_attention_quant_workspace(n_seqs: int, shape: DecoderShape, max_k: int, device) -> torch.Tensor:
    """Zeroed workspace for decode_attention_quant calls of up to n_seqs sequences and max_k keys (its counters
    stay zero between calls), for one stream: calls that may overlap need one each."""
    n = int(_lib.load().tg_decode_attention_quant_workspace_size(n_seqs, shape.n_heads, shape.n_kv_heads, int(max_k)))
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def decode_attention_quant(qkv: torch.Tensor, rope: torch.Tensor, lw: LayerWeights, shape: DecoderShape, cache: QuantKV,
                           kv_start: torch.Tensor, kv_used: torch.Tensor, max_k: int, scale: float,
                           workspace: torch.Tensor, bias_raw: Optional[torch.Tensor] = None,
                           q_head_scale: Optional[torch.Tensor] = None, q_row_scale: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decoder.decode_attention over a quantised cache in one launch (tg_decode_attention_quant): the new key and
    value of sequence b are quantised into cache row kv_start[b] + kv_used[b] - 1, and its query attends over rows
    kv_start[b] .. kv_start[b] + kv_used[b] - 1 as they are held (s c + m, not rounded to bf16); bias_raw
    (nseq, H, >= max_k) as decode_attention; a bias of -inf hides a row whatever it holds.  No sequence may append
    a row that another one reads or appends."""
    H, Hkv, D = shape.n_heads, shape.n_kv_heads, shape.head_dim
    dev = qkv.get_device()
    if qkv.dtype is not torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] < (H + 2 * Hkv) * D or qkv.stride(1) != 1:
        raise RuntimeError("decode_attention_quant: qkv must be bf16 rows of every head's q, k and v")
    B = qkv.shape[0]
    if cache.n_kv_heads != Hkv or cache.device_index != dev:
        raise RuntimeError("decode_attention_quant: the cache has other KV heads or is on another device")
    # (contiguous, dtype and device of each, and its least size)
    for t, dt, n, which in ((rope, torch.float32, B * D, "rope must be contiguous fp32 (B, 64, 2)"),
                            (kv_start, torch.int32, B, "kv_start must be contiguous int32, an entry per sequence"),
                            (kv_used, torch.int32, B, "kv_used must be contiguous int32, an entry per sequence"),
                            (q_head_scale, torch.float32, H, "q_head_scale must be contiguous fp32, an entry per head"),
                            (q_row_scale, torch.float32, B, "q_row_scale must be contiguous fp32, an entry per sequence"),
                            (workspace, torch.uint8, 0, "workspace must be contiguous bytes")):
        if t is not None and (t.dtype is not dt or t.numel() < n or not t.is_contiguous() or t.get_device() != dev):
            raise RuntimeError(f"decode_attention_quant: {which}, on qkv's device")
    bias_args = (None, 0, 0)
    if bias_raw is not None:
        if bias_raw.dtype is not torch.float32 or bias_raw.dim() != 3 or bias_raw.get_device() != dev:
            raise RuntimeError("decode_attention_quant: bias must be fp32 (B, H, >= max_k) on qkv's device")
        nb, nh, nk = bias_raw.shape
        sb, sh, sk = bias_raw.stride()
        if nb != B or nh != H or nk < max_k or (sk != 1 and nk > 1):
            raise RuntimeError("decode_attention_quant: bias must be fp32 (B, H, >= max_k) with a contiguous key axis")
        bias_args = (bias_raw.data_ptr(), sb, sh)
    if out is None:
        out = torch.empty((B, H, D), dtype=torch.bfloat16, device=qkv.device)
    elif out.dtype is not torch.bfloat16 or out.shape != (B, H, D) or out.stride()[1:] != (D, 1) or out.get_device() != dev:
        raise RuntimeError("decode_attention_quant: out must be bf16 (B, H, 128) rows on qkv's device")
    if B == 0:
        return out
    _lib.call_on(dev, "tg_decode_attention_quant", qkv.data_ptr(), qkv.stride(0) if B > 1 else (H + 2 * Hkv) * D,
                 rope.data_ptr(), B, H, Hkv, D, cache.bits, lw.q_norm.data_ptr(), lw.k_norm.data_ptr(), shape.rms_eps,
                 None if q_head_scale is None else q_head_scale.data_ptr(),
                 None if q_row_scale is None else q_row_scale.data_ptr(), *cache._args, kv_start.data_ptr(),
                 kv_used.data_ptr(), max_k, *bias_args, scale, out.data_ptr(),
                 out.stride(0) if B > 1 else H * D, workspace.data_ptr(), workspace.numel())
    return out
