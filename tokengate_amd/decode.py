"""Decode after the gated prefill, over the pruned KV caches: greedy, or with sampled tokens.

Follows generate_batch (tokengate/e2e_gate/decode/gate_decode.py:88-262) in its default form:
layers at or below the gate attend over the full prompt cache (prune_below_gate=False) plus the
generated tokens; layers above it attend over the kept rows, which keep their gate bias and
per-head temperature through decode (decode_phase2_form=True, FormDecodeState
qwen3_flex_attention.py:978-1117) while generated tokens carry bias 0; positions continue from
each sequence's last kept original position (+1 per step); generation stops when every row has
produced EOS, and answers are cut at the first EOS (gate_decode.py:241-257).

Cache layout: the prefill run with decode_headroom >= the steps to come leaves every layer's
cache with that many free rows after each sequence (decoder.CacheGap), and the decode appends in
place: each layer's q/k norm, RoPE, cache append (row seg[b] + used[b] of each sequence's segment)
and attention over its segment's used rows are ONE launch (tg_decode_attention).  A
prefill without enough headroom is re-laid out once (one copy per layer) into that layout.
The per-step counters live on the device, so nothing in a step synchronises with the host, and
every step launches the same kernels with the same arguments: with graph=True the second and
later steps replay one captured HIP graph of the whole step (144 launches for 28 layers), whose inputs
and outputs are static device buffers; the first step runs eagerly and warms every kernel and
library handle the capture records.

After a prefill with page_rows the caches are in pages: each layer's launch is tg_paged_decode_attention over the group's
page table, the same counters and steps otherwise.

Two options leave the reference's decode.  With kv_bits 4 or 8 every layer's prompt rows are quantised
into a cache of that many bits (kvquant.QuantKV; the prefill's bf16 caches may then be freed) and each
layer's launch is tg_decode_attention_quant, which quantises the new rows on the way in.  With a Sampling
the tokens are drawn by tg_sample_rows from one uniform random number per sequence and step, all of them
drawn ahead from its seed.
"""
import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Union

import torch

from tokengate_amd.decoder import (CacheGap, DecoderWeights, LayerKV, argmax_rows, decode_attention,
                                   decode_attention_workspace, decode_begin, h2d, linear_rows, linear_rows_norm,
                                   linear_rows_norm_act, linear_rows_swiglu, logits_last, rmsnorm, sample_rows,
                                   sample_rows_workspace, silu_mul)
from tokengate_amd.gate import ScoringHead
from tokengate_amd.paged import PagedKV, paged_decode_attention, paged_decode_attention_workspace
from tokengate_amd.kvquant import (QuantKV, decode_attention_quant, decode_attention_quant_workspace, kv_quantize)
from tokengate_amd.prefill import PrefillResult


@dataclass
class _Group:
    """Layers that share one cache geometry (at / below the gate, or above it)."""
    seg: List[int]            # host: segment start per sequence
    n0: List[int]             # host: rows per sequence when decoding starts
    gap: int


MAX_TEMPERATURE = torch.finfo(torch.float32).max


@dataclass
class Sampling:
    """How next tokens are drawn (decoder.sample_rows); every setting a number, or a sequence with one per
    sequence of the batch.  temperature 0 is greedy, top_k 0, top_p 1 and min_p 0 keep everything."""
    temperature: Union[float, Sequence[float]] = 1.0
    top_k: Union[int, Sequence[int]] = 0
    top_p: Union[float, Sequence[float]] = 1.0
    min_p: Union[float, Sequence[float]] = 0.0
    seed: int = 0

    def _values(self, name: str, B: int) -> list:
        x = getattr(self, name)
        x = [x] * B if isinstance(x, (int, float)) else list(x)
        if len(x) != B:
            raise ValueError(f"Sampling: {name} needs one value per sequence ({B}), got {len(x)}")
        return x

    def check(self, B: int) -> None:
        """ValueError unless every setting is a number of its range, one or B of them."""
        for name, ok, what in (("temperature", lambda v: 0 <= v <= MAX_TEMPERATURE, "a finite fp32 number of at least 0"),
                               ("top_k", lambda v: v == int(v) and 0 <= v < 2 ** 31, "a whole number of at least 0"),
                               ("top_p", lambda v: 0 <= v <= 1, "in 0..1"), ("min_p", lambda v: 0 <= v <= 1, "in 0..1")):
            for v in self._values(name, B):
                if math.isnan(v) or math.isinf(v) or not ok(v):
                    raise ValueError(f"Sampling: {name} must be {what} (got {v})")


class TokenSampler:
    """The next tokens of a batch's logits: the settings on the device, and every step's random numbers, drawn
    ahead from the seed."""

    def __init__(self, sampling: Sampling, B: int, vocab: int, n_draws: int, device):
        sampling.check(B)
        self.batch, self.vocab = B, vocab
        self.settings = [h2d(torch.tensor(sampling._values(name, B), dtype=dt), device)
                         for name, dt in (("temperature", torch.float32), ("top_k", torch.int32),
                                          ("top_p", torch.float32), ("min_p", torch.float32))]
        g = torch.Generator(device=device).manual_seed(int(sampling.seed))
        self.draws = torch.rand(n_draws, B, generator=g, dtype=torch.float32, device=device)
        self.u = torch.empty(B, dtype=torch.float32, device=device)     # this step's
        self.ws = sample_rows_workspace(B, vocab, device)

    def set_step(self, i: int) -> None:
        self.u.copy_(self.draws[i])

    def __call__(self, logits: torch.Tensor):
        """(tokens, log probabilities) with the random numbers of the step that was set."""
        return sample_rows(logits, self.u, *self.settings, workspace=self.ws, logprob=True)


def _relayout(kv: LayerKV, cu: List[int], gap: int) -> LayerKV:
    """Copy a back-to-back cache (cu layout) into one with `gap` free rows after each sequence."""
    B = len(cu) - 1
    rows = cu[-1] + B * gap
    k = torch.zeros(rows, *kv.k.shape[1:], dtype=kv.k.dtype, device=kv.k.device)
    v = torch.zeros_like(k)
    for b in range(B):
        s = cu[b] + b * gap
        k[s:s + cu[b + 1] - cu[b]] = kv.k[cu[b]:cu[b + 1]]
        v[s:s + cu[b + 1] - cu[b]] = kv.v[cu[b]:cu[b + 1]]
    return LayerKV(k, v)


class DecodeState:
    # most rows per step for which the norms and the SwiGLU product are folded into the projections (a number
    # set here or on a state holds for every model; else a state takes 8 up to 2048 columns and 2 beyond)
    max_fused_rows: Optional[int] = None

    def __init__(self, wts: DecoderWeights, head: ScoringHead, gate_layer: int, pf: PrefillResult,
                 max_new_tokens: int, prune_below_gate: bool = False, graph: bool = False, fused: bool = True,
                 kv_bits: int = 16, sampler: Optional[TokenSampler] = None, release_kv: bool = False):
        """kv_bits: 16 (the prefill's bf16 caches), 8 or 4 (quantised copies of them).  sampler: draws the tokens
        (step i takes its random numbers i + 1; the first token's are 0), else greedy.  release_kv: with
        quantised caches, drops pf's reference to each bf16 cache as soon as it is quantised.

        max_steps, the steps that the state takes: max_new_tokens, for which the caches have room; with a sampler of
        n random numbers per sequence n - 1 at most (n = max_new_tokens tokens in all, the first among them)."""
        shape = wts.shape
        if kv_bits not in (4, 8, 16):
            raise ValueError(f"DecodeState: kv_bits must be 16, 8 or 4 (got {kv_bits})")
        if sampler is not None and sampler.draws.shape[0] < max_new_tokens:
            raise ValueError("DecodeState: the sampler has fewer random numbers than max_new_tokens")
        if sampler is not None and (sampler.batch != len(pf.n_kept) or sampler.vocab < wts.lm_head.shape[0]):
            raise ValueError(f"DecodeState: the sampler is for {sampler.batch} sequences and {sampler.vocab} tokens, the model's "
                             f"are {len(pf.n_kept)} and {wts.lm_head.shape[0]}")
        self.wts, self.shape = wts, shape
        if self.max_fused_rows is None:
            self.max_fused_rows = 8 if shape.d_model <= 2048 else 2
        dev = wts.device
        B = len(pf.n_kept)
        self.B = B
        self.gate_layer = gate_layer
        L2 = shape.n_layers - gate_layer - 1
        cu_below = pf.cu_prompt if not prune_below_gate else pf.cu_kept
        self.kv_bits = kv_bits
        self.sampler = sampler
        self.paged = pf.pages_below is not None
        if self.paged and (kv_bits != 16 or prune_below_gate):
            raise ValueError("DecodeState: paged caches are decoded over as they are (kv_bits 16, not prune_below_gate)")
        if self.paged and pf.decode_headroom < max_new_tokens:
            raise ValueError("DecodeState: the prefill left pages for fewer new tokens than max_new_tokens")
        in_place = self.paged or kv_bits == 16 and pf.decode_headroom >= max_new_tokens and pf.cache_above is not None \
            and pf.cache_below is not None
        gap = pf.decode_headroom if in_place else max_new_tokens
        self.in_place = in_place
        self.kv: List[Union[LayerKV, QuantKV, PagedKV]] = []
        if kv_bits != 16:
            # where the prompt rows lie in the prefill's caches (None: back to back) and in these
            src = [c.rows_dev if pf.decode_headroom and c is not None else None for c in (pf.cache_below, pf.cache_above)]
            dst = [CacheGap.build(cu, gap, dev) for cu in (cu_below, pf.cu_kept)]
        for l in range(shape.n_layers):
            if kv_bits != 16:
                g = 0 if l <= gate_layer else 1
                cu = cu_below if g == 0 else pf.cu_kept
                q = QuantKV.alloc(dst[g].rows, shape.n_kv_heads, kv_bits, dev)
                kv_quantize(pf.kv[l].k, pf.kv[l].v, q, dst_rows=dst[g].rows_dev, src_rows=src[g], n_rows=cu[-1])
                self.kv.append(q)
                if release_kv:
                    pf.kv[l] = None
            elif in_place:
                self.kv.append(pf.kv[l])
            else:                      # the prefill left no room: one copy per layer
                self.kv.append(_relayout(pf.kv[l], cu_below if l <= gate_layer else pf.cu_kept, gap))
        groups = []
        for cu in (cu_below, pf.cu_kept):
            groups.append(_Group([cu[b] + b * gap for b in range(B)], [cu[b + 1] - cu[b] for b in range(B)], gap))
        self.groups = groups
        # device state: segment starts and rows used, (2, B) int32 (group 0: at / below the gate)
        hdr = torch.tensor([g.seg for g in groups] + [g.n0 for g in groups], dtype=torch.int32)
        d = h2d(hdr, dev)
        self.seg_dev, self.used = d[:2].contiguous(), d[2:].contiguous()
        self.cap_k = [max(g.n0) + max_new_tokens for g in groups]   # longest key run either group reaches
        # Phase-2 layers: key bias by (sequence, head, key), 0 on generated keys (decode_phase2_layer_tensors,
        # qwen3_flex_attention.py:1010-1017), and the per-head query scale
        if in_place and pf.phase2_bias_seq is not None and pf.phase2_bias_seq.shape[-1] >= self.cap_k[1]:
            self.bias = pf.phase2_bias_seq
        else:
            W = self.cap_k[1]
            self.bias = torch.zeros(L2, B, shape.n_heads, W, dtype=torch.float32, device=dev)
            for b in range(B):
                n = pf.n_kept[b]
                self.bias[:, b, :, :n] = pf.phase2_bias[:, :, pf.cu_kept[b]:pf.cu_kept[b + 1]]
        q_head = head.decode_query_head()
        self.qscale = [q_head[j].contiguous() for j in range(L2)] if q_head is not None else None
        last = torch.tensor([pf.cu_kept[b + 1] - 1 for b in range(B)], dtype=torch.int64)
        self.next_pos = pf.kept_positions.index_select(0, h2d(last, dev)) + 1
        self.ssmax = pf.kept_ratio is not None
        # cache slots of the Phase-2 layers, the new token's included once a step has begun
        self.slots = h2d(torch.tensor([float(x) for x in pf.n_kept], dtype=torch.float32), dev) if self.ssmax else None
        self.tables = (pf.pages_below.table, pf.pages_above.table) if self.paged else None
        workspace = paged_decode_attention_workspace if self.paged else decode_attention_workspace if kv_bits == 16 \
            else decode_attention_quant_workspace
        self.att_ws = workspace(B, shape, max(self.cap_k), dev)
        self.rows_b = torch.arange(B, device=dev)
        self.steps = 0
        self.max_new_tokens = max_new_tokens
        self.max_steps = max_new_tokens if sampler is None else min(max_new_tokens, sampler.draws.shape[0] - 1)
        self.use_graph = graph
        self.fused = fused
        self._graph = None
        self._tok_in = self._tok_out = None

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Appends one token per sequence (tokens (B,) int64) and returns the next tokens, greedy or sampled
        (self.last_logprobs then holds their log probabilities, until the next step)."""
        if self.steps >= self.max_new_tokens:
            raise RuntimeError("DecodeState: more steps than max_new_tokens (the caches are full)")
        if self.steps >= self.max_steps:
            raise RuntimeError("DecodeState: more steps than max_steps (the sampler has no random numbers for another)")
        if self.sampler is not None:
            self.sampler.set_step(self.steps + 1)
        if not self.use_graph or self.steps == 0:
            out = self._body(tokens)
        else:
            if self._graph is None:
                self._tok_in = tokens.clone()
                self._graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self._graph):
                    self._tok_out = self._body(self._tok_in)
            self._tok_in.copy_(tokens)
            self._graph.replay()
            out = self._tok_out.clone()
        self.steps += 1
        return out

    def _body(self, tokens: torch.Tensor) -> torch.Tensor:
        """One decode step as device work only (no host synchronisation, no host-side state), so
        that it can be captured and replayed."""
        s, w = self.shape, self.wts
        B = self.B
        dev = tokens.device
        x = torch.nn.functional.embedding(tokens, w.embed)
        # rows beyond max_fused_rows take the separate norm / SwiGLU launches
        wide = s.d_model > 2048
        fused = self.fused and B <= self.max_fused_rows and s.d_model % 512 == 0 and s.d_ff % 512 == 0
        res = None if fused else x.clone()
        normed = torch.empty_like(x)
        hid = torch.empty_like(x)
        qkv = torch.empty(B, s.qkv_dim, dtype=x.dtype, device=dev)
        att = torch.empty(B, s.n_heads, s.head_dim, dtype=x.dtype, device=dev)
        # the rotary table of the new token's position, its cache rows and its own scaled-softmax ratio
        # (slot n_kept + 1 + step at position next_pos); all counters are raised
        rope, r_dec = decode_begin(self.next_pos, w.inv_freq, self.used, self.slots)
        scale = 1.0 / math.sqrt(s.head_dim)
        if fused:
            # each norm is folded into the projection after it, and the SwiGLU product into the gate|up
            # projection (wide models: into the down projection); the residual stream alternates between two
            # buffers (a fused norm reads one and writes the other)
            rbuf = [torch.empty_like(x), torch.empty_like(x)]
            cur = 0
        for l in range(s.n_layers):
            lw = w.layers[l]
            g = 0 if l <= self.gate_layer else 1
            j = l - self.gate_layer - 1
            if fused:
                linear_rows_norm(x if l == 0 else hid, lw.ln1, s.rms_eps, lw.w_qkv, residual=None if l == 0 else rbuf[cur],
                                 residual_out=rbuf[1 - cur], out=qkv)
                cur = 1 - cur
            elif l == 0:
                rmsnorm(res, lw.ln1, s.rms_eps, out=normed)
            else:
                rmsnorm(hid, lw.ln1, s.rms_eps, residual=res, residual_out=res, out=normed)
            if not fused:
                linear_rows(normed, lw.w_qkv, out=qkv)
            kv = self.kv[l]
            rows = (self.used[g], self.cap_k[g], scale, self.att_ws, self.bias[j] if g else None,
                    self.qscale[j] if (g and self.qscale is not None) else None,
                    r_dec if (r_dec is not None and g) else None)
            if self.paged:
                paged_decode_attention(qkv, rope, lw, s, kv, self.tables[g], *rows, out=att)
            elif self.kv_bits == 16:
                decode_attention(qkv, rope, lw, s, kv.k, kv.v, self.seg_dev[g], *rows, out=att)
            else:
                decode_attention_quant(qkv, rope, lw, s, kv, self.seg_dev[g], *rows, out=att)
            linear_rows(att.view(B, -1), lw.w_o, out=hid)
            if fused:
                if wide:
                    gu = linear_rows_norm(hid, lw.ln2, s.rms_eps, lw.w_gu, residual=rbuf[cur], residual_out=rbuf[1 - cur])
                    linear_rows_swiglu(gu, lw.w_down, out=hid)
                else:
                    act = linear_rows_norm_act(hid, lw.ln2, s.rms_eps, lw.w_gu, residual=rbuf[cur],
                                               residual_out=rbuf[1 - cur])
                    linear_rows(act, lw.w_down, out=hid)
                cur = 1 - cur
            else:
                rmsnorm(hid, lw.ln2, s.rms_eps, residual=res, residual_out=res, out=normed)
                act = silu_mul(linear_rows(normed, lw.w_gu))
                linear_rows(act, lw.w_down, out=hid)
        if fused:   # every row produces a token: the final norm folds into the LM head
            logits = linear_rows_norm(hid, w.final_norm, s.rms_eps, w.lm_head, residual=rbuf[cur], out_fp32=True)
        else:
            logits = logits_last(w, hid + res, self.rows_b)
        self.last_logits = logits
        if self.sampler is not None:
            tokens, self.last_logprobs = self.sampler(logits)
            return tokens
        return argmax_rows(logits)
