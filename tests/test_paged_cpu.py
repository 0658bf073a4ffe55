"""Refusals of the paged KV cache, without a GPU: the argument checks of the Python entry points and of the C ABI come before
any launch."""
import copy
import ctypes
import pickle

import pytest
import torch

BF = torch.bfloat16


def _cache(pages=6, hkv=2, rows=16):
    from tokengate_amd import paged as P
    return P.PagedKV.alloc(pages, hkv, rows, "cpu")


def test_layouts():
    from tokengate_amd import paged as P
    c = _cache()
    assert (c.n_pages, c.n_kv_heads, c.page_rows, c.nbytes) == (6, 2, 16, 2 * 6 * 2 * 16 * 256)
    both = torch.zeros(6, 16, 2, 2, 128, dtype=BF)
    t = P.PagedKV(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2))
    assert t._args[1:4] == (16 * 512, 128, 512)
    one = torch.zeros(1, 1, 16, 128, dtype=BF)
    P.PagedKV(one.as_strided((1, 1, 16, 128), (8, 8, 128, 1)), one.clone())      # one page, one head: any strides
    for k, v, what in ((c.k.float(), c.v, "bf16"), (c.k[..., :64], c.v[..., :64], "bf16"), (c.k[0], c.v[0], "bf16"),
                       (c.k, c.v[:, :1], "one shape"), (c.k[:0], c.v[:0], "at least one page"), (c.k[:, :, :8], c.v[:, :, :8], "power of two"),
                       (torch.zeros(2, 2, 48, 128, dtype=BF), torch.zeros(2, 2, 48, 128, dtype=BF), "power of two"),
                       (c.k, c.k, "share memory"), (torch.zeros(6, 2, 16, 132, dtype=BF)[..., :128], c.v, "multiples of 8"),
                       (c.k[:1, :1].expand(6, 2, 16, 128), c.v, "overlap"),
                       (torch.zeros(9000, dtype=BF).as_strided((2, 2, 16, 128), (64, 2048, 128, 1)), c.v[:2], "overlap"),
                       (torch.zeros(50000, dtype=BF)[1:49153].view(12, 2, 16, 128)[:6], c.v, "aligned")):
        with pytest.raises(RuntimeError, match=what):
            P.PagedKV(k, v)


def test_copies():
    c = _cache()
    c.k.fill_(1.0)
    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert d._args[0] == d.k.data_ptr() != c.k.data_ptr() and d._args[4] == d.v.data_ptr() and torch.equal(d.k, c.k)
    with pytest.raises(Exception):
        c.k = c.v


def test_python_refusals():
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    c = _cache()
    shape = dec.DecoderShape(n_layers=1, n_heads=4, n_kv_heads=2)
    w = torch.ones(128, dtype=BF)
    lw = dec.LayerWeights(None, None, w, w, None, None, None, None)
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)
    qkv, rope, f = torch.zeros(3, 8 * 128, dtype=BF), torch.zeros(3, 64, 2), torch.zeros
    good = dict(qkv=qkv, rope=rope, lw=lw, shape=shape, cache=c, slots=i32(3))
    bad_w = dec.LayerWeights(None, None, w.float(), w, None, None, None, None)
    for kw, what in ((dict(qkv=qkv.float()), "qkv"), (dict(qkv=qkv[:, :900]), "qkv"), (dict(qkv=qkv[0]), "qkv"),
                     (dict(rope=rope[:2]), "rope"), (dict(rope=rope.double()), "rope"), (dict(slots=i32(2)), "slots"),
                     (dict(slots=i32(6)[::2]), "slots"), (dict(slots=torch.zeros(3)), "slots"), (dict(cache=_cache(hkv=4)), "other KV heads"),
                     (dict(q_head_scale=f(3)), "q_head_scale"), (dict(q_row_scale=f(3).double()), "q_row_scale"),
                     (dict(out=qkv), "out"), (dict(out=torch.zeros(3, 4, 128)), "out"), (dict(lw=bad_w), "norm weights"),
                     (dict(out=torch.zeros(1, 4, 128, dtype=BF).expand(3, 4, 128)), "overlap")):
        with pytest.raises(RuntimeError, match=what):
            P.paged_append(**dict(good, **kw))
    begin = dict(positions=torch.zeros(3, dtype=torch.int64), inv_freq=f(64), cu_q=i32(3), kv_used=i32(2), page_table=i32(2, 5), cache=c)
    for kw, what in ((dict(positions=i32(3)), "positions"), (dict(inv_freq=f(32)), "inv_freq"), (dict(cu_q=torch.zeros(3)), "cu_q"),
                     (dict(cu_q=i32(1)), "cu_q"), (dict(kv_used=i32(1)), "kv_used"), (dict(page_table=i32(1, 5)), "page_table"),
                     (dict(page_table=i32(2, 0)), "page_table"), (dict(page_table=i32(5, 2).t()), "page_table")):
        with pytest.raises(RuntimeError, match=what):
            P.paged_begin(**dict(begin, **kw))
    q = torch.zeros(3, 4, 128, dtype=BF)
    attn = dict(q=q, cache=c, page_table=i32(2, 5), cu_q=i32(3), kv_used=i32(2), max_q=3, max_k=80, scale=0.1)
    for kw, what in ((dict(q=q.float()), "q must"), (dict(q=q[:, :3]), "multiple"), (dict(page_table=i32(2, 4)), "fewer than max_k"),
                     (dict(kv_used=i32(1)), "kv_used"), (dict(bias_raw=f(2, 4, 79)), "bias"), (dict(bias_raw=f(2, 3, 80)), "bias"),
                     (dict(bias_raw=f(2, 4, 80).double()), "bias"), (dict(out=q[:2]), "out"), (dict(cu_q=i32(0)), "cu_q"),
                     (dict(page_table=torch.zeros(2, 5)), "page_table")):
        with pytest.raises(RuntimeError, match=what):
            P.paged_attention(**dict(attn, **kw))
    dec_ = dict(qkv=qkv, rope=rope, lw=lw, shape=shape, cache=c, page_table=i32(3, 5), kv_used=i32(3), max_k=80, scale=0.1,
                workspace=torch.zeros(16, dtype=torch.uint8))
    for kw, what in ((dict(workspace=torch.zeros(16)), "workspace"), (dict(kv_used=i32(2)), "kv_used"), (dict(max_k=81), "max_k"),
                     (dict(page_table=i32(2, 5)), "page_table"), (dict(bias_raw=f(1, 4, 80)), "bias"), (dict(rope=rope[:1]), "rope"),
                     (dict(out=q[:, :2]), "out"), (dict(q_row_scale=f(2)), "q_row_scale"), (dict(lw=bad_w), "norm weights")):
        with pytest.raises(RuntimeError, match=what):
            P.paged_decode_attention(**dict(dec_, **kw))
    for call in (lambda: P.paged_append(**good), lambda: P.paged_decode_attention(**dec_), lambda: P.paged_attention(**attn)):
        with pytest.raises(RuntimeError, match="on a GPU"):
            call()


def test_sizes_past_32_bits():
    """A table may hold more keys than a call takes: such a max_k is refused, as the C entries do, and not cut to 32 bits."""
    from tokengate_amd import decoder as dec
    from tokengate_amd import paged as P
    c = _cache(1, 1, 65536)
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)
    shape, w = dec.DecoderShape(n_layers=1, n_heads=1, n_kv_heads=1), torch.ones(128, dtype=BF)
    lw = dec.LayerWeights(None, None, w, w, None, None, None, None)
    table = i32(1, 65537)
    for max_k in (1 << 24, 2 ** 32 + 5, -1, -2 ** 32):
        with pytest.raises(RuntimeError, match="max_k must be in"):
            P.paged_attention(torch.zeros(1, 1, 128, dtype=BF), c, table, i32(2), i32(1), 1, max_k, 0.1)
        with pytest.raises(RuntimeError, match="max_k must be in"):
            P.paged_decode_attention(torch.zeros(1, 384, dtype=BF), torch.zeros(1, 64, 2), lw, shape, c, table, i32(1), max_k, 0.1,
                                     torch.zeros(16, dtype=torch.uint8))


def _call(name, good, **change):
    """The error of a C call whose arguments are `good` but for `change`, made before anything is launched."""
    from tokengate_amd import _lib
    lib = _lib.load()
    args = dict(good, **change)
    assert len(args) == len(_lib.SIGNATURES[name])
    assert getattr(lib, name)(*args.values()) != 0
    return lib.tg_last_error().decode()


@pytest.fixture(scope="module")
def ptr():
    """A 256-byte aligned host address: never read, as the calls are refused."""
    buf = ctypes.create_string_buffer(1024)
    return (ctypes.addressof(buf) + 255) // 256 * 256, buf


def test_c_abi_refusals(ptr):
    p = ptr[0]
    pool = dict(k=p, k_ps=32768, k_hs=4096, k_rs=128, v=p, v_ps=32768, v_hs=4096, v_rs=128)
    size = dict(pages=4, page=32)
    begin = dict(pos=p, n=4, inv=p, cu=p, used=p, nseq=1, table=p, table_rs=4, cols=4, **size, slots=p, rope=p, stream=None)
    for change, text in ((dict(pos=None), "null pointer"), (dict(nseq=0), "sequence count"), (dict(n=-1), "row"), (dict(table=None), "page table"),
                         (dict(cols=0), "columns"), (dict(page=24), "power of two"), (dict(page=8), "power of two"),
                         (dict(pages=1 << 28), "2^31")):
        assert text in _call("tg_paged_begin", begin, **change), change
    append = dict(qkv=p, qkv_rs=4096, rope=p, n=4, h=16, hkv=8, d=128, qw=p, kw=p, eps=1e-6, qh=None, qr=None, q=p, q_rs=2048, q_hs=128,
                  slots=p, **pool, **size, stream=None)
    bad_pool = ((dict(d=64), "head_dim"), (dict(hkv=0), "KV heads"), (dict(pages=0), "no pages"), (dict(page=48), "power of two"),
                (dict(pages=1 << 26), "2^31"), (dict(k=None), "null cache"), (dict(v=p + 2), "aligned"), (dict(k_rs=132), "multiples of 8"),
                (dict(v_ps=-8), "multiples of 8"), (dict(k_rs=1 << 25), "1 GiB"))
    for change, text in bad_pool + ((dict(slots=None), "null pointer"), (dict(h=0), "heads"), (dict(h=264), "256"), (dict(n=-1), "token"),
                                    (dict(qkv_rs=4088), "every head"), (dict(q_hs=64), "heads apart"), (dict(rope=p + 4), "aligned"),
                                    (dict(q_rs=2044), "multiples")):
        assert text in _call("tg_paged_append", append, **change), change
    attn = dict(q=p, q_rs=2048, q_hs=128, **pool, **size, table=p, table_rs=4, cols=4, cu=p, used=p, nseq=1, max_q=4, max_k=128, total=4, h=16,
                hkv=8, d=128, bias=None, b_s=0, b_h=0, scale=0.1, out=p, o_rs=2048, o_hs=128, ws=None, ws_n=0, stream=None)
    more = ((dict(scale=0.0), "softmax_scale"), (dict(h=15), "multiple of the KV heads"), (dict(max_k=129), "columns hold"),
            (dict(max_k=1 << 24, cols=1 << 20), "2^24"), (dict(max_k=-1), "max_seqlen_k"), (dict(table=None), "page table"), (dict(used=None), "null pointer"),
            (dict(out=p + 2), "aligned"), (dict(bias=p, b_h=-1), "bias stride"))
    for change, text in bad_pool + more + ((dict(o_hs=4), "multiples"), (dict(total=-1), "negative")):
        assert text in _call("tg_paged_attention", attn, **change), change
    dec = dict(qkv=p, qkv_rs=4096, rope=p, n=1, h=16, hkv=8, d=128, qw=p, kw=p, eps=1e-6, qh=None, qr=None, **pool, **size, table=p, table_rs=4,
               cols=4, used=p, max_k=128, bias=None, b_s=0, b_h=0, scale=0.1, out=p, o_rs=2048, ws=p, ws_n=1 << 30, stream=None)
    for change, text in bad_pool + more + ((dict(o_rs=2040), "every head"), (dict(n=-1), "sequence count"), (dict(qkv=None), "null pointer")):
        assert text in _call("tg_paged_decode_attention", dec, **change), change


def test_workspace_sizes():
    """A workspace serves every smaller call; sizes that no call takes need none."""
    from tokengate_amd import _lib
    lib = _lib.load()
    size = lib.tg_paged_decode_attention_workspace_size
    for h, hkv in ((16, 8), (16, 1), (5, 5), (28, 4)):
        for n in (1, 300, 5000, 1 << 20):
            sizes = [size(b, h, hkv, n) for b in (1, 2, 8, 31, 64, 200, 1000, 2048, 5000, 60000)]
            assert sizes == sorted(sizes)
        assert [size(8, h, hkv, n) for n in (1, 200, 3000, 40000)] == sorted(size(8, h, hkv, n) for n in (1, 200, 3000, 40000))
        assert size(0, h, hkv, 100) == size(-1, h, hkv, 100) == size(4, h, hkv, 0) == size(4, h, 0, 9) == size(4, 7, 3, 100) == 0
    size = lib.tg_paged_attention_workspace_size
    assert size(1, 33, 32769, 33, 16, 8) > 0 and size(1, 4096, 4096, 4096, 16, 8) >= 0
    assert size(8, 2 ** 31 - 1, 6000, 160, 16, 8) == size(8, 160, 6000, 160, 16, 8)
    for bad in ((0, 33, 900, 33, 16, 8), (1, 0, 900, 33, 16, 8), (1, 33, 0, 33, 16, 8), (1, 33, 900, 0, 16, 8), (1, 33, 900, 33, 15, 8),
                (-1, 33, 900, 33, 16, 8), (1, 33, 900, 33, 16, 0)):
        assert size(*bad) == 0
