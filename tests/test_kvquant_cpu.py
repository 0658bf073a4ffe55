"""Refusals of the quantised caches and of sampling, without a GPU: the argument checks of the Python entry points and
of the C ABI come before any launch."""
import ctypes
import math

import pytest
import torch


def _cache(rows=10, hkv=2, bits=4):
    from tokengate_amd import kvquant as Q
    return Q.QuantKV.alloc(rows, hkv, bits, "cpu")


def test_quantkv_layout_checks():
    from tokengate_amd import kvquant as Q
    c = _cache()
    assert c.rows == 10 and c.n_kv_heads == 2 and c.head_rows == 10 and c.nbytes == 2 * 10 * 2 * 80
    assert _cache(bits=8).nbytes == 2 * 10 * 2 * 144
    with pytest.raises(RuntimeError, match="4 or 8 bits"):
        Q.QuantKV.alloc(4, 2, 3, "cpu")
    with pytest.raises(RuntimeError, match="codes"):
        Q.QuantKV(8, c.k, c.k_meta, c.v, c.v_meta)
    with pytest.raises(RuntimeError, match="codes"):
        Q.QuantKV(4, c.k[:, ::2], c.k_meta[:, ::2], c.v[:, ::2], c.v_meta[:, ::2])
    with pytest.raises(RuntimeError, match="meta"):
        Q.QuantKV(4, c.k, c.k_meta.float(), c.v, c.v_meta)
    with pytest.raises(RuntimeError, match="between heads"):
        Q.QuantKV(4, c.k[:, 2:5], c.k_meta[:, 2:5].clone(), c.v[:, 2:5], c.v_meta[:, 2:5])
    part = Q.QuantKV(4, c.k[:, 2:5], c.k_meta[:, 2:5], c.v[:, 2:5], c.v_meta[:, 2:5])
    assert part.rows == 3 and part.head_rows == 10


def test_python_refusals():
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    c = _cache()
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="bf16"):
        Q.kv_quantize(k.float(), k, c)
    with pytest.raises(RuntimeError, match="bf16"):
        Q.kv_quantize(k[:, :1], k[:, :1], c)
    with pytest.raises(RuntimeError, match="same rows"):
        Q.kv_quantize(k, k[:3], c)
    with pytest.raises(RuntimeError, match="row maps"):
        Q.kv_quantize(k, k, c, dst_rows=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="row maps"):
        Q.kv_quantize(k, k, c, dst_rows=torch.zeros(3, dtype=torch.int32), n_rows=4)
    with pytest.raises(RuntimeError, match="fewer rows"):
        Q.kv_dequantize(c, n_rows=5, out=(k, k))
    x = torch.zeros(2, 7)
    one = torch.zeros(2)
    for kw, what in ((dict(temperature=one.double()), "temperature"), (dict(top_k=one), "top_k"), (dict(top_p=one[:1]), "top_p"),
                     (dict(min_p=torch.zeros(4)[::2]), "min_p"), (dict(workspace=one), "workspace")):
        with pytest.raises(RuntimeError, match=what):
            dec.sample_rows(x, one, **kw)
    with pytest.raises(RuntimeError, match="logits"):
        dec.sample_rows(x.double(), one)
    with pytest.raises(RuntimeError, match="logits"):
        dec.sample_rows(x.t(), torch.zeros(7))


def test_sampling_settings():
    from tokengate_amd.decode import Sampling
    Sampling(0.7, 20, 0.8, 0.0).check(3)
    Sampling([0.0, 1.0], [0, 5], 1.0, [0.1, 0.0]).check(2)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_k=-1),
                dict(top_k=1.5), dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2.0), dict(temperature=[1.0] * 3)):
        with pytest.raises(ValueError):
            Sampling(**bad).check(2)


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
    quant = dict(k=p, k_rs=1024, k_hs=128, v=p, v_rs=1024, v_hs=128, source_rows=4, src=None, dst=None, n=4, hkv=8, d=128,
                 bits=4, kc=p, km=p, vc=p, vm=p, rows=4, head_rows=4, stream=None)
    for change, text in ((dict(k=None), "null row"), (dict(bits=5), "4 or 8 bits"), (dict(d=64), "head_dim"),
                         (dict(km=None), "null cache"), (dict(vc=p + 4), "aligned"), (dict(k=p + 2), "aligned"),
                         (dict(k_rs=1028), "multiples of 8"), (dict(n=5), "more rows"), (dict(source_rows=3), "source"),
                         (dict(head_rows=3), "head_rows"), (dict(hkv=0), "KV heads"), (dict(n=-1), "row count"),
                         (dict(rows=1 << 31, head_rows=1 << 31), "cache rows")):
        assert text in _call("tg_kv_quantize", quant, **change), change
    read = dict(kc=p, km=p, vc=p, vm=p, rows=4, head_rows=4, hkv=8, d=128, bits=8, map=None, n=4, k=p, k_rs=1024, k_hs=128,
                v=p, v_rs=1024, v_hs=128, stream=None)
    for change, text in ((dict(n=5), "more rows"), (dict(v=None), "null row"), (dict(bits=16), "4 or 8"), (dict(v_hs=64), "head strides")):
        assert text in _call("tg_kv_dequantize", read, **change), change
    attn = dict(qkv=p, qkv_rs=4096, rope=p, n=1, h=16, hkv=8, d=128, bits=4, qw=p, kw=p, eps=1e-6, qh=None, qr=None, kc=p,
                km=p, vc=p, vm=p, rows=4, head_rows=4, start=p, used=p, max_k=4, bias=None, bias_s=0, bias_h=0, scale=0.1,
                out=p, out_rs=2048, ws=p, ws_n=1 << 30, stream=None)
    for change, text in ((dict(qkv=None), "null pointer"), (dict(h=15), "multiple of the KV heads"), (dict(qkv_rs=4088), "row strides"),
                         (dict(out_rs=2044), "row strides"), (dict(scale=0.0), "softmax_scale"), (dict(d=64), "head_dim"),
                         (dict(bits=2), "4 or 8"), (dict(rope=p + 4), "aligned"), (dict(n=-1), "sequence count"),
                         (dict(max_k=-1), "length"), (dict(h=264), "256"), (dict(max_k=1000, ws_n=1000), "workspace"),
                         (dict(max_k=1000, ws=None), "workspace"), (dict(max_k=1 << 24), "2^24")):
        assert text in _call("tg_decode_attention_quant", attn, **change), change
    sample = dict(x=p, rs=100, n=1, cols=100, u=p, t=None, k=None, tp=None, mp=None, token=p, lp=None, ws=p, ws_n=1 << 30, stream=None)
    for change, text in ((dict(u=None), "null pointer"), (dict(rs=99), "row stride"), (dict(cols=0), "columns"),
                         (dict(cols=262145, rs=262145), "columns"), (dict(n=-1), "rows")):
        assert text in _call("tg_sample_rows", sample, **change), change


def test_workspace_sizes():
    """Sizes never shrink as a launch grows, and bad sizes ask for nothing."""
    from tokengate_amd import _lib
    lib = _lib.load()
    assert lib.tg_decode_attention_quant_workspace_size(0, 16, 8, 100) == 0
    assert lib.tg_decode_attention_quant_workspace_size(1, 16, 7, 100) == 0
    assert lib.tg_sample_rows_workspace_size(0, 100) == 0 and lib.tg_sample_rows_workspace_size(1, 0) == 0
    sizes = [lib.tg_decode_attention_quant_workspace_size(4, 16, 8, n) for n in (1, 64, 65, 1000, 5000, 40000, 131072)]
    assert sizes == sorted(sizes)
    sizes = [lib.tg_sample_rows_workspace_size(n, 151936) for n in (1, 2, 3, 8, 64)]
    assert sizes == sorted(sizes)


def test_more_refusals(ptr):
    """Workspaces of sampling; tensors that are on no GPU."""
    from tokengate_amd import _lib
    from tokengate_amd import decoder as dec
    from tokengate_amd import kvquant as Q
    p = ptr[0]
    lib = _lib.load()
    for n, cols in ((1, 2049), (7, 40000), (300, 262144)):
        need = lib.tg_sample_rows_workspace_size(n, cols)
        sample = dict(x=p, rs=cols, n=n, cols=cols, u=p, t=None, k=None, tp=None, mp=None, token=p, lp=None, ws=p, ws_n=need, stream=None)
        for change in (dict(ws=None), dict(ws=p + 4), dict(ws_n=1000)):
            assert "workspace" in _call("tg_sample_rows", sample, **change), (n, cols, change)
    c = _cache()
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    for f in (lambda: Q.kv_quantize(k, k, c), lambda: Q.kv_dequantize(c, n_rows=2),
              lambda: dec.sample_rows(torch.zeros(2, 7), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="on a GPU"):
            f()


def test_calls_on_another_device(monkeypatch):
    """A call whose tensors are not on the current device is made on theirs, with its stream."""
    from tokengate_amd import _lib
    seen, on = [], [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            on.append(self.index)

        def __exit__(self, *e):
            on.pop()
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: on[-1], raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name, args, on[-1])))
    _lib.call_on(0, "a", 1)
    _lib.call_on(3, "b", 2)
    assert seen == [("a", (1, 100), 0), ("b", (2, 103), 3)] and on == [0]


def test_outputs_that_overlap(ptr):
    """Read-back into rows that share memory is refused."""
    p = ptr[0]
    read = dict(kc=p, km=p, vc=p, vm=p, rows=4, head_rows=4, hkv=2, d=128, bits=8, map=None, n=4, k=p, k_rs=256, k_hs=128,
                v=p, v_rs=128, v_hs=512, stream=None)
    for change in (dict(k_rs=0), dict(v_rs=64), dict(k_rs=128), dict(v_hs=384), dict(v_rs=0, v_hs=128)):
        assert "overlap" in _call("tg_kv_dequantize", read, **change), change


def test_copies_of_a_cache_are_their_own(monkeypatch):
    """A cache that was copied, pickled or moved passes its own tensors on; its fields cannot be replaced."""
    import copy
    import dataclasses
    import io
    from tokengate_amd import _lib
    from tokengate_amd import kvquant as Q
    calls = []
    monkeypatch.setattr(_lib, "call_on", lambda index, name, *args: calls.append((index, name, args)))
    whole = _cache(rows=20)
    cut = Q.QuantKV(4, *(t[:, 3:13] for t in (whole.k, whole.k_meta, whole.v, whole.v_meta)))
    buf = io.BytesIO()
    torch.save(cut, buf)
    buf.seek(0)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    for c in (copy.deepcopy(cut), torch.load(buf, weights_only=False), copy.copy(cut), dataclasses.replace(cut, v=whole.v.clone()[:, 3:13])):
        calls.clear()
        Q.kv_quantize(x, x, c)
        Q.kv_dequantize(c, n_rows=2)
        assert len(calls) == 2 and c.rows == 10 and c.n_kv_heads == 2 and c.device_index == -1
        ptrs = [t.data_ptr() for t in (c.k, c.k_meta, c.v, c.v_meta)] + [c.rows, c.head_rows]
        assert list(calls[0][2][-6:]) == ptrs and list(calls[1][2][:6]) == ptrs
    assert copy.copy(cut).k is cut.k and copy.deepcopy(cut).k.data_ptr() != cut.k.data_ptr()
    with pytest.raises(AttributeError):
        cut.k = whole.v[:, 3:13]
    with pytest.raises(AttributeError):
        cut.bits = 8


def test_outputs_that_overlap_in_part(ptr):
    """Strides by which some row of some head shares memory with another one's, neither of which is contained in the
    other: refused, against a list of every element's address."""
    p = ptr[0]
    read = dict(kc=p, km=p, vc=p, vm=p, rows=9, head_rows=9, hkv=4, d=128, bits=8, map=None, n=6, k=p, k_rs=1024, k_hs=128,
                v=p, v_rs=1024, v_hs=128, stream=None)
    for rs, hs in ((256, 256), (384, 256), (128, 640), (640, 384), (136, 128), (256, 392), (512, 1016), (8, 704), (1024, 336)):
        for n, hkv in ((6, 4), (3, 2)):
            at = torch.arange(n)[:, None, None] * rs + torch.arange(hkv)[:, None] * hs + torch.arange(128)
            if at.unique().numel() < at.numel():
                assert "overlap" in _call("tg_kv_dequantize", read, n=n, hkv=hkv, k_rs=rs, k_hs=hs), (rs, hs, n, hkv)
                assert "overlap" in _call("tg_kv_dequantize", read, n=n, hkv=hkv, v_rs=rs, v_hs=hs), (rs, hs, n, hkv)


def test_temperatures_of_fp32():
    """Temperatures are passed on as fp32 numbers: those that would be infinite there are refused, those that would be 0 are
    greedy."""
    from tokengate_amd.decode import Sampling
    most = torch.finfo(torch.float32).max
    Sampling([most, 1e-60, 0.0]).check(3)
    for t in (2 * most, 1e39, 1e300):
        with pytest.raises(ValueError, match="temperature"):
            Sampling(t).check(2)
        with pytest.raises(ValueError, match="temperature"):
            Sampling([1.0, t]).check(2)
