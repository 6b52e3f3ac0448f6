"""What the operators of a token batch refuse, without a GPU: the C entry points
return before the HIP runtime, the Python functions raise before the library."""
import ctypes
import math

import pytest
import torch

from spbitnet_amd import _lib
from spbitnet_amd import kernels as K

P = ctypes.c_void_p
A = P(0x10000)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _cache(**kw):
    d = dict(k=0x10000, v=0x20000, page_stride=2 * 16 * 128, head_stride=16 * 128, slot_stride=128,
             num_pages=10, page_size=16, num_kv_heads=2, head_dim=128)
    d.update(kw)
    return _lib.PagedCacheC(**d)


def _batch(**kw):
    d = dict(token_starts=0x1000, kv_lens=0x2000, page_table=0x3000, num_seqs=2, table_width=4,
             num_tokens=3, max_new=0)
    d.update(kw)
    return _lib.PagedBatchC(**d)


def _rope(**kw):
    d = dict(inv_freq=0x4000, rotary_dim=128, interleaved=1, scale=1.0)
    d.update(kw)
    return _lib.RopeC(**d)


def _said(lib, rc, text):
    assert rc == 1
    assert text in lib.spb_last_error_string().decode(), lib.spb_last_error_string()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_rope_tokens(lib, kind):
    fn = getattr(lib, f"spb_rope_tokens_{kind}")

    def call(x=A, y=A, pos=A, rope=_rope(), n=3, heads=2, hd=128, xs=256, ys=256):
        return fn(x, y, pos, ctypes.byref(rope) if rope else None, n, heads, hd, xs, ys, None)
    _said(lib, call(n=-1), "negative")
    _said(lib, call(heads=-1), "negative")
    _said(lib, call(rope=None), "null rope")
    _said(lib, call(hd=127), "head_dim")
    _said(lib, call(hd=258, rope=_rope(rotary_dim=2)), "head_dim")
    _said(lib, call(rope=_rope(rotary_dim=130)), "rotary_dim")
    _said(lib, call(rope=_rope(rotary_dim=63)), "rotary_dim")
    _said(lib, call(rope=_rope(rotary_dim=0)), "rotary_dim")
    _said(lib, call(rope=_rope(inv_freq=None)), "inv_freq")
    _said(lib, call(rope=_rope(inv_freq=0x4004)), "inv_freq")
    _said(lib, call(x=None), "null")
    _said(lib, call(y=None), "null")
    _said(lib, call(pos=None), "null")
    _said(lib, call(ys=255, y=P(0x50000)), "stride")
    _said(lib, call(xs=-256), "stride")
    _said(lib, call(xs=512), "in place")
    _said(lib, call(x=P(0x10001)), "aligned")
    assert call(n=0, x=None, y=None, pos=None) == 0
    assert call(heads=0, x=None, y=None, pos=None) == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_qk_norm_rope(lib, kind):
    fn = getattr(lib, f"spb_qk_norm_rope_{kind}")

    def call(q=A, k=A, qo=A, ko=A, qw=A, kw=A, pos=A, rope=_rope(), n=3, nh=4, nkv=2, hd=128,
             eps=1e-5, qs=512, qos=512):
        return fn(q, k, qo, ko, qw, kw, pos, ctypes.byref(rope) if rope else None, n, nh, nkv, hd,
                  qs, 256, qos, 256, ctypes.c_float(eps), None)
    for name in ("q", "k", "qo", "ko", "qw", "kw", "pos"):
        _said(lib, call(**{name: None}), "null")
    _said(lib, call(n=-1), "negative")
    _said(lib, call(nkv=-1), "negative")
    _said(lib, call(eps=-1.0), "eps")
    _said(lib, call(eps=math.nan), "eps")
    _said(lib, call(qos=511, qo=P(0x90000)), "stride")
    _said(lib, call(qs=1024), "in place")
    assert call(n=0) == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_paged_append(lib, kind):
    fn = getattr(lib, f"spb_paged_append_{kind}")

    def call(cache=_cache(), batch=_batch(), k=A, v=A, q=A, qo=A, nh=4, qw=None, kw=None, eps=0.0,
             rope=_rope(), qos=512, qs=512):
        return fn(ctypes.byref(cache) if cache else None, ctypes.byref(batch) if batch else None,
                  k, v, q, qo, 256, 256, qs, qos, nh, qw, kw, ctypes.c_float(eps),
                  ctypes.byref(rope) if rope else None, None)
    _said(lib, call(cache=None), "null cache")
    _said(lib, call(batch=None), "null batch")
    _said(lib, call(k=None), "together")
    _said(lib, call(qo=None), "together")
    _said(lib, call(k=None, v=None, q=None, qo=None), "neither")
    _said(lib, call(nh=0), "num_heads")
    _said(lib, call(nh=-1), "negative")
    _said(lib, call(q=None, qo=None, qw=A), "weight")
    _said(lib, call(k=None, v=None, kw=A), "weight")
    _said(lib, call(eps=-1.0), "eps")
    _said(lib, call(qos=100, qo=P(0x90000)), "stride")
    _said(lib, call(qs=1024), "in place")
    _said(lib, call(rope=_rope(rotary_dim=256)), "rotary_dim")
    assert call(batch=_batch(num_tokens=0)) == 0
    assert call(batch=_batch(num_seqs=0)) == 0


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null pages"), (dict(v=None), "null pages"), (dict(num_pages=0), "page"),
    (dict(page_size=0), "slot"), (dict(num_kv_heads=0), "kv head"), (dict(head_dim=4), "head_dim"),
    (dict(head_dim=100), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(k=0x10008), "aligned"),
    (dict(page_stride=4100), "multiples"), (dict(slot_stride=-128), "smaller"),
    (dict(slot_stride=64), "smaller"), (dict(head_stride=0), "smaller"),
    (dict(page_stride=0), "smaller")])
def test_caches(lib, change, text):
    rc = lib.spb_paged_append_f16(ctypes.byref(_cache(**change)), ctypes.byref(_batch()), A, A, None,
                                  None, 256, 256, 0, 0, 0, None, None, ctypes.c_float(0), None, None)
    _said(lib, rc, text)


@pytest.mark.parametrize("change,text", [
    (dict(num_seqs=-1), "negative"), (dict(table_width=-1), "negative"),
    (dict(num_tokens=-1), "negative"), (dict(max_new=-1), "negative"),
    (dict(num_seqs=65537), "65536"), (dict(token_starts=None), "null array"),
    (dict(kv_lens=None), "null array"), (dict(page_table=None), "null array")])
def test_batches(lib, change, text):
    rc = lib.spb_paged_append_f16(ctypes.byref(_cache()), ctypes.byref(_batch(**change)), A, A, None,
                                  None, 256, 256, 0, 0, 0, None, None, ctypes.c_float(0), None, None)
    _said(lib, rc, text)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_paged_attention(lib, kind):
    fn = getattr(lib, f"spb_paged_attention_{kind}")
    size = lib.spb_paged_attention_workspace_size(4, 2, 128)
    assert size > 0

    def call(cache=_cache(), batch=_batch(), q=A, out=P(0x80000), qs=512, os=512, nh=4, scale=0.1,
             window=0, ws=A, ws_size=size):
        return fn(ctypes.byref(cache) if cache else None, ctypes.byref(batch) if batch else None, q,
                  out, qs, os, nh, ctypes.c_float(scale), 1, window, ws, ws_size, None)
    _said(lib, call(cache=None), "null cache")
    _said(lib, call(batch=None), "null batch")
    _said(lib, call(nh=3), "multiple")
    _said(lib, call(nh=0), "multiple")
    for scale in (0.0, -1.0, math.inf, math.nan):
        _said(lib, call(scale=scale), "scale")
    _said(lib, call(window=-1), "window")
    _said(lib, call(q=None), "null")
    _said(lib, call(out=None), "null")
    _said(lib, call(q=P(0x10008)), "aligned")
    _said(lib, call(os=516), "multiples")
    _said(lib, call(os=256), "smaller")
    _said(lib, call(out=A, qs=1024), "in place")
    _said(lib, call(ws=None), "workspace")
    _said(lib, call(ws=P(0x10004)), "workspace")
    _said(lib, call(ws_size=size - 1), "workspace")
    _said(lib, call(batch=_batch(num_tokens=0x7FFFFFFF)), "rows")
    assert call(batch=_batch(num_tokens=0)) == 0
    assert call(batch=_batch(num_seqs=0)) == 0


def test_workspace_size(lib):
    assert lib.spb_paged_attention_workspace_size(3, 2, 128) == 0
    assert lib.spb_paged_attention_workspace_size(4, 2, 100) == 0
    with pytest.raises(_lib.SpbError):
        K.paged_attention_workspace_size(4, 2, 260)


def test_inv_freq():
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=258),
                dict(rotary_dim=64, theta=1.0), dict(rotary_dim=64, theta=math.inf),
                dict(rotary_dim=64, scaling="linear", factor=0.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0),
                dict(rotary_dim=64, scaling="yarn", factor=2.0),
                dict(rotary_dim=64, scaling="yarn", factor=2.0, original_positions=4096,
                     beta_fast=1.0, beta_slow=2.0)):
        with pytest.raises(_lib.SpbError):
            K.rope_inv_freq(**bad)
    with pytest.raises(ValueError):
        K.rope_inv_freq(64, scaling="other")


@pytest.mark.parametrize("rot", [2, 64, 128])
def test_inv_freq_values(rot):
    """Against the definitions; libm's pow and these differ by a few roundings."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    base = 500000.0 ** (-2 * i / rot)
    f, s = K.rope_inv_freq(rot, 500000.0)
    assert s == 1.0 and torch.allclose(f, base, rtol=1e-14, atol=0)
    f, s = K.rope_inv_freq(rot, 500000.0, scaling="linear", factor=4.0)
    assert s == 1.0 and torch.allclose(f, base / 4, rtol=1e-14, atol=0)
    if rot == 2:
        return
    f, s = K.rope_inv_freq(rot, 500000.0, scaling="ntk", factor=4.0)
    # the slowest pair turns exactly factor times slower, the fastest as before
    assert s == 1.0 and f[0] == 1.0 and math.isclose(f[-1], base[-1] / 4, rel_tol=1e-12)
    f, s = K.rope_inv_freq(rot, 500000.0, scaling="yarn", factor=4.0, original_positions=4096)
    turns = base * 4096 / (2 * math.pi)
    assert math.isclose(s, 0.1 * math.log(4.0) + 1.0, rel_tol=1e-6)
    assert torch.allclose(f[turns > 64], base[turns > 64], rtol=1e-14, atol=0)
    assert torch.allclose(f[turns < 0.5], base[turns < 0.5] / 4, rtol=1e-14, atol=0)
    assert ((f <= base * (1 + 1e-14)) & (f >= base / 4 * (1 - 1e-14))).all()


def test_python_refuses_host_tensors_and_wrong_types():
    x = torch.zeros(2, 3, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        K.rope_tokens_gpu(x, x, torch.zeros(2, dtype=torch.int32), None)
    with pytest.raises(TypeError):
        K.rope_tokens_gpu(x.float(), x, None, None)
    with pytest.raises(TypeError):
        K.rope_tokens_gpu(None, x, None, None)
    with pytest.raises(ValueError, match="tokens"):
        K.rope_tokens_gpu(x[0], x, None, None)
    with pytest.raises(ValueError):
        K.Rope(torch.zeros(3))
    with pytest.raises(ValueError, match="GPU"):
        K.PagedKVCache(x[None], x[None])
    with pytest.raises(ValueError, match="GPU"):
        i = torch.zeros(2, dtype=torch.int32)
        K.PagedBatch(torch.zeros(3, dtype=torch.int32), i, i[:, None], 4)
    with pytest.raises(ValueError, match="vector"):
        K.PagedBatch(None, None, None, 4)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("size", [dict(num_tokens=0), dict(num_tokens=0, num_seqs=0)])
def test_batches_without_tokens_have_no_pointers(lib, kind, size):
    """An empty tensor's pointer is null: nothing to do, whatever else is asked for."""
    fn = getattr(lib, f"spb_paged_append_{kind}")
    batch = _batch(**size, token_starts=None, kv_lens=None, page_table=None)

    def call(**rope):
        return fn(ctypes.byref(_cache()), ctypes.byref(batch), None, None, None, None, 256, 256, 512,
                  512, 4, A, A, ctypes.c_float(1e-5), ctypes.byref(_rope(**rope)), None)
    assert call() == 0
    _said(lib, call(rotary_dim=130), "rotary_dim")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("nh,nkv", [(2 ** 31 - 1, 0), (1 << 30, 1 << 30), (2 ** 31 - 1, 1)])
def test_more_heads_than_a_block_counts(lib, kind, nh, nkv):
    rope = ctypes.byref(_rope(rotary_dim=2))
    wide = 1 << 33
    if nkv == 0:
        _said(lib, getattr(lib, f"spb_rope_tokens_{kind}")(A, A, A, rope, 1, nh, 2, wide, wide, None),
              "heads")
    _said(lib, getattr(lib, f"spb_qk_norm_rope_{kind}")(
        A, A, A, A, A, A, A, rope, 1, nh, nkv, 2, wide, wide, wide, wide, ctypes.c_float(0), None),
        "heads")
    if nkv:  # its keys and values
        _said(lib, getattr(lib, f"spb_paged_append_{kind}")(
            ctypes.byref(_cache(num_kv_heads=nkv)), ctypes.byref(_batch()), A, A, A, A, wide, wide,
            wide, wide, nh, None, None, ctypes.c_float(0), None, None), "heads")


def test_python_refuses_what_is_no_cache():
    for bad in (None, torch.zeros(1), {}):
        with pytest.raises(TypeError, match="cache must be a PagedKVCache"):
            K.paged_append_gpu(bad, None, None, None)
        with pytest.raises(TypeError, match="cache must be a PagedKVCache"):
            K.paged_attention_gpu(bad, None, None, None, None)


@pytest.mark.parametrize("far", [2 ** 32 + 64, 2 ** 31, -2 ** 32 + 64, 2 ** 64 + 64])
def test_python_refuses_numbers_past_32_bits(far):
    """ctypes cuts them to 32 bits without a word: 2^32 + 64 would be 64."""
    with pytest.raises(ValueError, match="rotary_dim"):
        K.rope_inv_freq(far)
    with pytest.raises(ValueError, match="original_positions"):
        K.rope_inv_freq(64, scaling="yarn", factor=2.0, original_positions=far)
    with pytest.raises(ValueError, match="num_heads"):
        K.paged_attention_workspace_size(far, 1, 64)
    with pytest.raises(ValueError, match="num_kv_heads"):
        K.paged_attention_workspace_size(64, far, 64)
    with pytest.raises(ValueError, match="head_dim"):
        K.paged_attention_workspace_size(64, 1, far)
