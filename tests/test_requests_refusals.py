"""What the operators of requests in a shared batch refuse, without a GPU: the C entry
points return before the HIP runtime, the Python functions raise before the library."""
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


def _said(lib, rc, text):
    assert rc == 1
    assert text in lib.spb_last_error_string().decode(), lib.spb_last_error_string()


def _adapters(sections=(64, 32), **kw):
    d = dict(a=0x10000, b=0x20000, scales=0x30000, ranks=0x40000, a_adapter_stride=32 * 256,
             a_row_stride=256, b_adapter_stride=96 * 16, b_row_stride=16, num_adapters=3, rank=16,
             cols=256, num_sections=len(sections))
    d.update(kw)
    c = _lib.AdaptersC(**d)
    for i, s in enumerate(sections):
        c.section_rows[i] = s
    return c


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_adapters(lib, kind):
    fn = getattr(lib, f"spb_adapters_{kind}")

    def call(ad=_adapters(), ids=A, x=A, base=P(0x50000), out=P(0x60000), n=4, xs=256, bs=96, os=96,
             ws=P(0x70000), size=1 << 24):
        return fn(ctypes.byref(ad) if ad else None, ids, x, base, out, n, xs, bs, os, ws, size, None)
    _said(lib, call(ad=None), "null adapters")
    for bad, text in ((dict(num_adapters=0), "adapter"), (dict(rank=0), "rank"), (dict(rank=12), "rank"),
                      (dict(rank=264), "rank"), (dict(cols=0), "cols"), (dict(cols=100), "cols"),
                      (dict(num_sections=0), "sections"), (dict(num_sections=5), "sections"),
                      (dict(a=None), "null"), (dict(b=None), "null"), (dict(scales=None), "null"),
                      (dict(a=0x10008), "aligned"), (dict(b=0x10002), "aligned"),
                      (dict(scales=0x30002), "aligned"), (dict(ranks=0x30002), "aligned"),
                      (dict(a_row_stride=248), "stride"), (dict(a_row_stride=257), "strides"),
                      (dict(b_row_stride=8), "stride"), (dict(b_adapter_stride=-8), "strides"),
                      (dict(a_adapter_stride=4), "strides")):
        _said(lib, call(ad=_adapters(**bad)), text)
        assert lib.spb_adapters_workspace_size(ctypes.byref(_adapters(**bad)), 4) == 0
    _said(lib, call(ad=_adapters(sections=(64, 0))), "row")
    _said(lib, call(ad=_adapters(sections=(64, -1))), "row")
    _said(lib, call(ad=_adapters(sections=(2 ** 30, 2 ** 30))), "rows")
    _said(lib, call(n=-1), "negative")
    for name in ("ids", "x", "base", "out"):
        _said(lib, call(**{name: None}), "null")
    _said(lib, call(ids=P(0x10002)), "aligned")
    _said(lib, call(x=P(0x10008)), "aligned")
    _said(lib, call(base=P(0x10001)), "aligned")
    _said(lib, call(out=P(0x10001)), "aligned")
    _said(lib, call(xs=255), "stride")
    _said(lib, call(xs=248), "stride")
    _said(lib, call(bs=95), "stride")
    _said(lib, call(os=95), "stride")
    _said(lib, call(bs=128, out=P(0x50000)), "in place")
    _said(lib, call(ws=None), "workspace")
    _said(lib, call(ws=P(0x70008)), "workspace")
    _said(lib, call(size=lib.spb_adapters_workspace_size(ctypes.byref(_adapters()), 4) - 1), "workspace")
    assert lib.spb_adapters_workspace_size(None, 4) == 0
    assert lib.spb_adapters_workspace_size(ctypes.byref(_adapters()), -1) == 0
    assert call(n=0, ids=None, x=None, base=None, out=None, ws=None, size=0) == 0
    _said(lib, call(n=2 ** 31 - 1, size=1 << 62), "tokens")


def test_adapters_workspace_does_not_shrink(lib):
    ad = _adapters(rank=64, b_row_stride=64)
    last = 0
    for n in list(range(1, 700)) + [1000, 4097, 65536, 1 << 20]:
        size = lib.spb_adapters_workspace_size(ctypes.byref(ad), n)
        assert size >= last and size > 0
        last = size


def _sampling(**kw):
    d = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    d.update(kw)
    return _lib.SamplingC(**d)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_sample(lib, kind):
    fn = getattr(lib, f"spb_sample_{kind}")

    def call(logits=A, stride=1000, u=A, tokens=A, lp=A, rows=3, vocab=1000, s=_sampling(), ws=A, size=1 << 40):
        return fn(logits, stride, u, tokens, lp, rows, vocab, ctypes.byref(s) if s else None, ws, size, None)
    _said(lib, call(rows=-1), "negative")
    _said(lib, call(vocab=-1), "negative")
    _said(lib, call(rows=(1 << 20) + 1), "rows")
    _said(lib, call(vocab=(1 << 24) + 1, stride=1 << 25), "vocabulary")
    _said(lib, call(vocab=0), "token")
    _said(lib, call(s=None), "null sampling")
    for bad, text in ((dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"),
                      (dict(top_k=-1), "top_k"), (dict(top_p=-0.1), "top_p"), (dict(top_p=1.1), "top_p"),
                      (dict(top_p=math.nan), "top_p"), (dict(min_p=-0.1), "min_p"),
                      (dict(min_p=math.nan), "min_p"), (dict(temperatures=0x10002), "aligned"),
                      (dict(top_ks=0x10001), "aligned"), (dict(top_ps=0x10001), "aligned"),
                      (dict(min_ps=0x10001), "aligned")):
        _said(lib, call(s=_sampling(**bad)), text)
    for name in ("logits", "u", "tokens"):
        _said(lib, call(**{name: None}), "null")
    _said(lib, call(logits=P(0x10001)), "aligned")
    for name in ("u", "tokens", "lp"):
        _said(lib, call(**{name: P(0x10002)}), "aligned")
    _said(lib, call(stride=999), "overlap")
    _said(lib, call(ws=None), "workspace")
    _said(lib, call(ws=P(0x10008)), "workspace")
    _said(lib, call(size=lib.spb_sample_workspace_size(3, 1000) - 1), "workspace")
    assert call(rows=0, logits=None, u=None, tokens=None, ws=None, size=0) == 0
    assert lib.spb_sample_workspace_size(-1, 5) == 0
    assert lib.spb_sample_workspace_size(5, (1 << 24) + 1) == 0
    assert lib.spb_sample_workspace_size((1 << 20) + 1, 5) == 0
    assert lib.spb_sample_workspace_size(0, 0) > 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_token_logprobs(lib, kind):
    fn = getattr(lib, f"spb_token_logprobs_{kind}")

    def call(logits=A, stride=1000, tokens=A, lp=A, ids=A, values=A, rows=3, vocab=1000, top=5, ws=A,
             size=1 << 40):
        return fn(logits, stride, tokens, lp, ids, values, rows, vocab, top, ws, size, None)
    _said(lib, call(rows=-1), "negative")
    _said(lib, call(vocab=-1), "negative")
    _said(lib, call(rows=(1 << 20) + 1), "rows")
    _said(lib, call(vocab=(1 << 24) + 1, stride=1 << 25), "vocabulary")
    _said(lib, call(vocab=0), "token")
    _said(lib, call(top=-1), "top")
    _said(lib, call(top=65), "top")
    _said(lib, call(top=5, vocab=4), "top")
    _said(lib, call(logits=None), "null")
    _said(lib, call(tokens=None), "together")
    _said(lib, call(lp=None), "together")
    _said(lib, call(ids=None), "null")
    _said(lib, call(values=None), "null")
    _said(lib, call(tokens=None, lp=None, top=0), "neither")
    _said(lib, call(logits=P(0x10001)), "aligned")
    for name in ("tokens", "lp", "ids", "values"):
        _said(lib, call(**{name: P(0x10002)}), "aligned")
    _said(lib, call(stride=999), "overlap")
    _said(lib, call(ws=None), "workspace")
    _said(lib, call(ws=P(0x10008)), "workspace")
    _said(lib, call(size=lib.spb_token_logprobs_workspace_size(3, 1000, 5) - 1), "workspace")
    assert call(rows=0, logits=None, tokens=None, lp=None, ids=None, values=None, ws=None, size=0) == 0
    assert lib.spb_token_logprobs_workspace_size(5, 10, 65) == 0
    assert lib.spb_token_logprobs_workspace_size(-1, 10, 5) == 0
    assert lib.spb_token_logprobs_workspace_size(0, 0, 0) > 0


@pytest.mark.parametrize("name,args", [("sample", (1 << 20, 1 << 24)), ("token_logprobs", (1 << 20, 1 << 24, 64))])
def test_workspaces_do_not_shrink_and_stay_bounded(lib, name, args):
    """A larger batch's workspace serves a smaller one, and long batches go in parts."""
    fn = getattr(lib, f"spb_{name}_workspace_size")
    for vocab in (1, 100, 8193, 128256, 1 << 24):
        last = 0
        for rows in (0, 1, 2, 7, 64, 500, 513, 4096, 1 << 20):
            size = fn(rows, vocab, *args[2:])
            assert size >= last
            last = size
        assert last < 1 << 31


def test_python_refuses():
    half = torch.zeros(2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.Adapters(half, torch.zeros(2, 32, 16, dtype=torch.bfloat16), torch.zeros(2))
    with pytest.raises(TypeError, match="torch.Tensor"):
        K.Adapters(None, half, None)
    with pytest.raises(TypeError, match="dtype"):
        K.Adapters(half.float(), half, None)
    with pytest.raises(ValueError, match="adapters"):
        K.Adapters(half, half[:1], None)
    with pytest.raises(TypeError, match="Adapters"):
        K.adapters_gpu(None, None, None, None, None, None)
    with pytest.raises(TypeError, match="Adapters"):
        K.adapters_workspace_size(None, 4)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=1.5),
                dict(top_p=-0.5), dict(min_p=2.0), dict(min_p=math.nan), dict(top_k=2 ** 31)):
        with pytest.raises(ValueError):
            K.Sampling(**bad)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.Sampling(temperature=torch.ones(3))
    with pytest.raises(ValueError, match="vector"):
        K.Sampling(top_k=torch.ones(3, 1, dtype=torch.int32))
    with pytest.raises(TypeError, match="logits"):
        K.sample_gpu(None, None, None, None, None)
    with pytest.raises(TypeError, match="float32"):
        K.sample_gpu(torch.zeros(2, 3, dtype=torch.float64), None, None, None, None)
    with pytest.raises(ValueError, match=r"\[rows\]\[vocab\]"):
        K.sample_gpu(torch.zeros(3), None, None, None, None)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.sample_gpu(torch.zeros(2, 3), None, None, None, None)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.token_logprobs_gpu(torch.zeros(2, 3), None, None, None)
    for fn, args in ((K.sample_workspace_size, (2 ** 31, 5)), (K.sample_workspace_size, (5, 2 ** 32)),
                     (K.token_logprobs_workspace_size, (5, 5, 2 ** 32))):
        with pytest.raises(ValueError, match="32 bits"):
            fn(*args)
    with pytest.raises(_lib.SpbError, match="vocabulary"):
        K.sample_workspace_size(3, (1 << 24) + 1)
    with pytest.raises(_lib.SpbError, match="top"):
        K.token_logprobs_workspace_size(3, 100, 65)


def test_settings_are_fixed():
    s = K.Sampling(temperature=0.5, top_k=3)
    with pytest.raises(AttributeError, match="cannot be changed"):
        s.top_k = 5
    with pytest.raises(AttributeError):
        del s.temperature
    s.note = "a program's own"
    assert s.note
