"""Sampling and log-probabilities of a batch's logits, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from spbitnet_amd import kernels as K
from tests import requests64 as R

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def logits_of(kind, rows, vocab, seed, std=2.5, zipf=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * std
    x -= zipf * torch.log1p(torch.randperm(vocab, generator=g).float())
    return x.to(TYPES[kind])


def sample(logits, uniforms, sampling=None, logits_gpu=None, **settings):
    x = logits.cuda() if logits_gpu is None else logits_gpu
    n, v = x.shape
    u = torch.tensor(uniforms, dtype=torch.float32).cuda()
    tokens = torch.full((n,), -77, dtype=torch.int32, device="cuda")
    lp = torch.full((n,), 77.0, device="cuda")
    ws = torch.full((K.sample_workspace_size(n, v),), 0xFF, dtype=torch.uint8, device="cuda")
    K.sample_gpu(x, u, tokens, sampling or K.Sampling(**settings), ws, logprobs=lp)
    torch.cuda.synchronize()
    return tokens.tolist(), lp.double().tolist()


def check(logits, uniforms, got, settings, note=""):
    """settings: one dict, or one for each row."""
    x = R.f64(logits)
    u = np.float32(uniforms).astype(np.float64)
    for i in range(len(x)):
        s = settings[i] if isinstance(settings, list) else settings
        s = {k: float(np.float32(v)) if k != "top_k" else v for k, v in s.items()}
        token, lp, n = R.sample(x[i], u[i], **s)
        where = (note, i, s, u[i], "kept", n)
        assert got[0][i] == token, (where, got[0][i], token)
        if math.isinf(lp):
            assert got[1][i] == lp, where
        else:  # one rounding to float32; sums of these weights are held to 2^-38 of the largest
            assert abs(got[1][i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -36, (where, got[1][i], lp)


def uniforms_of(rows, seed):
    u = torch.rand(rows, generator=torch.Generator().manual_seed(seed)).tolist()
    if rows > 3:
        u[0], u[1] = 0.0, 1 - 2.0 ** -24
    return u


ONE = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.95),
       dict(top_k=1), dict(top_k=7), dict(top_k=1000, temperature=1.5), dict(top_p=0.9),
       dict(top_p=0.3, temperature=0.5), dict(min_p=0.05), dict(min_p=0.5, top_p=0.7, top_k=3),
       dict(min_p=1.0), dict(top_p=0.0), dict(temperature=3.0, top_p=0.999),
       dict(temperature=0.1), dict(temperature=20.0, top_p=0.5), dict(top_p=1e-6)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4093, 8192, 8193, 16384, 32003, 128256])
def test_one_setting_for_all_rows(gpu, kind, vocab):
    rows = 5
    x = logits_of(kind, rows, vocab, vocab)
    u = uniforms_of(rows, vocab)
    for s in ONE:
        check(x, u, sample(x, u, **s), s)


def mixed(rows, seed):
    g = np.random.default_rng(seed)
    out = []
    for _ in range(rows):
        out.append(dict(temperature=float(g.choice([0.0, 0.3, 0.8, 1.0, 1.7])),
                        top_k=int(g.choice([0, 0, 1, 5, 40, 300])),
                        top_p=float(g.choice([1.0, 1.0, 0.2, 0.8, 0.95])),
                        min_p=float(g.choice([0.0, 0.0, 0.01, 0.2]))))
    return out


def vectors(settings):
    return K.Sampling(
        torch.tensor([s["temperature"] for s in settings]).cuda(),
        torch.tensor([s["top_k"] for s in settings], dtype=torch.int32).cuda(),
        torch.tensor([s["top_p"] for s in settings]).cuda(),
        torch.tensor([s["min_p"] for s in settings]).cuda())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 5000), (3, 128256), (40, 32003), (300, 777), (1100, 100)])
def test_settings_of_each_row(gpu, kind, rows, vocab):
    x = logits_of(kind, rows, vocab, rows)
    u, s = uniforms_of(rows, rows), mixed(rows, rows)
    check(x, u, sample(x, u, vectors(s)), s)


@pytest.mark.parametrize("vocab", [5, 300, 20011, 128256])
@pytest.mark.parametrize("masked", [0.5, 0.99, 1.0])
def test_masked_rows(gpu, vocab, masked):
    rows = 6
    x = logits_of("f32", rows, vocab, 7)
    hide = torch.rand(rows, vocab, generator=torch.Generator().manual_seed(1)) < masked
    x[hide] = -math.inf
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, vocab - 1] = -50.0  # one token left
    x[4, ::2] = math.nan
    u = uniforms_of(rows, 3)
    for s in ONE[:9]:
        got = sample(x, u, **s)
        check(x, u, got, s)
        assert got[0][2] == -1 and got[1][2] == -math.inf
        assert got[0][3] == vocab - 1 and got[1][3] == 0.0


def test_infinities_zeros_and_lowest_values(gpu):
    lowest = torch.finfo(torch.float32).min
    x = torch.zeros(9, 300)
    x[0, 100] = math.inf                      # alone has weight
    x[1, [50, 200, 250]] = math.inf           # share it
    x[2] = lowest                             # a mask of the type's lowest value everywhere
    x[3] = lowest
    x[3, 7] = 1.0
    x[4, 10:20] = -0.0                        # equal to zero
    x[5] = math.nan
    x[6] = math.nan
    x[6, 299] = 3.0
    x[7] = torch.finfo(torch.float32).max
    x[7, 5] = -torch.finfo(torch.float32).max
    x[8] = torch.arange(300.0) * 1e-40        # subnormal steps
    for u in (0.0, 0.4, 0.999):
        for s in (dict(), dict(top_k=12), dict(top_p=0.5), dict(min_p=0.3), dict(temperature=0.0)):
            check(x, [u] * 9, sample(x, [u] * 9, **s), s, note=u)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [100, 5000, 128256])
def test_equal_logits(gpu, kind, vocab):
    """Rows of one value, of two and of few: ties go by index, also across a filter's border."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.stack([torch.full((vocab,), 1.5), torch.randint(0, 2, (vocab,), generator=g) * 1.0,
                     torch.randint(0, 5, (vocab,), generator=g) * 0.25]).to(TYPES[kind])
    for u in ([0.0, 0.3, 0.7], [0.5, 0.9999, 1 - 2.0 ** -24]):
        for s in (dict(), dict(top_k=3), dict(top_k=vocab // 2 + 1), dict(top_p=0.5),
                  dict(top_p=0.75, temperature=0.5), dict(top_k=vocab // 3, top_p=0.5), dict(min_p=0.9)):
            check(x, u, sample(x, u, **s), s, note=u)


@pytest.mark.parametrize("std,zipf,temperature", [(0.01, 0.0, 1.0), (1.0, 0.0, 1.0), (2.0, 0.0, 100.0),
                                                  (30.0, 0.0, 1.0), (0.5, 3.0, 0.2), (9.0, 0.0, 50.0),
                                                  (1000.0, 0.0, 10.0)])
@pytest.mark.parametrize("vocab", [3000, 128256])
def test_flat_and_steep_rows(gpu, std, zipf, temperature, vocab):
    rows = 6
    x = logits_of("f32", rows, vocab, 5, std, zipf)
    u = [0.0, 0.2, 0.5, 0.8, 0.97, 0.9999]
    for s in (dict(), dict(top_p=0.9), dict(top_k=vocab // 2), dict(top_k=vocab - 1, top_p=0.99),
              dict(min_p=0.001), dict(top_p=0.9999999)):
        s = dict(s, temperature=temperature)
        check(x, u, sample(x, u, **s), s)


@pytest.mark.parametrize("rows", [1, 400])
def test_top_k_ends_between_logits_of_which_thousands_decide(gpu, rows):
    """min-p's border is among 2000 nearly equal logits, top-k's before them between two."""
    vocab = 20000
    g = torch.Generator().manual_seed(rows)
    x = torch.full((rows, vocab), -60.0)
    at = torch.randperm(vocab, generator=g)
    x[:, at[:2000]] = -20.0 + torch.rand(rows, 2000, generator=g) * 0.01
    x[:, at[2000:2010]] = torch.arange(10).float() * -0.4
    u = uniforms_of(rows, rows)
    for k in (1, 2, 5, 9, 10, 0):
        for p in (1.0, 0.1, 0.6):
            s = dict(temperature=50.0, top_k=k, top_p=p, min_p=math.exp(-19.995 / 50))
            got = sample(x, u, **s)
            check(x[:5], u[:5], [v[:5] for v in got], s)


def test_temperatures_and_settings_out_of_range(gpu):
    rows = 14
    x = logits_of("f32", rows, 3000, 2)
    t = [1e-30, 1e-45, 3e38, math.inf, math.nan, -1.0, -0.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0]
    k = [0, 0, 0, 0, 0, 0, 0, -5, 2 ** 31 - 1, -2 ** 31, 0, 0, 0, 0]
    p = [1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, math.nan, 7.0, -1.0, 1.0]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, math.nan, -3.0, 0.0, 9.0]
    v = K.Sampling(torch.tensor(t).cuda(), torch.tensor(k, dtype=torch.int32).cuda(),
                   torch.tensor(p).cuda(), torch.tensor(m).cuda())
    meant = [dict(temperature=float(np.float32(a))) for a in t]
    meant[4] = dict(temperature=0.0)
    meant[12], meant[13] = dict(top_p=0.0), dict(min_p=1.0)
    for u in (0.0, 0.6, 0.99):
        got = sample(x, [u] * rows, v)
        check(x, [u] * rows, got, meant, note=u)


def test_uniforms_out_of_range(gpu):
    x = logits_of("f32", 7, 900, 3)
    u = [0.0, -1.0, math.nan, 1.0, 5.0, math.inf, -math.inf]
    check(x, u, sample(x, u, temperature=2.0), dict(temperature=2.0))


def test_shares_of_evenly_spaced_numbers(gpu):
    """Of N evenly spaced numbers each token gets its share, to within one."""
    n = 4096
    x = logits_of("f32", 1, 50, 4, 1.0, 0.5)
    u = [(i + 0.5) / n for i in range(n)]
    got, _ = sample(x.repeat(n, 1), u, temperature=0.9)
    p = torch.softmax(x[0].double() / np.float32(0.9), 0).numpy()
    count = np.bincount(got, minlength=50)
    assert np.abs(count - p * n).max() <= 1.0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_strides_and_alignment(gpu, kind):
    vocab = 9001
    x = logits_of(kind, 5, vocab, 6)
    for pad, at in ((1, 0), (7, 3), (64, 1)):
        big = torch.full((5, vocab + pad + at), math.inf, dtype=TYPES[kind], device="cuda")
        view = big[:, at:at + vocab]
        view.copy_(x)
        u = uniforms_of(5, pad)
        for s in ONE[:4]:
            check(x, u, sample(x, u, logits_gpu=view, **s), s)
        n = torch.tensor([3, 0, vocab - 1, 77, 9000], dtype=torch.int32)
        logprob_check(x, n, logprobs(x, n, 4, logits_gpu=view), 4)


def test_rows_past_32_bits(gpu):
    vocab, step = 4000, (1 << 30) + 1
    x = logits_of("f32", 3, vocab, 8)
    big = torch.empty(2 * step + vocab, device="cuda")
    view = big.as_strided((3, vocab), (step, 1))
    view.copy_(x)
    u = uniforms_of(3, 8)
    check(x, u, sample(x, u, logits_gpu=view, top_p=0.9), dict(top_p=0.9))
    n = torch.tensor([1, 2, 3], dtype=torch.int32)
    logprob_check(x, n, logprobs(x, n, 3, logits_gpu=view), 3)


def test_sample_graph_reads_everything_anew(gpu):
    rows, vocab = 9, 20000
    x = logits_of("bf16", rows, vocab, 10).cuda()
    u = torch.zeros(rows, device="cuda")
    s = vectors(mixed(rows, 1))
    ws = torch.empty(K.sample_workspace_size(rows, vocab), dtype=torch.uint8, device="cuda")
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lp = torch.zeros(rows, device="cuda")
    lw = torch.empty(K.token_logprobs_workspace_size(rows, vocab, 3), dtype=torch.uint8, device="cuda")
    ids, values, under = (torch.zeros(rows, 3, dtype=torch.int32, device="cuda"),
                          torch.zeros(rows, 3, device="cuda"), torch.zeros(rows, device="cuda"))

    def step():
        K.sample_gpu(x, u, tokens, s, ws, logprobs=lp)
        K.token_logprobs_gpu(x, tokens, under, lw, top_ids=ids, top_logprobs=values)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(4):
        new = mixed(rows, 20 + rep)
        s.temperature.copy_(torch.tensor([a["temperature"] for a in new]))
        s.top_k.copy_(torch.tensor([a["top_k"] for a in new], dtype=torch.int32))
        s.top_p.copy_(torch.tensor([a["top_p"] for a in new]))
        s.min_p.copy_(torch.tensor([a["min_p"] for a in new]))
        u.copy_(torch.tensor(uniforms_of(rows, rep)))
        x.copy_(logits_of("bf16", rows, vocab, 30 + rep, 1.0 + rep))
        graph.replay()
        torch.cuda.synchronize()
        first = tokens.tolist(), lp.double().tolist(), under.clone(), ids.clone(), values.clone()
        check(x, u.tolist(), first[:2], new, note=rep)
        logprob_check(x, tokens, (first[2], first[3], first[4]), 3)
        step()
        torch.cuda.synchronize()
        assert tokens.tolist() == first[0] and lp.double().tolist() == first[1]
        assert torch.equal(under, first[2]) and torch.equal(ids, first[3])


def test_two_graphs_share_a_workspace(gpu):
    sizes = ((3, 50000), (70, 3001))
    ws = torch.empty(max(K.sample_workspace_size(*s) for s in sizes), dtype=torch.uint8, device="cuda")
    parts = []
    for n, v in sizes:
        x, u = logits_of("f32", n, v, n), uniforms_of(n, n)
        d, du = x.cuda(), torch.tensor(u).cuda()
        t, lp = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
        s = K.Sampling(top_p=0.9)
        K.sample_gpu(d, du, t, s, ws, logprobs=lp)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.sample_gpu(d, du, t, s, ws, logprobs=lp)
        parts.append((x, u, t, lp, g, d, du, s))
    for i in (0, 1, 1, 0, 1):
        x, u, t, lp, g = parts[i][:5]
        t.fill_(-9)
        g.replay()
        torch.cuda.synchronize()
        check(x, u, (t.tolist(), lp.double().tolist()), dict(top_p=0.9), note=i)


def test_own_stream_and_ends_of_the_workspaces(gpu):
    n, v = 5, 40000
    x, u = logits_of("f32", n, v, 1), uniforms_of(n, 1)
    d, du = x.cuda(), torch.tensor(u).cuda()
    size, lsize = K.sample_workspace_size(n, v), K.token_logprobs_workspace_size(n, v, 5)
    ws = torch.full((size + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    lw = torch.full((lsize + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    t = torch.full((n + 2,), -9, dtype=torch.int32, device="cuda")
    lp = torch.full((n + 2,), 9.0, device="cuda")
    ids = torch.full((n + 1, 5), -9, dtype=torch.int32, device="cuda")
    values = torch.full((n + 1, 5), 9.0, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    K.sample_gpu(d, du, t[:n], K.Sampling(top_k=9), ws[:size], logprobs=lp[:n], stream=s)
    K.token_logprobs_gpu(d, t[:n], lp[:n], lw[:lsize], top_ids=ids[:n], top_logprobs=values[:n], stream=s)
    s.synchronize()
    logprob_check(x, t[:n], (lp[:n], ids[:n], values[:n]), 5)
    assert t[n:].tolist() == [-9, -9] and lp[n:].tolist() == [9.0, 9.0]
    assert (ids[n] == -9).all() and (values[n] == 9).all()
    assert (ws[size:] == 0x5A).all() and (lw[lsize:] == 0x5A).all()


# ---- log-probabilities ----------------------------------------------------------

def logprobs(logits, tokens, top, logits_gpu=None):
    x = logits.cuda() if logits_gpu is None else logits_gpu
    n, v = x.shape
    ws = torch.full((K.token_logprobs_workspace_size(n, v, top),), 0xFF, dtype=torch.uint8, device="cuda")
    lp = torch.full((n,), 77.0, device="cuda")
    ids = torch.full((n, top), -77, dtype=torch.int32, device="cuda")
    values = torch.full((n, top), 77.0, device="cuda")
    both = dict(top_ids=ids, top_logprobs=values) if top else {}
    if tokens is None:
        K.token_logprobs_gpu(x, None, None, ws, **both)
    else:
        K.token_logprobs_gpu(x, tokens.cuda(), lp, ws, **both)
    torch.cuda.synchronize()
    return lp, ids, values


def _near(got, want, err):
    if math.isinf(want):
        return got == want
    return abs(got - want) <= err


def logprob_check(logits, tokens, got, top, note=""):
    x = R.f64(logits)
    lp, ids, values = (t.cpu() for t in got)
    for i in range(len(x)):
        want, err, best = R.logprobs(x[i], top)
        t = None if tokens is None else int(tokens[i])
        if t is not None and not 0 <= t < x.shape[1]:
            assert lp[i] == 77.0 and (ids[i] == -77).all() and (values[i] == 77.0).all()
            continue
        if t is not None:
            assert _near(float(lp[i]), want[t], err[t]), (note, i, t, float(lp[i]), want[t], err[t])
        if top:
            assert ids[i].tolist() == best.tolist(), (note, i, ids[i].tolist(), best.tolist())
            for j, b in enumerate(best):
                assert _near(float(values[i, j]), want[b], err[b]), (note, i, j, float(values[i, j]), want[b])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 63), (5, 64), (4, 1000), (300, 65), (3, 8193),
                                        (2, 16385), (40, 32003), (1, 128256), (1030, 257), (9, 128256)])
def test_logprobs(gpu, kind, rows, vocab):
    x = logits_of(kind, rows, vocab, rows + vocab)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    tokens[-1] = vocab - 1
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        logprob_check(x, tokens, logprobs(x, tokens, top), top, note=top)
    top = min(3, vocab)
    logprob_check(x, None, logprobs(x, None, top), top)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_logprobs_in_sorted_and_equal_rows(gpu, kind):
    """Rows that rise and fall, of one value and of few: the best may stand anywhere."""
    v = 30000
    up = torch.linspace(-9, 9, v)
    x = torch.stack([up, up.flip(0), torch.zeros(v), (torch.arange(v) % 3).float(),
                     (torch.arange(v) % 1024 == 1023).float(), (torch.arange(v) // 8192).float(),
                     -(torch.arange(v) % 64).float()]).to(TYPES[kind])
    tokens = torch.tensor([0, 5, v - 1, 9, 1023, 8191, 64], dtype=torch.int32)
    for top in (1, 5, 20, 64):
        logprob_check(x, tokens, logprobs(x, tokens, top), top, note=top)


@pytest.mark.parametrize("kind,vocab", [("f32", 700001), ("bf16", 3000001), ("f32", 3000001)])
def test_logprobs_of_vocabularies_of_millions(gpu, kind, vocab):
    """Groups of many units; in rising order more than the list holds are left of them."""
    up = torch.linspace(-9, 9, vocab)
    for x in (up[None], logits_of("f32", 1, vocab, vocab)):
        x = x.to(TYPES[kind])
        tokens = torch.tensor([vocab - 9], dtype=torch.int32)
        for top in (3, 64):
            logprob_check(x, tokens, logprobs(x, tokens, top), top, note=top)


def test_the_largest_vocabulary(gpu):
    vocab = 1 << 24
    x = logits_of("f16", 1, vocab, 1)
    s = dict(temperature=1.1, top_k=3000, top_p=0.9)
    check(x, [0.7], sample(x, [0.7], **s), s)
    tokens = torch.tensor([vocab - 1], dtype=torch.int32)
    logprob_check(x, tokens, logprobs(x, tokens, 20), 20)


def test_many_rows_of_a_vocabulary_of_a_million(gpu):
    """A block a row, with more units than it keeps the largest logits of."""
    vocab, rows = 1100003, 194
    two = logits_of("f16", 2, vocab, 7)
    two[1] = two[1].sort().values
    x = two.cuda().repeat(rows // 2, 1)
    u = [0.1, 0.93] * (rows // 2)
    for s in (dict(temperature=1.3, top_p=0.9), dict(top_k=900, min_p=0.001)):
        tokens, lp = sample(x, u, logits_gpu=x, **s)
        assert tokens == tokens[:2] * (rows // 2) and lp == lp[:2] * (rows // 2)
        check(two, u[:2], [tokens[:2], lp[:2]], s)
    t = torch.tensor([5, vocab - 1] * (rows // 2), dtype=torch.int32)
    got = logprobs(x, t, 20, logits_gpu=x)
    logprob_check(two, t[:2], [v[:2] for v in got], 20)
    for v in got:
        assert torch.equal(v, v[:2].repeat(rows // 2, *[1] * (v.dim() - 1)))


def test_logprobs_masked_infinite_and_padded(gpu):
    v = 5000
    x = logits_of("f32", 9, v, 3)
    x[0] = -math.inf
    x[1, 10:] = -math.inf            # fewer tokens than are asked for
    x[2, ::3] = math.nan
    x[3, 17] = math.inf
    x[4, [5, 4000]] = math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6, 2] = 60.0                   # nearly all of the mass
    tokens = torch.tensor([4, 11, 3, 17, 9, 0, 2, -1, v], dtype=torch.int32)
    for top in (0, 20):
        logprob_check(x, tokens, logprobs(x, tokens, top), top, note=top)


def test_a_likely_token_keeps_its_digits(gpu):
    """log-probabilities near zero, relative to themselves."""
    x = torch.full((4, 2000), -20.0)
    x[:, 9] = torch.tensor([0.0, 3.0, 8.0, 12.0])
    got = logprobs(x, torch.full((4,), 9, dtype=torch.int32), 1)[0].double().tolist()
    for v, lp in zip([0.0, 3.0, 8.0, 12.0], got):
        want = -math.log1p(1999 * math.exp(-20.0 - v))
        assert abs(lp - want) <= 2.0 ** -18 * abs(want), (v, lp, want)
