"""Sampling where most of a row's tokens are far below its first: sums of many small weights,
of wide and of narrow rows, against 64 bits of mantissa.

A weight in a sum is off by 2^-37 of itself at most (its exponential by 2^-38.6, its rounding to a
whole number by 2^-39 / 0.49), so a sum of them is, and the float64 additions by 2^-50 of the
sum.  A token is right if u times the kept mass is within that of its place."""
import math

import numpy as np
import pytest
import torch

from spbitnet_amd import kernels as K
from tests import requests64 as R
from tests import test_gpu_sampling as S

pytestmark = pytest.mark.gpu
LAST = 1 - 2.0 ** -24  # the largest u


def run(x, u, **settings):
    """Tokens and log-probabilities of x (on the GPU) under settings."""
    n, v = x.shape
    tokens = torch.full((n,), -77, dtype=torch.int32, device="cuda")
    lp = torch.full((n,), 77.0, device="cuda")
    ws = torch.full((K.sample_workspace_size(n, v),), 0xFF, dtype=torch.uint8, device="cuda")
    K.sample_gpu(x, torch.tensor(u, dtype=torch.float32).cuda(), tokens, K.Sampling(**settings), ws,
                 logprobs=lp)
    torch.cuda.synchronize()
    return tokens.tolist(), lp.double().tolist()


class Row:
    """A row (numpy float64) under settings, by the definition and with the bound above."""

    def __init__(self, x, temperature=1.0, top_p=1.0, top_k=0):
        temperature, top_p = float(np.float32(temperature)), float(np.float32(top_p))
        keys = np.argsort(-x, kind="stable")
        self.keys = keys[~np.isneginf(x[keys])]
        self.d = (x[self.keys] - x[self.keys[0]]) / temperature
        w = np.exp(self.d.astype(np.longdouble))
        if top_k:
            w = w[:top_k]
        # without the first weight, an exact 1: beside it each of 128256 would lose up to 2^-64
        self.tail = np.concatenate(([0], w[1:].cumsum()))
        self.upto = 1 + self.tail
        self.slack = self.tail * 2.0 ** -37 + 2.0 ** -50 * self.upto
        self.kept = [len(w)]  # how many may be kept
        if top_p < 1:
            total, off = self.upto[-1], self.slack[-1]
            some = [int((self.upto - w < top_p * total + s).sum()) for s in (-off, off)]
            self.kept = range(some[0], some[1] + 1)

    def check(self, u, token, lp, note=""):
        u, upto = float(np.float32(u)), self.upto
        at = np.flatnonzero(self.keys[:len(upto)] == token)
        assert len(at) == 1, (note, u, "not kept", token)
        at = int(at[0])
        before, off = upto[at - 1] if at else 0.0, self.slack[at] + self.slack[-1]
        ok = [m for m in self.kept if m > at and before - off <= u * upto[m - 1] <= upto[at] + off]
        assert ok, (note, u, token, "at", at, float(before), float(upto[at]))
        for m in ok:
            tail = float(self.tail[m - 1])
            want = float(self.d[at]) - math.log1p(tail)
            # float32's rounding; the weight's 2^-38 and the sum's share of 2^-37
            err = 2.0 ** -24 * abs(want) + (2.0 ** -38 if at else 0.0) + 2.0 ** -37 * min(1.0, tail) + 2.0 ** -49
            if abs(lp - want) <= err:
                return
        raise AssertionError((note, u, token, lp, want))


# weights around half a step of a sum of as many in whole numbers of 2^-48, 2^-46, 2^-42, 2^-38
@pytest.mark.parametrize("vocab,far,t", [(v, far, t) for v, far in (
    (32003, 33.3), (32003, 34.1), (128256, 31.9), (128256, 32.6), (128256, 28.5), (1100003, 27.2),
    (1100003, 30.0)) for t in (1.0, 0.5, 100.0)] + [
    (1 << 24, 27.2, 1.0), (1 << 24, 20.0, 1.0), (1 << 24, 26.4, 100.0)])
def test_one_likely_token_and_all_others_alike(gpu, vocab, far, t):
    x = torch.full((vocab,), -far * t)
    x[vocab // 3] = 0.0
    u = [0.5, 0.99999, LAST]
    got = run(x.cuda().repeat(3, 1), u, temperature=t)
    row = Row(R.f64(x), t)
    for one in zip(u, *got):
        row.check(*one, note=(vocab, far, t))


@pytest.mark.parametrize("vocab,far,wide", [(32003, 33.0, 2.0), (128256, 31.6, 2.0), (128256, 28.0, 3.0),
                                            (128256, 20.0, 30.0), (1100003, 26.0, 10.0)])
@pytest.mark.parametrize("t", [1.0, 0.25, 100.0, 1e-3])
def test_one_likely_token_and_a_wide_tail(gpu, vocab, far, wide, t):
    """The tail's logits differ, so that bins and not equal ones decide."""
    g = torch.Generator().manual_seed(vocab)
    x = -(far + wide * torch.rand(vocab, generator=g)) * t
    x[vocab // 2] = 0.0
    u = [0.3, 0.99999, LAST]
    row = x.cuda()
    whole = run(row.repeat(200 if vocab < 200000 else 3, 1), u * 66 + u[:2] if vocab < 200000 else u,
                temperature=t)
    split = run(row.repeat(3, 1), u, temperature=t)
    assert [v[:3] for v in whole] == list(split)  # a block a row and several
    want = Row(R.f64(x), t)
    for one in zip(u, *split):
        want.check(*one, note=(vocab, far, t))


@pytest.mark.parametrize("t", [1.0, 100.0])
def test_a_border_inside_a_far_tail(gpu, t):
    """top-p and u end among weights of 2^-30 and below, of which there are a million."""
    vocab = 1100003
    g = torch.Generator().manual_seed(3)
    x = -(21.0 + 8.0 * torch.rand(vocab, generator=g)) * t
    x[:40] = -torch.arange(40).float() * t
    u = [0.9, 0.99999, LAST]
    rows = x.cuda().repeat(3, 1)
    for p in (1.0, 0.99999, 0.9999999, 0.9):
        for k in (0, 500000):
            got = run(rows, u, temperature=t, top_p=p, top_k=k)
            row = Row(R.f64(x), t, p, k)
            for one in zip(u, *got):
                row.check(*one, note=(t, p, k))


def test_the_same_row_in_any_batch(gpu):
    """Bit for bit alike alone, in a few rows and among many, aligned or not."""
    vocab = 50021
    g = torch.Generator().manual_seed(5)
    x = torch.randn(vocab, generator=g) * 2 - 2 * torch.log1p(torch.randperm(vocab, generator=g).float())
    x[::7] -= 25.0
    u = [0.999999]
    want = run(x.cuda()[None], u, temperature=1.7, top_p=0.99999)
    for n in (2, 31, 192, 193, 500):
        big = torch.full((n, vocab + n % 3 + 1), 5.0, device="cuda")
        view = big[:, 1:vocab + 1]
        view.copy_(x)
        got = run(view, u * n, temperature=1.7, top_p=0.99999)
        assert got[0] == want[0] * n and got[1] == want[1] * n, n


@pytest.mark.parametrize("mask", [-1e4, -65504.0, -1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("t", [1.0, 30.0])
def test_nearly_equal_logits_beside_finite_masks(gpu, mask, kind, t):
    vocab = 128256
    g = torch.Generator().manual_seed(1)
    x = 3.0 + 0.2 * torch.rand(3, vocab, generator=g)
    x[torch.rand(3, vocab, generator=g) < 0.1] = mask
    x[1, 0] = -100.0
    x = x.to(S.TYPES[kind])
    u = [0.1, 0.7, LAST]
    for s in (dict(), dict(top_p=0.95), dict(top_k=3000)):
        s = dict(s, temperature=t)
        got = run(x.cuda(), u, **s)
        for i in range(3):
            Row(R.f64(x[i]), **s).check(u[i], got[0][i], got[1][i], note=(mask, kind, s))


def test_flat_rows_of_few_values(gpu):
    """bfloat16 rows of 200000: bins of one value that thousands of tokens have."""
    rows, vocab = 6, 200000
    g = torch.Generator().manual_seed(2)
    rank = torch.randperm(vocab, generator=g).float()
    x = torch.randn(rows, vocab, generator=g) * 0.75 - torch.log1p(rank) + 12.0
    x = x.to(torch.bfloat16)
    u = [0.05, 0.3, 0.5, 0.8, 0.97, LAST]
    for s in (dict(temperature=1.3, top_p=0.95), dict(temperature=1.5), dict(temperature=1.5, top_k=90000)):
        got = run(x.cuda(), u, **s)
        for i in range(rows):
            Row(R.f64(x[i]), **s).check(u[i], got[0][i], got[1][i], note=s)


@pytest.mark.parametrize("rows", [1, 250])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_logits_and_temperatures_at_the_ends_of_the_range(gpu, rows, vocab):
    """Subnormal logits under subnormal temperatures, the largest ones under the largest."""
    top = torch.finfo(torch.float32).max
    n = torch.arange(vocab).float()
    step = torch.tensor(2.0 ** -149)
    for t, x in ((2.0 ** -149, (n % 90) * -step), (2.0 ** -146, (n % 90) * -step * 3),
                 (2.0 ** -126, (n % 77) * -(2.0 ** -128)), (2.0 ** -113, (n % 77) * -(2.0 ** -114)),
                 (2.0 ** -115, 2.0 ** -81 + (n % 3) * -(2.0 ** -104)), (2.0 ** -115, 1.0 - (n % 3) * 2.0 ** -24),
                 (2.0 ** -60, 2.0 ** -40 - n * 2.0 ** -63), (top, top - (n % 60) / 30 * top),
                 (top / 2, top * (1 - (n % 60) / 30)), (top / 100, top * (1 - (n % 60) / 30)),
                 (1e30, (n % 60) * -2e30), (3e37, 5.0 - (n % 60) * 5e36), (math.inf, (n % 60) * -5e36),
                 (1e20, -1e5 - n)):
        x = x.float()
        u = 0.617
        token, lp = run(x.cuda().repeat(rows, 1), [u] * rows, temperature=t)
        assert token == token[:1] * rows and lp == lp[:1] * rows
        Row(R.f64(x), t).check(u, token[0], lp[0], note=(t, vocab))


@pytest.mark.parametrize("vocab,rise", [(128256, 0.5), (1100003, 0.01), (1100003, 0.1), (1100003, 0.3),
                                        (1100003, 0.7), (1100003, 20.0), (1 << 24, 0.2)])
@pytest.mark.parametrize("rows", [3, 194])
def test_logprobs_in_slowly_rising_rows(gpu, rows, vocab, rise):
    """The largest logit so far changes with every 1024 of a row, in one block or in several."""
    x = torch.linspace(0.0, rise, vocab)
    tokens = torch.tensor([0, vocab // 2, vocab - 1] * rows, dtype=torch.int32)[:rows]
    got = S.logprobs(x, tokens, 2, logits_gpu=x.cuda().repeat(rows, 1))
    for v in got:  # alike in all rows of a token
        assert torch.equal(v[3:], v[:-3])
    want, err, best = R.logprobs(R.f64(x), 2)
    lp, ids, values = (v.cpu() for v in got)
    for i in range(3):
        t = int(tokens[i])
        assert abs(float(lp[i]) - want[t]) <= err[t], (t, float(lp[i]), want[t], err[t])
        assert ids[i].tolist() == best.tolist()
        for j, b in enumerate(best):
            assert abs(float(values[i, j]) - want[b]) <= err[b], (j, float(values[i, j]), want[b], err[b])


@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rows_wholly_below_the_masks_bound(gpu, rows, kind):
    """Logits around -5000 and -3e4, some parts of a row without any other, some of the row's
    parts wholly masked: the bins' width comes from them where no logit is above."""
    vocab = 9000
    g = torch.Generator().manual_seed(rows)
    u = [0.2, 0.9]
    for low, wide, mask in ((-5000.0, 0.2, None), (-3e4, 900.0, -65504.0), (-4096.0, 3.0, -1e4),
                            (-4100.0, 9.0, -math.inf)):
        x = low + wide * torch.rand(2, vocab, generator=g)
        if mask is not None:
            x[:, 2000:5000] = mask
        x[1, 17] = math.nan
        x = x.to(S.TYPES[kind])
        for s in (dict(), dict(top_p=0.7, temperature=2.0), dict(top_k=900)):
            got = run(x.cuda().repeat(rows // 2, 1), u * (rows // 2), **s)
            assert [v[:2] * (rows // 2) for v in got] == [list(v) for v in got]
            for i in range(2):
                one = R.f64(x[i])
                one[np.isnan(one)] = -math.inf
                Row(one, **s).check(u[i], got[0][i], got[1][i], note=(low, kind, s))
