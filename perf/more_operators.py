"""What each request of a shared batch brings of its own: low-rank adapters beside
a shared projection, sampling of the next token under the request's settings, and
the log-probabilities that it is told.

listed() and draw() give the cases, prepare() what a program holds before the
call, run() one pass, work() what the pass cannot do without and exact() its
result in 64 bits.  run() computes the plain form in elementary torch
operations, or, where `own` is true, calls the framework's operators.

Adapters: token t of a batch with adapter a = ids[t] gets
base[t] + scale[a] * B[a] (A[a] x[t]); ids outside the pool: base[t].  A stacked
projection (q|k|v, gate|up) has sections of rows, each with an A of its own.
Sampling: the tokens of a row stand in the order of falling logits, equal ones by
index; top-k keeps the first k, top-p those with less than p of that mass before
them, min-p those with at least min_p of the first one's mass; the first kept one
whose mass with that before it passes u times the kept mass is taken, and told
with the logarithm of its share of the kept mass.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence, the stacked q|k|v of the 2B shape: all latency
        dict(name="adapters_1_qkv", kind="adapters", dtype="bf16", tokens=1, run=1, adapters=8,
             rank=16, cols=2560, sections="2560 640 640", ragged=False, none=0.0, mix=1),
        # 32 sequences decoded together, 20 fine-tunes among them, some on the plain model
        dict(name="adapters_32_qkv", kind="adapters", dtype="bf16", tokens=32, run=1, adapters=20,
             rank=16, cols=2560, sections="2560 640 640", ragged=False, none=0.15, mix=2),
        # 61 sequences, adapters of different ranks, the down projection
        dict(name="adapters_61_down", kind="adapters", dtype="f16", tokens=61, run=1, adapters=24,
             rank=64, cols=6912, sections="2560", ragged=True, none=0.0, mix=3),
        # prompts of several requests, 2049 tokens in all, the stacked gate|up
        dict(name="adapters_2049_gateup", kind="adapters", dtype="bf16", tokens=2049, run=300,
             adapters=5, rank=32, cols=2560, sections="6912 6912", ragged=False, none=0.0,
             mix=4),
        # the next token of one sequence, the 2B shape's vocabulary
        dict(name="sample_1", kind="sample", dtype="f32", rows=1, vocab=128256, flat=1.0,
             masked=0.0, settings="chat", mix=5),
        # 32 sequences, each with settings of its own, greedy ones and unfiltered ones among them
        dict(name="sample_32_mixed", kind="sample", dtype="f32", rows=32, vocab=128256, flat=1.0,
             masked=0.0, settings="mixed", mix=6),
        # many sequences of a small odd vocabulary, most of it masked off by a grammar
        dict(name="sample_203_masked", kind="sample", dtype="f16", rows=203, vocab=32003, flat=1.0,
             masked=0.9, settings="min_p", mix=7),
        # many samples at a high temperature: flat rows, of which top-p keeps thousands
        dict(name="sample_512_top_p", kind="sample", dtype="f32", rows=512, vocab=128256, flat=1.6,
             masked=0.0, settings="top_p", mix=8),
        # the token of one sequence and its 20 best alternatives
        dict(name="logprobs_1_top20", kind="logprobs", dtype="f32", rows=1, vocab=128256, flat=1.0,
             masked=0.0, top=20, mix=9),
        # 32 sequences decoded together
        dict(name="logprobs_32_top5", kind="logprobs", dtype="f32", rows=32, vocab=128256, flat=1.0,
             masked=0.0, top=5, mix=10),
        # a prompt scored, no alternatives, odd vocabulary
        dict(name="logprobs_1023", kind="logprobs", dtype="bf16", rows=1023, vocab=32003, flat=1.0,
             masked=0.0, top=0, mix=11),
        # a prompt of 2048 tokens scored with alternatives
        dict(name="logprobs_2048_top5", kind="logprobs", dtype="f32", rows=2048, vocab=128256,
             flat=1.0, masked=0.0, top=5, mix=12),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["adapters", "sample", "logprobs"])
    mix = rng.randrange(1 << 20)
    if kind == "adapters":
        cols = 8 * _log(rng, 16, 864)
        rows = [_log(rng, 64, 6912) for _ in range(rng.choice([1, 1, 2, 3]))]
        rank = rng.choice([8, 16, 16, 32, 64, 128])
        use = rng.choice(["decode", "decode", "prompts"])
        one = rank * (len(rows) * cols + sum(rows))  # an adapter's weights
        most = max(1, min(4096, 1500 * 13824 // (sum(rows) + cols), 2049 * 32 * 18944 // one))
        tokens = _log(rng, 1, min(128, most)) if use == "decode" else _log(rng, min(16, most), most)
        many = max(1, min(40 if use == "decode" else 8, (1 << 24) // one))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), tokens=tokens,
                    run=1 if use == "decode" else _log(rng, 4, 512),
                    adapters=_log(rng, 1, many), rank=rank, cols=cols,
                    sections=" ".join(map(str, rows)), ragged=rng.random() < 0.5,
                    none=rng.choice([0.0, 0.0, 0.2]), mix=mix)
    vocab = _log(rng, 500, 200000)
    most = (512 if kind == "sample" else 2048) * 128256
    rows = _log(rng, 1, max(1, min(2048, most // (2 * vocab))))
    c = dict(kind=kind, dtype=rng.choice(["f32", "f32", "f16", "bf16"]), rows=rows, vocab=vocab,
             flat=rng.choice([0.5, 1.0, 1.0, 1.6]), masked=rng.choice([0.0, 0.0, 0.5, 0.95]), mix=mix)
    if kind == "sample":
        return dict(c, settings=rng.choice(["chat", "mixed", "mixed", "min_p", "top_p", "plain"]))
    return dict(c, top=rng.choice([0, 1, 5, 20]))


# ---- inputs -----------------------------------------------------------------

def _settings(c):
    """(temperature, top_k, top_p, min_p) of each row."""
    r = random.Random(c["mix"])
    out = []
    for _ in range(c["rows"]):
        t, k, p, m = 1.0, 0, 1.0, 0.0
        if c["settings"] == "chat":
            t, k, p = 0.7, 50, 0.95
        elif c["settings"] == "top_p":
            t, p = 1.3, 0.95
        elif c["settings"] == "min_p":
            t, m = r.choice([0.8, 1.0, 1.5]), r.choice([0.02, 0.05, 0.1])
        elif c["settings"] == "mixed":
            t = r.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.4])
            k = r.choice([0, 0, 1, 20, 50, 1000])
            p = r.choice([1.0, 1.0, 0.5, 0.9, 0.99])
            m = r.choice([0.0, 0.0, 0.05, 0.001])
        out.append((t, k, p, m))
    return out


def _rows(c):
    """Rows of each section of the projection."""
    return [int(x) for x in c["sections"].split()]


def _ids(c):
    """The adapter of each token: runs of `run` tokens (prompts), or one by one (decoding)."""
    r = random.Random(c["mix"])
    ids = []
    while len(ids) < c["tokens"]:
        a = -1 if r.random() < c["none"] else r.randrange(c["adapters"])
        ids += [a] * (1 if c["run"] == 1 else r.randint(1, 2 * c["run"]))
    return ids[:c["tokens"]]


def _ranks(c):
    r = random.Random(c["mix"] + 1)
    return [r.randint(1, c["rank"]) if c["ragged"] else c["rank"] for _ in range(c["adapters"])]


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[c["dtype"]]
    st = {"case": c}
    if c["kind"] == "adapters":
        n, k, r, rows, num = c["tokens"], c["cols"], c["rank"], sum(_rows(c)), c["adapters"]
        sec = len(_rows(c))

        def normal(*shape, std=1.0):
            return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)

        st.update(ids=torch.tensor(_ids(c), dtype=torch.int32, device=DEV),
                  ranks=torch.tensor(_ranks(c), dtype=torch.int32, device=DEV),
                  x=normal(n, k), base=normal(n, rows, std=2.0),
                  out=torch.empty(n, rows, dtype=dt, device=DEV),
                  a=normal(num, sec * r, k, std=k ** -0.5), b=normal(num, rows, r, std=r ** -0.5),
                  scales=torch.rand(num, generator=g, device=DEV) + 0.5)
        if own:
            from spbitnet_amd import kernels as K
            st["adapters"] = K.Adapters(st["a"], st["b"], st["scales"], ranks=st["ranks"],
                                        sections=_rows(c))
            size = K.adapters_workspace_size(st["adapters"], n)
            st["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)
        return st
    # logits of a language model: a few likely tokens ahead of a long tail that falls with the
    # logarithm of the rank, ranks spread over the vocabulary, masked ones at minus infinity
    n, v = c["rows"], c["vocab"]
    rank = torch.empty(v, device=DEV)
    rank[torch.randperm(v, generator=g, device=DEV)] = torch.arange(v, device=DEV).float()
    slope = -(1.0 + 0.6 * torch.rand(n, 1, generator=g, device=DEV)) / c["flat"]
    logits = torch.randn(n, v, generator=g, device=DEV)
    logits.mul_(1.2 / c["flat"]).addcmul_(slope, torch.log(1.0 + rank)).add_(6.0)
    if c["masked"]:
        hide = torch.rand(n, v, generator=g, device=DEV) < c["masked"]
        logits.masked_fill_(hide, -math.inf)
        del hide
    st["logits"] = logits.to(dt)
    del logits
    if c["kind"] == "sample":
        s = _settings(c)
        st.update(uniforms=torch.rand(n, generator=g, device=DEV),
                  tokens=torch.empty(n, dtype=torch.int32, device=DEV),
                  logprobs=torch.empty(n, device=DEV),
                  temperature=torch.tensor([x[0] for x in s], device=DEV),
                  top_k=torch.tensor([x[1] for x in s], dtype=torch.int32, device=DEV),
                  top_p=torch.tensor([x[2] for x in s], device=DEV),
                  min_p=torch.tensor([x[3] for x in s], device=DEV))
        if own:
            from spbitnet_amd import kernels as K
            st["sampling"] = K.Sampling(st["temperature"], st["top_k"], st["top_p"], st["min_p"])
            size = K.sample_workspace_size(n, v)
            st["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)
        return st
    # the tokens that were sampled or stand in the prompt: likely ones mostly
    noise = torch.rand(n, 64, generator=g, device=DEV)
    pick = torch.randint(0, v, (n, 64), generator=g, device=DEV)
    score = torch.gather(st["logits"].float(), 1, pick) - torch.log(-torch.log(noise))
    tokens = torch.gather(pick, 1, score.argmax(1, keepdim=True))[:, 0]
    st.update(tokens=tokens.to(torch.int32), logprobs=torch.empty(n, device=DEV),
              top_ids=torch.empty(n, c["top"], dtype=torch.int32, device=DEV),
              top_logprobs=torch.empty(n, c["top"], device=DEV))
    if own:
        from spbitnet_amd import kernels as K
        size = K.token_logprobs_workspace_size(n, v, c["top"])
        st["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)
    return st


# ---- one pass ---------------------------------------------------------------

def _plain_adapters(st):
    c, r, parts = st["case"], st["case"]["rank"], _rows(st["case"])
    sec = len(parts)
    x, ids, num = st["x"].float(), st["ids"].long(), c["adapters"]
    cut = [sum(parts[:s]) for s in range(sec + 1)]
    live = torch.arange(r, device=DEV) < st["ranks"][:, None]  # [adapter][rank]
    total = st["base"].float()
    if c["tokens"] * sec * r * (c["cols"] + sum(parts)) <= 1 << 28:  # each token's own weights
        at = ids.clamp_min(0)
        h = torch.matmul(st["a"][at].float(), x[:, :, None])[:, :, 0].unflatten(1, (sec, r))
        h = h * live[at][:, None] * torch.where(ids >= 0, st["scales"][at], 0.0)[:, None, None]
        w = st["b"][at].float()
        for s in range(sec):
            rows = slice(cut[s], cut[s + 1])
            total[:, rows] += torch.matmul(w[:, rows], h[:, s, :, None])[:, :, 0]
    else:  # all tokens through each adapter, those of others at zero
        for a in range(num):
            mine = torch.where(ids == a, st["scales"][a], 0.0)[:, None, None]
            h = (x @ st["a"][a].float().T).unflatten(1, (sec, r)) * live[a] * mine
            for s in range(sec):
                rows = slice(cut[s], cut[s + 1])
                total[:, rows] += h[:, s] @ st["b"][a, rows].float().T
    return st["out"].copy_(total)


def _plain_sample(st):
    l, order = st["logits"].float().sort(dim=1, descending=True, stable=True)
    v, t, k = l.shape[1], st["temperature"].double()[:, None], st["top_k"].long()[:, None]
    place = torch.arange(v, device=DEV)
    # sums in 64 bits: a border between two tokens is one of 128 thousand
    w = torch.where(t > 0, ((l - l[:, :1].double()) / t.clamp_min(1e-30)).exp(), (place == 0).double())
    w.masked_fill_((k > 0) & (place >= k), 0.0)
    before = w.cumsum(1) - w
    p = st["top_p"].double()[:, None]
    w.masked_fill_((p < 1) & (before >= p * w.sum(1, keepdim=True)), 0.0)
    w.masked_fill_(w < st["min_p"].double()[:, None], 0.0)
    upto = w.cumsum(1)
    at = (upto <= st["uniforms"].double()[:, None] * upto[:, -1:]).sum(1, keepdim=True)
    st["tokens"].copy_(torch.gather(order, 1, at)[:, 0])
    st["logprobs"].copy_((torch.gather(w, 1, at) / upto[:, -1:]).log()[:, 0])
    return {"tokens": st["tokens"], "logprobs": st["logprobs"]}


def _plain_logprobs(st):
    l, n = st["logits"].float(), st["case"]["top"]
    top = l.amax(1, keepdim=True)
    norm = (l - top).exp_().sum(1, keepdim=True, dtype=torch.float64).log()

    def logprob(at):
        return (torch.gather(l, 1, at) - top - norm).float()

    st["logprobs"].copy_(logprob(st["tokens"].long()[:, None])[:, 0])
    if n == 0:
        return {"logprobs": st["logprobs"]}
    left = torch.ones_like(l, dtype=torch.bool)
    at = torch.arange(l.shape[1], device=DEV)
    for i in range(n):  # of equal ones the lowest index first
        best = torch.where(left, l, -math.inf).amax(1, keepdim=True)
        best = torch.where(left & (l == best), at, l.shape[1]).amin(1, keepdim=True)
        st["top_ids"][:, i:i + 1] = best
        st["top_logprobs"][:, i:i + 1] = logprob(best)
        left.scatter_(1, best, False)
    return {"logprobs": st["logprobs"], "top_ids": st["top_ids"], "top_logprobs": st["top_logprobs"]}


def run(state):
    st = state
    kind = st["case"]["kind"]
    if own:
        from spbitnet_amd import kernels as K
        if kind == "adapters":
            K.adapters_gpu(st["adapters"], st["ids"], st["x"], st["base"], st["out"],
                           st["workspace"])
            return st["out"]
        if kind == "sample":
            K.sample_gpu(st["logits"], st["uniforms"], st["tokens"], st["sampling"],
                         st["workspace"], logprobs=st["logprobs"])
            return {"tokens": st["tokens"], "logprobs": st["logprobs"]}
        if st["case"]["top"] == 0:
            K.token_logprobs_gpu(st["logits"], st["tokens"], st["logprobs"], st["workspace"])
            return {"logprobs": st["logprobs"]}
        K.token_logprobs_gpu(st["logits"], st["tokens"], st["logprobs"], st["workspace"],
                             top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
        return {"logprobs": st["logprobs"], "top_ids": st["top_ids"],
                "top_logprobs": st["top_logprobs"]}
    if kind == "adapters":
        return _plain_adapters(st)
    return _plain_sample(st) if kind == "sample" else _plain_logprobs(st)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    c = case
    if c["kind"] == "adapters":
        ids, ranks, rows, sec = _ids(c), _ranks(c), sum(_rows(c)), len(_rows(c))
        weights = sum(ranks[a] for a in set(ids) if a >= 0) * (sec * c["cols"] + rows)
        flops = sum(2 * ranks[a] * (sec * c["cols"] + rows) for a in ids if a >= 0)
        x = sum(a >= 0 for a in ids) * c["cols"]
        return {"bytes": 2 * (weights + x + 2 * c["tokens"] * rows) + 4 * c["tokens"]
                + 8 * c["adapters"], "flops": flops}
    size = 4 if c["dtype"] == "f32" else 2
    n, v = c["rows"], c["vocab"]
    if c["kind"] == "sample":
        return {"bytes": n * v * size + 28 * n, "flops": 4 * n * v}
    return {"bytes": n * v * size + 8 * n + 8 * n * c["top"], "flops": 3 * n * v}


# ---- the results in 64 bits -------------------------------------------------

def _exact_token(l, u, temperature, k, p, m):
    """One row's token and its log-probability, from the definition; l float64 [vocab]."""
    value, index = torch.sort(-l, stable=True)
    if temperature <= 0:
        return int(index[0]), 0.0
    w = torch.exp((value[0] - value) / temperature)
    n = len(w) if k <= 0 else min(k, len(w))
    w = w[:n]
    kept = torch.ones(n, dtype=torch.bool, device=DEV)
    if p < 1:
        upto = torch.cumsum(w, 0)
        kept[1:] &= upto[:-1] < p * upto[-1]
    if m > 0:
        kept &= w >= m
    w = w[:int(kept.sum())]
    upto = torch.cumsum(w, 0)
    at = int(torch.nonzero(upto > u * upto[-1])[0, 0])
    return int(index[at]), float(torch.log(w[at]) - torch.log(upto[-1]))


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["kind"] == "adapters":
        out, x = st["base"].double(), st["x"].double()
        ids, ranks = _ids(c), _ranks(c)
        for a in sorted(set(ids) - {-1}):
            at = torch.tensor([t for t, i in enumerate(ids) if i == a], device=DEV)
            row = 0
            for s, many in enumerate(_rows(c)):
                down = st["a"][a, s * c["rank"]:s * c["rank"] + ranks[a]].double()
                up = st["b"][a, row:row + many, :ranks[a]].double()
                delta = torch.mm(torch.mm(x[at], down.t()), up.t()) * float(st["scales"][a])
                out[at, row:row + many] += delta
                row += many
        return out
    if c["kind"] == "sample":
        u = st["uniforms"].double().tolist()
        set32 = zip(st["temperature"].tolist(), st["top_k"].tolist(), st["top_p"].tolist(),
                    st["min_p"].tolist())
        got = [_exact_token(st["logits"][i].double(), u[i], *s) for i, s in enumerate(set32)]
        return {"tokens": torch.tensor([x[0] for x in got], dtype=torch.int32, device=DEV),
                "logprobs": torch.tensor([x[1] for x in got], dtype=torch.float64, device=DEV)}
    n, top = c["rows"], c["top"]
    picked = torch.empty(n, dtype=torch.float64, device=DEV)
    ids = torch.empty(n, top, dtype=torch.int32, device=DEV)
    values = torch.empty(n, top, dtype=torch.float64, device=DEV)
    tokens = st["tokens"].tolist()
    for i in range(n):
        l = st["logits"][i].double()
        l = l - torch.logsumexp(l, 0)
        picked[i] = l[tokens[i]]
        if top:
            at = torch.sort(l, descending=True, stable=True)[1][:top]
            ids[i], values[i] = at, l[at]
    return {"logprobs": picked, "top_ids": ids, "top_logprobs": values} if top else {"logprobs": picked}
