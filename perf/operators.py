"""The operators of a serving step over a paged key / value cache: rotary
positions of a batch of tokens, norms of query and key heads with the rotation,
appending keys and values to the cache's pages with the rotation on the way, and
the attention of the new tokens over the pages.

listed() and draw() give the cases, prepare() what a program holds before the
call, run() one pass, work() what the pass cannot do without and exact() its
result in 64 bits.  run() computes the plain form in elementary torch
operations, or, where `own` is true, calls the framework's operators.

A batch is a packed list of new tokens: sequence s has the tokens
starts[s] .. starts[s + 1] - 1, which are the last ones of its lens[s] cached
positions; position j of sequence s is slot j % page of page table[s][j // page].
Pages are [kv head][slot][head_dim], K and V each in a pool of them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
HALF = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # one decode step of one sequence, the q and k heads of the 2B shape: all latency
        dict(name="rope_1x25x128", kind="rope", dtype="bf16", tokens=1, heads=25, head_dim=128,
             rotary=128, half=False, theta=500000.0, scaling="none", factor=1.0, first=2048),
        # a pass over long prompts, half layout on half of each head, positions
        # scaled for a context 8 times as long
        dict(name="rope_8192x25x128_half", kind="rope", dtype="f16", tokens=8192, heads=25,
             head_dim=128, rotary=64, half=True, theta=10000.0, scaling="yarn", factor=8.0,
             first=24576),
        # 32 sequences decoded together, a model that normalises q and k
        dict(name="qknorm_32x20x5x128", kind="qknorm", dtype="bf16", tokens=32, heads=20,
             kv_heads=5, head_dim=128, rotary=128, half=True, theta=500000.0, scaling="none",
             factor=1.0, first=2048),
        # a prompt of 2048 tokens and an odd one more
        dict(name="qknorm_2049x20x5x128", kind="qknorm", dtype="f16", tokens=2049, heads=20,
             kv_heads=5, head_dim=128, rotary=128, half=False, theta=10000.0, scaling="ntk",
             factor=4.0, first=0),
        # one token of one sequence into the cache
        dict(name="append_b1", kind="append", dtype="bf16", seqs=1, new_lo=1, new_hi=1, chunk=0,
             ctx_lo=2048, ctx_hi=2048, heads=20, kv_heads=5, head_dim=128, page=64, rotary=128,
             half=False, theta=500000.0, scaling="none", factor=1.0, norm=False, mix=1),
        # prompts in chunks of ragged lengths, small pages, q and k normalised on the way
        dict(name="append_b21_chunks", kind="append", dtype="f16", seqs=21, new_lo=1, new_hi=400,
             chunk=0, ctx_lo=0, ctx_hi=2500, heads=20, kv_heads=5, head_dim=128, page=16,
             rotary=128, half=True, theta=500000.0, scaling="none", factor=1.0, norm=True, mix=2),
        # one decode step of one sequence: the smallest attention
        dict(name="attention_b1_ctx2048", kind="attention", dtype="bf16", seqs=1, new_lo=1,
             new_hi=1, chunk=0, ctx_lo=2048, ctx_hi=2048, heads=20, kv_heads=5, head_dim=128,
             page=64, window=0, causal=True, mix=3),
        # one sequence far into a long context
        dict(name="attention_b1_ctx131071", kind="attention", dtype="f16", seqs=1, new_lo=1,
             new_hi=1, chunk=0, ctx_lo=131071, ctx_hi=131071, heads=20, kv_heads=5, head_dim=128,
             page=64, window=0, causal=True, mix=4),
        # 32 sequences decoded together, ragged contexts, small pages
        dict(name="attention_b32_ragged", kind="attention", dtype="bf16", seqs=32, new_lo=1,
             new_hi=1, chunk=0, ctx_lo=100, ctx_hi=8191, heads=20, kv_heads=5, head_dim=128,
             page=16, window=0, causal=True, mix=5),
        # a chunk of a prompt beside 15 decoding sequences in one call
        dict(name="attention_b16_chunk512", kind="attention", dtype="bf16", seqs=16, new_lo=1,
             new_hi=1, chunk=512, ctx_lo=300, ctx_hi=4000, heads=20, kv_heads=5, head_dim=128,
             page=32, window=0, causal=True, mix=6),
        # a few drafted tokens of each sequence checked in one call, a sliding
        # window, seven heads on one, 80 wide, pages of 24 that end inside any tile
        dict(name="attention_b9_draft5_w1000", kind="attention", dtype="f16", seqs=9, new_lo=2,
             new_hi=5, chunk=0, ctx_lo=700, ctx_hi=6000, heads=7, kv_heads=1, head_dim=80,
             page=24, window=1000, causal=True, mix=7),
        # a chunk of 2048 prompt tokens behind 8192 cached ones
        dict(name="attention_chunk2048_ctx8192", kind="attention", dtype="bf16", seqs=1,
             new_lo=2048, new_hi=2048, chunk=0, ctx_lo=8192, ctx_hi=8192, heads=20, kv_heads=5,
             head_dim=128, page=64, window=0, causal=True, mix=8),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "qknorm", "append", "append", "attention", "attention",
                       "attention", "attention"])
    hd = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kvh = rng.choice([1, 2, 4, 5, 8])
    nh = kvh * rng.choice([1, 2, 4, 4, 7, 8])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]))
    if kind != "attention":
        rot = dict(rotary=rng.choice([hd, hd, hd // 2]), half=rng.random() < 0.5,
                   theta=rng.choice([10000.0, 500000.0]),
                   scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                   factor=rng.choice([2.0, 4.0, 8.0]))
    if kind == "rope":
        n = _log(rng, 1, max(1, min(8192, 8192 * 25 * 128 // (nh * hd))))
        return dict(c, tokens=n, heads=nh, head_dim=hd, first=_log(rng, 1, 131072), **rot)
    if kind == "qknorm":
        n = _log(rng, 1, max(1, min(4096, 4096 * 25 * 128 // ((nh + kvh) * hd))))
        return dict(c, tokens=n, heads=nh, kv_heads=kvh, head_dim=hd, first=_log(rng, 1, 131072),
                    **rot)
    c.update(heads=nh, kv_heads=kvh, head_dim=hd, page=rng.choice([8, 16, 16, 24, 32, 64, 128]),
             mix=rng.randrange(1 << 20))
    if kind == "append":
        s = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(2048, 4096 * 25 * 128 // (s * (nh + kvh) * hd))))
        return dict(c, seqs=s, new_lo=1, new_hi=new, chunk=0, ctx_lo=0, ctx_hi=_log(rng, 1, 4096),
                    norm=rng.random() < 0.5, **rot)
    c.update(window=rng.choice([0, 0, 0, 128, 1000]), causal=rng.random() < 0.85)
    use = rng.choice(["decode", "decode", "draft", "chunk", "prompt"])
    most = 20 * 128 * 2048 * 8192  # heads * width * tokens * positions of the largest
    if use == "decode" or use == "draft":
        s = _log(rng, 1, 64)
        new = 1 if use == "decode" else rng.randint(2, 8)
        # the cache is at most that of 32 sequences of 8192 positions of the 2B shape
        ctx = _log(rng, 16, max(16, min(131072, 32 * 8192 * 5 * 128 // (s * kvh * hd))))
        return dict(c, seqs=s, new_lo=1, new_hi=new, chunk=0, ctx_lo=ctx // 8, ctx_hi=ctx)
    if use == "chunk":
        s, ctx = _log(rng, 2, 16), _log(rng, 64, 4096)
        chunk = _log(rng, 16, max(16, min(512, most // (nh * hd * 8 * (ctx + 512)))))
        return dict(c, seqs=s, new_lo=1, new_hi=1, chunk=chunk, ctx_lo=ctx // 8, ctx_hi=ctx)
    s = _log(rng, 1, 4)
    new = _log(rng, 16, max(16, min(2048, 2048 * 20 * 128 // (s * nh * hd))))
    ctx = _log(rng, 1, max(1, min(8192, most // (2 * nh * hd * s * new))))
    return dict(c, seqs=s, new_lo=max(1, new // 4), new_hi=new, chunk=0, ctx_lo=0, ctx_hi=ctx)


def _lengths(c):
    """(new tokens, cached positions with them) of each sequence; the first has the most."""
    r = random.Random(c["mix"])
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    ctx = [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["seqs"])]
    new[0], ctx[0] = c["chunk"] or c["new_hi"], c["ctx_hi"]
    return new, [n + x for n, x in zip(new, ctx)]


def _rope_numbers(c):
    """Angles per position (float64, on the host) and the factor of cosines and sines."""
    rot, theta, s = c["rotary"], c["theta"], c["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    if c["scaling"] == "ntk":
        theta = theta * s ** (rot / (rot - 2))
    f = theta ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        return f / s, 1.0
    if c["scaling"] == "yarn":  # pairs that turn often over the trained 4096 positions keep their speed
        def turn(n):
            return rot * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / s * ramp, 0.1 * math.log(s) + 1.0
    return f, 1.0


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, hd, nh = HALF[c["dtype"]], c["head_dim"], c["heads"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)

    st = {"case": c, "hd": hd, "nh": nh}
    if "rotary" in c:
        f, scale = _rope_numbers(c)
        st.update(inv_freq=f.to(DEV), rope_scale=scale, half=c["half"])
    if c["kind"] in ("qknorm", "append"):
        st.update(qw=torch.rand(hd, generator=g, device=DEV) + 0.5,
                  kw=torch.rand(hd, generator=g, device=DEV) + 0.5)
    if c["kind"] in ("rope", "qknorm"):
        n = c["tokens"]
        st["pos"] = torch.arange(c["first"], c["first"] + n, dtype=torch.int32, device=DEV)
        if c["kind"] == "rope":
            st.update(x=normal(n, nh, hd), y=torch.empty(n, nh, hd, dtype=dt, device=DEV))
        else:  # the heads of a stacked projection: q, k, v of a token side by side
            kvh = c["kv_heads"]
            qkv = normal(n, nh + 2 * kvh, hd, std=2.0)
            st.update(q=qkv[:, :nh], k=qkv[:, nh:nh + kvh],
                      qo=torch.empty(n, nh, hd, dtype=dt, device=DEV),
                      ko=torch.empty(n, kvh, hd, dtype=dt, device=DEV))
        if own:
            _plan(st)
        return st
    kvh, page = c["kv_heads"], c["page"]
    new, lens = _lengths(c)
    n, width = sum(new), max(-(-x // page) for x in lens)
    pool = sum(-(-x // page) for x in lens) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["seqs"], width), -1, dtype=torch.int32)
    at = 0
    where = []
    for s, x in enumerate(lens):
        k = -(-x // page)
        where.append((s, at, k))
        at += k
    table = table.to(DEV)
    for s, at, k in where:
        table[s, :k] = order[at:at + k]
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)
    qkv = normal(n, nh + 2 * kvh, hd, std=1.5)
    st.update(kvh=kvh, page=page, n=n, new_max=max(new), len_max=max(lens), table=table,
              starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
              lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
              k_pages=normal(pool, kvh, page, hd), v_pages=normal(pool, kvh, page, hd),
              q=qkv[:, :nh], k=qkv[:, nh:nh + kvh], v=qkv[:, nh + kvh:],
              qo=torch.empty(n, nh, hd, dtype=dt, device=DEV))
    if own:
        _plan(st)
    return st


def _plan(st):
    """What a program keeps beside its tensors: the descriptors of the rotation, the
    cache and the batch, and the attention's workspace."""
    from spbitnet_amd import kernels as K
    if "inv_freq" in st:
        st["rope"] = K.Rope(st["inv_freq"], scale=st["rope_scale"], interleaved=not st["half"])
    if "table" in st:
        st["cache"] = K.PagedKVCache(st["k_pages"], st["v_pages"])
        st["batch"] = K.PagedBatch(st["starts"], st["lens"], st["table"], st["n"],
                                   max_new=st["new_max"])
    if st["case"]["kind"] == "attention":
        size = K.paged_attention_workspace_size(st["nh"], st["kvh"], st["hd"])
        st["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)


# ---- one pass ---------------------------------------------------------------

def _rotate(x, pos, st):
    """x float32 [n][heads][hd], pos [n]: the pairs of the first rotary elements turned."""
    f = st["inv_freq"]
    r = f.numel()
    angle = pos.double()[:, None] * f  # far positions: an angle in 32 bits is off by far / 2^24
    cos = (angle.cos() * st["rope_scale"]).float()[:, None]
    sin = (angle.sin() * st["rope_scale"]).float()[:, None]
    rest = x[..., 2 * r:]
    if st["half"]:
        a, b = x[..., :r], x[..., r:2 * r]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
    a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
    turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, rest), -1)


def _normed(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _places(st):
    """Sequence, number in its sequence and position of each new token."""
    t = torch.arange(st["n"], device=DEV)
    seq = torch.searchsorted(st["starts"].long(), t, right=True) - 1
    i = t - st["starts"].long()[seq]
    new = (st["starts"][1:] - st["starts"][:-1]).long()
    return seq, i, st["lens"].long()[seq] - new[seq] + i


def _plain_append(st):
    q, k, dt = st["q"].float(), st["k"].float(), st["q"].dtype
    if st["case"]["norm"]:
        q, k = _normed(q, st["qw"]), _normed(k, st["kw"])
    seq, _, pos = _places(st)
    page = st["table"].long()[seq, pos // st["page"]]
    slot = pos % st["page"]
    st["qo"].copy_(_rotate(q, pos, st))
    st["k_pages"][page, :, slot] = _rotate(k, pos, st).to(dt)
    st["v_pages"][page, :, slot] = st["v"]
    return {"q": st["qo"], "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _plain_attention(st):
    c, page, kvh, hd, nh = st["case"], st["page"], st["kvh"], st["hd"], st["nh"]
    group, most, far = nh // kvh, st["new_max"], st["len_max"]
    j = torch.arange(far, device=DEV)
    held = st["table"].long()[:, j // page].clamp_min(0)
    k = st["k_pages"][held, :, j % page].float().permute(0, 2, 1, 3)  # [seq][kv head][position][hd]
    v = st["v_pages"][held, :, j % page].float().permute(0, 2, 1, 3)
    new = (st["starts"][1:] - st["starts"][:-1]).long()
    i = torch.arange(most, device=DEV)
    rows = (st["starts"].long()[:-1, None] + i).clamp_max(st["n"] - 1)
    q = st["q"].float()[rows].unflatten(2, (kvh, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    pos = (st["lens"].long() - new)[:, None] + i  # [seq][new]
    seen = (j < st["lens"][:, None])[:, None].expand(-1, most, -1)
    if c["causal"]:
        seen = seen & (j <= pos[..., None])
    if c["window"]:
        seen = seen & (j > pos[..., None] - c["window"])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(hd ** -0.5).unflatten(2, (group, most))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)  # a row that sees nothing has none
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, most))
    out = torch.where(total > 0, out / total, 0.0)  # [seq][kv head][group][new][hd]
    seq, i, _ = _places(st)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, i]
    return st["qo"].copy_(out)


def run(state):
    st = state
    kind = st["case"]["kind"]
    if own:
        from spbitnet_amd import kernels as K
        if kind == "rope":
            K.rope_tokens_gpu(st["x"], st["y"], st["pos"], st["rope"])
            return st["y"]
        if kind == "qknorm":
            K.qk_norm_rope_gpu(st["q"], st["k"], st["qo"], st["ko"], st["qw"], st["kw"], st["pos"],
                               st["rope"], EPS)
            return {"q": st["qo"], "k": st["ko"]}
        if kind == "append":
            norm = st["case"]["norm"]
            K.paged_append_gpu(st["cache"], st["batch"], st["k"], st["v"], rope=st["rope"],
                               q=st["q"], q_output=st["qo"], q_weight=st["qw"] if norm else None,
                               k_weight=st["kw"] if norm else None, eps=EPS)
            return {"q": st["qo"], "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
        K.paged_attention_gpu(st["cache"], st["batch"], st["q"], st["qo"], st["workspace"],
                              causal=st["case"]["causal"], window=st["case"]["window"])
        return st["qo"]
    if kind == "rope":
        return st["y"].copy_(_rotate(st["x"].float(), st["pos"], st))
    if kind == "qknorm":
        st["qo"].copy_(_rotate(_normed(st["q"].float(), st["qw"]), st["pos"], st))
        st["ko"].copy_(_rotate(_normed(st["k"].float(), st["kw"]), st["pos"], st))
        return {"q": st["qo"], "k": st["ko"]}
    return _plain_append(st) if kind == "append" else _plain_attention(st)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    c = case
    hd, nh = c["head_dim"], c["heads"]
    if c["kind"] == "rope":
        n = c["tokens"]
        return {"bytes": 4 * n * nh * hd + 4 * n + 4 * c["rotary"], "flops": 3 * n * nh * c["rotary"]}
    kvh = c["kv_heads"]
    if c["kind"] == "qknorm":
        n = c["tokens"]
        return {"bytes": 4 * n * (nh + kvh) * hd + 4 * n + 4 * c["rotary"] + 8 * hd,
                "flops": n * (nh + kvh) * (4 * hd + 3 * c["rotary"])}
    new, lens = _lengths(c)
    n, pages = sum(new), sum(-(-x // c["page"]) for x in lens)
    if c["kind"] == "append":
        return {"bytes": 4 * n * (nh + 2 * kvh) * hd + 8 * c["seqs"] + 4 * n,
                "flops": n * (nh + kvh) * ((4 * hd if c["norm"] else 0) + 3 * c["rotary"])}
    keys, pairs = 0, 0
    for a, b in zip(new, lens):
        w = c["window"] or b
        first = max(0, b - a - w + 1)  # the first key that the first new token sees
        keys += b - first
        for p in range(b - a, b):
            pairs += (p + 1 if c["causal"] else b) - max(0, p - w + 1)
    return {"bytes": 4 * n * nh * hd + 4 * keys * kvh * hd + 4 * pages + 8 * c["seqs"],
            "flops": 4 * pairs * nh * hd}


# ---- the results in 64 bits -------------------------------------------------

def _exact_angles(c, positions):
    """cos and sin, with their factor, [position][pair], from the definition of each scaling."""
    d, base, s = c["rotary"], c["theta"], c["factor"]
    speeds, factor = [], 1.0
    for i in range(d // 2):
        if c["scaling"] == "ntk":
            speeds.append((base * s ** (d / (d - 2.0))) ** (-2.0 * i / d))
            continue
        w = base ** (-2.0 * i / d)
        if c["scaling"] == "linear":
            w /= s
        elif c["scaling"] == "yarn":
            edges = [d * math.log(4096.0 / (2 * math.pi * n)) / (2 * math.log(base)) for n in (32, 1)]
            low, high = max(0, math.floor(edges[0])), min(d - 1, math.ceil(edges[1]))
            part = min(1.0, max(0.0, (i - low) / max(1e-3, high - low)))
            w, factor = (1 - part) * w + part * w / s, 1.0 + 0.1 * math.log(s)
        speeds.append(w)
    a = torch.outer(positions.double(), torch.tensor(speeds, dtype=torch.float64, device=DEV))
    return a.cos() * factor, a.sin() * factor


def _exact_turn(c, x, positions):
    cos, sin = (t[:, None] for t in _exact_angles(c, positions))
    y, d = x.clone(), c["rotary"]
    one = slice(0, d // 2) if c["half"] else slice(0, d, 2)
    two = slice(d // 2, d) if c["half"] else slice(1, d, 2)
    y[..., one] = x[..., one] * cos - x[..., two] * sin
    y[..., two] = x[..., two] * cos + x[..., one] * sin
    return y


def _exact_norm(x, w):
    return w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["kind"] == "rope":
        return _exact_turn(c, st["x"].double(), st["pos"])
    if c["kind"] == "qknorm":
        return {"q": _exact_turn(c, _exact_norm(st["q"].double(), st["qw"]), st["pos"]),
                "k": _exact_turn(c, _exact_norm(st["k"].double(), st["kw"]), st["pos"])}
    new, lens = _lengths(c)
    page, hd, kvh = c["page"], c["head_dim"], c["kv_heads"]
    starts = [sum(new[:s]) for s in range(len(new))]
    if c["kind"] == "append":
        q, k, v = (st[m].double() for m in "qkv")
        if c["norm"]:
            q, k = _exact_norm(q, st["qw"]), _exact_norm(k, st["kw"])
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        for s, (a, b) in enumerate(zip(new, lens)):
            rows = slice(starts[s], starts[s] + a)
            at = torch.arange(b - a, b, device=DEV)
            q[rows], k[rows] = _exact_turn(c, q[rows], at), _exact_turn(c, k[rows], at)
            pages = st["table"][s].long()[torch.div(at, page, rounding_mode="floor")]
            kp[pages, :, at % page], vp[pages, :, at % page] = k[rows], v[rows]
        return {"q": q, "k_pages": kp, "v_pages": vp}
    out = torch.zeros(sum(new), c["heads"], hd, dtype=torch.float64, device=DEV)
    for s, (a, b) in enumerate(zip(new, lens)):
        pages = st["table"][s, :-(-b // page)].long()
        q = st["q"][starts[s]:starts[s] + a].double()
        at = torch.arange(b - a, b, device=DEV)[:, None]
        key = torch.arange(b, device=DEV)[None]
        hidden = torch.zeros(a, b, dtype=torch.bool, device=DEV)
        if c["causal"]:
            hidden |= key > at
        if c["window"]:
            hidden |= key <= at - c["window"]
        for h in range(c["heads"]):
            head = h * kvh // c["heads"]
            k = st["k_pages"][pages, head].double().reshape(-1, hd)[:b]
            v = st["v_pages"][pages, head].double().reshape(-1, hd)[:b]
            logits = (q[:, h] @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            out[starts[s]:starts[s] + a, h] = torch.softmax(logits, -1) @ v
    return out
