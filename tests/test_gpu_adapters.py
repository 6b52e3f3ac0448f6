"""Low-rank adapters of many requests beside a shared projection, against 64 bits."""
import numpy as np
import pytest
import torch

from spbitnet_amd import kernels as K
from tests import requests64 as R

pytestmark = pytest.mark.gpu
HALF = {"f16": torch.float16, "bf16": torch.bfloat16}


def make(kind, tokens, cols, sections, rank, num, ids, seed=0, ranks=None, x_std=1.0, a_std=None):
    g = torch.Generator().manual_seed(seed)
    dt, rows = HALF[kind], sum(sections)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(dt).cuda()
    d = dict(a=normal(num, len(sections) * rank, cols, std=a_std or cols ** -0.5),
             b=normal(num, rows, rank, std=rank ** -0.5),
             scales=(torch.rand(num, generator=g) * 2 - 0.5).cuda(),
             ranks=None if ranks is None else torch.tensor(ranks, dtype=torch.int32).cuda(),
             sections=sections)
    if ids is None:
        ids = torch.randint(-1, num, (tokens,), generator=g).tolist()
    d.update(ids=torch.tensor(ids, dtype=torch.int32).cuda(), x=normal(tokens, cols, std=x_std),
             base=normal(tokens, rows, std=2.0))
    return d


def handle(d):
    return K.Adapters(d["a"], d["b"], d["scales"], ranks=d["ranks"], sections=d["sections"])


def workspace(ad, n):
    return torch.full((K.adapters_workspace_size(ad, n),), 0xFF, dtype=torch.uint8, device="cuda")


def close(got, d, rows=None, note=""):
    want, err = R.adapters(d["a"], d["b"], d["scales"], d["ranks"], d["sections"], d["ids"],
                           d["x"], d["base"])
    got = R.f64(got)
    rows = slice(None) if rows is None else rows
    bad = ~(np.abs(got - want) <= err)
    assert not bad[rows].any(), (note, np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], err[bad][:5])


def run(d, out=None, base=None, x=None):
    ad = handle(d)
    n = d["ids"].numel()
    base = d["base"] if base is None else base
    out = torch.full_like(d["base"], float("nan")) if out is None else out
    K.adapters_gpu(ad, d["ids"], d["x"] if x is None else x, base, out, workspace(ad, n))
    torch.cuda.synchronize()
    return out


SHAPES = [
    # tokens, cols, sections, rank, adapters
    (1, 8, (1,), 8, 1),
    (1, 2560, (2560, 640, 640), 16, 3),
    (2, 136, (17, 5), 8, 2),
    (7, 256, (64,), 24, 4),
    (16, 640, (129, 1, 30, 7), 16, 5),
    (17, 1024, (80,), 256, 2),
    (33, 2560, (640,), 64, 40),
    (63, 200, (100, 100), 40, 3),
    (64, 6912, (256,), 32, 7),
    (65, 512, (333,), 8, 70),
    (130, 328, (1000, 24), 48, 3),
    (513, 256, (200,), 16, 9),
    (1100, 640, (130, 70), 32, 2),
]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(gpu, kind, shape):
    d = make(kind, *shape, ids=None, seed=shape[0])
    close(run(d), d)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("ids", ["one", "runs", "alternating", "none", "each", "outside"])
@pytest.mark.parametrize("tokens", [5, 64, 200, 900])
def test_orders_of_ids(gpu, kind, ids, tokens):
    num = 6
    made = {"one": [3] * tokens, "runs": [t // 37 % num for t in range(tokens)],
            "alternating": [t % 2 + 1 for t in range(tokens)], "none": [-1] * tokens,
            "each": [t % num for t in range(tokens)],
            "outside": [(-1, 0, num, 2 ** 31 - 1, -2 ** 31, 5)[t % 6] for t in range(tokens)]}[ids]
    d = make(kind, tokens, 264, (96, 41), 16, num, made, seed=tokens)
    got = run(d)
    close(got, d)
    idle = torch.tensor([not 0 <= i < num for i in made])
    assert torch.equal(got.cpu()[idle].view(torch.int16), d["base"].cpu()[idle].view(torch.int16))
    inplace = d["base"].clone()
    run(d, out=inplace, base=inplace)
    assert torch.equal(inplace, got)


@pytest.mark.parametrize("tokens", [3, 40, 700])
@pytest.mark.parametrize("rank", [8, 16, 24, 64, 200])
def test_ragged_ranks_and_what_is_behind_them(gpu, tokens, rank):
    """Ranks past their range are clamped; what stands behind a rank is not used."""
    ranks = [rank, 0, 1, rank - 1, -5, rank + 9, min(9, rank)]
    d = make("bf16", tokens, 320, (70, 26), rank, len(ranks), None, seed=rank, ranks=ranks)
    clean = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in d.items()}
    for i, r in enumerate(ranks):
        r = min(max(r, 0), rank)
        for s in range(2):
            d["a"][i, s * rank + r:(s + 1) * rank] = float("nan")
        d["b"][i, :, r:] = float("inf")
    got = run(d)
    close(got, clean)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [4, 90])
def test_bad_values_stay_in_their_token(gpu, kind, tokens):
    d = make(kind, tokens, 256, (64, 48), 16, 3, [t % 3 for t in range(tokens)], seed=5)
    want = run(d)
    d["x"][1, 7] = float("nan")
    d["x"][2, 9] = float("inf")
    d["base"][3, 5] = float("nan")
    got = run(d)
    assert not torch.isfinite(got[1]).any() and not torch.isfinite(got[2]).any()
    assert torch.isnan(got[3, 5])
    got[3, 5] = want[3, 5]
    keep = torch.ones(tokens, dtype=torch.bool)
    keep[1] = keep[2] = False
    assert torch.equal(got.cpu()[keep], want.cpu()[keep])


@pytest.mark.parametrize("tokens", [2, 100])
def test_inner_products_past_the_range_of_fp16(gpu, tokens):
    """A x of 10^6 and of 10^-9 beside it: the output is in range again."""
    d = make("f16", tokens, 512, (48,), 16, 2, [t % 2 for t in range(tokens)], seed=3, x_std=200.0,
             a_std=200.0)
    d["b"] *= 1e-4
    d["x"][0] = 2e-7
    close(run(d), d)


@pytest.mark.parametrize("tokens", [3, 70])
def test_strides_and_alignment(gpu, tokens):
    """Parts of wider tensors, rows that begin at odd elements, a pool with gaps."""
    d = make("bf16", tokens, 200, (51, 30), 16, 4, None, seed=9)
    wide = torch.full((4, 40, 240), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:35, 8:208] = d["a"]
    d["a"] = wide[:, 3:35, 8:208]
    wide = torch.full((4, 90, 32), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:83, 8:24] = d["b"]
    d["b"] = wide[:, 2:83, 8:24]
    x = torch.full((tokens, 400), float("nan"), dtype=torch.bfloat16, device="cuda")
    x[:, 16:216] = d["x"]
    big = torch.full((tokens, 97), 7.0, dtype=torch.bfloat16, device="cuda")
    base = torch.full((tokens, 131), float("nan"), dtype=torch.bfloat16, device="cuda")
    base[:, 1:82] = d["base"]
    got = run(d, out=big[:, 3:84], base=base[:, 1:82], x=x[:, 16:216])
    close(got, d)
    assert (big[:, :3] == 7).all() and (big[:, 84:] == 7).all()


def test_rows_behind_and_workspace_ends_stay(gpu):
    d = make("bf16", 70, 256, (64,), 32, 3, None, seed=2)
    ad = handle(d)
    size = K.adapters_workspace_size(ad, 70)
    ws = torch.full((size + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    out = torch.full((80, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    K.adapters_gpu(ad, d["ids"], d["x"], d["base"], out[:70], ws[:size])
    torch.cuda.synchronize()
    close(out[:70], d)
    assert (out[70:] == 7).all() and (ws[size:] == 0x5A).all()


@pytest.mark.parametrize("tokens", [2, 70, 600])
@pytest.mark.parametrize("sections", [(13,), (256, 131), (264, 70)])
def test_ragged_last_rows_leave_the_padding(gpu, tokens, sections):
    """Padded rows whose last section is no multiple of 8: tokens with and without an adapter."""
    d = make("bf16", tokens, 96, sections, 8, 3, [t % 5 - 1 for t in range(tokens)], seed=tokens)
    rows, wide = sum(sections), sum(sections) // 8 * 8 + 16
    base = torch.full((tokens, wide), 7.0, dtype=torch.bfloat16, device="cuda")
    base[:, :rows] = d["base"]
    out = torch.full((tokens, wide), 3.0, dtype=torch.bfloat16, device="cuda")
    run(d, out=out[:, :rows], base=base[:, :rows])
    assert bool((out[:, rows:] == 3.0).all())
    close(out[:, :rows], d)


@pytest.mark.parametrize("cols", [8, 16, 24, 40])
@pytest.mark.parametrize("tokens", [70, 1500])
def test_few_columns(gpu, cols, tokens):
    d = make("f16", tokens, cols, (300, 9), 24, 80, None, seed=cols)
    close(run(d), d)


def test_smaller_batches_in_a_workspace_of_a_larger_one(gpu):
    d = make("bf16", 1000, 512, (64, 64), 64, 5, None, seed=4)
    ad = handle(d)
    ws = workspace(ad, 1000)
    for n in (1, 2, 31, 64, 65, 128, 200, 333, 512, 999, 1000):
        assert K.adapters_workspace_size(ad, n) <= ws.numel()
        out = torch.empty_like(d["base"][:n])
        K.adapters_gpu(ad, d["ids"][:n], d["x"][:n], d["base"][:n], out, ws)
        part = dict(d, ids=d["ids"][:n], x=d["x"][:n], base=d["base"][:n])
        close(out, part, note=n)


def test_repeatable(gpu):
    d = make("bf16", 300, 2560, (640,), 64, 4, None, seed=8)
    first = run(d)
    for _ in range(5):
        assert torch.equal(run(d), first)


def test_weights_past_32_bits(gpu):
    """Adapters 2^31 and more elements into their pool, a token as far into its tensor."""
    cols, rank, rows, num = 256, 8, 64, 3
    step = (1 << 30) + 8
    pool = torch.empty(2 * step + 2 * rank * cols, dtype=torch.bfloat16, device="cuda")
    d = make("bf16", 3, cols, (rows,), rank, num, [2, 1, 0], seed=1)
    a = pool.as_strided((num, rank, cols), (step, cols, 1))
    b = pool.as_strided((num, rows, rank), (step, rank, 1), rank * cols)
    a.copy_(d["a"])
    b.copy_(d["b"])
    d["a"], d["b"] = a, b
    far = torch.empty(2 * step + rows, dtype=torch.bfloat16, device="cuda")
    base = far.as_strided((3, rows), (step, 1))
    base.copy_(d["base"])
    got = run(d, out=base, base=base)
    close(got, d)


def test_graph_reads_ids_ranks_and_weights_anew(gpu):
    d = make("bf16", 40, 512, (96,), 32, 4, None, seed=6, ranks=[32, 8, 17, 32])
    ad = handle(d)
    ws = workspace(ad, 40)
    big = make("bf16", 300, 512, (96,), 32, 4, None, seed=7, ranks=[32, 8, 17, 32])
    big.update(a=d["a"], b=d["b"], scales=d["scales"], ranks=d["ranks"])
    wsb = workspace(ad, 300)
    outs = [torch.empty_like(x["base"]) for x in (d, big)]

    def both():  # two sizes, one after the other
        K.adapters_gpu(ad, d["ids"], d["x"], d["base"], outs[0], ws)
        K.adapters_gpu(ad, big["ids"], big["x"], big["base"], outs[1], wsb)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    g = torch.Generator().manual_seed(11)
    for rep in range(4):
        for x in (d, big):
            x["ids"].copy_(torch.randint(-2, 5, x["ids"].shape, generator=g, dtype=torch.int32))
            x["x"].copy_(torch.randn(x["x"].shape, generator=g))
        d["ranks"].copy_(torch.randint(0, 33, (4,), generator=g, dtype=torch.int32))
        d["a"].copy_(torch.randn(d["a"].shape, generator=g) * 0.05)
        for o in outs:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        close(kept[0], d, note=rep)
        close(kept[1], big, note=rep)
        both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, outs))


def test_two_graphs_share_a_workspace(gpu):
    ds = [make("bf16", n, 512, (96, 32), 32, 4, None, seed=n) for n in (33, 260)]
    ads = [handle(d) for d in ds]
    ws = torch.empty(max(K.adapters_workspace_size(a, d["ids"].numel()) for a, d in zip(ads, ds)),
                     dtype=torch.uint8, device="cuda")
    outs = [torch.empty_like(d["base"]) for d in ds]
    graphs = []
    for d, ad, out in zip(ds, ads, outs):
        K.adapters_gpu(ad, d["ids"], d["x"], d["base"], out, ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.adapters_gpu(ad, d["ids"], d["x"], d["base"], out, ws)
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        outs[i].fill_(float("nan"))
        graphs[i].replay()
        torch.cuda.synchronize()
        close(outs[i], ds[i], note=i)


def test_own_stream(gpu):
    d = make("f16", 50, 1024, (128,), 32, 3, None, seed=12)
    ad, out = handle(d), torch.empty_like(d["base"])
    ws = workspace(ad, 50)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    K.adapters_gpu(ad, d["ids"], d["x"], d["base"], out, ws, stream=s)
    s.synchronize()
    close(out, d)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,rank", [(1, 8), (5, 16), (40, 64), (90, 40), (300, 200), (1100, 16)])
def test_differences_of_near_inner_products(gpu, kind, tokens, rank):
    """Inner products of 24 bits whose last ones differ, each exact in float32, and a B that
    subtracts two of them, exact in float32 too.  fp16 holds them to 2^-22, bf16 as they are,
    and the output is rounded once."""
    dt, num, rows, cols = HALF[kind], 3, rank + 7, 64
    g = torch.Generator().manual_seed(tokens)

    def odd(*shape):  # odd numbers of 7 and 8 bits
        return (torch.randint(32, 112, shape, generator=g) * 2 + 1).double()
    a, x = torch.zeros(num, rank, cols, dtype=torch.float64), torch.zeros(tokens, cols, dtype=torch.float64)
    a[:, :, 3] = odd(num, 1)
    a[:, :, 50] = (odd(num, 1) + 2 * torch.randint(0, 15, (num, rank), generator=g)) / 256
    x[:, 3], x[:, 50] = odd(tokens), odd(tokens) * (torch.randint(0, 2, (tokens,), generator=g) * 2 - 1)
    b = torch.zeros(num, rows, rank, dtype=torch.float64)
    one, two = torch.arange(rows) % rank, (torch.arange(rows) + 1) % rank
    b[:, torch.arange(rows), one] = 1.0 / 256
    b[:, torch.arange(rows), two] = -1.0 / 256
    ids = [t % (num + 1) - 1 if tokens > 1 else 1 for t in range(tokens)]
    h = torch.matmul(a, x.t()).transpose(1, 2) / 256  # [adapter][token][rank]
    at = torch.tensor(ids).clamp_min(0), torch.arange(tokens)
    live = torch.tensor([[float(i >= 0)] for i in ids])
    h1, h2 = h[at][:, one] * live, h[at][:, two] * live
    assert torch.equal(h.float().double(), h) and torch.equal((h1 - h2).float().double(), h1 - h2)
    d = dict(a=a.to(dt).cuda(), b=b.to(dt).cuda(), scales=torch.ones(num).cuda(), ranks=None, sections=(rows,),
             ids=torch.tensor(ids, dtype=torch.int32).cuda(), x=x.to(dt).cuda(),
             base=torch.zeros(tokens, rows, dtype=dt, device="cuda"))
    for name, v in (("a", a), ("b", b), ("x", x)):
        assert torch.equal(d[name].cpu().double(), v), name  # all of it is exact in the type
    want = (h1 - h2).numpy()
    held = (h1.abs() + h2.abs()).numpy() * (2.0 ** -22 if kind == "f16" else 0.0)
    err = held * (1 + R.HALF_STEP[dt]) + R.HALF_STEP[dt] * np.abs(want) + R.SMALLEST[dt]
    got = R.f64(run(d))
    assert (np.abs(got - want) <= err).all(), np.abs(got - want).max()
    assert np.abs(want).max() > 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,rank", [(2, 16), (90, 16), (90, 128)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_an_infinite_inner_product_beside_large_ones(gpu, kind, tokens, rank, bad):
    """The others are past fp16's range and of the other sign: the output is still infinite."""
    d = make(kind, tokens, 64, (40,), rank, 2, [t % 2 for t in range(tokens)], seed=1)
    d["scales"].fill_(1.0)
    d["x"].fill_(1.0)
    d["b"].fill_(0.5)
    d["a"].fill_(-3e4)  # inner products of -1.9e6
    if bad < 0:
        d["a"].fill_(3e4)
    d["a"][1, 5, 9] = bad
    got = run(d)
    other = run(dict(d, ids=torch.zeros_like(d["ids"])))
    assert torch.equal(got[0::2].view(torch.int16), other[0::2].view(torch.int16))
    assert torch.isnan(got[1::2]).all() if bad != bad else bool((got[1::2] == bad).all()), got[1, :4]


@pytest.mark.parametrize("kind,rank", [("bf16", 8), ("f16", 72)])
@pytest.mark.parametrize("tokens", [1024, 1025, 4032, 4033, 8128, 8129, 16384, 16385])
def test_ends_of_the_workspace_where_the_split_changes(gpu, tokens, kind, rank):
    """Tokens of one window more or less than go by 8, 4, 2 and 1 parts, a workspace of just
    the size that is asked for, and the same workspace for fewer of them."""
    d = make(kind, tokens, 16, (24, 9), rank, 3, None, seed=tokens)
    ad = handle(d)
    size, guard = K.adapters_workspace_size(ad, tokens), 1 << 20
    ws = torch.full((size + guard,), 0x5A, dtype=torch.uint8, device="cuda")
    for n in (tokens, 1024, 1000):
        out = torch.full_like(d["base"][:n], float("nan"))
        assert K.adapters_workspace_size(ad, n) <= size
        K.adapters_gpu(ad, d["ids"][:n], d["x"][:n], d["base"][:n], out, ws[:size])
        torch.cuda.synchronize()
        assert bool((ws[size:] == 0x5A).all())
        close(out, dict(d, ids=d["ids"][:n], x=d["x"][:n], base=d["base"][:n]), note=n)


@pytest.mark.parametrize("tokens,rank", [(1, 8), (70, 16), (70, 136)])
def test_inner_products_next_to_the_largest_float32(gpu, tokens, rank):
    """Beyond the largest bf16 number and its half step: still finite, and so is the output."""
    d = make("bf16", tokens, 64, (24,), rank, 2, [t % 2 for t in range(tokens)], seed=1)
    d["scales"].fill_(1.0)
    d["base"].zero_()
    d["a"].zero_()
    d["x"].zero_()
    d["a"][:, :, 7], d["x"][:, 7] = 255 / 128 * 2.0 ** 63, 2.0 ** 64
    d["a"][:, :, 40], d["x"][:, 40] = 127 / 64 * 2.0 ** 56, 2.0 ** 63
    d["b"].zero_()
    d["b"][:, :, 3] = 2.0 ** -120
    assert float(R.f64(d["a"])[0, 3] @ R.f64(d["x"])[0]) > 1.998 * 2.0 ** 127
    close(run(d), d)
