"""GPU checks of the paged operators at the edges of what a call may hold: what
lies before a window, and arguments at the ends of their ranges.  Tolerances are
those of tests/paged64.py; everything else is compared bit for bit."""
import ctypes
import math

import pytest
import torch

from tests import paged64 as R
from tests.test_gpu_paged import _attend, _k, _randn, _workspace

pytestmark = pytest.mark.gpu

HALF = R.HALF

# seqs, heads, kv heads, window, max_new: every sequence's window begins inside a
# block of 64 keys
BEHIND = {
    "decode": ([(1, 90), (1, 500), (1, 33)], 4, 2, 30, 1),
    "decode, pieces": ([(1, 6000), (1, 5100)], 4, 2, 5000, 1),
    "17 heads on one": ([(1, 500), (1, 2077)], 17, 1, 1000, 1),
    "130 heads on one": ([(3, 300)], 130, 1, 70, 3),
    "decode beside a chunk": ([(1, 1000), (40, 900), (1, 400)], 4, 2, 333, 0),
    "chunk, pieces": ([(1, 4000), (150, 5000)], 2, 1, 3000, 0),
    "drafts": ([(5, 700), (2, 400), (1, 260)], 8, 2, 100, 5),
}


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", BEHIND)
def test_what_lies_before_the_window_has_no_effect(gpu, kind, hd, causal, case):
    """Positions that no row of a sequence sees hold inf and NaN: the same bits as
    with finite ones, in tiles of one token and of several, whole and cut."""
    K = _k()
    seqs, nh, nkv, window, max_new = BEHIND[case]
    assert all(0 < (n - new - window + 1) % 64 for new, n in seqs if n - new >= window)
    b = R.Batch(seqs, 16, nkv, hd, HALF[kind], seed=hd)
    q = _randn(b.rows, nh, hd, dtype=HALF[kind], seed=7)
    clean = _attend(b, q, causal, window, max_new=max_new)
    batch = K.PagedBatch(b.starts, b.lens, b.table, b.rows, max_new=max_new)
    ws = _workspace(nh, nkv, hd)
    for bad in (math.nan, math.inf, -math.inf):
        for s, (new, n) in enumerate(seqs):
            j = torch.arange(max(0, n - new - window + 1))
            page = b.host_table[s].long()[j // 16].cuda()
            b.k[page, :, (j % 16).cuda()] = bad
            b.v[page, :, (j % 16).cuda()] = bad
        out = torch.empty_like(q)
        K.paged_attention_gpu(K.PagedKVCache(b.k, b.v), batch, q, out, ws, causal=causal,
                              window=window)
        same = torch.equal(out, clean)
        assert same, bad


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 25])
@pytest.mark.parametrize("max_new", [0, 1])
def test_windows_up_to_the_largest_int(gpu, kind, causal, window, max_new):
    """No position is before them, also where a sequence has fewer positions than new
    tokens (its first ones are negative: -23 - (2^31 - 1) + 1 does not fit in 32 bits)."""
    b = R.Batch([(40, 17), (3, 0), (1, 90), (200, 150)], 16, 2, 64, HALF[kind], seed=3, padding=1)
    q = _randn(b.rows, 4, 64, dtype=HALF[kind], seed=4)
    out = _attend(b, q, causal, window, max_new=max_new)
    same = torch.equal(out, _attend(b, q, causal, 0, max_new=max_new))
    assert same


@pytest.mark.parametrize("length", [-1, -2 ** 31 + 2, -2 ** 31])
def test_append_skips_sequences_of_negative_length(gpu, length):
    """Their positions are negative, however far the length is below 0: keys, values and
    queries are left out.  (A length of 2^31 - 1 is past the table: the query is rotated,
    key and value have no slot.)"""
    K = _k()
    b = R.Batch([(3, 20), (2, 9)], 16, 2, 64, torch.bfloat16, seed=6)
    k, v = (_randn(5, 2, 64, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    q = _randn(5, 4, 64, dtype=torch.bfloat16, seed=3)
    kp, vp = b.k.clone(), b.v.clone()
    for n, first in ((length, 7.0), (2 ** 31 - 1, None)):
        lens = torch.tensor([n, 9], dtype=torch.int32).cuda()
        qo = torch.full_like(q, 7.0)
        K.paged_append_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, lens, b.table, 5), k, v,
                           q=q, q_output=qo)
        page = int(b.host_table[1, 0])
        kp[page, :, 7:9], vp[page, :, 7:9] = k[3:].transpose(0, 1), v[3:].transpose(0, 1)
        assert torch.equal(b.k, kp) and torch.equal(b.v, vp)
        assert torch.equal(qo[3:], q[3:])
        assert torch.equal(qo[:3], q[:3] if first is None else torch.full_like(q[:3], first))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("seqs", [0, 3])
def test_batches_without_tokens(gpu, kind, seqs):
    """Every operator on a batch of no tokens, as a serving loop may have one."""
    K = _k()
    dt, nh, nkv, hd = HALF[kind], 4, 2, 64
    k, v = (_randn(5, nkv, 16, hd, dtype=dt, seed=s) for s in (1, 2))
    kp, vp = k.clone(), v.clone()
    q, x = (torch.empty(0, h, hd, dtype=dt, device="cuda") for h in (nh, nkv))
    w = torch.ones(hd, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rope = K.Rope.scaled(hd)
    cache = K.PagedKVCache(k, v)
    batch = K.PagedBatch(torch.zeros(seqs + 1, dtype=torch.int32, device="cuda"),
                         torch.full((seqs,), 9, dtype=torch.int32, device="cuda"),
                         torch.zeros(seqs, 1, dtype=torch.int32, device="cuda"), 0)
    K.rope_tokens_gpu(q, q, none, rope)
    K.qk_norm_rope_gpu(q, x, q, x, w, w, none, rope)
    K.paged_append_gpu(cache, batch, x, x)
    K.paged_append_gpu(cache, batch, x, x, rope=rope, q=q, q_output=q, q_weight=w, k_weight=w)
    K.paged_append_gpu(cache, batch, None, None, rope=rope, q=q, q_output=q)
    K.paged_attention_gpu(cache, batch, q, q, _workspace(nh, nkv, hd))
    assert torch.equal(k, kp) and torch.equal(v, vp)


def test_more_tokens_than_a_launch_holds(gpu):
    """2^25 + 3 tokens of one head, and one token of that many heads, against float64."""
    K = _k()
    n, f = (1 << 25) + 3, K.rope_inv_freq(2)[0]
    rope, none = K.Rope(f), torch.zeros(0, dtype=torch.float64, device="cuda")
    x = torch.randn(n, 1, 2, device="cuda").to(torch.float16)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    y = torch.full_like(x, 7.0)
    K.rope_tokens_gpu(x, y, pos, rope)
    R.check_rotated(y, x.double(), R.rotate(x.double(), pos, f.cuda(), 1.0, True), f.cuda(), 1.0, True)
    for far in (0, 1 << 24, n):  # launches meet at 2^24: rows by a call of their own
        rows = slice(max(0, far - 3), min(n, far + 3))
        z = torch.full_like(x[rows], 7.0)
        K.rope_tokens_gpu(x[rows], z, pos[rows], rope)
        assert torch.equal(z, y[rows])
    w = torch.ones(2, device="cuda")
    y.fill_(7.0)
    k, ko = x[:, :0], y[:, :0]
    K.qk_norm_rope_gpu(x, k, y, ko, w, w, None, None)
    want = R.norm(x.double(), w, 1e-5)
    R.check_rotated(y, want, want, none, 1.0, True)
    heads = x.view(1, n, 2)
    z = torch.full_like(heads, 7.0)
    K.rope_tokens_gpu(heads, z, pos[3:4], rope)
    R.check_rotated(z, heads.double(), R.rotate(heads.double(), pos[3:4], f.cuda(), 1.0, True),
                    f.cuda(), 1.0, True)


def test_append_of_more_tokens_than_a_launch_holds(gpu):
    K = _k()
    n, page = (1 << 24) + 5, 1 << 12
    held = -(-n // page)
    k, v = (torch.randn(n, 1, 8, device="cuda").to(torch.bfloat16) for _ in range(2))
    pools = [torch.zeros(held, 1, page, 8, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    batch = K.PagedBatch(torch.tensor([0, n], dtype=torch.int32).cuda(),
                         torch.tensor([n], dtype=torch.int32).cuda(),
                         torch.arange(held, dtype=torch.int32).cuda()[None], n)
    K.paged_append_gpu(K.PagedKVCache(*pools), batch, k, v)
    for got, want in zip(pools, (k, v)):
        got = got.view(-1, 8)
        assert torch.equal(got[:n], want.view(-1, 8)) and not got[n:].any()


def test_what_is_no_descriptor_is_refused(gpu):
    K = _k()
    b = R.Batch([(2, 9)], 16, 2, 64, torch.float16)
    q, x = (_randn(2, h, 64, dtype=torch.float16, seed=h) for h in (4, 2))
    w, pos = torch.ones(64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    rope, cache = K.Rope.scaled(64), K.PagedKVCache(b.k, b.v)
    batch, ws = K.PagedBatch(b.starts, b.lens, b.table, 2), _workspace(4, 2, 64)
    for bad in (None, 1.0, cache):
        with pytest.raises(TypeError, match="rope must be a Rope"):
            K.rope_tokens_gpu(q, q, pos, bad)
    with pytest.raises(TypeError, match="rope must be a Rope"):
        K.qk_norm_rope_gpu(q, x, q, x, w, w, pos, batch)
    with pytest.raises(TypeError, match="rope must be a Rope"):
        K.paged_append_gpu(cache, batch, x, x, rope=rope.inv_freq)
    for bad in (None, rope):
        with pytest.raises(TypeError, match="batch must be a PagedBatch"):
            K.paged_append_gpu(cache, bad, x, x)
        with pytest.raises(TypeError, match="batch must be a PagedBatch"):
            K.paged_attention_gpu(cache, bad, q, q, ws)
        with pytest.raises(TypeError, match="cache must be a PagedKVCache"):
            K.paged_append_gpu(bad, batch, x, x)
        with pytest.raises(TypeError, match="cache must be a PagedKVCache"):
            K.paged_attention_gpu(bad, batch, q, q, ws)


@pytest.mark.parametrize("far", [2 ** 32 + 5, 2 ** 31, -2 ** 32 + 5])
def test_numbers_past_32_bits_are_refused(gpu, far):
    """ctypes cuts them to 32 bits without a word: a window of 2^32 + 5 would be one of 5."""
    K = _k()
    b = R.Batch([(2, 9)], 16, 2, 64, torch.float16)
    q = _randn(2, 4, 64, dtype=torch.float16, seed=1)
    cache, batch, ws = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, 2), _workspace(4, 2, 64)
    with pytest.raises(ValueError, match="window"):
        K.paged_attention_gpu(cache, batch, q, q, ws, window=far)
    with pytest.raises(ctypes.ArgumentError):
        K.paged_attention_gpu(cache, batch, q, q, ws, window=5.5)
    with pytest.raises(ValueError, match="num_tokens"):
        K.PagedBatch(b.starts, b.lens, b.table, far)
    with pytest.raises(ValueError, match="max_new"):
        K.PagedBatch(b.starts, b.lens, b.table, 2, max_new=far)


def test_shapes_past_32_bits_are_refused(gpu):
    """Views of one element: nothing is read or written."""
    K = _k()
    n = 2 ** 32 + 1
    one = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    w, pos = torch.ones(64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    rope = K.Rope.scaled(64)
    for x in (one.expand(n, 1, 64), one.expand(1, n, 64)):
        p = pos.expand(x.shape[0])
        with pytest.raises(ValueError, match="x has shape"):
            K.rope_tokens_gpu(x, x, p, rope)
        with pytest.raises(ValueError, match="q has shape"):
            K.qk_norm_rope_gpu(x, one.expand(x.shape[0], 1, 64), x, one, w, w, p, rope)
    with pytest.raises(ValueError, match="k has shape"):
        K.qk_norm_rope_gpu(one, one.expand(1, n, 64), one, one, w, w, pos, rope)
    for at in range(3):
        shape = [1, 1, 1, 64]
        shape[at] = n
        big = one.view(1, 1, 1, 64).expand(shape)
        with pytest.raises(ValueError, match="k and v has shape"):
            K.PagedKVCache(big, big)
    b = R.Batch([(1, 9)], 16, 1, 64, torch.float16)
    cache, batch, ws = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, 1), _workspace(1, 1, 64)
    q = one.expand(1, n, 64)
    with pytest.raises(ValueError, match="q has shape"):
        K.paged_append_gpu(cache, batch, one, one, q=q, q_output=q)
    with pytest.raises(ValueError, match="q has shape"):
        K.paged_attention_gpu(cache, batch, q, q, ws)
    with pytest.raises(ValueError, match="page_table has shape"):
        K.PagedBatch(b.starts, b.lens, b.table[:, :1].expand(1, n), 1)
    with pytest.raises(ValueError, match="kv_lens has shape"):
        K.PagedBatch(b.starts, b.lens.expand(n), b.table.expand(n, 1), 1)


def test_descriptors_are_fixed(gpu):
    """Their C structs keep the first tensors' pointers and sizes."""
    K = _k()
    b = R.Batch([(2, 9)], 16, 2, 64, torch.float16)
    for x, names in ((K.Rope.scaled(64), ("inv_freq", "scale", "interleaved", "rotary_dim")),
                     (K.PagedKVCache(b.k, b.v), ("k", "v", "head_dim", "num_kv_heads", "dtype")),
                     (K.PagedBatch(b.starts, b.lens, b.table, 2),
                      ("token_starts", "kv_lens", "page_table", "num_tokens", "max_new", "_ptr", "_c", "_fixed"))):
        for name in names:
            before = getattr(x, name, None)
            with pytest.raises(AttributeError, match="cannot be changed"):
                setattr(x, name, 1)
            assert getattr(x, name, None) is before
            with pytest.raises(AttributeError, match="cannot be changed"):
                delattr(x, name)
        for value in (1, 2):  # a program's own
            x.tag = value
            assert x.tag == value
        del x.tag


def test_thousands_of_sequences(gpu):
    """3000 short ones, empty ones among them, and a chunk near the end: every search
    over them goes on past many groups of 64."""
    K = _k()
    seqs = [((1, 2, 0)[s % 3], 2 + s % 37) for s in range(3000)]
    seqs[2900] = (150, 400)
    b = R.Batch(seqs, 16, 1, 64, torch.float16, seed=8, padding=2)
    q = _randn(b.rows, 2, 64, dtype=torch.float16, seed=9)
    _attend(b, q, max_new=150)
    _attend(b, q, window=5, max_new=2)
    x = _randn(b.rows, 2, 64, dtype=torch.float16, seed=10)
    kp, vp = b.k.clone(), b.v.clone()
    K.paged_append_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, b.rows),
                       x[:, :1], x[:, 1:])
    pos = torch.cat([torch.arange(n - new, n) for new, n in seqs])
    page = torch.cat([b.host_table[s].long()[torch.arange(n - new, n) // 16]
                      for s, (new, n) in enumerate(seqs)]).cuda()
    slot = (pos % 16).cuda()
    kp[page, :, slot], vp[page, :, slot] = x[:b.tokens, :1], x[:b.tokens, 1:]
    assert torch.equal(b.k, kp) and torch.equal(b.v, vp)


def test_two_graphs_share_a_workspace(gpu):
    """Replayed in turn, with eager calls between: each finds its own results, whatever
    the other left in the workspace."""
    K = _k()
    ws = _workspace(8, 2, 64)
    parts = []
    for seed, seqs, window in ((1, [(1, 6000), (1, 90)], 1000), (2, [(200, 700), (1, 3000)], 0)):
        b = R.Batch(seqs, 16, 2, 64, torch.bfloat16, seed=seed)
        q = _randn(b.rows, 8, 64, dtype=torch.bfloat16, seed=seed)
        want, out = _attend(b, q, window=window), torch.zeros_like(q)
        cache, batch = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, b.rows)

        def call(q=q, out=out, cache=cache, batch=batch, window=window):
            K.paged_attention_gpu(cache, batch, q, out, ws, window=window)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            call()
        parts.append((b, graph, call, want, out))
    for i in range(4):
        for b, graph, call, want, out in parts:
            out.fill_(7.0)
            graph.replay()
            assert torch.equal(out, want)
            if i % 2:
                out.fill_(7.0)
                call()
                assert torch.equal(out, want)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_kernels_that_max_new_selects_agree(gpu, kind):
    """What max_new says selects tiles of 16 or 128 rows: both results are within the
    tolerance of float64, so they are within twice that of each other."""
    b = R.Batch([(1, 700), (3, 90), (5, 2000)], 16, 2, 128, HALF[kind], seed=1)
    q = _randn(b.rows, 8, 128, dtype=HALF[kind], seed=2)
    _, tol = R.attention(b, q, 128 ** -0.5, True, 0, R.half_step(q.dtype))
    one, other = _attend(b, q, max_new=1), _attend(b, q)
    assert ((one.double() - other.double()).abs() <= 2 * tol).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 40, 130])
@pytest.mark.parametrize("seqs,nh,hd,max_new", [
    ([(150, 700)], 2, 128, 0), ([(7, 300)], 2, 80, 7), ([(1, 4000), (90, 90)], 3, 64, 0),
    ([(40, 17), (33, 200)], 20, 64, 0)])
def test_one_bad_value_reaches_the_rows_that_see_it(gpu, kind, window, seqs, nh, hd, max_new):
    """NaN in V of one position of the last sequence: those rows are NaN, all others have
    the bits that they have without it."""
    K = _k()
    b = R.Batch(seqs, 16, 1, hd, HALF[kind], seed=5)
    q = _randn(b.rows, nh, hd, dtype=HALF[kind], seed=6)
    clean = _attend(b, q, window=window, max_new=max_new)
    cache = K.PagedKVCache(b.k, b.v)
    batch = K.PagedBatch(b.starts, b.lens, b.table, b.rows, max_new=max_new)
    ws, out = _workspace(nh, 1, hd), torch.empty_like(q)
    s, (new, n) = len(seqs) - 1, seqs[-1]
    pos = torch.arange(n - new, n)
    g = torch.Generator().manual_seed(7)
    places = torch.cat([torch.randint(max(0, n - new - window), n, (6,), generator=g),
                        torch.tensor([0, n - 1, n - new, max(0, n - new - window)])])
    for at in places.tolist():
        page = int(b.host_table[s, at // 16])
        before = b.v[page, 0, at % 16].clone()
        b.v[page, 0, at % 16] = math.nan
        K.paged_attention_gpu(cache, batch, q, out, ws, window=window)
        b.v[page, 0, at % 16] = before
        sees = (at <= pos) & ((at > pos - window) | (window == 0))
        rows = torch.zeros(b.rows, dtype=torch.bool)
        rows[b.host_starts[s]:b.host_starts[s + 1]] = sees
        rows = rows.cuda()
        same = torch.equal(out[~rows], clean[~rows])
        assert same and out[rows].isnan().all(), at
