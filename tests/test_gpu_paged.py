"""GPU checks of the operators of a token batch over a paged cache (rope_tokens,
qk_norm_rope, paged_append and paged_attention of spbitnet_amd.kernels) against
float64, at the sizes, layouts and masks where they can go wrong.  Tolerances are
derived in tests/paged64.py."""
import ctypes
import math

import pytest
import torch

from tests import paged64 as R

pytestmark = pytest.mark.gpu

HALF = R.HALF


def _k():
    from spbitnet_amd import kernels as K
    return K


def _randn(*shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def _workspace(nh, nkv, hd):
    # NaN bits: what the call reads it has written
    n = _k().paged_attention_workspace_size(nh, nkv, hd)
    return torch.full((n,), 255, dtype=torch.uint8, device="cuda")


# ---- rotary positions --------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("n,heads,hd,rot", [
    (1, 25, 128, 128), (1, 1, 2, 2), (3, 2, 6, 4), (5, 3, 10, 2), (33, 7, 80, 80), (33, 7, 80, 40),
    (7, 5, 96, 48), (2049, 3, 64, 64), (1030, 2, 256, 256), (9, 4, 72, 24), (6, 1, 254, 250),
    (1100, 5, 24, 8)])
def test_rope_tokens(gpu, kind, interleaved, n, heads, hd, rot):
    K = _k()
    f, scale = K.rope_inv_freq(rot, 10000.0)
    assert scale == 1.0
    x = _randn(n, heads, hd, dtype=HALF[kind], seed=n + hd)
    pos = torch.arange(n, dtype=torch.int32).cuda() * 37
    y = torch.full_like(x, 7.0)
    K.rope_tokens_gpu(x, y, pos, K.Rope(f, 1.0, interleaved))
    x64 = x.double()
    want = R.rotate(x64, pos, f.cuda(), 1.0, interleaved)
    R.check_rotated(y, x64, want, f.cuda(), 1.0, interleaved)
    K.rope_tokens_gpu(x, x, pos, K.Rope(f, 1.0, interleaved))
    assert torch.equal(x, y)


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0),
                                            ("yarn", 8.0)])
def test_rope_far_positions_and_scalings(gpu, scaling, factor):
    """Positions up to the largest int32: an angle in float32 would be off by whole turns."""
    K = _k()
    f, scale = K.rope_inv_freq(128, 500000.0, scaling=scaling, factor=factor,
                               original_positions=4096)
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1], dtype=torch.int32).cuda()
    x = _randn(6, 3, 128, dtype=torch.float16, seed=3)
    y = torch.empty_like(x)
    K.rope_tokens_gpu(x, y, pos, K.Rope(f, scale, False))
    # float64 itself holds an angle of 2^31 radians to 2^-22
    want = R.rotate(x.double(), pos, f.cuda(), scale, False)
    R.check_rotated(y, x.double(), want, f.cuda(), scale, False)


def test_rope_strides_padding_and_alignment(gpu):
    """A part of a stacked projection, a buffer that is 2-byte aligned only, padding
    tokens left as they were."""
    K = _k()
    f, _ = K.rope_inv_freq(64, 10000.0)
    rope = K.Rope(f, 1.0, True)
    pos = torch.tensor([5, -1, 9, -7, 3], dtype=torch.int32).cuda()
    qkv = _randn(5, 9, 64, dtype=torch.bfloat16, seed=1)
    before = qkv.clone()
    K.rope_tokens_gpu(qkv[:, 2:5], qkv[:, 2:5], pos, rope)
    want = R.rotate(before[:, 2:5].double(), pos, f.cuda(), 1.0, True)
    live = [0, 2, 4]
    R.check_rotated(qkv[live, 2:5], before[live, 2:5].double(), want[live], f.cuda(), 1.0, True)
    assert torch.equal(qkv[[1, 3]], before[[1, 3]])
    assert torch.equal(qkv[:, :2], before[:, :2]) and torch.equal(qkv[:, 5:], before[:, 5:])
    flat = torch.zeros(5 * 3 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    odd = flat[1:].view(5, 3, 64)
    odd.copy_(before[:, 2:5])
    K.rope_tokens_gpu(odd, odd, pos, rope)
    assert torch.equal(odd, qkv[:, 2:5])


def test_rope_empty(gpu):
    K = _k()
    x = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    rope = K.Rope(K.rope_inv_freq(64)[0])
    K.rope_tokens_gpu(x, x, torch.empty(0, dtype=torch.int32, device="cuda"), rope)


def test_rope_matches_the_single_token_entry_point(gpu):
    """spb_rope_bf16 on one token (angles in float32 at a near position)."""
    from spbitnet_amd import _lib
    K = _k()
    x = _randn(1, 25, 128, dtype=torch.bfloat16, seed=9)
    y, z = torch.empty_like(x), x.clone()
    K.rope_tokens_gpu(x, y, torch.tensor([3], dtype=torch.int32).cuda(),
                      K.Rope.scaled(128, 500000.0))
    _lib.check(_lib.load().spb_rope_bf16(z.data_ptr(), 25, 128, 3, 500000.0, None), "rope")
    torch.cuda.synchronize()
    size = R.pair_size(x.double(), torch.empty(64), True)
    assert ((y.double() - z.double()).abs() <= 2 * 2.0 ** -8 * y.double().abs() + 2.0 ** -19 * size).all()


# ---- norms with the rotation ---------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,nh,nkv,hd,rot,interleaved", [
    (1, 20, 5, 128, 128, True), (32, 20, 5, 128, 128, False), (3, 3, 1, 2, 2, True),
    (17, 7, 1, 80, 40, False), (1025, 4, 2, 64, 32, True), (5, 2, 2, 254, 254, False),
    (4, 4, 0, 96, 96, True), (1100, 2, 1, 256, 128, False), (2, 0, 3, 72, 72, False)])
def test_qk_norm_rope(gpu, kind, n, nh, nkv, hd, rot, interleaved):
    K = _k()
    dt = HALF[kind]
    f = K.rope_inv_freq(rot, 10000.0)[0]
    qkv = _randn(n, nh + 2 * nkv, hd, dtype=dt, seed=hd + n, std=3.0)
    q, k = qkv[:, :nh], qkv[:, nh:nh + nkv]
    qw, kw = (torch.rand(hd, generator=torch.Generator().manual_seed(s)).cuda() + 0.5 for s in (1, 2))
    pos = (torch.arange(n, dtype=torch.int32) * 11 + 5).cuda()
    qo = torch.empty(n, nh, hd, dtype=dt, device="cuda")
    ko = torch.empty(n, nkv, hd, dtype=dt, device="cuda")
    K.qk_norm_rope_gpu(q, k, qo, ko, qw, kw, pos, K.Rope(f, 1.0, interleaved), 1e-5)
    for x, o, w in ((q, qo, qw), (k, ko, kw)):
        y = R.norm(x.double(), w, 1e-5)
        want = R.rotate(y, pos, f.cuda(), 1.0, interleaved)
        # the mean over hd squares in float32: hd / 2 roundings of 2^-24 behind the root
        R.check_rotated(o, y, want, f.cuda(), 1.0, interleaved, 2.0 ** -20 + hd * 2.0 ** -25)
    only, _ = torch.empty_like(qo), torch.empty_like(ko)
    K.qk_norm_rope_gpu(q, k, only, _, qw, kw, None, None, 1e-5)
    none = torch.zeros(0, dtype=torch.float64, device="cuda")
    y = R.norm(q.double(), qw, 1e-5)
    R.check_rotated(only, y, y, none, 1.0, True, 2.0 ** -20 + hd * 2.0 ** -25)
    K.qk_norm_rope_gpu(q, k, q, k, qw, kw, pos, K.Rope(f, 1.0, interleaved), 1e-5)
    assert torch.equal(q, qo) and torch.equal(k, ko)


def test_qk_norm_of_zeros(gpu):
    """A head of zeros stays zeros (eps under the root), with eps 0 it is NaN as the formula."""
    K = _k()
    x = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    w = torch.ones(64, device="cuda")
    y, z = torch.ones_like(x), torch.ones_like(x)
    K.qk_norm_rope_gpu(x, x, y, z, w, w, None, None, 1e-5)
    assert (y == 0).all() and (z == 0).all()
    K.qk_norm_rope_gpu(x, x, y, z, w, w, None, None, 0.0)
    assert y.isnan().all()


# ---- appending to pages ----------------------------------------------------------

SEQS = {
    "one": [(1, 1)],
    "decode": [(1, 77), (1, 1), (1, 130), (1, 16)],
    "chunks": [(40, 100), (0, 50), (3, 3), (1, 65), (0, 0), (17, 33)],
    "many": [(1 + s % 3, 5 + s) for s in range(70)],
}


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("seqs,page,nh,nkv,hd,rot,interleaved,normed,token_major", [
    ("one", 64, 20, 5, 128, 128, True, False, False),
    ("decode", 16, 20, 5, 128, 128, False, True, False),
    ("chunks", 24, 7, 1, 80, 40, False, True, True),
    ("chunks", 1, 3, 3, 64, 64, True, False, False),
    ("many", 7, 8, 2, 96, 96, False, False, True),
    ("many", 128, 2, 1, 256, 128, True, True, False),
    ("chunks", 16, 4, 2, 8, 2, True, True, False)])
def test_paged_append(gpu, kind, seqs, page, nh, nkv, hd, rot, interleaved, normed, token_major):
    K = _k()
    dt = HALF[kind]
    b = R.Batch(SEQS[seqs], page, nkv, hd, dt, seed=page, padding=4, token_major=token_major)
    f = K.rope_inv_freq(rot, 500000.0)[0]
    qkv = _randn(b.rows, nh + 2 * nkv, hd, dtype=dt, seed=hd, std=2.0)
    q, k, v = qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:]
    qw, kw = (torch.rand(hd, generator=torch.Generator().manual_seed(s)).cuda() + 0.5 for s in (1, 2))
    qo = torch.full((b.rows, nh, hd), 7.0, dtype=dt, device="cuda")
    kp, vp = b.k.clone(), b.v.clone()  # clone keeps the strides
    cache, batch = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, b.rows)
    w = dict(q_weight=qw, k_weight=kw) if normed else {}
    K.paged_append_gpu(cache, batch, k, v, rope=K.Rope(f, 1.0, interleaved), q=q, q_output=qo, **w)
    pos = torch.cat([torch.arange(n - new, n) for new, n in b.seqs]).cuda()
    t = slice(0, b.tokens)
    f32 = 2.0 ** -20 + hd * 2.0 ** -25
    q64, k64 = q[t].double(), k[t].double()
    if normed:
        q64, k64 = R.norm(q64, qw, 1e-5), R.norm(k64, kw, 1e-5)
    R.check_rotated(qo[t], q64, R.rotate(q64, pos, f.cuda(), 1.0, interleaved), f.cuda(), 1.0,
                    interleaved, f32)
    assert (qo[b.tokens:] == 7.0).all()  # rows behind the last sequence
    page_of = torch.cat([b.host_table[s].long()[torch.arange(n - new, n) // page]
                         for s, (new, n) in enumerate(b.seqs)]).cuda()
    slot = pos % page
    R.check_rotated(b.k[page_of, :, slot], k64, R.rotate(k64, pos, f.cuda(), 1.0, interleaved),
                    f.cuda(), 1.0, interleaved, f32)
    assert torch.equal(b.v[page_of, :, slot], v[t])
    kp[page_of, :, slot] = b.k[page_of, :, slot]
    vp[page_of, :, slot] = b.v[page_of, :, slot]
    assert torch.equal(b.k, kp) and torch.equal(b.v, vp)  # nothing else was written


def test_append_without_queries_or_rotation(gpu):
    K = _k()
    b = R.Batch([(2, 9), (5, 5)], 4, 2, 64, torch.float16, seed=2)
    k, v = (_randn(7, 2, 64, dtype=torch.float16, seed=s) for s in (1, 2))
    cache, batch = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, 7)
    K.paged_append_gpu(cache, batch, k, v)
    for s, (new, n) in enumerate(b.seqs):
        r = slice(b.host_starts[s], b.host_starts[s] + new)
        assert torch.equal(b.gathered(b.k, s)[:, n - new:], k[r].double().transpose(0, 1))
        assert torch.equal(b.gathered(b.v, s)[:, n - new:], v[r].double().transpose(0, 1))
    # queries only: the pages stay
    kp = b.k.clone()
    q = _randn(7, 4, 64, dtype=torch.float16, seed=5)
    qo = torch.empty_like(q)
    f = K.rope_inv_freq(64)[0]
    K.paged_append_gpu(cache, batch, None, None, rope=K.Rope(f), q=q, q_output=qo)
    pos = torch.cat([torch.arange(n - new, n) for new, n in b.seqs]).cuda()
    R.check_rotated(qo, q.double(), R.rotate(q.double(), pos, f.cuda(), 1.0, True), f.cuda(), 1.0, True)
    assert torch.equal(b.k, kp)


def test_append_skips_what_has_no_slot(gpu):
    """Bad page ids, positions past the table and negative positions drop the
    key and value; a negative position leaves the query as well."""
    K = _k()
    page, hd = 4, 64
    b = R.Batch([(3, 10), (2, 8), (4, 2), (2, 12)], page, 1, hd, torch.bfloat16, seed=4)
    table = b.table.clone()
    assert table.shape[1] == 3
    table[0, 2] = b.k.shape[0]        # just past the pool: positions 8, 9
    table[1, 1] = -5                  # positions 6, 7
    lens = b.lens.clone()
    lens[3] = 14                      # positions 12, 13 are past the table
    kp, vp = b.k.clone(), b.v.clone()
    n = b.tokens
    k, v, q = (_randn(n, 1, hd, dtype=torch.bfloat16, seed=s) for s in (1, 2, 3))
    qo = torch.full_like(q, 7.0)
    K.paged_append_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, lens, table, n), k, v,
                       q=q, q_output=qo)
    # the only tokens with a slot: sequence 0 position 7, sequence 2 positions 0, 1 (its last two)
    p0, p2 = int(table[0, 1]), int(table[2, 0])
    kp[p0, :, 3], vp[p0, :, 3] = k[0], v[0]
    kp[p2, :, 0], kp[p2, :, 1], vp[p2, :, 0], vp[p2, :, 1] = k[7], k[8], v[7], v[8]
    assert torch.equal(b.k, kp) and torch.equal(b.v, vp)
    want = q.clone()
    want[5:7] = 7.0  # sequence 2's first two tokens are at -2 and -1
    assert torch.equal(qo, want)


# ---- attention ---------------------------------------------------------------------

def _attend(b, q, causal=True, window=0, scale=None, max_new=0, left_out=None, stale=None):
    K = _k()
    nh, hd = q.shape[1], q.shape[2]
    if stale is not None:  # every slot that holds no position
        held = torch.zeros(b.k.shape[0], b.page, dtype=torch.bool)
        for s, (_, n) in enumerate(b.seqs):
            j = torch.arange(max(n, 0))
            held[b.host_table[s].long()[j // b.page], j % b.page] = True
        b.k.masked_fill_(~held.cuda()[:, None, :, None], stale)
        b.v.masked_fill_(~held.cuda()[:, None, :, None], stale)
    out = torch.full_like(q, 7.0)
    K.paged_attention_gpu(K.PagedKVCache(b.k, b.v),
                          K.PagedBatch(b.starts, b.lens, b.table, b.rows, max_new=max_new), q, out,
                          _workspace(nh, b.kvh, hd), scale=scale, causal=causal, window=window)
    want, tol = R.attention(b, q, hd ** -0.5 if scale is None else scale, causal, window,
                            R.half_step(q.dtype), left_out)
    t = slice(0, b.tokens)
    err = (out[t].double() - want[t]).abs()
    assert (err <= tol[t]).all(), float((err / tol[t].clamp_min(1e-30)).max())
    assert (out[b.tokens:] == 7.0).all()
    return out


ATTN = [  # seqs, page, heads, kv heads, head_dim, causal, window, token_major
    ([(1, 1)], 16, 4, 1, 128, True, 0, False),
    ([(1, 2049)], 64, 20, 5, 128, True, 0, False),
    ([(1, 20001)], 64, 20, 5, 128, True, 0, False),
    ([(1, 100), (1, 3000), (1, 1), (1, 64), (1, 65), (1, 777)], 16, 20, 5, 128, True, 0, False),
    ([(1 + s % 2, 3 + 37 * s) for s in range(70)], 16, 4, 2, 64, True, 0, True),
    ([(5, 700), (2, 6000), (0, 10), (3, 3)], 24, 7, 1, 80, True, 1000, False),
    ([(130, 130)], 16, 4, 4, 128, True, 0, False),
    ([(300, 1111), (1, 500), (1, 33), (0, 0), (7, 7)], 32, 20, 5, 128, True, 0, False),
    ([(257, 400)], 7, 3, 1, 96, True, 0, True),
    ([(64, 64), (65, 65), (31, 32), (32, 33)], 1, 2, 2, 64, True, 0, False),
    ([(16, 900)], 100, 4, 1, 72, True, 0, False),
    ([(20, 200), (9, 1000)], 16, 6, 2, 192, True, 50, False),
    ([(33, 500), (1, 999)], 48, 4, 2, 256, True, 0, True),
    ([(50, 300), (4, 9)], 16, 8, 2, 128, False, 0, False),
    ([(50, 300), (4, 9)], 16, 8, 2, 64, False, 20, False),
    ([(12, 40)], 16, 64, 1, 128, True, 0, False),
    ([(1, 5000)], 1000, 64, 1, 64, True, 0, False),
    ([(3, 10)], 16, 5, 5, 8, True, 0, False),
    ([(200, 200)], 16, 4, 2, 128, True, 1, False),
    ([(200, 1000)], 16, 4, 2, 128, True, 1 << 30, False),
    ([(40, 17), (3, 0), (2, 1)], 16, 4, 2, 128, True, 0, False),  # rows before position 0
    ([(40, 17), (3, 0)], 16, 4, 2, 128, False, 5, False),
]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_paged_attention(gpu, kind, case):
    seqs, page, nh, nkv, hd, causal, window, token_major = ATTN[case]
    b = R.Batch(seqs, page, nkv, hd, HALF[kind], seed=case, padding=3, token_major=token_major)
    q = _randn(b.rows, nh, hd, dtype=HALF[kind], seed=case, std=2.0)
    most = max(n for n, _ in seqs)
    a = _attend(b, q, causal, window, max_new=most, stale=math.nan)
    # the number of new tokens not told, or told wrongly, selects another kernel
    c = _attend(b, q, causal, window)
    d = _attend(b, q, causal, window, max_new=1)
    assert torch.equal(a, _attend(b, q, causal, window, max_new=most))  # the same bits each time
    assert c.shape == d.shape


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("scale,std", [(1.0, 1.0), (0.01, 4.0), (4.0, 6.0)])
def test_attention_flat_and_peaked(gpu, kind, scale, std):
    """Scores all alike, and scores thousands apart (the reference of a row moves often)."""
    b = R.Batch([(40, 1500), (1, 2500)], 16, 2, 64, HALF[kind], seed=1)
    b.k.mul_(std)
    q = _randn(b.rows, 4, 64, dtype=HALF[kind], seed=2, std=std)
    _attend(b, q, scale=scale)


def test_attention_rising_scores(gpu):
    """Each key's score above the last one's: every tile moves the reference."""
    b = R.Batch([(1, 3000), (70, 2000)], 16, 1, 64, torch.bfloat16, seed=1)
    for s, (_, n) in enumerate(b.seqs):
        j = torch.arange(n)
        ramp = torch.zeros(n, 64)
        ramp[:, 0] = j.float() / 8
        b.k[b.host_table[s].long()[j // 16].cuda(), 0, (j % 16).cuda()] = ramp.bfloat16().cuda()
    q = torch.zeros(b.rows, 2, 64, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 8.0
    _attend(b, q, scale=1.0)
    q[..., 0] = -8.0
    _attend(b, q, scale=1.0)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_non_finite_values_reach_only_rows_that_see_them(gpu, kind, bad):
    """A later token's key or value has no effect on earlier ones, whatever it holds."""
    dt = HALF[kind]
    K = _k()
    for seqs, at in (([(150, 150)], 77), ([(6, 300)], 296), ([(300, 500)], 333)):
        b = R.Batch(seqs, 16, 1, 128, dt, seed=3)
        q = _randn(b.rows, 2, 128, dtype=dt, seed=4)
        clean = _attend(b, q)
        p, slot = int(b.host_table[0, at // 16]), at % 16
        first = seqs[0][1] - seqs[0][0]
        cut = max(0, at - first)
        b.v[p, 0, slot, 5] = bad
        out = torch.empty_like(q)
        cache, batch = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, b.rows)
        ws = _workspace(2, 1, 128)
        K.paged_attention_gpu(cache, batch, q, out, ws)
        assert torch.equal(out[:cut], clean[:cut])
        hit = out[cut:, :, 5]
        assert (hit.isnan() if math.isnan(bad) else hit == bad).all()
        rest = [d for d in range(128) if d != 5]
        assert torch.equal(out[:, :, rest], clean[:, :, rest])
        b.v[p, 0, slot, 5] = 1.0
        b.k[p, 0, slot, 9] = math.nan
        K.paged_attention_gpu(cache, batch, q, out, ws)
        assert torch.equal(out[:cut], clean[:cut]) and out[cut:].isnan().all()


def test_windowed_rows_do_not_see_old_values(gpu):
    K = _k()
    b = R.Batch([(64, 400)], 16, 1, 64, torch.float16, seed=5)
    q = _randn(b.rows, 2, 64, dtype=torch.float16, seed=6)
    clean = _attend(b, q, window=40)
    at = 336 - 40 + 10  # seen by the first tokens only
    b.v[int(b.host_table[0, at // 16]), 0, at % 16] = math.inf
    out = torch.empty_like(q)
    K.paged_attention_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, 64), q,
                          out, _workspace(2, 1, 64), window=40)
    first = at + 40 - 336  # the first row that does not see it
    assert torch.equal(out[first:], clean[first:])
    assert (out[:first] == math.inf).all()


@pytest.mark.parametrize("new", [1, 20, 100])
def test_bad_pages_are_left_out(gpu, new):
    b = R.Batch([(new, 700), (1, 200)], 16, 2, 128, torch.bfloat16, seed=7)
    q = _randn(b.rows, 4, 128, dtype=torch.bfloat16, seed=8)
    want = R.Batch.gathered
    b.table[0, 3], b.table[0, 20], b.table[1, 12] = -1, b.k.shape[0], 1 << 30
    gone = {0: (3, 20), 1: (12,)}

    def left_out(s, j):
        page = j // 16
        return sum((page == p) for p in gone[s]) > 0
    assert want is R.Batch.gathered
    _attend(b, q, left_out=left_out)


def test_all_pages_bad(gpu):
    K = _k()
    b = R.Batch([(1, 40), (1, 40)], 16, 1, 64, torch.float16, seed=7)
    q = _randn(2, 1, 64, dtype=torch.float16, seed=8)
    b.table[0] = -1
    out = torch.zeros_like(q)
    K.paged_attention_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, 2), q,
                          out, _workspace(1, 1, 64))
    assert out[0].isnan().all() and out[1].isfinite().all()


def test_arrays_out_of_range_stay_inside(gpu):
    """Lengths past the table are cut to it; starts past the batch are cut to it."""
    K = _k()
    b = R.Batch([(1, 48), (2, 32)], 16, 1, 64, torch.float16, seed=9)
    q = _randn(3, 2, 64, dtype=torch.float16, seed=8)
    clean = _attend(b, q)
    lens = b.lens.clone()
    lens[0] = 2 ** 31 - 1  # the table holds 48
    starts = b.starts.clone()
    starts[2] = 1000
    out = torch.empty_like(q)
    K.paged_attention_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(starts, lens, b.table, 3), q, out,
                          _workspace(2, 1, 64))
    assert torch.equal(out, clean)
    lens[0] = -5
    K.paged_attention_gpu(K.PagedKVCache(b.k, b.v), K.PagedBatch(starts, lens, b.table, 3), q, out,
                          _workspace(2, 1, 64))
    assert (out[0] == 0).all() and torch.equal(out[1:], clean[1:])


def test_attention_in_place_strided_and_on_a_stream(gpu):
    K = _k()
    b = R.Batch([(1, 900), (70, 300)], 16, 2, 128, torch.bfloat16, seed=3)
    qkv = _randn(b.rows, 8 + 4, 128, dtype=torch.bfloat16, seed=4)
    q = qkv[:, :8]
    want = _attend(b, q.contiguous())
    cache, batch = K.PagedKVCache(b.k, b.v), K.PagedBatch(b.starts, b.lens, b.table, b.rows)
    before = qkv.clone()
    ws = _workspace(8, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    K.paged_attention_gpu(cache, batch, q, q, ws, stream=side)
    side.synchronize()
    assert torch.equal(q, want) and torch.equal(qkv[:, 8:], before[:, 8:])


def test_long_cache_offsets_pass_32_bits(gpu):
    """Pages past 2^32 bytes and 2^31 elements of the pool."""
    K = _k()
    hd, page, nkv = 128, 64, 8
    per = page * nkv * hd
    pool = (1 << 31) // per + 40
    k = torch.zeros(pool, nkv, page, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    b = R.Batch([(1, 500), (20, 700)], page, nkv, hd, torch.bfloat16, seed=1)
    far = pool - b.k.shape[0]
    k[far:], v[far:] = b.k, b.v
    q = _randn(b.rows, 16, hd, dtype=torch.bfloat16, seed=2)
    want = _attend(b, q)
    table = torch.where(b.table >= 0, b.table + far, b.table)
    out = torch.empty_like(q)
    cache, batch = K.PagedKVCache(k, v), K.PagedBatch(b.starts, b.lens, table, b.rows)
    K.paged_attention_gpu(cache, batch, q, out, _workspace(16, nkv, hd))
    assert torch.equal(out, want)
    new = _randn(b.rows, nkv, hd, dtype=torch.bfloat16, seed=3)
    K.paged_append_gpu(cache, batch, new, new)
    K.paged_append_gpu(K.PagedKVCache(b.k, b.v),
                       K.PagedBatch(b.starts, b.lens, b.table, b.rows), new, new)
    assert torch.equal(k[far:], b.k) and not k[:far].any()


# ---- as a serving program uses them -----------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_prompt_in_chunks_then_decode(gpu, kind):
    """Two prompts in chunks and decoded tokens beside each other through append (with
    norms and the rotation) and attention, against the whole sequences in float64;
    and the separate norm-and-rotation operator gives the same cache."""
    K = _k()
    dt, nh, nkv, hd, page = HALF[kind], 8, 2, 128, 16
    total = [150, 70]
    g = torch.Generator().manual_seed(5)
    x = [torch.randn(n, nh + 2 * nkv, hd, generator=g).to(dt).cuda() for n in total]
    qw, kw = (torch.rand(hd, generator=g).cuda() + 0.5 for _ in range(2))
    f = K.rope_inv_freq(hd, 500000.0)[0]
    rope = K.Rope(f, 1.0, False)
    pool = 20
    kc = torch.full((pool, nkv, page, hd), math.nan, dtype=dt, device="cuda")
    vc = kc.clone()
    kc2, vc2 = kc.clone(), vc.clone()
    table = torch.randperm(pool, generator=g).int()[:20].view(2, 10).cuda()
    cache, cache2 = K.PagedKVCache(kc, vc), K.PagedKVCache(kc2, vc2)
    ws = _workspace(nh, nkv, hd)
    got = [torch.empty(n, nh, hd, dtype=dt, device="cuda") for n in total]
    steps = [(100, 0), (20, 33), (29, 1), (1, 35), (0, 1)]
    at = [0, 0]
    for step in steps:
        rows = torch.cat([x[s][at[s]:at[s] + n] for s, n in enumerate(step)])
        at2 = [a + n for a, n in zip(at, step)]
        batch = K.PagedBatch(torch.tensor([0, step[0], sum(step)], dtype=torch.int32).cuda(),
                             torch.tensor(at2, dtype=torch.int32).cuda(), table, sum(step),
                             max_new=max(step))
        q, k, v = rows[:, :nh], rows[:, nh:nh + nkv], rows[:, nh + nkv:]
        qo, out = (torch.empty(sum(step), nh, hd, dtype=dt, device="cuda") for _ in range(2))
        K.paged_append_gpu(cache, batch, k, v, rope=rope, q=q, q_output=qo, q_weight=qw,
                           k_weight=kw)
        pos = torch.cat([torch.arange(a, b) for a, b in zip(at, at2)]).int().cuda()
        q2, k2 = torch.empty_like(qo), torch.empty(sum(step), nkv, hd, dtype=dt, device="cuda")
        K.qk_norm_rope_gpu(q, k, q2, k2, qw, kw, pos, rope)
        K.paged_append_gpu(cache2, batch, k2, v)
        assert torch.equal(q2, qo)
        K.paged_attention_gpu(cache, batch, qo, out, ws)
        got[0][at[0]:at2[0]], got[1][at[1]:at2[1]] = out[:step[0]], out[step[0]:]
        at = at2
    assert torch.equal(kc.view(torch.int16), kc2.view(torch.int16))
    assert torch.equal(vc.view(torch.int16), vc2.view(torch.int16))
    u = R.half_step(dt)
    for s, n in enumerate(total):
        pos = torch.arange(n).cuda()
        q64 = R.rotate(R.norm(x[s][:, :nh].double(), qw, 1e-5), pos, f.cuda(), 1.0, False)
        k64 = R.rotate(R.norm(x[s][:, nh:nh + nkv].double(), kw, 1e-5), pos, f.cuda(), 1.0, False)
        v64 = x[s][:, nh + nkv:].double()
        for h in range(nh):
            kk, vv = k64[:, h // 4], v64[:, h // 4]
            hide = pos[None] > pos[:, None]
            sc = (q64[:, h] @ kk.T * hd ** -0.5).masked_fill(hide, -math.inf)
            p = torch.softmax(sc, -1)
            # q and k are rounded once each: a score is off by 2 u sum |q k|, a
            # probability by twice that (the quotient), and once by its own rounding
            e = (2 * 2 * u * (q64[:, h].abs() @ kk.abs().T) * hd ** -0.5).masked_fill(hide, 0).amax(-1, keepdim=True)
            tol = (p @ vv.abs()) * ((2 * e).exp() - 1 + u + 2.0 ** -14) + u * (p @ vv).abs() + 2.0 ** -20
            assert ((got[s][:, h].double() - p @ vv).abs() <= tol).all()


def test_decode_matches_the_single_token_operators(gpu):
    """One token, a cache of one page: attention_scores, softmax and attention_output."""
    from spbitnet_amd import _lib
    K, L = _k(), _lib.load()
    nh, nkv, hd, n, size = 20, 5, 128, 700, 1024
    b = R.Batch([(1, n)], size, nkv, hd, torch.bfloat16, seed=1)
    q = _randn(1, nh, hd, dtype=torch.bfloat16, seed=2)
    got = _attend(b, q)
    page = int(b.host_table[0, 0])
    sc = torch.empty(nh, size, device="cuda")
    out = torch.empty_like(q)
    _lib.check(L.spb_attention_scores_bf16(q.data_ptr(), b.k[page].data_ptr(), sc.data_ptr(), nh,
                                           nkv, hd, size, n, hd ** -0.5, None), "scores")
    _lib.check(L.spb_softmax(sc.data_ptr(), nh, size, n, None), "softmax")
    _lib.check(L.spb_attention_output_bf16(sc.data_ptr(), b.v[page].data_ptr(), out.data_ptr(), nh,
                                           nkv, hd, size, n, None), "output")
    torch.cuda.synchronize()
    _, tol = R.attention(b, q, hd ** -0.5, True, 0, 2.0 ** -8)
    assert ((got.double() - out.double()).abs() <= 2 * tol).all()


def test_captured_step_follows_its_arrays(gpu):
    """append and attention in one graph; the program refills lengths, starts and the
    table between replays, with eager calls in between on the same workspace."""
    K = _k()
    dt, nh, nkv, hd, page = torch.bfloat16, 8, 2, 128, 16
    rope = K.Rope.scaled(hd, 10000.0)
    kc = torch.zeros(64, nkv, page, hd, dtype=dt, device="cuda")
    vc = torch.zeros_like(kc)
    cache = K.PagedKVCache(kc, vc)
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()
    lens = torch.tensor([300, 17, 64], dtype=torch.int32).cuda()
    table = torch.randperm(64, generator=torch.Generator().manual_seed(1)).int()[:60].view(3, 20).cuda()
    n = 6
    x = _randn(n, nh + 2 * nkv, hd, dtype=dt, seed=1)
    qo, out = (torch.zeros(n, nh, hd, dtype=dt, device="cuda") for _ in range(2))
    ws = _workspace(nh, nkv, hd)
    batch = K.PagedBatch(starts, lens, table, n)
    kc.normal_()
    vc.normal_()

    def step():
        K.paged_append_gpu(cache, batch, x[:, nh:nh + nkv], x[:, nh + nkv:], rope=rope,
                           q=x[:, :nh], q_output=qo)
        K.paged_attention_gpu(cache, batch, qo, out, ws)
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for i, (st, ln) in enumerate([([0, 1, 2, 3], [301, 18, 65]), ([0, 4, 4, 6], [310, 0, 320]),
                                  ([0, 0, 0, 0], [5, 5, 5]), ([0, 1, 2, 5], [20, 100, 7])]):
        x.copy_(_randn(n, nh + 2 * nkv, hd, dtype=dt, seed=10 + i))
        starts.copy_(torch.tensor(st, dtype=torch.int32))
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        k0, v0 = kc.clone(), vc.clone()
        qo.zero_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in (kc, vc, qo, out)]
        kc.copy_(k0)
        vc.copy_(v0)
        qo.zero_()
        out.zero_()
        step()
        torch.cuda.synchronize()
        for a, c in zip(seen, (kc, vc, qo, out)):
            assert torch.equal(a, c)


def test_two_streams_with_their_own_workspaces(gpu):
    K = _k()
    parts = []
    for seed, seqs in ((1, [(1, 9000)]), (2, [(200, 1500), (1, 4000)])):
        b = R.Batch(seqs, 16, 2, 128, torch.float16, seed=seed)
        q = _randn(b.rows, 8, 128, dtype=torch.float16, seed=seed)
        want = _attend(b, q)
        parts.append((b, q, want, torch.empty_like(q), _workspace(8, 2, 128), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for b, q, want, out, ws, st in parts:
            K.paged_attention_gpu(K.PagedKVCache(b.k, b.v),
                                  K.PagedBatch(b.starts, b.lens, b.table, b.rows), q, out, ws,
                                  stream=st)
    torch.cuda.synchronize()
    for b, q, want, out, ws, st in parts:
        assert torch.equal(out, want)


@pytest.mark.parametrize("seed", range(24))
def test_mixed_batches(gpu, seed):
    """Decoding sequences beside chunks, empty ones and ones shorter than their new
    tokens, over head counts, widths, page sizes and windows."""
    import random
    r = random.Random(seed)
    kind = r.choice(["f16", "bf16"])
    nkv = r.choice([1, 2, 3, 5])
    nh = nkv * r.choice([1, 2, 4, 7, 16, 17])
    hd = r.choice([16, 64, 80, 96, 120, 128, 160, 192, 256])
    page = r.choice([1, 4, 8, 16, 20, 33, 64, 512])
    n = r.choice([1, 3, 10, 64, 65, 130])
    if n >= 64:  # the float64 reference goes head by head
        nh = nkv * r.choice([1, 2])
    seqs = []
    for _ in range(n):
        new = r.choice([0, 1, 1, 1, 2, 5, r.randint(1, 60 if n < 20 else 9)])
        seqs.append((new, r.choice([0, 1, new, new + r.randint(0, 100), r.randint(0, 1200)])))
    if n < 20 and r.random() < 0.7:
        seqs[r.randrange(n)] = (r.randint(50, 300), r.randint(300, 1500))
    if sum(x for x, _ in seqs) == 0:
        seqs[0] = (1, 5)
    b = R.Batch(seqs, page, nkv, hd, HALF[kind], seed=seed, padding=r.choice([0, 2]),
                extra_width=r.choice([0, 5]), token_major=r.random() < 0.3)
    q = _randn(b.rows, nh, hd, dtype=HALF[kind], seed=seed, std=r.choice([0.5, 2.0]))
    _attend(b, q, causal=r.random() < 0.8, window=r.choice([0, 0, 1, 37, 500]),
            max_new=r.choice([0, max(x for x, _ in seqs)]), stale=math.nan)


def test_more_sequences_than_a_wave_beside_a_chunk(gpu):
    """150 sequences, a chunk among them, so that the search passes 64 and 128."""
    seqs = [(1, 10 + 5 * s) for s in range(150)]
    seqs[100] = (90, 700)
    seqs[149] = (70, 70)
    b = R.Batch(seqs, 16, 2, 128, torch.bfloat16, seed=3)
    q = _randn(b.rows, 8, 128, dtype=torch.bfloat16, seed=4)
    _attend(b, q, stale=math.nan)
    _attend(b, q, window=64)


def test_long_ragged_decode_splits(gpu):
    """Lengths from one to tens of thousands in one call: pieces of every kind."""
    seqs = [(1, n) for n in (1, 40000, 63, 64, 65, 30000, 2, 129, 12345, 7)]
    for kind in ("f16", "bf16"):
        b = R.Batch(seqs, 64, 2, 64, HALF[kind], seed=5)
        q = _randn(b.rows, 8, 64, dtype=HALF[kind], seed=6)
        _attend(b, q, max_new=1)
        _attend(b, q, window=5000, max_new=1)


def test_rows_of_a_load_far_apart(gpu):
    """A slot stride past 2^24 elements: the rows of one load have 64-bit offsets."""
    K = _k()
    slot = (1 << 24) + 64
    store = [torch.zeros(8 * slot + 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = (t.as_strided((3, 1, 8, 64), (64 * 8, 64 * 8 * 3, slot, 1)) for t in store)
    b = R.Batch([(1, 20)], 8, 1, 64, torch.bfloat16, seed=5, spare=0)
    k.copy_(b.k)
    v.copy_(b.v)
    q = _randn(1, 2, 64, dtype=torch.bfloat16, seed=6)
    want, out = _attend(b, q), torch.empty_like(q)
    K.paged_attention_gpu(K.PagedKVCache(k, v), K.PagedBatch(b.starts, b.lens, b.table, 1), q, out,
                          _workspace(2, 1, 64))
    assert torch.equal(out, want)
