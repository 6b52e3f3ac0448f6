"""float64 statements of the operators over a paged cache, for their tests, and
batches to run them on."""
import math

import torch

HALF = {"f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """A rounding's largest relative error."""
    return torch.finfo(dtype).eps / 2


def rotate(x, pos, inv_freq, scale, interleaved):
    """x float64 [n][heads][hd]; pos [n]."""
    r = inv_freq.numel()
    a = pos.double()[:, None, None] * inv_freq
    c, s = a.cos() * scale, a.sin() * scale
    y = x.clone()
    i, j = ((slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved
            else (slice(0, r), slice(r, 2 * r)))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def norm(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def pair_size(x, inv_freq, interleaved):
    """Length of each element's pair (its own size past the rotated part)."""
    r = inv_freq.numel()
    y = x.abs().clone()
    i, j = ((slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved
            else (slice(0, r), slice(r, 2 * r)))
    y[..., i] = (x[..., i].square() + x[..., j].square()).sqrt()
    y[..., j] = y[..., i]
    return y


def check_rotated(got, x64, want, inv_freq, scale, interleaved, f32=2.0 ** -20):
    """One rounding to 16 bits, and float32 arithmetic: each of the two products
    and their sum 2^-24, the hardware's sine 2^-23, both relative to the pair
    (2^-20 has room for a norm's square root and product before them)."""
    u = half_step(got.dtype)
    size = pair_size(x64, inv_freq, interleaved) * max(scale, 1.0)
    tiny = torch.finfo(got.dtype).smallest_normal * u
    err = (got.double() - want).abs()
    tol = u * 1.001 * want.abs() + f32 * size + tiny
    assert (err <= tol).all(), float((err / tol).max())


class Batch:
    """Sequences [(new, len)] over a pool with spare pages, a random page order and
    -1 past a sequence's pages; padding rows behind the last sequence."""

    def __init__(self, seqs, page, kv_heads, hd, dtype, seed=0, spare=3, padding=0, extra_width=0,
                 token_major=False, device="cuda"):
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.seqs, self.page, self.kvh, self.hd = seqs, page, kv_heads, hd
        held = [-(-max(n, 0) // page) for _, n in seqs]
        pool = sum(held) + spare
        order = torch.randperm(pool, generator=g).int()
        width = max(held + [1]) + extra_width
        table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        at = 0
        for s, h in enumerate(held):
            table[s, :h] = order[at:at + h]
            at += h
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1]
        self.rows = self.tokens + padding
        self.host_table, self.host_starts = table, starts
        self.table = table.to(device)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=device)
        self.lens = torch.tensor([n for _, n in seqs], dtype=torch.int32, device=device)

        def pages():
            shape = (pool, page, kv_heads, hd) if token_major else (pool, kv_heads, page, hd)
            t = torch.randn(shape, generator=g).to(dtype).to(device)
            return t.transpose(1, 2) if token_major else t
        self.k, self.v = pages(), pages()

    def gathered(self, pages, s):
        """[kv head][position][hd] float64 of sequence s."""
        n = max(self.seqs[s][1], 0)
        j = torch.arange(n)
        p = self.host_table[s].long()[j // self.page] if n else j
        return pages[p.to(pages.device), :, (j % self.page).to(pages.device)].double().permute(1, 0, 2)


def attention(b, q, scale, causal, window, u, left_out=None):
    """float64 result of the batch's rows, and how far a kernel with rounding unit u
    for its probabilities and output may be: u for each probability and for the
    result, scores in float32 (hd products of 2^-24 each, in natural units twice
    for the quotient), float32 sums over the keys.  left_out(s, j): positions in
    bad pages."""
    nh = q.shape[1]
    group = nh // b.kvh
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for s, (new, n) in enumerate(b.seqs):
        if new == 0:
            continue
        rows = slice(b.host_starts[s], b.host_starts[s] + new)
        n = max(n, 0)
        if n == 0:
            continue
        k, v = b.gathered(b.k, s), b.gathered(b.v, s)
        pos = torch.arange(n - new, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        seen = torch.ones(new, n, dtype=torch.bool, device=q.device)
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        if left_out is not None:
            seen &= ~left_out(s, j)
        some = seen.any(-1, keepdim=True)
        for h in range(nh):
            kk, vv, qq = k[h // group], v[h // group], q[rows, h].double()
            sc = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            size = (qq.abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0)
            top = sc.amax(-1, keepdim=True).clamp_min(-1e300)
            p = (sc - top).exp()
            p = torch.where(some, p / p.sum(-1, keepdim=True), torch.zeros_like(p))
            vz = torch.where(seen.any(0)[:, None], vv, torch.zeros_like(vv))  # unseen: anything
            o = p @ vz
            e = 2 * (b.hd + 8) * 2.0 ** -24 * size.amax(-1, keepdim=True) + 2.0 ** -21
            a = p @ vz.abs()
            out[rows, h] = o
            tol[rows, h] = (a * (u + e + (n + b.hd) * 2.0 ** -24) + u * 1.001 * o.abs()
                            + 2.0 ** -24 + n * 2.0 ** -30 * vz.abs().max())
    return out, tol
