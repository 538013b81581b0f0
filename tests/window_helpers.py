"""Windowed attention over a paged cache by its definition, in 64 bits, and a
cache whose invisible slots are poisoned.

A query at position p of a sequence sees token t when t <= p and (t < sinks or
t > p - window).
"""
import math

import torch

SENTINEL = -1e30


def visible(pos, window, sinks):
    """Tokens that the query at `pos` sees, ascending."""
    first = max(0, pos - window + 1)
    return list(range(min(sinks, first))) + list(range(first, pos + 1))


def seen_by_any(length, queries, window, sinks):
    """Tokens of a sequence that any of its last `queries` positions sees."""
    first = max(0, length - queries - window + 1)
    return list(range(min(sinks, first))) + list(range(first, length))


class PoisonedCache:
    """Paged K/V for sequences of `lens` tokens, of which the last `queries[b]` are
    about to be attended from. Slots that nothing sees hold NaN, pages that nothing
    sees are not there (-1 in the table), unused pages hold NaN."""

    def __init__(self, lens, queries, hkv, d, bs, dtype, window, sinks, seed, device="cuda",
                 slack=3, width=None):
        g = torch.Generator().manual_seed(seed)
        need = [sorted({t // bs for t in seen_by_any(s, q, window, sinks)})
                for s, q in zip(lens, queries)]
        pool = sum(map(len, need)) + slack
        perm = torch.randperm(pool, generator=g).tolist()
        width = width or max(1, max(-(-s // bs) for s in lens))
        k = torch.full((pool, bs, hkv, d), float("nan"))
        v = torch.full((pool, bs, hkv, d), float("nan"))
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, (s, q) in enumerate(zip(lens, queries)):
            for j in need[b]:
                table[b, j] = perm.pop()
            tok = torch.tensor(seen_by_any(s, q, window, sinks), dtype=torch.long)
            if len(tok):
                page, slot = table[b, tok // bs].long(), tok % bs
                k[page, slot] = torch.randn(len(tok), hkv, d, generator=g)
                v[page, slot] = torch.randn(len(tok), hkv, d, generator=g)
        self.k, self.v = k.to(dtype).to(device), v.to(dtype).to(device)
        self.table = table.to(device)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)


def reference(q, k, v, table, lens, bs, window, sinks, starts=None, scale=None):
    """(O, LSE, tolerance of O) of packed queries q [T, Hq, D], on the CPU in 64 bits;
    sequence b has the queries starts[b] .. starts[b+1] - 1, its last positions
    (default: one each). Rows that see nothing: O = 0, LSE = -1e30. Rows outside
    every sequence are NaN.

    The tolerance counts: the output's rounding, half a step of its type; the
    scores' rounding in 32 bits, 2^-24 D sum|q_i k_i| scale each, which moves p by
    that factor and O by twice its product with max|v|; p held as a pair of
    16-bit halves (2^-16 for bf16, less for fp16) and the 32-bit sums.
    """
    q, k, v, table = (x.cpu() for x in (q, k, v, table))
    lens = [int(x) for x in lens]
    starts = list(range(len(lens) + 1)) if starts is None else [int(x) for x in starts]
    t, hq, d = q.shape
    hkv = k.shape[2]
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    o = torch.full((t, hq, d), float("nan"), dtype=torch.float64)
    lse = torch.full((t, hq), float("nan"), dtype=torch.float64)
    tol = torch.zeros(t, hq, d, dtype=torch.float64)
    half = torch.finfo(q.dtype).eps / 2
    for b, s in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            r, pos = starts[b] + i, s - n + i
            if pos < 0:
                o[r], lse[r] = 0.0, SENTINEL
                continue
            tok = torch.tensor(visible(pos, window, sinks))
            page, slot = table[b, tok // bs].long(), tok % bs
            kk, vv = k[page, slot].double(), v[page, slot].double()     # [V, Hkv, D]
            kk, vv = kk.repeat_interleave(g, 1), vv.repeat_interleave(g, 1)
            sc = torch.einsum("hd,vhd->hv", q[r].double(), kk) * scale
            big = torch.einsum("hd,vhd->hv", q[r].double().abs(), kk.abs()).amax(1) * scale
            lse[r] = torch.logsumexp(sc, 1)
            o[r] = torch.einsum("hv,vhd->hd", torch.exp(sc - lse[r][:, None]), vv)
            vmax = vv.abs().amax((0, 2))
            tol[r] = ((2 * d * 2.0 ** -24 * big + 2.0 ** -16) * vmax)[:, None]
    tol = tol + half * o.abs().nan_to_num()
    return o, lse, tol


def assert_matches(got, want, tol, what):
    got = got.double().cpu()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    over = (got - want).abs() - tol
    assert not (over > 0).any(), (f"{what}: {int((over > 0).sum())} of {over.numel()} values over "
                                  f"the tolerance, the worst by {over.max().item():.3e}")


def assert_lse(got, want, d, what):
    """LSE in 32 bits: relative 1e-4 of the framework's parity contract is for
    16-bit partials; here the scores' own rounding, 2^-24 D times their size."""
    got = got.double().cpu()
    empty = want <= -1e29
    assert (got[empty].float() == SENTINEL).all(), f"{what}: sentinel"
    err = (got - want)[~empty].abs()
    bound = d * 2.0 ** -24 * (16 + want[~empty].abs())
    assert not (err > bound).any(), f"{what}: LSE off by {err.max().item():.3e}"
