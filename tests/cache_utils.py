"""Caches for the tests, and their operators in 64 bits, one sequence at a time."""

from __future__ import annotations

import math

import torch

LN = 2.0 ** -24  # half a step of fp32, relative


def make_cache(lengths, kv_heads, dim, page, dtype, seed=0, spare=2, room=0, device="cuda"):
    """(k_pages, v_pages, table, lengths): scattered pages, all of them filled with numbers, some
    of the rows that no sequence owns with infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    per = max(1, -(-(max(lengths, default=0) + room) // page))
    total = per * len(lengths) + spare
    k, v = (torch.randn(total, kv_heads, page, dim, generator=g) for _ in range(2))
    table = torch.randperm(total, generator=g)[: per * len(lengths)].reshape(len(lengths), per).int()
    for b, n in enumerate(lengths):  # behind a length: never to be seen
        for s in range(n, per * page):
            for x, bad in ((k, math.nan), (v, math.inf)):
                x[table[b, s // page], :, s % page] = bad
    ns = torch.tensor(lengths, dtype=torch.int32)
    return tuple(t.to(device) for t in (k.to(dtype), v.to(dtype), table, ns))


def roomy(table, page, rows):
    """The same table with room for so many slots that `rows` query rows over them are 3.3 million
    pairs, whatever the lengths: the size at which many rows go to the tensor-core tiles.  The
    entries that no length uses name no page."""
    columns = -(-int(3.3e6 / max(rows, 1)) // page)
    if columns <= table.shape[1]:
        return table
    more = torch.full((table.shape[0], columns - table.shape[1]), -1, dtype=table.dtype, device=table.device)
    return torch.cat([table, more], 1)


def slots_of(pages, table, b, n):
    """The first n slots of sequence b: [H_kv, n, D] in 64 bits."""
    page = pages.shape[2]
    rows = [pages[int(table[b, s // page]), :, s % page] for s in range(n)]
    if not rows:
        return pages.new_zeros(pages.shape[1], 0, pages.shape[3]).double()
    return torch.stack(rows, 1).double()


def attention_64(q, k, v, seen, scale):
    """out, lse and what their errors scale with, for q [H, T, D], k, v [H_kv, n, D], seen [T, n].

    Hidden keys are left out of the sums altogether, so whatever they hold stays out."""
    h, t, d = q.shape
    hk, n = k.shape[:2]
    q = q.double()
    out, lse = torch.zeros(h, t, d).double(), torch.full((h, t), -math.inf).double()
    spread, reach, size, count = (torch.zeros(h, t, *x).double() for x in ((d,), (d,), (), ()))
    for i in range(h):
        kv = i // (h // hk)
        for j in range(t):
            at = seen[j].nonzero().flatten()
            if not len(at):
                continue
            kk, vv = k[kv, at], v[kv, at]
            s = kk @ q[i, j] * scale
            lse[i, j] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[i, j])
            out[i, j] = p @ vv
            spread[i, j] = p @ vv.abs()
            # exp(s - lse) = p / l in the kernel's terms, l >= 1: a subnormal P is off by up to
            # a fixed amount against the largest one, which is exp(max - lse)
            reach[i, j] = torch.exp(s.max() - lse[i, j]) * vv.abs().sum(0)
            # sum of |products| of a score bounds its fp32 error
            size[i, j] = scale * (kk.abs() @ q[i, j].abs()).max()
            count[i, j] = len(at)
    return out, lse, spread, reach, size, count


def score_error(size, dim):
    """Relative error of exp(score): the product's dim sums (the tensor core may cut instead of
    round, twice the half step), the scaling and the subtraction (3 roundings of numbers no larger
    than twice the score's bound), ex2.approx (2 units of 2^-23)."""
    return size * (dim * 2 + 6) * LN + 4 * LN


def out_bound(out, spread, reach, size, count, dtype, dim):
    """Output rounding, P rounding, exponentials (in P and in the sum), fp32 sums over the keys; in
    fp16 a P below 2^-14 is rounded to steps of 2^-24."""
    step = torch.finfo(dtype).eps / 2
    e = (2 * score_error(size, dim) + 2 * count * LN + step)[..., None]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return step * out.abs() + e * spread * (1 + 2 * step) + tiny * reach + tiny


def lse_bound(lse, size, count, dim):
    return score_error(size, dim) + (2 * count + 4) * LN + 4 * LN * lse.abs()
