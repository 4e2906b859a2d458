"""Plain 64-bit attention and cache helpers for the tests (torch, CPU)."""
from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # unit roundoff


def attend(q, k, v, scale):
    """q [n, h, d], k / v [m, g, d] in float64; query i sees keys j <= i + m - n.

    Returns (output [n, h, d], weights [h, n, m], bound_v, score_bound):
    bound_v = sum_j p_j |v_j| over the seen keys, the size that a relative
    error of the weights has in the output; score_bound [h, n]: the worst
    error of a float32 sum of the d products of a score, times the scale."""
    n, h, d = q.shape
    m, g = k.shape[0], k.shape[1]
    rep = h // g
    see = torch.arange(m)[None] <= torch.arange(n)[:, None] + (m - n)
    out = torch.zeros(n, h, d, dtype=torch.float64)
    size = torch.zeros(n, h, d, dtype=torch.float64)
    w = torch.zeros(h, n, m, dtype=torch.float64)
    sb = torch.zeros(h, n, dtype=torch.float64)
    for head in range(h):
        kk, vv = k[:, head // rep], v[:, head // rep]
        for i in range(n):
            js = see[i].nonzero()[:, 0]
            if not len(js):
                continue
            s = (kk[js] @ q[i, head]) * scale
            p = torch.softmax(s, 0)
            w[head, i, js] = p
            out[i, head] = p @ vv[js]
            size[i, head] = p @ vv[js].abs()
            sb[head, i] = float(((kk[js].abs() @ q[i, head].abs()) * abs(scale)).max()) * d * 2.0 ** -23
    return out, w, size, sb


def out_bound(ref, size, sb, out_dtype, p_unit):
    """Per-element error bound of an attention output: the output's rounding,
    the rounding of the weights to p_unit, and what the scores' float32 sums
    and two exponentials (2^-21) do to the weights and their sum."""
    rel = p_unit + 2.0 * sb.T[..., None] + 2.0 ** -20
    return UNIT[out_dtype] * ref.abs() * (1 + rel) + rel * size + 1e-30


def max_excess(got, ref, bound):
    """Largest |got - ref| / bound; finite places of ref must be finite."""
    got = got.double().cpu()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), "non-finite values"
    return float(((got - ref).abs() / bound).max()) if ref.numel() else 0.0


def make_pool(lens, page, kv_heads, dim, seed, extra=3, device="cuda", scale=3.4 / 127):
    """A shuffled paged cache holding `lens` tokens: (k_codes, v_codes,
    k_scale, v_scale, table) on the device."""
    g = torch.Generator().manual_seed(seed)
    need = [math.ceil(n / page) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need, default=1))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    codes = [torch.randint(-127, 128, (pages, kv_heads, page, dim), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [(0.5 + torch.rand(pages, kv_heads, generator=g)) * scale for _ in range(2)]
    return [t.to(device) for t in (*codes, *scales, table)]


def read(cache, which, table, b, h, n):
    """The first n tokens of (sequence, head) as float64 [n, dim]."""
    codes, scales = cache[which].cpu(), cache[2 + which].cpu()
    page = codes.shape[2]
    ids = table[b, :math.ceil(n / page)].cpu().long()
    x = codes[ids, h].double() * scales[ids, h].double()[:, None, None]
    return x.reshape(-1, codes.shape[-1])[:n]


def cu(lens, device="cuda"):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int64), 0).to(torch.int32) if lens else 0
    return t.to(device)


def i32(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)
