"""Cases, plain forms and 64-bit values of the attention and key/value-cache operators.

Five operators that belong together: causal attention over packed prompts
(ops.attention_prefill), an int8 paged cache with one scale per page of tokens
and KV head that is written (ops.kv8_append), read back (ops.kv8_gather),
attended to by the newest tokens (ops.attention_kv8) and shrunk by accumulated
attention weight (ops.kv8_evict).

`own` selects between the framework's operators and plain torch operations in
32 bits that compute the same.  Sequence lengths travel in a case as text
("17,333"); page tables point into a shuffled page pool, as a serving process
has it after a while.
"""
import math

import torch

own = False

QMAX = 127.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# widest padded score matrix (sequences x queries x keys) a drawn prompt case may have, and most cached tokens
MOST_PAIRS = 8192 * 8192
MOST_TOKENS = 64 * 4096


def ints(text):
    return [int(x) for x in str(text).split(",")]


def text(values):
    return ",".join(str(int(v)) for v in values)


def uneven(total, parts, seed):
    """`parts` positive lengths of quite different sizes that add up to `total`, the same for the same seed."""
    import random
    r = random.Random(seed)
    w = [math.exp(r.uniform(-1.5, 1.0)) for _ in range(parts)]
    got = [1 + int((total - parts) * x / sum(w)) for x in w]
    got[got.index(max(got))] += total - sum(got)
    return got


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    h = {"heads": 28, "kv_heads": 4, "dim": 128}
    ragged64 = text(uneven(64 * 4096, 64, 3))
    return [
        # one short text prompt: launch latency
        {"name": "prompt_37", "op": "prefill", "q_lens": "37", "k_lens": "37", "dtype": "bf16", **h},
        # several clips' prompts packed into one call, lengths as they come
        {"name": "prompt_packed", "op": "prefill", "q_lens": "1,17,333,1023,640,97,1500,485",
         "k_lens": "1,17,333,1023,640,97,1500,485", "dtype": "bf16", **h},
        # one multi-camera prompt
        {"name": "prompt_8192", "op": "prefill", "q_lens": "8192", "k_lens": "8192", "dtype": "bf16", **h},
        # a stream's next chunks over cached history, 64-wide heads
        {"name": "chunk_fp16_d64", "op": "prefill", "q_lens": "512,389", "k_lens": "4096,2500", "dtype": "fp16",
         "heads": 16, "kv_heads": 4, "dim": 64},
        # prompts written to the cache, some behind tokens it already holds
        {"name": "append_prompts", "op": "append", "lens": "2048,77,3000,900,1,2166", "starts": "0,0,1000,37,513,250",
         "page": 64, "dtype": "bf16", **h},
        # one decode step's tokens of 64 clips
        {"name": "append_step_64", "op": "append", "lens": text([1] * 64), "starts": text(uneven(64 * 1000, 64, 4)),
         "page": 16, "dtype": "bf16", **h},
        # one clip, a short history: launch latency
        {"name": "decode_300", "op": "decode", "new": 1, "lens": "300", "page": 16, "weights": False, "dtype": "bf16",
         **h},
        # a decode step of 64 clips that keeps the attention totals eviction needs
        {"name": "decode_64_ragged", "op": "decode", "new": 1, "lens": ragged64, "page": 64, "weights": True,
         "dtype": "bf16", **h},
        # one clip with a long history: few rows, a long axis
        {"name": "decode_131072", "op": "decode", "new": 1, "lens": "131072", "page": 64, "weights": False,
         "dtype": "bf16", **h},
        # speculative verify: 8 drafted tokens of each clip
        {"name": "verify_8", "op": "decode", "new": 8, "lens": text(uneven(8 * 4000, 8, 5)), "page": 32,
         "weights": True, "dtype": "fp16", **h},
        # 64 clips brought back to 2048 cached tokens
        {"name": "evict_64_ragged", "op": "evict", "lens": ragged64, "page": 64, "budget": 2048, "sink": 4,
         "recent": 256, "dtype": "bf16", **h},
        # one long clip
        {"name": "evict_32768", "op": "evict", "lens": "32768", "page": 16, "budget": 4096, "sink": 4, "recent": 500,
         "dtype": "bf16", **h},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kv = rng.choice([1, 2, 4, 8])
    c = {"op": rng.choice(["prefill", "prefill", "append", "decode", "decode", "decode", "evict"]),
         "dtype": rng.choice(["bf16", "bf16", "fp16"]), "kv_heads": kv,
         "heads": kv * rng.choice([1, 3, 4, 7] if kv < 8 else [1, 3]), "dim": rng.choice([64, 128, 128])}
    seed = rng.randrange(1 << 30)
    if c["op"] == "prefill":
        while True:
            total = log(2, 8192)
            n = min(total, log(1, 16))
            q = uneven(total, n, seed)
            past = [log(1, 8192) if rng.random() < 0.3 else 0 for _ in q]
            k = [a + b for a, b in zip(q, past)]
            if n * max(q) * max(k) <= MOST_PAIRS:
                break
        return {**c, "q_lens": text(q), "k_lens": text(k)}
    c["page"] = rng.choice([16, 32, 64, 128])
    if c["op"] == "append":
        total = log(1, 8192)
        n = min(total, log(1, 64))
        lens = uneven(total, n, seed)
        return {**c, "lens": text(lens), "starts": text([log(1, 4096) if rng.random() < 0.6 else 0 for _ in lens])}
    n = log(1, 64)
    total = log(max(16, n), MOST_TOKENS * 4 // kv // 8)
    # what the plain form pads to stays within the listed cases' own
    lens = [min(v, max(1, MOST_TOKENS * 4 // kv // n)) for v in uneven(total, n, seed)]
    if c["op"] == "decode":
        return {**c, "lens": text(lens), "new": rng.choice([1, 1, 1, 2, 3, 5, 8, 16]), "weights": rng.random() < 0.5}
    sink, recent = rng.choice([0, 1, 4]), rng.choice([0, 17, 64])
    return {**c, "lens": text(lens), "sink": sink, "recent": recent, "budget": sink + recent + log(1, 4096)}


# --------------------------------------------------------------------------
# states
# --------------------------------------------------------------------------
def offsets(lens, dev):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int64), 0).to(torch.int32)
    return t.to(dev)


def rows_of(lens, dev):
    """Sequence and position in it of each packed row."""
    n = torch.tensor(lens, dtype=torch.int64)
    seq = torch.repeat_interleave(torch.arange(len(lens)), n)
    pos = torch.arange(int(n.sum())) - (torch.cumsum(n, 0) - n)[seq]
    return seq.to(dev), pos.to(dev)


def projected(tokens, heads, kv_heads, dim, dtype, g, dev):
    """A fused q/k/v projection's output [tokens, (heads + 2 kv_heads) * dim]: some query heads sharper than others, a few outlier key channels."""
    x = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g, device=dev)
    x[:, :heads] *= (0.5 + 1.5 * torch.rand(heads, 1, generator=g, device=dev))
    x[:, heads:heads + kv_heads, :: dim // 4] *= 3.0
    return x.to(dtype).view(tokens, -1)


def pool(lens, page, kv_heads, dim, g, dev, spare=0):
    """A paged int8 cache that holds `lens` tokens (and `spare` more pages): codes, scales, page table."""
    need = [-(-n // page) for n in lens]
    width, pages = max(need), sum(need) + spare + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    seq, pos = rows_of(need, dev)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    table[seq, pos] = order[:sum(need)]
    shape = (pages, kv_heads, page, dim)
    codes = [(torch.randn(shape, generator=g, device=dev) * 38.0).round_().clamp_(-127, 127).to(torch.int8)
             for _ in range(2)]
    scales = [(0.8 + 0.4 * torch.rand(pages, kv_heads, generator=g, device=dev)) * (3.4 / QMAX) for _ in range(2)]
    return codes, scales, table, order[sum(need):]


def totals(lens, kv_heads, cap, g, dev):
    """Accumulated attention weights as some tens of decode steps leave them: heavy-tailed, zero past the end."""
    w = torch.rand(len(lens), kv_heads, cap, generator=g, device=dev)
    w = w.mul_(6.0).exp_().mul_(1e-4)
    live = torch.arange(cap, device=dev)[None, :] < torch.tensor(lens, device=dev)[:, None]
    return w * live[:, None, :]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c = dict(case)
    Hq, Hkv, D, dtype = c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    st = {"case": c, "scale": D ** -0.5}
    if c["op"] == "prefill":
        ql, kl = ints(c["q_lens"]), ints(c["k_lens"])
        st["cu_q"], st["q_rows"] = offsets(ql, dev), rows_of(ql, dev)
        st["q_len"], st["k_len"] = torch.tensor(ql, device=dev), torch.tensor(kl, device=dev)
        if ql == kl:
            st["qkv"] = projected(sum(ql), Hq, Hkv, D, dtype, g, dev)
            st["cu_k"], st["k_rows"] = st["cu_q"], st["q_rows"]
        else:  # keys of the history and the chunk together, as the cache gives them back
            st["qkv"] = projected(sum(ql), Hq, 0, D, dtype, g, dev)
            st["kv"] = projected(sum(kl), 0, Hkv, D, dtype, g, dev)
            st["cu_k"], st["k_rows"] = offsets(kl, dev), rows_of(kl, dev)
        st["pad"] = (len(ql), max(ql), max(kl))
        return st
    page, lens = c["page"], ints(c["lens"])
    if c["op"] == "append":
        starts = ints(c["starts"])
        ends = [a + b for a, b in zip(starts, lens)]
        codes, scales, st["table"], _ = pool(ends, page, Hkv, D, g, dev)
        kv = projected(sum(lens), 0, Hkv, D, dtype, g, dev).view(sum(lens), 2, Hkv, D)
        st["kv"], st["cu"], st["rows"] = kv, offsets(lens, dev), rows_of(lens, dev)
        st["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        # the tokens read back: every page the call touches, from its first token on
        first = [a // page * page for a in starts]
        back = [b - a for a, b in zip(first, ends)]
        st["first"] = torch.tensor(first, dtype=torch.int32, device=dev)
        st["cu_back"], st["back"], st["back_rows"] = offsets(back, dev), sum(back), rows_of(back, dev)
        st["blocks"] = max(-(-(b - a) // page) for a, b in zip(first, ends))
    elif c["op"] == "decode":
        T = c["new"]
        codes, scales, st["table"], _ = pool(lens, page, Hkv, D, g, dev)
        cap = st["table"].shape[1] * page
        st["q"] = projected(len(lens) * T, Hq, 0, D, dtype, g, dev).view(len(lens), T, Hq, D)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        if c["weights"]:
            st["weights"] = totals(lens, Hkv, cap, g, dev)
            st["weights_out"] = torch.zeros_like(st["weights"])
    else:
        keep = [min(n, c["budget"]) for n in lens]
        width = -(-c["budget"] // page)
        codes, scales, st["table"], free = pool(lens, page, Hkv, D, g, dev, spare=len(lens) * width)
        st["out_table"] = free[:len(lens) * width].view(len(lens), width).contiguous()
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["weights"] = totals(lens, Hkv, st["table"].shape[1] * page, g, dev)
        st["zero"] = torch.zeros(len(lens), dtype=torch.int32, device=dev)
        st["cu_back"], st["back"], st["back_rows"] = offsets(keep, dev), sum(keep), rows_of(keep, dev)
    st["cache"] = (*codes, *scales)
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def split(st):
    """Query, key and value views of the projections' outputs."""
    c = st["case"]
    Hq, Hkv, D = c["heads"], c["kv_heads"], c["dim"]
    if "kv" in st:
        kv = st["kv"].view(-1, 2 * Hkv, D)
        return st["qkv"].view(-1, Hq, D), kv[:, :Hkv], kv[:, Hkv:]
    x = st["qkv"].view(-1, Hq + 2 * Hkv, D)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


def run(st):
    c = st["case"]
    if not own:
        return {"prefill": plain_prefill, "append": plain_append, "decode": plain_decode, "evict": plain_evict}[c["op"]](st)
    from alpamayo_b200 import ops
    if c["op"] == "prefill":
        q, k, v = split(st)
        return ops.attention_prefill(q, k, v, st["cu_q"], st["cu_k"], st["scale"])
    if c["op"] == "append":
        k, v = st["kv"][:, 0], st["kv"][:, 1]
        ops.kv8_append(k, v, st["cu"], st["starts"], *st["cache"], st["table"])
        return ops.kv8_gather(*st["cache"], st["table"], st["first"], st["cu_back"], st["back"], k.dtype)
    if c["op"] == "decode":
        if not c["weights"]:
            return ops.attention_kv8(st["q"], *st["cache"], st["table"], st["lens"], st["scale"])
        out = ops.attention_kv8(st["q"], *st["cache"], st["table"], st["lens"], st["scale"], st["weights"],
                                st["weights_out"])
        return out, st["weights_out"]
    kept, w, n = ops.kv8_evict(st["weights"], *st["cache"], st["table"], st["lens"], st["out_table"], c["budget"],
                               c["sink"], c["recent"])
    return kept, w, n, ops.kv8_gather(*st["cache"], st["out_table"], st["zero"], st["cu_back"], st["back"],
                                      DTYPES[c["dtype"]])


def softmax_parts(s, hidden):
    """exp(s - row maximum) with hidden places zero, and 1 / row sum (zero for rows that see nothing); s is overwritten."""
    s.masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    s.sub_(m).exp_()
    total = s.sum(-1, keepdim=True)
    return s, torch.where(total > 0, 1.0 / total, torch.zeros_like(total))


def plain_prefill(st):
    c = st["case"]
    q, k, v = split(st)
    Hkv, G, D = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    B, Lq, Lk = st["pad"]
    (qs, qp), (ks, kp) = st["q_rows"], st["k_rows"]
    dev = q.device
    qd = torch.zeros(B, Hkv, G, Lq, D, device=dev)
    qd[qs, :, :, qp] = q.float().view(-1, Hkv, G, D)
    kd = torch.zeros(B, Hkv, Lk, D, device=dev)
    vd = torch.zeros(B, Hkv, Lk, D, device=dev)
    kd[ks, :, kp] = k.float()
    vd[ks, :, kp] = v.float()
    s = torch.matmul(qd.view(B, Hkv, G * Lq, D), kd.transpose(-1, -2)).mul_(st["scale"]).view(B, Hkv, G, Lq, Lk)
    i, j = torch.arange(Lq, device=dev), torch.arange(Lk, device=dev)
    last = i[None, :] + (st["k_len"] - st["q_len"])[:, None]                   # last key each query sees
    p, inv = softmax_parts(s, (j[None, None, :] > last[:, :, None])[:, None, None])
    o = torch.matmul(p.view(B, Hkv, G * Lq, Lk), vd).view(B, Hkv, G, Lq, D) * inv
    return o[qs, :, :, qp].reshape(-1, c["heads"], D).to(q.dtype)


def cached(codes, scales, pages):
    """Values of the pages [..., P] as [..., Hkv, P * page, D]."""
    x = codes[pages].float() * scales[pages][..., None, None]
    x = x.transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1])


def plain_decode(st):
    c = st["case"]
    Hkv, G, D, T = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["new"]
    kc, vc, ksc, vsc = st["cache"]
    pages = st["table"].clamp(min=0).long()
    B = pages.shape[0]
    k, v = cached(kc, ksc, pages), cached(vc, vsc, pages)
    q = st["q"].float().view(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4)
    s = torch.matmul(q.reshape(B, Hkv, T * G, D), k.transpose(-1, -2)).mul_(st["scale"]).view(B, Hkv, T, G, -1)
    j = torch.arange(s.shape[-1], device=s.device)
    n = st["lens"].long()
    last = n[:, None] - T + torch.arange(T, device=s.device)[None, :]
    p, inv = softmax_parts(s, (j[None, None, :] > last[:, :, None])[:, None, :, None])
    o = torch.matmul(p.view(B, Hkv, T * G, -1), v).view(B, Hkv, T, G, D) * inv
    out = o.permute(0, 2, 1, 3, 4).reshape(B, T, c["heads"], D).to(st["q"].dtype)
    if not c["weights"]:
        return out
    mass = (p * inv).sum((2, 3))
    live = (j[None, :] < n[:, None])[:, None]
    return out, torch.where(live, st["weights"] + mass, st["weights_out"])


def quantised(x, scale):
    """Codes of x under a scale per leading index; a zero scale gives zero codes."""
    return torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x))


def plain_append(st):
    page, D = st["case"]["page"], st["case"]["dim"]
    Hkv, NB = st["case"]["kv_heads"], st["blocks"]
    B, dev = st["table"].shape[0], st["table"].device
    starts, first = st["starts"].long(), st["first"].long()
    seq, pos = st["rows"]
    at = pos + (starts - first)[seq]                                            # place from the first touched page on
    place = torch.arange(NB * page, device=dev).view(NB, page)
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    is_old = place[None] < (starts - first)[:, None, None]
    touched = torch.arange(NB, device=dev)[None] * page < (starts - first + n)[:, None]
    column = torch.where(touched, first[:, None] // page + torch.arange(NB, device=dev)[None], torch.zeros_like(n)[:, None])
    pages = torch.gather(st["table"].long(), 1, column)
    got = []
    for which in range(2):  # keys, values
        codes, scales = st["cache"][which], st["cache"][2 + which]
        x = torch.zeros(B, NB * page, Hkv, D, device=dev)
        x[seq, at] = st["kv"][:, which].float()
        x = x.view(B, NB, page, Hkv, D).transpose(2, 3)                         # [B, NB, Hkv, page, D]
        top = x.abs().amax((-1, -2))
        new = top / torch.full_like(top, QMAX)
        prior = scales[pages]
        has_old = is_old.any(-1)[..., None]
        s = torch.where(has_old, torch.maximum(prior, new), new)
        ratio = torch.where(s > 0, prior / s, torch.zeros_like(s))
        old = torch.round(codes[pages].float() * ratio[..., None, None])
        now = torch.where(is_old[:, :, None, :, None], old, quantised(x, s[..., None, None]))
        live = touched.nonzero(as_tuple=True)
        scales[pages[live]] = s[live]
        rewritten = place[None] < (starts - first + n)[:, None, None]
        stays = codes[pages].float()
        codes[pages[live]] = torch.where(rewritten[:, :, None, :, None], now, stays)[live].to(torch.int8)
        values = (now * s[..., None, None]).transpose(2, 3).reshape(B, NB * page, Hkv, D)
        bseq, bpos = st["back_rows"]
        got.append(values[bseq, bpos].to(st["kv"].dtype))
    return got


def plain_evict(st):
    c = st["case"]
    budget, page, D, Hkv = c["budget"], c["page"], c["dim"], c["kv_heads"]
    kc, vc, ksc, vsc = st["cache"]
    w, n = st["weights"], st["lens"].long()[:, None, None]
    B, _, cap = w.shape
    j = torch.arange(cap, device=w.device)[None, None]
    key = torch.where((j < c["sink"]) | (j >= n - c["recent"]), torch.full_like(w, math.inf), w)
    key = torch.where(j < n, key, torch.full_like(w, -1.0))
    at = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    at = torch.where(at < n, at, torch.full_like(at, cap)).sort(-1).values
    short = budget - at.shape[-1]
    at = torch.nn.functional.pad(at, (0, max(0, short)), value=cap)
    there = at < cap
    kept = torch.where(there, at, torch.full_like(at, -1)).to(torch.int32)
    new_w = torch.where(there, torch.gather(w, -1, at.clamp(max=cap - 1)), torch.zeros_like(at, dtype=w.dtype))
    new_n = st["lens"].clamp(max=budget)
    blocks = -(-budget // page)
    at = torch.nn.functional.pad(at, (0, blocks * page - budget), value=cap)
    there = at < cap
    src = at.clamp(max=cap - 1)
    pages = torch.gather(st["table"].long()[:, None].expand(B, Hkv, -1), 2, src // page).clamp(min=0)
    head = torch.arange(Hkv, device=w.device)[None, :, None].expand_as(pages)
    seq, pos = st["back_rows"]
    got = []
    for codes, scales in ((kc, ksc), (vc, vsc)):
        x = codes[pages, head, src % page].float() * scales[pages, head][..., None]
        x = torch.where(there[..., None], x, torch.zeros_like(x)).view(B, Hkv, blocks, page, D)
        top = x.abs().amax((-1, -2), keepdim=True)
        s = top / torch.full_like(top, QMAX)
        code = quantised(x, s)
        codes[st["out_table"].long()] = code.transpose(1, 2).to(torch.int8)
        scales[st["out_table"].long()] = s[..., 0, 0].transpose(1, 2)
        got.append((code * s).view(B, Hkv, -1, D)[seq, :, pos].to(DTYPES[c["dtype"]]))
    return kept, new_w, new_n, got


# --------------------------------------------------------------------------
# 64 bits, sequence by sequence
# --------------------------------------------------------------------------
def attend64(q, k, v, scale):
    """q [n, h, d] over k, v [m, g, d], the last query seeing every key: output [n, h, d], weights [n, h, m]."""
    n, h, d = q.shape
    m, g = k.shape[0], k.shape[1]
    outs, weights = [], []
    for head in range(h):
        z = (q[:, head] @ k[:, head * g // h].T) * scale
        see = torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + (m - n)
        z = z.masked_fill(~see, -math.inf)
        a = torch.softmax(z, -1).masked_fill(~see.any(-1, keepdim=True), 0.0)
        outs.append(a @ v[:, head * g // h])
        weights.append(a)
    return torch.stack(outs, 1), weights


def page64(x):
    s = x.abs().amax() / 127
    return (torch.round(x / s), s) if s > 0 else (torch.zeros_like(x), s)


def tokens64(st, which, b, h, n):
    codes, scales, page = st["cache"][which], st["cache"][2 + which], st["case"]["page"]
    ids = st["table"][b, :-(-n // page)].long()
    return (codes[ids, h].double() * scales[ids, h].double()[:, None, None]).reshape(-1, codes.shape[-1])[:n]


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    Hq, Hkv, D = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "prefill":
        q, k, v = (x.double() for x in split(st))
        out, a, b = [], 0, 0
        for n, m in zip(ints(c["q_lens"]), ints(c["k_lens"])):
            rows = max(1, (1 << 28) // m)
            part = []
            for r in range(0, n, rows):   # the queries in pieces, each with the keys its last one sees
                e = min(n, r + rows)
                upto = b + m - n + e
                part.append(attend64(q[a + r:a + e], k[b:upto], v[b:upto], st["scale"])[0])
            out += part
            a, b = a + n, b + m
        return torch.cat(out)
    lens, page = ints(c["lens"]), c["page"]
    if c["op"] == "decode":
        outs = []
        total = st["weights"].double() if c["weights"] else None
        for b, n in enumerate(lens):
            k = torch.stack([tokens64(st, 0, b, h, n) for h in range(Hkv)], 1)
            v = torch.stack([tokens64(st, 1, b, h, n) for h in range(Hkv)], 1)
            o, w = attend64(st["q"][b].double(), k, v, st["scale"])
            outs.append(o)
            if c["weights"]:
                for head, x in enumerate(w):
                    total[b, head * Hkv // Hq, :n] += x.sum(0)
        return torch.stack(outs) if total is None else (torch.stack(outs), total)
    sides = ([], [])
    if c["op"] == "append":
        starts, at = ints(c["starts"]), 0
        if sum(lens) // page + 2 * len(lens) > 2000:
            return None
        for b, n in enumerate(lens):
            a = starts[b]
            for which, side in enumerate(sides):
                heads = []
                for h in range(Hkv):
                    x = st["kv"][at:at + n, which, h].double()
                    first = min(n, -a % page if a % page else 0)       # new tokens that go behind old ones
                    rows = []
                    if a % page:
                        ids = st["table"][b, a // page].long()
                        s0 = st["cache"][2 + which][ids, h].double()
                        s1 = torch.maximum(s0, x[:first].abs().amax() / 127)
                        rows += [torch.round(st["cache"][which][ids, h, :a % page].double() * (s0 / s1)) * s1,
                                 torch.round(x[:first] / s1) * s1]
                    for r in range(first, n, page):
                        code, s = page64(x[r:min(n, r + page)])
                        rows.append(code * s)
                    heads.append(torch.cat(rows))
                side.append(torch.stack(heads, 1))
            at += n
        return [torch.cat(s) for s in sides]
    B, budget, w = len(lens), c["budget"], st["weights"].cpu().double().numpy()
    if B * Hkv * -(-min(budget, max(lens)) // page) > 20000:
        return None
    kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32)
    new_w = torch.zeros(B, Hkv, budget, dtype=torch.float64)
    for b, n in enumerate(lens):
        cols = ([], [])
        for h in range(Hkv):
            if n <= budget:
                keep = list(range(n))
            else:
                fixed = set(range(c["sink"])) | set(range(n - c["recent"], n))
                x = w[b, h]
                free = sorted((i for i in range(n) if i not in fixed), key=lambda i: (-x[i], i))
                keep = sorted(list(fixed) + free[:budget - len(fixed)])
            kept[b, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            new_w[b, h, :len(keep)] = torch.tensor(w[b, h][keep])
            for which, side in enumerate(cols):
                x = tokens64(st, which, b, h, n)[torch.tensor(keep, device="cuda")]
                part = []
                for r in range(0, len(keep), page):
                    code, s = page64(x[r:r + page])
                    part.append(code * s)
                side.append(torch.cat(part))
        for side, col in zip(sides, cols):
            side.append(torch.stack(col, 1))
    return kept, new_w, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), [torch.cat(s) for s in sides]


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    c = case
    Hq, Hkv, D = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "prefill":
        ql, kl = ints(c["q_lens"]), ints(c["k_lens"])
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(ql, kl))
        return {"bytes": 2 * D * (2 * Hq * sum(ql) + 2 * Hkv * sum(kl)), "flops": 4 * D * Hq * pairs}
    lens, page = ints(c["lens"]), c["page"]
    if c["op"] == "append":
        starts = ints(c["starts"])
        n = sum(lens)
        old = sum(a % page for a in starts)
        back = n + old
        # new tokens read, codes written (and the old ones of a begun page read and rewritten), then all read back
        return {"bytes": 2 * Hkv * D * (2 * n + n + 2 * old + back + 2 * back), "flops": 4 * Hkv * D * (n + back)}
    if c["op"] == "decode":
        T, n = c["new"], sum(lens)
        tables = sum(-(-x // page) for x in lens) * (4 + 8 * Hkv)
        moved = 2 * Hkv * D * n + tables + 4 * D * Hq * T * len(lens) + (8 * Hkv * n if c["weights"] else 0)
        return {"bytes": moved, "flops": 4 * D * Hq * T * n}
    keep = sum(min(n, c["budget"]) for n in lens)
    # totals read; kept codes read and written; indices and totals written; then the codes read back
    return {"bytes": 4 * Hkv * sum(lens) + Hkv * keep * (4 * D + 8) + 2 * Hkv * keep * 3 * D,
            "flops": 4 * Hkv * D * keep}
