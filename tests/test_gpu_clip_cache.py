"""Prompts, decode steps, verification and eviction through ClipCache and a
decoder stack."""
import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
H, G, D = 6, 2, 128


def qkv(rows, seed):
    return torch.randn(rows, (H + 2 * G) * D, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


def new(clips, **kw):
    from alpamayo_b200 import ClipCache
    kw = dict(dict(layers=2, clips=clips, capacity=256, heads=H, kv_heads=G, head_dim=D, page_size=16), **kw)
    return ClipCache(**kw)


def test_prompt_is_causal_attention_and_fills_the_cache():
    import alpamayo_b200.ops as ops
    c, lens = new(3), [40, 0, 17]
    x = qkv(57, 1)
    out = c.prompt(lens)(0, x)
    y = x.view(57, H + 2 * G, D)
    want = ops.attention_prefill(y[:, :H], y[:, H:H + G], y[:, H + G:], R.cu(lens))
    assert torch.equal(out, want.view(57, -1))
    k, v = c.caches[0].gather(c.table, R.i32([0, 0, 0]), R.cu(lens), 57, torch.float32)
    # half a step of a page's scale; page maxima of normal values stay below 6
    assert float((k - y[:, H:H + G].float()).abs().max()) <= 6 / 254 * 1.01
    assert float((v - y[:, H + G:].float()).abs().max()) <= 6 / 254 * 1.01
    assert c.lens == lens and c.seq_lens.tolist() == lens


def test_chunks_steps_and_a_whole_prompt_agree():
    """The same tokens as one prompt, in two chunks, and a prompt with decode
    steps: they differ by the cache's rounding only."""
    lens = [60, 33]
    x = qkv(93, 2)
    rows = [x[:60], x[60:]]
    whole = new(2).prompt(lens)(0, x).split(lens)
    c = new(2)
    first = c.prompt([41, 7])(0, torch.cat([rows[0][:41], rows[1][:7]])).split([41, 7])
    second = c.prompt([19, 26])(0, torch.cat([rows[0][41:], rows[1][7:]])).split([19, 26])
    s = new(2, totals=True)
    s.prompt([57, 30])(0, torch.cat([rows[0][:57], rows[1][:30]]))
    steps = [s.step()(0, torch.stack([rows[0][57 + i], rows[1][30 + i]])) for i in range(3)]
    v = new(2)
    v.prompt([57, 30])(0, torch.cat([rows[0][:57], rows[1][:30]]))
    ver = v.verify(3)(0, torch.cat([rows[0][57:], rows[1][30:]])).view(2, 3, -1)
    for b in range(2):
        w = whole[b].float()
        chunked = torch.cat([first[b], second[b]]).float()
        n = lens[b]
        # the values' rounding (half a step of max|v| / 127 with max|v| below
        # 5) and what the keys' rounding does to the weights: score errors of
        # standard deviation 0.02
        assert float((chunked - w).abs().max()) < 0.15
        for i in range(3):
            assert float((steps[i][b].float() - w[n - 3 + i]).abs().max()) < 0.15
            assert float((ver[b, i].float() - w[n - 3 + i]).abs().max()) < 0.15
    # each of three tokens gave a total weight of one per query head
    assert torch.allclose(s.totals[0].sum(-1), torch.full((2, G), 3.0 * H / G, device="cuda"), rtol=1e-4)


def test_rejected_tokens_are_written_again():
    x = qkv(50, 3)
    c, ref = new(1, totals=True), new(1, totals=True)
    c.prompt([40])(0, x[:40])
    ref.prompt([40])(0, x[:40])
    c.verify(4)(0, x[40:44] * 0.5)                     # smaller values: the pages' scales do not grow
    c.accept([4])
    assert c.lens == [40] and c.seq_lens.tolist() == [40]
    a, b = c.step()(0, x[44:45]), ref.step()(0, x[44:45])
    assert torch.equal(a, b)
    with pytest.raises(ValueError):
        c.accept([99])


def test_evict_frees_pages_and_keeps_what_was_attended():
    c = new(2, totals=True, spare=64, capacity=128)
    x = qkv(150, 4)
    c.prompt([100, 40])(0, x[:140])
    c.prompt([0, 0])(0, x[:0])
    for layer in range(2):
        c.totals[layer].copy_(torch.rand_like(c.totals[layer]))
        live = torch.arange(c.totals[layer].shape[2], device="cuda")[None] < c.seq_lens[:, None]
        c.totals[layer] *= live[:, None]
    k0, _ = c.caches[0].gather(c.table, R.i32([0, 0]), R.cu([100, 40]), 140, torch.float32)
    free = len(c.free)
    kept = c.evict(48, sink=2, recent=8)
    assert c.lens == [48, 40] and len(c.free) == free + (7 + 3) - (3 + 3)
    k1, _ = c.caches[0].gather(c.table, R.i32([0, 0]), R.cu([48, 40]), 88, torch.float32)
    for g in range(G):
        idx = kept[0][0, g].long()
        assert idx[:2].tolist() == [0, 1] and idx[-8:].tolist() == list(range(92, 100))
        assert float((k1[:48, g] - k0[idx, g]).abs().max()) <= 6 / 254 * 1.01
    out = c.step()(0, x[140:142])
    assert torch.isfinite(out).all() and c.lens == [49, 41]


def test_limits():
    c = new(2, capacity=32)
    with pytest.raises(ValueError):
        c.prompt([33, 1])
    with pytest.raises(ValueError):
        c.prompt([1])
    with pytest.raises(RuntimeError):
        c.evict(8)
    from alpamayo_b200 import KV8Cache
    with pytest.raises(ValueError):
        KV8Cache(4, 1, 96)
    t = new(1, capacity=32, totals=True)
    t.prompt([32])(0, qkv(32, 5))
    with pytest.raises(RuntimeError):
        t.evict(16)                                     # no spare pages
    assert t.lens == [32]


def test_decoder_stack_with_attention():
    from alpamayo_b200 import ClipCache
    from alpamayo_b200.stack import HEAD_DIM, HEADS, HIDDEN, KV_HEADS, DecoderStack
    stack = DecoderStack(layers=2, seed=3)
    c = ClipCache(2, 2, 64, HEADS, KV_HEADS, HEAD_DIM, 16, totals=True)
    x = torch.randn(30, HIDDEN, generator=torch.Generator().manual_seed(6)).to(BF16).cuda()
    out = stack.forward(x, attention=c.prompt([20, 10]))
    assert out.shape == (30, HIDDEN) and torch.isfinite(out).all()
    y = torch.randn(2, HIDDEN, generator=torch.Generator().manual_seed(7)).to(BF16).cuda()
    a = stack.forward(y, attention=c.step())
    assert a.shape == (2, HIDDEN) and torch.isfinite(a).all() and c.lens == [21, 11]
    # fused and separate prologues agree bit for bit with a real attention too
    c.accept([1, 1])
    assert torch.equal(stack.forward(y, fused=False, attention=c.step()), a)
    # and without one, nothing has changed
    ident = stack.forward(y)
    assert torch.equal(ident, stack.forward(y, attention=lambda i, qkv: qkv[:, :HEADS * HEAD_DIM].contiguous()))


def test_a_prompt_does_not_depend_on_the_other_clips():
    # a clip's first prompt beside another clip's second chunk: bit for bit what it is alone
    import alpamayo_b200.ops as ops
    x, y, z = qkv(60, 90), qkv(33, 91), qkv(21, 92)
    alone = new(1).prompt([33])(0, y)
    c = new(3)
    c.prompt([60, 0, 0])(0, x)
    out = c.prompt([21, 33, 0])(0, torch.cat([z, y]))
    assert torch.equal(out[21:], alone)
    # the chunk sees its own tokens as they are and the cached ones as the cache holds them
    k, v = c.caches[0].gather(c.table, R.i32([0, 0, 0]), R.cu([60, 0, 0]), 60, BF16)
    t = z.view(21, H + 2 * G, D)
    want = ops.attention_prefill(t[:, :H], torch.cat([k, t[:, H:H + G]]), torch.cat([v, t[:, H + G:]]), R.cu([21]), R.cu([81]))
    assert torch.equal(out[:21], want.view(21, -1))
    # and the cache holds both
    k, v = c.caches[0].gather(c.table, R.i32([0, 0, 0]), R.cu([81, 33, 0]), 114, torch.float32)
    assert float((k[81:] - y.view(33, H + 2 * G, D)[:, H:H + G].float()).abs().max()) <= 6 / 254 * 1.01
    assert c.lens == [81, 33, 0]


def test_evict_leaves_clips_under_budget_where_they_are():
    c = new(3, totals=True, capacity=128)
    x = qkv(190, 93)
    c.prompt([100, 50, 40])(0, x)
    live = torch.arange(128, device="cuda")[None] < c.seq_lens[:, None]
    for t in c.totals:
        t.copy_(torch.rand_like(t))
        t *= live[:, None]
    totals, pages = [t.clone() for t in c.totals], [list(p) for p in c.pages]
    tensors = [t.clone() for t in c.caches[0].tensors]
    c.free = c.free[:4]                                     # room for the first clip's 50 tokens, and no more
    kept = c.evict(50, sink=2, recent=8)
    assert c.lens == [50, 50, 40] and c.seq_lens.tolist() == c.lens
    assert c.pages[1:] == pages[1:] and sorted(c.free) == sorted(pages[0])
    for b, n in ((1, 50), (2, 40)):
        p = torch.tensor(pages[b])
        assert all(torch.equal(t[p], u[p]) for t, u in zip(c.caches[0].tensors, tensors))
        for layer in range(2):
            assert kept[layer][b].tolist() == [list(range(n)) + [-1] * (50 - n)] * G
            assert torch.equal(c.totals[layer][b], totals[layer][b])
    for layer in range(2):
        assert kept[layer].shape == (3, G, 50) and kept[layer].dtype == torch.int32
        idx = kept[layer][0].long()
        assert torch.equal(c.totals[layer][0, :, :50], totals[layer][0].gather(1, idx)) and (c.totals[layer][0, :, 50:] == 0).all()
    # nothing to evict: nothing moves, no pages needed
    c.free = []
    pages = [list(p) for p in c.pages]
    kept = c.evict(64)
    assert c.pages == pages and c.lens == [50, 50, 40] and kept[1][2].tolist() == [list(range(40)) + [-1] * 24] * G


def test_no_call_waits_for_the_device():
    c = new(2, totals=True, spare=64)
    x = qkv(140, 94)

    def all_calls():
        c.prompt([30, 20])(0, x[:50])
        c.prompt([20, 0])(0, x[50:70])
        c.step()(0, x[70:72])
        c.verify(3)(0, x[72:78])
        c.accept([1, 0])
        c.evict(40, sink=2, recent=8)
    all_calls()                                             # what is allocated or loaded once
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        all_calls()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    assert c.seq_lens.tolist() == c.lens


def test_lengths_and_tables_sent_far_ahead_of_the_device():
    c = new(2, totals=True)
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)                          # about a tenth of a second: every copy below waits behind it
    seen = []
    for i in range(150):
        c._grow([1, 2 if i < 20 else 0])
        seen.append((c.seq_lens, c.table, list(c.lens), [list(p) for p in c.pages]))
    torch.cuda.synchronize()
    for lens, table, want, pages in seen:
        assert lens.tolist() == want
        assert table.tolist() == [p + [-1] * (c.width - len(p)) for p in pages]
