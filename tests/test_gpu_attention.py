"""Causal attention over packed prompts, and attention over the int8 paged
cache, against a 64-bit evaluation of the formula."""

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _clean_error_word(request):
    import alpamayo_b200.ops as ops
    ops.device_error_word()
    yield
    if "bad_" not in request.node.name:
        assert ops.device_error_word() == 0


def packed(q_lens, k_lens, heads, kv_heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(sum(q_lens), heads, dim, generator=g) * 1.5).to(dtype)
    k = torch.randn(sum(k_lens), kv_heads, dim, generator=g).to(dtype)
    v = torch.randn(sum(k_lens), kv_heads, dim, generator=g).to(dtype)
    return q, k, v


def check_prefill(out, q, k, v, q_lens, k_lens, scale, dtype):
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        ref, _, size, sb = R.attend(q[a:a + n].double(), k[b:b + m].double(), v[b:b + m].double(), scale)
        got = out[a:a + n]
        assert R.max_excess(got, ref, R.out_bound(ref, size, sb, dtype, R.UNIT[dtype])) <= 1.0, (n, m)
        a, b = a + n, b + m


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(7, 1, 128), (4, 4, 64), (6, 2, 128), (3, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [2, 1], [37], [127, 128, 129], [1, 300, 0, 5], [257, 64]])
def test_prefill(lens, heads, kv_heads, dim, dtype):
    import alpamayo_b200.ops as ops
    q, k, v = packed(lens, lens, heads, kv_heads, dim, dtype, 1)
    scale = dim ** -0.5
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(lens))
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    check_prefill(out, q, k, v, lens, lens, scale, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens", [([5], [200]), ([130, 3], [400, 3]), ([1, 1, 1], [129, 1, 700]),
                                           ([64], [20]), ([4, 0, 9], [0, 7, 300]), ([260], [261])])
def test_prefill_behind_history(q_lens, k_lens, dim, dtype):
    # fewer keys than queries: the first Lq - Lk queries see nothing and give zeros
    import alpamayo_b200.ops as ops
    q, k, v = packed(q_lens, k_lens, 4, 2, dim, dtype, 2)
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(q_lens), R.cu(k_lens), 0.2)
    check_prefill(out, q, k, v, q_lens, k_lens, 0.2, dtype)
    a = 0
    for n, m in zip(q_lens, k_lens):
        assert (out[a:a + max(0, n - m)] == 0).all()
        a += n


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("q_lens,k_lens", [([5, 100], [3000, 1111]), ([1], [5000]), ([300], [2500]), ([3, 0, 700, 2], [9, 0, 700, 6000])])
def test_prefill_keys_shared_out(q_lens, k_lens, dim, dtype):
    # few rows over long sequences: several blocks share a row's keys
    import alpamayo_b200.ops as ops
    from alpamayo_b200 import _native
    assert _native.capi().paro_attention_prefill_workspace_size(len(q_lens), sum(q_lens), sum(k_lens), 2, dim) > 0
    q, k, v = packed(q_lens, k_lens, 2, 1, dim, dtype, 40)
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(q_lens), R.cu(k_lens))
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        for i in sorted({0, n // 3, n // 2, n - 1} - {-1}) if n else []:
            see = i + 1 + m - n
            ref, _, size, sb = R.attend(q[a + i:a + i + 1].double(), k[b:b + see].double(), v[b:b + see].double(), dim ** -0.5)
            bound = R.out_bound(ref, size, sb, dtype, R.UNIT[dtype]) + (2.0 ** -25 if dtype == F16 else 0.0)
            assert R.max_excess(out[a + i:a + i + 1], ref, bound) <= 1.0, (n, m, i)
        a, b = a + n, b + m
    # a value that is not finite, seen by some of the last sequence's rows only
    n, m = q_lens[-1], k_lens[-1]
    v2 = v.clone()
    v2[-1, 0, 5] = float("inf")
    got = ops.attention_prefill(q.cuda(), k.cuda(), v2.cuda(), R.cu(q_lens), R.cu(k_lens))
    assert torch.equal(got[:-1], out[:-1]) and not torch.isfinite(got[-1, :, 5]).any()
    rest = torch.arange(dim) != 5
    assert torch.equal(got[-1][:, rest], out[-1][:, rest])


@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [(BF16, 128, 12, 4), (F16, 64, 2, 2), (BF16, 64, 28, 4)])
def test_prefill_one_long_history_among_short_ones(dtype, dim, heads, kv_heads):
    # keys shared out for one sequence only, in more parts than blocks
    import alpamayo_b200.ops as ops
    q_lens, k_lens = [164, 69, 357, 0, 165, 64, 5, 178, 56], [5408, 110, 726, 0, 165, 60, 2, 178, 1134]
    q, k, v = packed(q_lens, k_lens, heads, kv_heads, dim, dtype, 47)
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(q_lens), R.cu(k_lens))
    assert torch.equal(out, ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(q_lens), R.cu(k_lens)))
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        for i in sorted({0, n // 2, n - 1} - {-1}) if n else []:
            see = max(0, i + 1 + m - n)
            if not see:
                assert (out[a + i] == 0).all()
                continue
            ref, _, size, sb = R.attend(q[a + i:a + i + 1].double(), k[b:b + see].double(), v[b:b + see].double(), dim ** -0.5)
            bound = R.out_bound(ref, size, sb, dtype, R.UNIT[dtype]) + (2.0 ** -25 if dtype == F16 else 0.0)
            assert R.max_excess(out[a + i:a + i + 1], ref, bound) <= 1.0, (n, m, i)
        a, b = a + n, b + m


def test_prefill_many_sequences_in_order_of_place():
    # over 32 sequences, of all numbers of tiles
    import alpamayo_b200.ops as ops
    lens = [(i * 37) % 520 if i % 5 else 0 for i in range(70)]
    q, k, v = packed(lens, lens, 2, 2, 64, BF16, 41)
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(lens))
    a = 0
    for n in lens:
        for i in sorted({0, n // 2, n - 1} - {-1}) if n else []:
            ref, _, size, sb = R.attend(q[a + i:a + i + 1].double(), k[a:a + i + 1].double(), v[a:a + i + 1].double(), 0.125)
            assert R.max_excess(out[a + i:a + i + 1], ref, R.out_bound(ref, size, sb, BF16, R.UNIT[BF16])) <= 1.0, (n, i)
        a += n


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,nseq", [(BF16, 128, 28, 4, 40), (F16, 64, 20, 5, 21), (BF16, 64, 9, 3, 70)])
def test_prefill_many_items_per_block(dtype, dim, heads, kv_heads, nseq):
    # several items behind one another in a block, rows that see nothing,
    # values that are not finite in some: every sequence as it comes out alone
    import alpamayo_b200.ops as ops
    q_lens = [(i * 101) % 700 if i % 7 else i % 3 for i in range(nseq)]
    k_lens = [max(0, n + (i * 59) % 300 - 90) for i, n in enumerate(q_lens)]
    q, k, v = packed(q_lens, k_lens, heads, kv_heads, dim, dtype, 43)
    cq, ck = [0], [0]
    for n, m in zip(q_lens, k_lens):
        cq.append(cq[-1] + n)
        ck.append(ck[-1] + m)
    for i in range(0, nseq, 4):
        if k_lens[i] > 8:
            v[ck[i + 1] - 1 - i % 8, i % kv_heads, i % dim] = float("nan") if i % 8 else float("inf")
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    out = ops.attention_prefill(q, k, v, R.cu(q_lens), R.cu(k_lens))
    for i, (n, m) in enumerate(zip(q_lens, k_lens)):
        if n == 0:
            continue
        a, b = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        alone = ops.attention_prefill(q[a], k[b], v[b], R.cu([n]), R.cu([m]))
        assert torch.equal(torch.nan_to_num(out[a], 7.0, 8.0, 9.0), torch.nan_to_num(alone, 7.0, 8.0, 9.0)), i
        row = n - 1
        if m and torch.isfinite(v[b]).all():
            ref, _, size, sb = R.attend(q[a][row:].double().cpu(), k[b].double().cpu(), v[b].double().cpu(), dim ** -0.5)
            bound = R.out_bound(ref, size, sb, dtype, R.UNIT[dtype]) + (2.0 ** -25 if dtype == F16 else 0.0)
            assert R.max_excess(out[a][row:], ref, bound) <= 1.0, i


def test_prefill_long_rows_and_large_scores():
    import alpamayo_b200.ops as ops
    lens = [1500]
    q, k, v = packed(lens, lens, 2, 1, 128, BF16, 3)
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(lens), None, 1.0)   # scores of +-60: near one-hot rows
    rows = torch.tensor([0, 1, 126, 127, 128, 255, 256, 700, 1023, 1499])
    for i in rows.tolist():
        ref, _, size, sb = R.attend(q[i:i + 1].double(), k[:i + 1].double(), v[:i + 1].double(), 1.0)
        assert R.max_excess(out[i:i + 1], ref, R.out_bound(ref, size, sb, BF16, R.UNIT[BF16])) <= 1.0, i


def test_prefill_reads_fused_projection_in_place():
    import alpamayo_b200.ops as ops
    lens, H, G, D = [70, 200], 6, 2, 128
    g = torch.Generator().manual_seed(4)
    x = torch.randn(270, (H + 2 * G) * D, generator=g).to(BF16).cuda()
    y = x.view(270, H + 2 * G, D)
    q, k, v = y[:, :H], y[:, H:H + G], y[:, H + G:]
    want = ops.attention_prefill(q.contiguous(), k.contiguous(), v.contiguous(), R.cu(lens))
    assert torch.equal(ops.attention_prefill(q, k, v, R.cu(lens)), want)
    # heads outermost, and a slice of a wider token dimension
    qt = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    kt = torch.stack([k, k], 1)[:, 0]
    assert torch.equal(ops.attention_prefill(qt, kt, v, R.cu(lens)), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prefill_what_is_not_seen_has_no_effect(bad):
    import alpamayo_b200.ops as ops
    lens = [100, 150, 40]
    q, k, v = packed(lens, lens, 4, 2, 128, BF16, 5)
    want = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu(lens))
    # the second sequence's last keys and values from token 90 on, and every key and value of the third
    k2, v2 = k.clone(), v.clone()
    k2[100 + 90:] = bad
    v2[100 + 90:] = bad
    got = ops.attention_prefill(q.cuda(), k2.cuda(), v2.cuda(), R.cu(lens))
    assert torch.equal(got[:190], want[:190])
    # one value row alone: rows before it are untouched, rows from it on show it
    v3 = v.clone()
    v3[100 + 37, 0, 3] = bad
    got = ops.attention_prefill(q.cuda(), k.cuda(), v3.cuda(), R.cu(lens))
    assert torch.equal(got[:137], want[:137]) and torch.equal(got[250:], want[250:])
    assert not torch.isfinite(got[137:250, :2, 3]).any()
    assert torch.equal(got[137:250, 2:], want[137:250, 2:])
    rest = torch.ones(128, dtype=torch.bool)
    rest[3] = False
    assert torch.equal(got[137:250, :2][..., rest], want[137:250, :2][..., rest])


def test_prefill_rows_behind_the_last_sequence_are_zero():
    import alpamayo_b200.ops as ops
    q, k, v = packed([300], [300], 4, 2, 64, F16, 6)
    out = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu([40, 33]))
    assert (out[73:] == 0).all()
    check_prefill(out[:73], q[:73], k[:73], v[:73], [40, 33], [40, 33], 0.125, F16)


def test_prefill_offsets_beyond_32_bits():
    import alpamayo_b200.ops as ops
    n, H, D = 9, 2, 128
    step = (1 << 31) // 4 + 8                  # elements between tokens: the last one lies beyond 2^32
    buf = torch.empty(step * (n - 1) + H * D, dtype=BF16, device="cuda")
    q, k, v = packed([n], [n], H, H, D, BF16, 7)
    big = buf.as_strided((n, H, D), (step, D, 1))
    want = ops.attention_prefill(q.cuda(), k.cuda(), v.cuda(), R.cu([n]))
    big.copy_(q)
    assert torch.equal(ops.attention_prefill(big, k.cuda(), v.cuda(), R.cu([n])), want)
    big.copy_(k)
    assert torch.equal(ops.attention_prefill(q.cuda(), big, v.cuda(), R.cu([n])), want)
    big.copy_(v)
    assert torch.equal(ops.attention_prefill(q.cuda(), k.cuda(), big, R.cu([n])), want)


def test_prefill_on_another_stream_and_graph():
    import alpamayo_b200.ops as ops
    lens = [200, 77]
    q, k, v = (t.cuda() for t in packed(lens, lens, 7, 1, 128, BF16, 8))
    c = R.cu(lens)
    want = ops.attention_prefill(q, k, v, c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.attention_prefill(q, k, v, c)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.attention_prefill(q, k, v, c)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# --------------------------------------------------------------------------
# attention over the cache
# --------------------------------------------------------------------------
def check_kv8(out, q, cache, table, lens, scale, weights=None, got_weights=None):
    """The codes and scales are exact inputs; the weights are rounded to fp16
    before the value product, whatever the output's type."""
    B, T, H, D = q.shape
    G = cache[0].shape[1]
    for b, n in enumerate(lens):
        k = torch.stack([R.read(cache, 0, table, b, h, n) for h in range(G)], 1)
        v = torch.stack([R.read(cache, 1, table, b, h, n) for h in range(G)], 1)
        ref, w, size, sb = R.attend(q[b].double().cpu(), k, v, scale)
        assert R.max_excess(out[b], ref, R.out_bound(ref, size, sb, q.dtype, 2.0 ** -11)) <= 1.0, (b, n)
        if weights is not None:
            mass = w.view(G, H // G, T, n).sum((1, 2))
            err = (w * (2.0 * sb[..., None] + 2.0 ** -19)).view(G, H // G, T, n).sum((1, 2))
            want = weights[b, :, :n].double().cpu() + mass
            tol = err + want.abs() * 2.0 ** -23 + mass * 2.0 ** -18 + 1e-30
            assert (((got_weights[b, :, :n].double().cpu() - want).abs() / tol) <= 1.0).all(), (b, n)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,dim,T", [(7, 1, 128, 1), (4, 4, 64, 1), (6, 2, 128, 4), (12, 2, 64, 3),
                                                  (4, 1, 128, 16), (14, 2, 128, 1)])
def test_kv8_attention(heads, kv_heads, dim, T, page, dtype):
    import alpamayo_b200.ops as ops
    lens = [16 + T, 1 + T, 300, 129, 32, 1000]
    lens = [max(n, T) for n in lens]
    *cache, table = R.make_pool(lens, page, kv_heads, dim, 11)
    g = torch.Generator().manual_seed(12)
    q = (torch.randn(len(lens), T, heads, dim, generator=g) * 1.5).to(dtype).cuda()
    cap = table.shape[1] * page + 5
    w = torch.rand(len(lens), kv_heads, cap, generator=g).cuda()
    out = ops.attention_kv8(q, *cache, table, R.i32(lens))
    check_kv8(out, q, cache, table, lens, dim ** -0.5)
    w_out = torch.full_like(w, 7.0)
    out2 = ops.attention_kv8(q, *cache, table, R.i32(lens), None, w, w_out)
    assert torch.equal(out, out2)
    check_kv8(out2, q, cache, table, lens, dim ** -0.5, w, w_out)
    for b, n in enumerate(lens):
        assert (w_out[b, :, n:] == 7.0).all()          # behind the last token nothing is written
    w_in = w.clone()
    ops.attention_kv8(q, *cache, table, R.i32(lens), None, w_in)   # in place
    for b, n in enumerate(lens):
        assert torch.equal(w_in[b, :, :n], w_out[b, :, :n])
        assert torch.equal(w_in[b, :, n:], w[b, :, n:])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("heads,kv_heads,dim,T", [(14, 2, 128, 16), (5, 1, 64, 7), (5, 1, 128, 5), (16, 1, 64, 16),
                                                  (3, 1, 128, 3), (28, 4, 128, 8)])
def test_kv8_attention_many_rows(heads, kv_heads, dim, T, page, dtype):
    # up to 256 rows a KV head; an output below 2^-14 rounds to a multiple of fp16's 2^-24
    import alpamayo_b200.ops as ops
    lens = [16 + T, 1 + T, 300, 129, 32, 1000]
    *cache, table = R.make_pool(lens, page, kv_heads, dim, 11)
    q = (torch.randn(len(lens), T, heads, dim, generator=torch.Generator().manual_seed(12)) * 1.5).to(dtype).cuda()
    w = torch.zeros(len(lens), kv_heads, table.shape[1] * page, device="cuda")
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), None, w)
    for b, n in enumerate(lens):
        k = torch.stack([R.read(cache, 0, table, b, h, n) for h in range(kv_heads)], 1)
        v = torch.stack([R.read(cache, 1, table, b, h, n) for h in range(kv_heads)], 1)
        ref, p, size, sb = R.attend(q[b].double().cpu(), k, v, dim ** -0.5)
        bound = R.out_bound(ref, size, sb, dtype, 2.0 ** -11) + (2.0 ** -25 if dtype == F16 else 0.0)
        assert R.max_excess(out[b], ref, bound) <= 1.0, (b, n)
        mass = p.view(kv_heads, heads // kv_heads, T, n).sum((1, 2))
        err = (p * (2.0 * sb[..., None] + 2.0 ** -18)).view(kv_heads, heads // kv_heads, T, n).sum((1, 2))
        got = w[b, :, :n].double().cpu()
        assert ((got - mass).abs() <= err + mass * 2.0 ** -20 + 1e-30).all(), (b, n)
        assert (w[b, :, n:] == 0).all()


def test_kv8_attention_lengths_zero_and_shorter_than_the_new_tokens():
    import alpamayo_b200.ops as ops
    lens, T = [0, 2, 5, 40], 5
    *cache, table = R.make_pool(lens, 16, 2, 128, 13)
    q = torch.randn(4, T, 6, 128, generator=torch.Generator().manual_seed(14)).to(BF16).cuda()
    w = torch.zeros(4, 2, table.shape[1] * 16, device="cuda")
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), None, w)
    assert (out[0] == 0).all() and (out[1, :3] == 0).all()
    check_kv8(out, q, cache, table, lens, 128 ** -0.5, torch.zeros_like(w), w)
    none = ops.attention_kv8(q, *cache, table, R.i32([0, 0, 0, 0]))
    assert (none == 0).all()


def test_kv8_attention_long_and_uneven():
    import alpamayo_b200.ops as ops
    lens = [9000, 1, 33, 2500]
    *cache, table = R.make_pool(lens, 32, 1, 128, 15)
    q = (torch.randn(4, 1, 7, 128, generator=torch.Generator().manual_seed(16)) * 2).to(BF16).cuda()
    w = torch.zeros(4, 1, table.shape[1] * 32, device="cuda")
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), 0.3, w)
    check_kv8(out, q, cache, table, lens, 0.3, torch.zeros_like(w), w)
    again = ops.attention_kv8(q, *cache, table, R.i32(lens), 0.3)
    assert torch.equal(out, again)                      # no order of arrival in the sums
    mass = w.sum(-1).cpu()
    assert torch.allclose(mass, torch.full_like(mass, 7.0), rtol=1e-4, atol=0)   # 7 heads' weights sum to 1 each


@pytest.mark.parametrize("ratio", [1e-6, 1e6])
def test_kv8_attention_page_scales_of_very_different_sizes(ratio):
    import alpamayo_b200.ops as ops
    lens = [200]
    *cache, table = R.make_pool(lens, 16, 1, 128, 17)
    cache[3][table[0, 2:5].long()] *= ratio
    cache[3][table[0, 7].long()] = 0.0
    q = torch.randn(1, 1, 4, 128, generator=torch.Generator().manual_seed(18)).to(F16).cuda()
    out = ops.attention_kv8(q, *cache, table, R.i32(lens))
    k, v = R.read(cache, 0, table, 0, 0, 200)[:, None], R.read(cache, 1, table, 0, 0, 200)[:, None]
    ref, _, size, sb = R.attend(q[0].double().cpu(), k, v, 128 ** -0.5)
    bound = R.out_bound(ref, size, sb, F16, 2.0 ** -11) + 2.0 ** -25   # fp16 output: values below 2^-14 are subnormal
    inside = ref.abs() < 65000
    got = out[0].double().cpu()
    assert float(((got - ref).abs() / bound)[inside].max()) <= 1.0


def test_kv8_attention_q_of_extreme_sizes():
    import alpamayo_b200.ops as ops
    lens = [100, 100, 100]
    *cache, table = R.make_pool(lens, 16, 1, 64, 19)
    g = torch.Generator().manual_seed(20)
    q = torch.randn(3, 1, 2, 64, generator=g)
    q[0] *= 1e-30
    q[1] = 0
    q[2] *= 1e30
    q = q.to(BF16).cuda()
    scale = 1e-31
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), scale)
    check_kv8(out, q, cache, table, lens, scale)


def test_kv8_attention_scale_behind_the_last_token_is_not_seen():
    import alpamayo_b200.ops as ops
    lens = [20]
    *cache, table = R.make_pool([64], 16, 2, 128, 21)
    q = torch.randn(1, 1, 4, 128, generator=torch.Generator().manual_seed(22)).to(BF16).cuda()
    want = ops.attention_kv8(q, *cache, table, R.i32(lens))
    for b in (2, 3):                                    # pages behind the last token: nothing of them is seen
        cache[2][table[0, b].long()] = float("nan")
        cache[3][table[0, b].long()] = float("inf")
    assert torch.equal(ops.attention_kv8(q, *cache, table, R.i32(lens)), want)
    cache[3][table[0, 0].long(), 1] = float("nan")      # a seen one shows, in its head alone
    got = ops.attention_kv8(q, *cache, table, R.i32(lens))
    assert torch.equal(got[:, :, :2], want[:, :, :2]) and torch.isnan(got[:, :, 2:]).all()
    cache[3][table[0, 0].long(), 1] = 0.01
    cache[2][table[0, 1].long(), 0] = float("nan")
    assert torch.isnan(ops.attention_kv8(q, *cache, table, R.i32(lens))[:, :, :2]).all()


def test_kv8_attention_pool_beyond_32_bits():
    import alpamayo_b200.ops as ops
    page, D, pages = 128, 128, 140000                   # 2.3e9 codes a side
    codes = [torch.empty(pages, 1, page, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, 1, device="cuda") for _ in range(2)]
    lens = [300, 140]
    table = R.i32([[pages - 1, pages - 7, 3], [pages - 2, 135000, -1]])
    g = torch.Generator(device="cuda").manual_seed(23)
    kv = torch.randn(440, 2, 1, D, generator=g, device="cuda").to(BF16)
    cache = (*codes, *scales)
    ops.kv8_append(kv[:, 0], kv[:, 1], R.cu(lens), R.i32([0, 0]), *cache, table)
    k, v = ops.kv8_gather(*cache, table, R.i32([0, 0]), R.cu(lens), 440, torch.float32)
    assert float((k - kv[:, 0].float()).abs().max()) < 0.03 and float((v - kv[:, 1].float()).abs().max()) < 0.03
    q = torch.randn(2, 1, 4, D, generator=g, device="cuda").to(BF16)
    small = [t[table.flatten().clamp(min=0).long()].contiguous() for t in cache]
    small_table = R.i32([[0, 1, 2], [3, 4, -1]])
    assert torch.equal(ops.attention_kv8(q, *cache, table, R.i32(lens)),
                       ops.attention_kv8(q, *small, small_table, R.i32(lens)))


def test_kv8_attention_strided_queries_stream_and_graph():
    import alpamayo_b200.ops as ops
    lens = [333, 20]
    *cache, table = R.make_pool(lens, 64, 2, 128, 24)
    x = torch.randn(2, 1, 10, 128, generator=torch.Generator().manual_seed(25)).to(BF16).cuda()
    q, n = x[:, :, :6], R.i32(lens)                     # the query heads of a fused projection
    want = ops.attention_kv8(q.contiguous(), *cache, table, n)
    assert torch.equal(ops.attention_kv8(q, *cache, table, n), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.attention_kv8(q, *cache, table, n)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.attention_kv8(q, *cache, table, n)
    n.copy_(R.i32([250, 20]))                           # lengths are read on the device
    want = ops.attention_kv8(q, *cache, table, n)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_kv8_attention_bad_pages_and_lengths_are_reported():
    import alpamayo_b200.ops as ops
    lens = [40, 40]
    *cache, table = R.make_pool(lens, 16, 1, 64, 26)
    q = torch.randn(2, 1, 2, 64, generator=torch.Generator().manual_seed(27)).to(BF16).cuda()
    want = ops.attention_kv8(q, *cache, table, R.i32(lens))
    for entry in (-1, cache[0].shape[0]):
        t = table.clone()
        t[1, 1] = entry
        got = ops.attention_kv8(q, *cache, t, R.i32(lens))
        torch.cuda.synchronize()
        assert ops.device_error_word() & 8
        assert torch.equal(got[0], want[0])
    ops.attention_kv8(q, *cache, table, R.i32([40, 1000]))
    torch.cuda.synchronize()
    assert ops.device_error_word() & 8
    assert ops.device_error_word() == 0
    assert torch.equal(ops.attention_kv8(q, *cache, table, R.i32(lens)), want)


def test_refusals():
    import alpamayo_b200.ops as ops
    q, k, v = (t.cuda() for t in packed([8], [8], 4, 2, 128, BF16, 9))
    c = R.cu([8])
    ok = lambda *a: pytest.raises(RuntimeError)  # noqa: E731
    with ok():
        ops.attention_prefill(q.float(), k.float(), v.float(), c)
    with ok():
        ops.attention_prefill(q, k.half(), v, c)
    with ok():
        ops.attention_prefill(q[:, :3], k, v, c)                    # heads no multiple of kv_heads
    with ok():
        ops.attention_prefill(q[..., :96], k[..., :96], v[..., :96], c)
    with ok():
        ops.attention_prefill(q, k[:4], v[:4], c)                   # other rows, no cu_seqlens_k
    with ok():
        ops.attention_prefill(q, k, v, c.long())
    with ok():
        ops.attention_prefill(q.permute(0, 2, 1).contiguous().permute(0, 2, 1), k, v, c)
    with ok():
        ops.attention_prefill(torch.empty(8 * 4 * 128 + 1, dtype=BF16, device="cuda")[1:].view(8, 4, 128), k, v, c)
    lens = [20, 20]
    *cache, table = R.make_pool(lens, 16, 2, 128, 30)
    n = R.i32(lens)
    q = torch.zeros(2, 1, 4, 128, dtype=BF16, device="cuda")
    w = torch.zeros(2, 2, 32, device="cuda")
    with ok():
        ops.attention_kv8(q.float(), *cache, table, n)
    with ok():
        ops.attention_kv8(q[:, :, :3], *cache, table, n)
    with ok():
        ops.attention_kv8(q[..., :64], *cache, table, n)
    with ok():
        ops.attention_kv8(q, *cache, table, n[:1])
    with ok():
        ops.attention_kv8(q, *cache, table.long(), n)
    with ok():
        ops.attention_kv8(q, *cache, table, n, None, w[:, :, :31].contiguous())    # fewer places than the table has tokens
    with ok():
        ops.attention_kv8(q, *cache, table, n, None, w.half())
    with ok():
        ops.attention_kv8(q, cache[0], cache[1][:, :, :8].contiguous(), *cache[2:], table, n)
    with ok():
        ops.attention_kv8(torch.zeros(2, 300, 4, 128, dtype=BF16, device="cuda"), *cache, table, n)   # 600 rows a KV head
    with ok():
        ops.attention_kv8(q.cpu(), *cache, table, n)
    assert ops.attention_kv8(q[:, :0], *cache, table, n).shape == (2, 0, 4, 128)
    assert ops.attention_prefill(torch.zeros(0, 4, 128, dtype=BF16, device="cuda"),
                                 torch.zeros(0, 2, 128, dtype=BF16, device="cuda"),
                                 torch.zeros(0, 2, 128, dtype=BF16, device="cuda"), R.cu([])).shape == (0, 4, 128)
