"""Attention and cache operators where an input or a table is out of the
ordinary: infinite scores, rows of no sequence, pages that are not there,
values of extreme sizes."""
import ctypes

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


@pytest.fixture(autouse=True)
def _clean_error_word(request):
    import alpamayo_b200.ops as ops
    ops.device_error_word()
    yield
    if "bad_" not in request.node.name:
        assert ops.device_error_word() == 0


def prefill_into_dirty_memory(q, k, v, cu_q, cu_k=None, scale=None):
    """attention_prefill with an output that lies where the same number of
    bytes held 123 before: a place that is not written shows."""
    import alpamayo_b200.ops as ops
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    dirty = [torch.full(q.shape, 123.0, dtype=q.dtype, device="cuda") for _ in range(4)]
    del dirty
    return ops.attention_prefill(q, k, v, cu_q, cu_k, scale)


def prefill_unsplit(q, k, v, cu_q, cu_k):
    """The entry point without a workspace, whose rows are never shared out."""
    from alpamayo_b200 import _native
    out = torch.full_like(q, 123.0)
    st = (ctypes.c_int64 * 6)(*(t.stride(d) for t in (q, k, v) for d in (0, 1)))
    rc = _native.capi().paro_attention_prefill(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 2 if q.dtype == BF16 else 1, st, cu_q.data_ptr(), cu_k.data_ptr(),
        cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[2] ** -0.5,
        out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out


def shared_out(q_rows, k_rows, heads, kv_heads, dim, dtype, seed):
    from alpamayo_b200 import _native
    assert _native.capi().paro_attention_prefill_workspace_size(1, q_rows, k_rows, heads, dim) > 0
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(q_rows, heads, dim, generator=g) * 1.5).to(dtype)
    q[:, :, 3] = torch.where(q[:, :, 3] == 0, torch.ones_like(q[:, :, 3]), q[:, :, 3])
    return q, *(torch.randn(k_rows, kv_heads, dim, generator=g).to(dtype) for _ in range(2))


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("at", [5, 2600, 4000])
def test_prefill_infinite_key_in_keys_shared_out(at, dim, dtype):
    # a score of +inf makes the row NaN whichever part it lies in; one of
    # -inf takes the key out, i.e. the row is that of the other keys
    n, m, heads = 64, 4096, 4
    q, k, v = shared_out(n, m, heads, 2, dim, dtype, 70)
    k[at, 0, 3] = INF
    cq, ck = R.cu([n]), R.cu([m])
    out = prefill_into_dirty_memory(q.cuda(), k.cuda(), v.cuda(), cq, ck)
    want_nan = torch.zeros(n, heads, dtype=torch.bool)
    want_nan[:, :2] = q[:, :2, 3] > 0
    if at > m - n:                                        # the first rows do not see it
        want_nan[:at - (m - n)] = False
    assert torch.equal(torch.isnan(out).all(-1).cpu(), want_nan)
    assert torch.equal(torch.isnan(out).any(-1).cpu(), want_nan)
    assert torch.equal(torch.isnan(prefill_unsplit(q.cuda(), k.cuda(), v.cuda(), cq, ck)).any(-1).cpu(), want_nan)
    for i in (0, n // 2, n - 1):
        for h in range(heads):
            if want_nan[i, h]:
                continue
            keep = torch.arange(i + 1 + m - n)
            if h < 2:
                keep = keep[keep != at]
            ref, _, size, sb = R.attend(q[i:i + 1, h:h + 1].double(), k[keep, h // 2:h // 2 + 1].double(),
                                        v[keep, h // 2:h // 2 + 1].double(), dim ** -0.5)
            bound = R.out_bound(ref, size, sb, dtype, R.UNIT[dtype]) + (2.0 ** -25 if dtype == F16 else 0.0)
            assert R.max_excess(out[i:i + 1, h:h + 1], ref, bound) <= 1.0, (i, h)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("first,q_lens,k_lens", [(7, [33, 40], None), (300, [20, 0, 290], None), (5, [50, 9], [70, 4]),
                                                 (40, [60, 30], [3000, 30]), (260, [3], [2600])])
def test_prefill_rows_before_the_first_sequence_are_zero(first, q_lens, k_lens, dim, dtype):
    import alpamayo_b200.ops as ops
    end = first + sum(q_lens)
    rows, m = end + 11, sum(k_lens or q_lens)
    k_first = 2 if k_lens else first
    k_rows = m + k_first + 3 if k_lens else rows
    g = torch.Generator().manual_seed(71)
    q = torch.randn(rows, 4, dim, generator=g).to(dtype).cuda()
    k, v = (torch.randn(k_rows, 2, dim, generator=g).to(dtype).cuda() for _ in range(2))
    cq = R.cu(q_lens) + first
    ck = R.cu(k_lens) + k_first if k_lens else None
    out = prefill_into_dirty_memory(q, k, v, cq, ck)
    assert (out[:first] == 0).all() and (out[end:] == 0).all()
    want = ops.attention_prefill(q[first:end].contiguous(), k[k_first:k_first + m].contiguous(),
                                 v[k_first:k_first + m].contiguous(), R.cu(q_lens), R.cu(k_lens) if k_lens else None)
    # the rows before the first sequence move its tiles: the same sums in another order
    diff = (out[first:end].double() - want.double()).abs()
    assert float(diff.max()) <= 4 * R.UNIT[dtype] * float(v.abs().max())


def test_gather_rows_outside_the_ranges_are_zero():
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([100, 40, 0, 70], 16, 3, 64, 72)
    starts, lens, first = [37, 0, 0, 5], [50, 40, 0, 60], 70
    want_k, want_v = ops.kv8_gather(*cache, table, R.i32(starts), R.cu(lens), 150, F32)
    k, v = ops.kv8_gather(*cache, table, R.i32(starts), R.cu(lens) + first, 230, F32)
    for got, want in ((k, want_k), (v, want_v)):
        assert (got[:first] == 0).all() and (got[220:] == 0).all()
        assert torch.equal(got[first:220], want)


def attend_seen(q, k, v, see, scale):
    """q [h, d], k / v [m, g, d] in 64 bits, see [m]: output, weights [h, m],
    and the parts of R.out_bound, over the tokens of `see` alone."""
    h, d, m = q.shape[0], q.shape[1], k.shape[0]
    out, w = torch.zeros(1, h, d, dtype=torch.float64), torch.zeros(h, m, dtype=torch.float64)
    size, sb = torch.zeros(1, h, d, dtype=torch.float64), torch.zeros(h, 1, dtype=torch.float64)
    js = see.nonzero()[:, 0]
    if len(js):
        o, p, size, sb = R.attend(q[None], k[js], v[js], scale)
        out, w[:, js] = o, p[:, 0]
    return out, w, size, sb


@pytest.mark.parametrize("heads,kv_heads,dim,T", [(2, 1, 64, 1), (14, 2, 128, 1), (12, 1, 64, 1), (6, 2, 128, 9), (16, 1, 64, 6)])
@pytest.mark.parametrize("page", [16, 64])
def test_kv8_attention_tokens_of_bad_pages_are_left_out(page, heads, kv_heads, dim, T):
    # page 0 belongs to another sequence: nothing of it may show
    import alpamayo_b200.ops as ops
    lens = [5 * page - 3, 3 * page, 2 * page - 1, 4 * page]
    *cache, table = R.make_pool(lens, page, kv_heads, dim, 73)
    cache[2][0], cache[3][0] = 50.0, 50.0
    bad = {0: [1, 4], 1: [0], 2: [0, 1], 3: []}
    for b, blocks in bad.items():
        for i, blk in enumerate(blocks):
            table[b, blk] = -1 - i if i % 2 else cache[0].shape[0] + b
    q = torch.randn(4, T, heads, dim, generator=torch.Generator().manual_seed(74)).to(BF16).cuda()
    w = torch.full((4, kv_heads, table.shape[1] * page), 3.0, device="cuda")
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), None, w)
    assert ops.device_error_word() & 8
    again = ops.attention_kv8(q, *cache, table, R.i32(lens))
    assert ops.device_error_word() & 8 and torch.equal(out, again)
    w = w.cpu().double()
    for b, n in enumerate(lens):
        ok = torch.ones(n, dtype=torch.bool)
        for blk in bad[b]:
            ok[blk * page:(blk + 1) * page] = False
        t = table.clone()
        t[b, bad[b]] = 0
        k, v = (torch.stack([R.read(cache, which, t, b, h, n) for h in range(kv_heads)], 1) for which in (0, 1))
        mass = torch.zeros(kv_heads, n, dtype=torch.float64)
        err = torch.zeros(kv_heads, n, dtype=torch.float64)
        for i in range(T):
            see = ok & (torch.arange(n) <= n - T + i)
            ref, p, size, sb = attend_seen(q[b, i].double().cpu(), k, v, see, dim ** -0.5)
            if not see.any():
                assert (out[b, i] == 0).all()
            assert R.max_excess(out[b, i:i + 1], ref, R.out_bound(ref, size, sb, BF16, 2.0 ** -11)) <= 1.0, (b, i)
            mass += p.view(kv_heads, -1, n).sum(1)
            err += (p * (2.0 * sb + 2.0 ** -18)).view(kv_heads, -1, n).sum(1)
        got = w[b, :, :n] - 3.0
        # 3 + the mass, rounded to float32
        assert ((got - mass).abs() <= err + (3.0 + mass) * 2.0 ** -23).all(), b
        assert (got[:, ~ok] == 0).all()


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n,m", [(40, 40), (64, 4096)])
def test_prefill_rows_of_minus_infinity_are_nan(n, m, dim, dtype):
    # every seen score -inf: 0 / 0 by the formula, whether keys are shared out or not
    q, k, v = shared_out(n, m, 4, 2, dim, dtype, 75) if m > n else (t.clone() for t in shared_out(64, 4096, 4, 2, dim, dtype, 75))
    q, k, v = q[:n], k[:m], v[:m]
    q[:, :2, 3] = q[:, :2, 3].abs()
    k[:, 0, 3] = -INF
    cq, ck = R.cu([n]), R.cu([m])
    for out in (prefill_into_dirty_memory(q.cuda(), k.cuda(), v.cuda(), cq, ck), prefill_unsplit(q.cuda(), k.cuda(), v.cuda(), cq, ck)):
        assert torch.isnan(out[:, :2]).all() and torch.isfinite(out[:, 2:]).all()
    # one seen score is finite: its value alone
    k[0, 0, 3] = 0.0
    for out in (prefill_into_dirty_memory(q.cuda(), k.cuda(), v.cuda(), cq, ck), prefill_unsplit(q.cuda(), k.cuda(), v.cuda(), cq, ck)):
        assert torch.equal(out[:, :2].cpu(), v[0, 0].expand(n, 2, dim))


@pytest.mark.parametrize("heads,T", [(2, 1), (7, 1), (12, 1), (9, 3), (8, 8)])
@pytest.mark.parametrize("n", [20, 900])
def test_kv8_attention_rows_of_minus_infinity_are_nan(n, heads, T):
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([n, 30], 16, 1, 64, 76)
    cache[0][..., 3] = -5
    q = torch.randn(2, T, heads, 64, generator=torch.Generator().manual_seed(77)).to(BF16)
    q[0, 0, 0, 3] = INF                                    # times -5 everywhere: -inf for every token
    q = q.cuda()
    w = torch.zeros(2, 1, table.shape[1] * 16, device="cuda")
    out = ops.attention_kv8(q, *cache, table, R.i32([n, 30]), None, w)
    assert torch.isnan(out[0, 0, 0]).all()
    rest = out.clone()
    rest[0, 0, 0] = 0
    assert torch.isfinite(rest).all()
    assert torch.isnan(w[0, 0, :n - T + 1]).all() and torch.isfinite(w[0, 0, n - T + 1:]).all() and torch.isfinite(w[1]).all()


@pytest.mark.parametrize("factor", [2.0 ** 62, 1e25, 1e34])
@pytest.mark.parametrize("every", [True, False])
def test_kv8_attention_values_of_extreme_sizes(every, factor):
    import alpamayo_b200.ops as ops
    lens = [200, 7]
    *cache, table = R.make_pool(lens, 16, 1, 128, 78)
    big = table[0, :13] if every else table[0, 2:5]
    cache[3][big.long()] *= factor
    q = torch.randn(2, 1, 4, 128, generator=torch.Generator().manual_seed(79)).to(BF16).cuda()
    w = torch.zeros(2, 1, table.shape[1] * 16, device="cuda")
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), None, w)
    for b, n in enumerate(lens):
        k, v = R.read(cache, 0, table, b, 0, n)[:, None], R.read(cache, 1, table, b, 0, n)[:, None]
        ref, p, size, sb = R.attend(q[b].double().cpu(), k, v, 128 ** -0.5)
        assert R.max_excess(out[b], ref, R.out_bound(ref, size, sb, BF16, 2.0 ** -11)) <= 1.0, b
        mass = p.sum((0, 1))
        assert ((w[b, 0, :n].double().cpu() - mass).abs() <= mass * (2.0 * float(sb.max()) + 2.0 ** -17)).all()


def test_kv8_attention_queries_near_the_largest_bf16():
    import alpamayo_b200.ops as ops
    lens = [100, 100]
    *cache, table = R.make_pool(lens, 16, 1, 64, 80)
    q = torch.randn(2, 1, 2, 64, generator=torch.Generator().manual_seed(81))
    q[0] *= 5e37 / float(q[0].abs().max())
    q[1] *= 1e36 / float(q[1].abs().max())
    q = q.to(BF16).cuda()
    scale = 1e-37
    out = ops.attention_kv8(q, *cache, table, R.i32(lens), scale)
    for b, n in enumerate(lens):
        k, v = R.read(cache, 0, table, b, 0, n)[:, None], R.read(cache, 1, table, b, 0, n)[:, None]
        ref, _, size, sb = R.attend(q[b].double().cpu(), k, v, scale)
        assert R.max_excess(out[b], ref, R.out_bound(ref, size, sb, BF16, 2.0 ** -11)) <= 1.0, b


def test_evict_refuses_sinks_whose_sum_overflows():
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([64], 16, 1, 64, 82, extra=4)
    w = torch.rand(1, 1, 64, device="cuda")
    with pytest.raises(RuntimeError):
        ops.kv8_evict(w, *cache, table, R.i32([64]), R.i32([[0, 1]]), 32, 2 ** 62 + 5, 2 ** 62 + 5)
    with pytest.raises(RuntimeError):
        ops.kv8_evict(w, *cache, table, R.i32([64]), R.i32([[0, 1]]), 32, 4, 2 ** 63 - 1)


def test_operators_trace_as_they_run():
    # schemas (what is written, what aliases) and traced shapes against the real calls
    import alpamayo_b200.ops as ops  # noqa: F401
    _ops = torch.ops.paro_b200
    lens = [30, 9]
    *cache, table = R.make_pool(lens, 16, 2, 64, 83, extra=6)
    cache = [t.clone() for t in cache]
    used = set(table.flatten().tolist())
    free = [p for p in range(cache[0].shape[0]) if p not in used]
    q = torch.randn(39, 4, 64, device="cuda").to(BF16)
    k, v = (torch.randn(39, 2, 64, device="cuda").to(BF16) for _ in range(2))
    w = torch.rand(2, 2, table.shape[1] * 16, device="cuda")
    cu, n = R.cu(lens), R.i32(lens)
    calls = [(_ops.attention_prefill, (q, k, v, cu, None, 0.1)),
             (_ops.attention_prefill, (q[:2], k, v, R.cu([1, 1]), cu, 0.1)),
             (_ops.kv8_append, (k, v, cu, R.i32([0, 0]), *cache, table)),
             (_ops.kv8_gather, (*cache, table, R.i32([0, 0]), cu, 39, F16)),
             (_ops.attention_kv8, (q[:2, None], *cache, table, n, 0.1, None, None)),
             (_ops.attention_kv8, (q[:2, None], *cache, table, n, 0.1, w, torch.empty_like(w))),
             (_ops.kv8_evict, (w, *cache, table, n, R.i32(free[:4]).view(2, 2), 20, 2, 3))]
    for op, args in calls:
        for check in ("test_schema", "test_faketensor"):
            torch.library.opcheck(op.default, args, test_utils=check)
