"""Writing, reading back and evicting from the int8 paged cache."""
import math

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_error_word(request):
    import alpamayo_b200.ops as ops
    ops.device_error_word()
    yield
    if "bad_" not in request.node.name:
        assert ops.device_error_word() == 0


def page_step(x, old=0.0):
    """Half a quantisation step of a page whose largest value is max|x|, with float32's own rounding on top."""
    top = max(float(x.abs().max()) if x.numel() else 0.0, old)
    return top / 127 * 0.5 * (1 + 1e-5) + top * 2.0 ** -22


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv_heads,dim", [(1, 64), (4, 128), (3, 64)])
def test_append_and_gather(kv_heads, dim, page, dtype):
    import alpamayo_b200.ops as ops
    starts, lens = [0, page - 1, 5, 3 * page, 0, 17, 0], [1, 2, page + 7, 1, 2 * page, 0, 3 * page + 1]
    ends = [a + b for a, b in zip(starts, lens)]
    *cache, table = R.make_pool(ends, page, kv_heads, dim, 31)
    before = [t.clone() for t in cache]
    g = torch.Generator().manual_seed(32)
    kv = (torch.randn(sum(lens), 2, kv_heads, dim, generator=g) * torch.tensor([1.0, 4.0])[None, :, None, None]).to(dtype)
    dev = kv.cuda()
    ops.kv8_append(dev[:, 0], dev[:, 1], R.cu(lens), R.i32(starts), *cache, table)
    got = ops.kv8_gather(*cache, table, R.i32([0] * len(ends)), R.cu(ends), sum(ends), F32)
    at = row = 0
    for b, n in enumerate(ends):
        for which in range(2):
            for h in range(kv_heads):
                new = kv[at:at + lens[b], which, h].double()
                old = R.read(before, which, table, b, h, n)
                x = torch.cat([old[:starts[b]], new])
                y = got[which][row:row + n, h].double().cpu()
                assert torch.equal(y, R.read(cache, which, table, b, h, n).float().double()) or \
                    float((y - R.read(cache, which, table, b, h, n)).abs().max()) <= float(y.abs().max()) * 2.0 ** -23
                for p0 in range(0, n, page):
                    p1 = min(n, p0 + page)
                    if p1 <= starts[b]:
                        assert torch.equal(x[p0:p1].float(), y[p0:p1].float())       # pages not written stay
                        continue
                    had = starts[b] > p0
                    prior = float(before[2 + which][table[b, p0 // page].long(), h]) * 127 if had else 0.0
                    first = max(p0, starts[b])
                    step = page_step(x[first:p1], prior)
                    assert float((x[p0:p1] - y[p0:p1]).abs().max()) <= step, (b, which, h, p0)
        at, row = at + lens[b], row + n
    # pages of no sequence are not written
    used = set(table.flatten().tolist())
    for p in range(cache[0].shape[0]):
        if p not in used:
            assert all(torch.equal(x[p], y[p]) for x, y in zip(cache, before))
    # the same call again changes nothing
    then = [t.clone() for t in cache]
    ops.kv8_append(dev[:, 0], dev[:, 1], R.cu(lens), R.i32(starts), *cache, table)
    assert all(torch.equal(x, y) for x, y in zip(cache, then))


def test_append_token_by_token_keeps_up_with_growing_values():
    import alpamayo_b200.ops as ops
    page, n = 16, 40
    *cache, table = R.make_pool([n], page, 2, 64, 33)
    g = torch.Generator().manual_seed(34)
    x = torch.randn(n, 2, 64, generator=g) * torch.linspace(0.1, 5.0, n)[:, None, None]
    for t in range(n):
        one = x[t:t + 1].cuda()
        ops.kv8_append(one, one, R.cu([1]), R.i32([t]), *cache, table)
    k, v = ops.kv8_gather(*cache, table, R.i32([0]), R.cu([n]), n, F32)
    assert torch.equal(k, v)
    for p0 in range(0, n, page):
        p1 = min(n, p0 + page)
        for h in range(2):
            y = x[p0:p1, h].double()
            # every growth of the scale rounds the older codes once more: half a step of each scale in turn
            tops = torch.cummax(y.abs().amax(1), 0).values
            grown = sorted(set(tops.tolist()))
            step = sum(s / 127 * 0.5 for s in grown) * (1 + 1e-4) + 1e-6
            assert float((k[p0:p1, h].double().cpu() - y).abs().max()) <= step
            last = tops[-1] / 127 * 0.5 * (1 + 1e-5) + 1e-6
            assert float((k[p1 - 1, h].double().cpu() - y[-1]).abs().max()) <= last


def test_append_codes_are_the_nearest_integers():
    import alpamayo_b200.ops as ops
    page = 16
    *cache, table = R.make_pool([page], page, 1, 64, 35)
    x = torch.zeros(page, 1, 64)
    x[0, 0, 0] = 127.0                                       # scale 1
    x[1, 0, :9] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 0.49, -126.5, 126.4, -127.0])
    ops.kv8_append(x.cuda(), x.cuda(), R.cu([page]), R.i32([0]), *cache, table)
    id_ = int(table[0, 0])
    assert float(cache[2][id_, 0]) == 1.0
    assert cache[0][id_, 0, 1, :9].tolist() == [0, 2, 2, 0, -2, 0, -126, 126, -127]
    zero = torch.zeros(page, 1, 64, device="cuda")
    ops.kv8_append(zero, zero, R.cu([page]), R.i32([0]), *cache, table)
    assert float(cache[2][id_, 0]) == 0.0 and (cache[0][id_] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_append_values_that_are_not_finite_show(bad):
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([48], 16, 2, 64, 36)
    x = torch.randn(48, 2, 64, generator=torch.Generator().manual_seed(37))
    x[20, 1, 3] = bad
    ops.kv8_append(x.cuda(), x.cuda(), R.cu([48]), R.i32([0]), *cache, table)
    k, _ = ops.kv8_gather(*cache, table, R.i32([0]), R.cu([48]), 48, F32)
    wrong = torch.isnan(k).all(-1).cpu()
    want = torch.zeros(48, 2, dtype=torch.bool)
    want[16:32, 1] = True
    assert torch.equal(wrong, want) and torch.isfinite(k.cpu()[~want]).all()


def test_append_reads_strided_projections():
    import alpamayo_b200.ops as ops
    lens = [30, 3]
    *cache, table = R.make_pool(lens, 16, 2, 128, 38)
    x = torch.randn(33, 8, 128, generator=torch.Generator().manual_seed(39)).to(BF16).cuda()
    other = [t.clone() for t in cache]
    ops.kv8_append(x[:, 4:6], x[:, 6:], R.cu(lens), R.i32([0, 0]), *cache, table)
    ops.kv8_append(x[:, 4:6].contiguous(), x[:, 6:].contiguous(), R.cu(lens), R.i32([0, 0]), *other, table)
    assert all(torch.equal(a, b) for a, b in zip(cache, other))


def test_gather_ranges():
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([100, 40, 0, 70], 16, 3, 64, 40)
    starts, lens = [37, 0, 0, 69], [50, 40, 0, 1]
    k, v = ops.kv8_gather(*cache, table, R.i32(starts), R.cu(lens), 95, BF16)   # 91 rows, then zeros
    row = 0
    for b, (a, n) in enumerate(zip(starts, lens)):
        for h in range(3):
            for which, y in enumerate((k, v)):
                want = R.read(cache, which, table, b, h, a + n)[a:]
                # one float32 product, rounded once more to bf16
                assert float(((y[row:row + n, h].double().cpu() - want).abs() - want.abs() * (2.0 ** -8 + 2.0 ** -23)).max()
                             if n else 0.0) <= 0
        row += n
    assert (k[91:] == 0).all() and (v[91:] == 0).all()
    assert ops.kv8_gather(*cache, table, R.i32([0] * 4), R.cu([0] * 4), 0)[0].shape == (0, 3, 64)


def test_append_and_gather_bad_pages_are_reported_and_left_out():
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([32, 32], 16, 1, 64, 41)
    before = [t.clone() for t in cache]
    x = torch.ones(64, 1, 64, device="cuda")
    t = table.clone()
    t[0, 1], t[1, 0] = -5, cache[0].shape[0] + 3
    ops.kv8_append(x, x, R.cu([32, 32]), R.i32([0, 0]), *cache, t)
    assert ops.device_error_word() & 8
    for b, p, written in ((0, 0, True), (0, 1, False), (1, 0, False), (1, 1, True)):
        page = int(table[b, p])
        assert torch.equal(cache[0][page], before[0][page]) != written
    k, _ = ops.kv8_gather(*cache, t, R.i32([0, 0]), R.cu([32, 32]), 64, F32)
    assert ops.device_error_word() & 8
    assert (k[16:48] == 0).all() and (k[:16] != 0).all()
    ops.kv8_append(x, x, R.cu([32, 32]), R.i32([0, 30]), *cache, table)         # past the table's row
    assert ops.device_error_word() & 8
    assert ops.device_error_word() == 0


# --------------------------------------------------------------------------
# eviction
# --------------------------------------------------------------------------
def keep_ref(w, n, budget, sink, recent):
    if n <= budget:
        return list(range(n))
    fixed = set(range(sink)) | set(range(n - recent, n))
    key = lambda i: (0 if math.isnan(w[i]) else 1, -w[i] if not math.isnan(w[i]) else 0.0, i)  # noqa: E731
    free = sorted((i for i in range(n) if i not in fixed), key=key)
    return sorted(list(fixed) + free[:budget - len(fixed)])


def run_evict(lens, page, kv_heads, dim, budget, sink, recent, weights, seed):
    import alpamayo_b200.ops as ops
    width = math.ceil(budget / page)
    *cache, table = R.make_pool(lens, page, kv_heads, dim, seed, extra=len(lens) * width + 2)
    used = set(table.flatten().tolist())
    free = [p for p in range(cache[0].shape[0]) if p not in used]
    out_table = R.i32(free[:len(lens) * width]).view(len(lens), width)
    cap = table.shape[1] * page + 3
    w = torch.zeros(len(lens), kv_heads, cap)
    for b, n in enumerate(lens):
        w[b, :, :n] = weights(b, kv_heads, n)
    w = w.cuda()
    before = [t.clone() for t in cache]
    kept, nw, nl = ops.kv8_evict(w, *cache, table, R.i32(lens), out_table, budget, sink, recent)
    assert nl.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        for h in range(kv_heads):
            want = keep_ref(w[b, h].tolist(), n, budget, sink, recent)
            assert kept[b, h].tolist() == want + [-1] * (budget - len(want)), (b, h)
            got_w = nw[b, h].cpu()
            src_w = w[b, h].cpu()[want]
            assert torch.equal(got_w[:len(want)].nan_to_num(-9.0), src_w.nan_to_num(-9.0))
            assert (got_w[len(want):] == 0).all()
            for which in range(2):
                x = R.read(before, which, table, b, h, n)[want]
                y = R.read(cache, which, out_table, b, h, len(want))
                for p0 in range(0, len(want), page):
                    assert float((x[p0:p0 + page] - y[p0:p0 + page]).abs().max()) <= page_step(x[p0:p0 + page])
    # what is not a destination stays as it was
    dest = set(out_table.flatten().tolist())
    keep = [p for p in range(cache[0].shape[0]) if p not in dest]
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(cache, before))
    return kept


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("budget,sink,recent", [(50, 4, 10), (64, 0, 0), (1, 0, 0), (33, 16, 17), (20, 0, 20), (300, 4, 1)])
def test_evict(budget, sink, recent, page):
    g = torch.Generator().manual_seed(50)
    run_evict([200, 51, 1, 0, 50, 1000], page, 2, 64, budget, sink, recent,
              lambda b, h, n: torch.rand(h, n, generator=g) ** 8, 51)


def test_evict_equal_weights_keep_the_lowest_index():
    g = torch.Generator().manual_seed(52)
    run_evict([3000, 1200], 32, 2, 128, 700, 3, 5, lambda b, h, n: torch.randint(0, 3, (h, n), generator=g).float(), 53)
    kept = run_evict([5000], 64, 1, 64, 100, 0, 0, lambda b, h, n: torch.zeros(h, n), 54)
    assert kept[0, 0].tolist() == list(range(100))


def test_evict_weights_of_all_kinds():
    def odd(b, h, n):
        w = torch.randn(h, n, generator=torch.Generator().manual_seed(55 + b))
        w[:, 5] = float("nan")
        w[:, 17] = float("inf")
        w[:, 30] = -float("inf")
        w[:, 40:45] = 0.0
        w[:, 45:50] = -0.0                                   # equal to 0
        w[:, 50] = torch.finfo(torch.float32).min
        w[:, 60] = 1e-42
        return w
    for budget in (3, 40, 150):
        run_evict([160, 170], 16, 2, 64, budget, 1, 2, odd, 56)


def test_evict_long_sequence():
    g = torch.Generator().manual_seed(57)
    run_evict([20000], 64, 1, 64, 3000, 4, 100, lambda b, h, n: torch.exp(torch.rand(h, n, generator=g) * 6), 58)


def test_evict_refusals_and_bad_pages():
    import alpamayo_b200.ops as ops
    *cache, table = R.make_pool([64], 16, 1, 64, 59, extra=6)
    w = torch.rand(1, 1, 64, device="cuda")
    out = R.i32([[0, 1]])
    n = R.i32([64])
    for args in ((0, 0, 0), (4, 3, 2), (33, 0, 0), (8, -1, 0), (8, 0, -2)):
        with pytest.raises(RuntimeError):
            ops.kv8_evict(w, *cache, table, n, out, *args)
    with pytest.raises(RuntimeError):
        ops.kv8_evict(w[:, :, :40].contiguous(), *cache, table, n, out, 20, 0, 0)
    with pytest.raises(RuntimeError):
        ops.kv8_evict(w.half(), *cache, table, n, out, 20, 0, 0)
    x = torch.zeros(8, 1, 64, dtype=BF16, device="cuda")
    for bad in (lambda: ops.kv8_append(x, x, R.cu([8]).long(), R.i32([0]), *cache, table),
                lambda: ops.kv8_append(x[..., :32], x[..., :32], R.cu([8]), R.i32([0]), *cache, table),
                lambda: ops.kv8_append(x.int(), x.int(), R.cu([8]), R.i32([0]), *cache, table),
                lambda: ops.kv8_append(x, x, R.cu([8]), R.i32([0, 0]), *cache, table),
                lambda: ops.kv8_gather(*cache, table, R.i32([0]), R.cu([8]), -1),
                lambda: ops.kv8_gather(cache[0][:, :, :12].contiguous(), cache[1][:, :, :12].contiguous(), *cache[2:],
                                       table, R.i32([0]), R.cu([8]), 8)):
        with pytest.raises(RuntimeError):
            bad()
    ops.kv8_evict(w, *cache, table, n, R.i32([[-1, 10 ** 6]]), 20, 0, 0)
    assert ops.device_error_word() & 8


@pytest.mark.parametrize("lens,kv_heads", [([45000, 300], 1), ([9000] * 20, 8)])
def test_evict_split_over_several_blocks_and_not(lens, kv_heads):
    # few (sequence, head)s share their tokens out to several blocks, many do not
    g = torch.Generator().manual_seed(60)
    run_evict(lens, 128, kv_heads, 64, 130, 5, 9,
              lambda b, h, n: torch.randint(0, 400, (h, n), generator=g).float(), 61)


def test_append_codes_are_the_rounded_quotients():
    # the quotient of every pair of a bf16 value and a page maximum, divided and rounded in float32
    import alpamayo_b200.ops as ops
    page = 128
    g = torch.Generator().manual_seed(62)
    n = 40 * page
    *cache, table = R.make_pool([n], page, 1, 128, 63)
    x = torch.randn(n, 1, 128, generator=g).to(BF16)
    top = x.view(40, page * 128).abs().amax(-1).float()
    x.view(40, page, 128)[:, 1, :64] = (top / 127)[:, None].to(BF16) * torch.arange(64).to(BF16)
    x.view(40, page, 128)[:, 2, 0] = (top * 0.5).to(BF16)
    ops.kv8_append(x.cuda(), x.cuda(), R.cu([n]), R.i32([0]), *cache, table)
    s = (x.view(40, page, 128).float().abs().amax((1, 2)) / torch.full((40,), 127.0))
    want = torch.round(x.view(40, page, 128).float() / s[:, None, None]).to(torch.int8)
    got = cache[0][table[0].long(), 0].cpu()
    assert torch.equal(cache[2][table[0].long(), 0].cpu(), s)
    assert torch.equal(got, want)
