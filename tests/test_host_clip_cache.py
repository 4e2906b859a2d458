"""ClipCache's bookkeeping of pages and lengths, which is host work: a cache on
the CPU, whose operators (CUDA only) are not reached or fail."""
import pytest
import torch

H, G, D = 6, 2, 128


def new(clips, **kw):
    from alpamayo_b200 import ClipCache
    kw = dict(dict(layers=2, clips=clips, capacity=256, heads=H, kv_heads=G, head_dim=D, page_size=16, device="cpu"), **kw)
    return ClipCache(**kw)


def books(c):
    return sorted(c.free), [list(p) for p in c.pages], list(c.lens), c.table.tolist(), c.seq_lens.tolist()


def test_evict_that_fails_keeps_every_page():
    c = new(3, totals=True, capacity=64)
    c.prompt([64, 64, 48])
    c.free += [100, 101, 102]                              # room for the first clip's two pages, not for all
    before = books(c)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.evict(32)
    assert books(c) == before


@pytest.mark.parametrize("budget,sink,recent", [(0, 0, 0), (-3, 0, 0), (2, 4, 0), (20, 12, 9), (20, -1, 0), (20, 0, -1)])
def test_evict_refuses_before_it_takes_pages(budget, sink, recent):
    c = new(2, totals=True, spare=64)
    c.prompt([64, 40])
    before = books(c)
    with pytest.raises(ValueError):
        c.evict(budget, sink=sink, recent=recent)
    assert books(c) == before


def test_evict_gives_pages_back_when_a_layer_fails(monkeypatch):
    import alpamayo_b200.kv_cache as kv
    c = new(2, totals=True, spare=64)
    c.prompt([64, 40])
    before, totals, calls = books(c), [t.clone() for t in c.totals], []

    def fails_in_the_second_layer(cache, weights, table, seq_lens, out_table, budget, sink=4, recent=0):
        calls.append(0)
        if len(calls) == 2:
            raise RuntimeError("no")
        shape = (2, G, budget)
        return torch.zeros(shape, dtype=torch.int32), torch.ones(shape), seq_lens
    monkeypatch.setattr(kv.KV8Cache, "evict", fails_in_the_second_layer)
    with pytest.raises(RuntimeError, match="no"):
        c.evict(32)
    assert books(c) == before and all(torch.equal(a, b) for a, b in zip(c.totals, totals))


def test_verify_refuses_more_rows_than_the_kernels_take():
    # 512 query rows to a KV head: 170 tokens at three heads each
    c = new(2, capacity=256)
    before = books(c)
    for tokens in (171, 200, -1):
        with pytest.raises(ValueError):
            c.verify(tokens)
        assert books(c) == before
    c.verify(170)
    assert c.lens == [170, 170]
