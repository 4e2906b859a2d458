"""Argument checks of the attention and cache entry points through the C ABI:
every refusal comes before anything touches a device."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    from alpamayo_b200 import _native
    return _native.capi()


OK, INVALID, SHAPE, UNSUPPORTED, MISALIGNED, CUDA, WORKSPACE, DEVICE, TOO_LARGE = range(9)
P = 4096   # a pointer that is never followed


def cache(**kw):
    from alpamayo_b200 import _native
    v = dict(k_codes=P, v_codes=P, k_scale=P, v_scale=P, num_pages=10, kv_heads=4, page_size=16, head_dim=128)
    v.update(kw)
    return _native.Kv8Cache(**v)


def strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


def prefill(L, q=P, k=P, v=P, dtype=2, st=(3584, 128, 512, 128, 512, 128), cu=P, cu_k=P, B=1, rows=8, k_rows=8, heads=28,
            kv=4, dim=128, out=P):
    return L.paro_attention_prefill(q, k, v, dtype, strides(*st), cu, cu_k, B, rows, k_rows, heads, kv, dim, 1.0, out,
                                    None)


def test_prefill_statuses(L):
    assert prefill(L, q=None) == INVALID
    assert prefill(L, cu_k=None) == INVALID
    assert prefill(L, rows=-1) == INVALID
    assert prefill(L, kv=0) == INVALID
    assert prefill(L, dtype=0) == UNSUPPORTED
    assert prefill(L, dtype=9) == UNSUPPORTED
    assert prefill(L, heads=27) == SHAPE
    assert prefill(L, dim=96) == SHAPE
    assert prefill(L, q=P + 2) == MISALIGNED
    assert prefill(L, st=(3584, 127, 512, 128, 512, 128)) == MISALIGNED
    assert prefill(L, st=(-8, 128, 512, 128, 512, 128)) == MISALIGNED
    assert prefill(L, rows=1 << 31) == TOO_LARGE
    assert prefill(L, rows=0) == OK


def test_cache_statuses(L):
    st4 = strides(512, 128, 512, 128)
    app = lambda c, **kw: L.paro_kv8_append(ctypes.byref(c), kw.get("table", P), kw.get("width", 4), kw.get("k", P), P,  # noqa: E731
                                            kw.get("dtype", 2), kw.get("st", st4), P, P, kw.get("B", 2),
                                            kw.get("rows", 8), None)
    assert app(cache(k_codes=None)) == INVALID
    assert app(cache(num_pages=0)) == INVALID
    assert app(cache(), table=None) == INVALID
    assert app(cache(), width=0) == INVALID
    assert app(cache(), rows=-1) == INVALID
    assert app(cache(page_size=24)) == SHAPE
    assert app(cache(page_size=256)) == SHAPE
    assert app(cache(head_dim=96)) == SHAPE
    assert app(cache(kv_heads=2000)) == TOO_LARGE
    assert app(cache(), B=40000) == TOO_LARGE
    assert app(cache(), width=1 << 28) == TOO_LARGE
    assert app(cache(k_codes=P + 8)) == MISALIGNED
    assert app(cache(), k=P + 4) == MISALIGNED
    assert app(cache(), st=strides(512, 4, 512, 128)) == MISALIGNED
    assert app(cache(), dtype=7) == UNSUPPORTED
    assert app(cache(), rows=0) == OK
    gat = lambda **kw: L.paro_kv8_gather(ctypes.byref(cache()), P, 4, P, kw.get("cu", P), 2, kw.get("rows", 8),  # noqa: E731
                                         kw.get("k", P), P, kw.get("dtype", 2), None)
    assert gat(cu=None) == INVALID
    assert gat(k=P + 4) == MISALIGNED
    assert gat(dtype=5) == UNSUPPORTED
    assert gat(rows=0) == OK


def test_kv8_attention_statuses(L):
    st3 = strides(3584, 3584, 128)

    def att(c=None, q=P, dtype=2, st=st3, B=2, T=1, heads=28, lens=P, w=None, wo=None, cap=64, out=P, ws=P, wsb=1 << 40,
            width=4):
        return L.paro_attention_kv8(ctypes.byref(c or cache()), P, width, q, dtype, st, B, T, heads, lens, 1.0, w, wo, cap,
                                    out, ws, wsb, None)
    assert att(q=None) == INVALID
    assert att(lens=None) == INVALID
    assert att(w=P) == INVALID                       # weights without weights_out
    assert att(dtype=0) == UNSUPPORTED
    assert att(heads=30) == SHAPE
    assert att(w=P, wo=P, cap=63) == SHAPE
    assert att(T=200) == TOO_LARGE
    assert att(ws=P + 16) == MISALIGNED
    assert att(st=strides(3584, 3584, 12)) == MISALIGNED
    assert att(wsb=16) == WORKSPACE
    assert att(T=0) == OK
    size = L.paro_attention_kv8_workspace_size
    assert size(ctypes.byref(cache()), 4, 2, 200, 28, 0) == 0
    assert size(ctypes.byref(cache()), 4, 2, 1, 27, 0) == 0
    small, large = (size(ctypes.byref(cache()), 4, 2, 1, 28, w) for w in (0, 1))
    assert 0 < small < large


def test_evict_statuses(L):
    def ev(w=P, cap=64, budget=32, sink=4, recent=8, kept=P, width=2, B=2):
        return L.paro_kv8_evict(ctypes.byref(cache()), P, 4, w, cap, P, B, budget, sink, recent, kept, P, P, P, width, None)
    assert ev(w=None) == INVALID
    assert ev(kept=None) == INVALID
    assert ev(budget=0) == INVALID
    assert ev(sink=30, recent=3) == INVALID
    assert ev(sink=-1) == INVALID
    assert ev(budget=33) == SHAPE                    # two pages of 16
    assert ev(cap=63) == SHAPE
    assert ev(B=0) == OK


def test_misaligned_index_and_weight_pointers(L):
    odd = P + 2                                      # int32 and float32 arrays begin on 4-byte boundaries
    c, table = cache(), P
    st4, st3 = strides(512, 128, 512, 128), strides(3584, 3584, 128)
    app = lambda cu=P, starts=P: L.paro_kv8_append(ctypes.byref(c), table, 4, P, P, 2, st4, cu, starts, 2, 8, None)  # noqa: E731
    gat = lambda cu=P, starts=P: L.paro_kv8_gather(ctypes.byref(c), table, 4, starts, cu, 2, 8, P, P, 2, None)  # noqa: E731
    att = lambda lens=P, w=P, wo=P: L.paro_attention_kv8(ctypes.byref(c), table, 4, P, 2, st3, 2, 1, 28, lens, 1.0, w,  # noqa: E731
                                                         wo, 64, P, P, 1 << 40, None)
    ev = lambda w=P, lens=P, kept=P, nw=P, nl=P, out=P: L.paro_kv8_evict(ctypes.byref(c), table, 4, w, 64, lens, 2, 32, 4,  # noqa: E731
                                                                         8, kept, nw, nl, out, 2, None)
    assert app(cu=odd) == app(starts=odd) == MISALIGNED
    assert gat(cu=odd) == gat(starts=odd) == MISALIGNED
    assert att(lens=odd) == att(w=odd) == att(wo=odd) == MISALIGNED
    assert [ev(**{k: odd}) for k in ("w", "lens", "kept", "nw", "nl", "out")] == [MISALIGNED] * 6


def test_sizes_next_to_the_largest_int(L):
    # the kernels step through rows and tokens in ints, some thousands at a time
    top = 0x7FFFFFFF
    st4 = strides(512, 128, 512, 128)
    c = cache()
    ev = lambda budget, width: L.paro_kv8_evict(ctypes.byref(c), P, 4, P, 64, P, 2, budget, 4, 8, P, P, P, P, width, None)  # noqa: E731
    assert ev(top, 1 << 27) == TOO_LARGE
    assert ev(top - 4000, 1 << 27) == TOO_LARGE
    assert L.paro_kv8_append(ctypes.byref(c), P, top // 16, P, P, 2, st4, P, P, 2, 8, None) == TOO_LARGE
    assert prefill(L, rows=top) == TOO_LARGE
    assert prefill(L, k_rows=top) == TOO_LARGE
