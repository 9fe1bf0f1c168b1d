"""CPU tests of the cache-page entry points: what they refuse before any launch,
and the Python front end's checks."""
import ctypes as C

import numpy as np
import pytest
import torch

from c_gpt2_b200 import _lib, ops
from c_gpt2_b200.pages import PageCache
from tests.pages_oracle import Book

INVALID, UNSUPPORTED = _lib.W8A8_ERR_INVALID, _lib.W8A8_ERR_UNSUPPORTED
P = 0x10000  # an address that nothing dereferences on the host


def _pages(**kw):
    f = dict(K=P, V=P, page_stride=2 * 3 * 16 * 64, n_pages=8, page=16, n_layer=2, n_kv_head=3,
             table=P, max_pages=4, n_slot=2, n_ctx=P, refs=P)
    f.update(kw)
    return C.byref(_lib.Pages(*(f[n] for n, _ in _lib.Pages._fields_)))


@pytest.mark.parametrize("bad,status", [
    (dict(K=None), INVALID), (dict(V=None), INVALID), (dict(table=None), INVALID),
    (dict(n_ctx=None), INVALID), (dict(refs=None), INVALID),
    (dict(page=8), UNSUPPORTED), (dict(page=48), UNSUPPORTED), (dict(page=256), UNSUPPORTED),
    (dict(n_pages=0), INVALID), (dict(n_slot=0), INVALID), (dict(n_slot=8193), INVALID),
    (dict(max_pages=0), INVALID), (dict(max_pages=2 ** 31 - 1), INVALID),
    (dict(n_layer=0), INVALID), (dict(n_kv_head=0), INVALID),
    (dict(page_stride=2 * 3 * 16 * 64 - 8), INVALID), (dict(page_stride=2 * 3 * 16 * 64 + 4), INVALID),
    (dict(K=P + 8), INVALID), (dict(V=P + 2), INVALID),
])
def test_every_call_refuses_a_bad_cache(bad, status):
    lib, c = _lib.core(), _pages(**bad)
    assert lib.w8a8_pages_extend(c, P, P, None) == status
    assert lib.w8a8_pages_write(c, 0, P, 192, P, 192, 1, 1, None, P, None) == status
    assert lib.w8a8_pages_fork(c, P, P, 1, P, None) == status
    assert lib.w8a8_pages_free(c, P, 1, None) == status
    assert lib.w8a8_pages_compact(c, P, P, 1 << 20, None) == status
    assert lib.w8a8_attention_pages(c, 0, P, 192, 1, 1, None, 64, None, 0, 3, 64, P, 192, P,
                                    1 << 30, None) == status


def test_a_missing_cache_is_refused():
    assert _lib.core().w8a8_pages_free(None, P, 1, None) == INVALID
    assert _lib.core().w8a8_pages_extend(None, P, P, None) == INVALID


@pytest.mark.parametrize("n_src,n_dst,ss,ds,elems,off", [
    (0, 4, 64, 64, 64, 0), (4, 0, 64, 64, 64, 0), (4, 4, 56, 64, 64, 0), (4, 4, 64, 56, 64, 0),
    (4, 4, 68, 64, 64, 0), (4, 4, 64, 64, 60, 0), (4, 4, 64, 64, 0, 0), (4, 4, 64, 64, 64, 8),
])
def test_copy_refusals(n_src, n_dst, ss, ds, elems, off):
    assert _lib.core().w8a8_pages_copy(P + off, P, ss, n_src, P, P, ds, n_dst, elems, P, P, 1,
                                       None) == INVALID


def test_copy_of_nothing_is_ok():
    assert _lib.core().w8a8_pages_copy(P, P, 64, 1, P, P, 64, 1, 64, P, P, 0, None) == 0


def test_workspace_sizes():
    lib = _lib.core()
    assert lib.w8a8_pages_compact_workspace_size(0) == 0
    assert lib.w8a8_pages_compact_workspace_size(100) >= 3 * 400
    size = lib.w8a8_attention_pages_workspace_size
    assert size(4, 1, 12, 12, 1024, 512) > 0
    # seq, T, heads, key heads, max_ctx, shared
    for bad in [(0, 1, 12, 12, 64, 0), (1, 0, 12, 12, 64, 0), (1, 1, 12, 5, 64, 0),
                (1, 1, 12, 0, 64, 0), (1, 1, 0, 1, 64, 0), (1, 1, 12, 12, 0, 0),
                (1, 1, 12, 12, 64, 128), (1, 1, 12, 12, 64, -16), (1 << 20, 1 << 10, 12, 12, 64, 0),
                (1, 1, 12, 12, (1 << 30) + 1, 0)]:
        assert size(*bad) == 0


@pytest.mark.parametrize("n_seq,T,n_head,n_kv,max_ctx,n_shared", [
    (64, 1, 3, 3, 1 << 30, 0),            # 16-row pieces of the sequences' keys
    (256, 1, 15, 3, 1 << 30, 1 << 29),    # of what follows a prefix
    (8192, 33, 1100, 1100, 2000, 0),      # items of one sequence's rows
])
def test_calls_of_too_many_pieces_are_unsupported(n_seq, T, n_head, n_kv, max_ctx, n_shared):
    """Said before the workspace is looked at, which has no size for them, and before any
    launch; the same call with a bad argument is invalid."""
    lib = _lib.core()
    assert lib.w8a8_attention_pages_workspace_size(n_seq, T, n_head, n_kv, max_ctx, n_shared) == 0
    c = _pages(n_slot=8192, n_layer=1, n_kv_head=n_kv, page_stride=n_kv * 16 * 64)
    d = n_head * 64

    def call(ws, size, layer=0):
        return lib.w8a8_attention_pages(c, layer, P, d, n_seq, T, None, max_ctx, P, n_shared,
                                        n_head, 64, P, d, ws, size, None)
    assert call(None, 0) == UNSUPPORTED and call(P, 1 << 40) == UNSUPPORTED
    assert call(P, 1 << 40, layer=1) == INVALID


def test_a_missing_or_small_workspace_is_invalid():
    lib = _lib.core()
    size = lib.w8a8_attention_pages_workspace_size(2, 1, 3, 3, 4096, 0)
    assert size > 16
    for ws, n in ((None, size), (P, size - 1), (P + 8, size)):
        assert lib.w8a8_attention_pages(_pages(), 0, P, 192, 2, 1, None, 4096, None, 0, 3, 64, P,
                                        192, ws, n, None) == INVALID


def _cpu_cache(**kw):
    t = dict(K=torch.zeros(8, 2, 3, 16, 64, dtype=torch.bfloat16),
             V=torch.zeros(8, 2, 3, 16, 64, dtype=torch.bfloat16),
             table=torch.full((2, 4), -1, dtype=torch.int32),
             n_ctx=torch.zeros(2, dtype=torch.int32), refs=torch.zeros(8, dtype=torch.int32))
    t.update(kw)
    return PageCache(**t)


@pytest.mark.parametrize("bad,err", [
    (dict(K=torch.zeros(8, 2, 3, 16, 64)), TypeError),
    (dict(V=torch.zeros(8, 2, 3, 16, 32, dtype=torch.bfloat16)), ValueError),
    (dict(V=torch.zeros(8, 2, 3, 64, 16, dtype=torch.bfloat16).transpose(3, 4)), ValueError),
    (dict(table=torch.zeros(2, 4, dtype=torch.int64)), TypeError),
    (dict(table=torch.zeros(4, 2, dtype=torch.int32).t()), ValueError),
    (dict(table=torch.zeros(3, 4, dtype=torch.int32)), ValueError),
    (dict(n_ctx=torch.zeros(2)), TypeError),
    (dict(refs=torch.zeros(7, dtype=torch.int32)), ValueError),
    (dict(K=torch.zeros(0, 2, 3, 16, 64, dtype=torch.bfloat16),
          V=torch.zeros(0, 2, 3, 16, 64, dtype=torch.bfloat16),
          refs=torch.zeros(0, dtype=torch.int32)), ValueError),
])
def test_page_cache_refuses_tensors(bad, err):
    with pytest.raises(err):
        _cpu_cache(**bad)


def test_the_front_end_refuses_a_cache_off_the_gpu():
    c = _cpu_cache()
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.pages_extend(c, i), lambda: ops.pages_free(c, i),
                 lambda: ops.pages_fork(c, i, i), lambda: ops.pages_compact(c),
                 lambda: ops.pages_write(c, 0, c.K, c.V, i),
                 lambda: ops.attention_pages(torch.zeros(2, 192, dtype=torch.bfloat16), c, 0, 3),
                 lambda: ops.pages_copy(c.K, c.V, i, c.K, c.V, i)):
        with pytest.raises(ValueError):
            call()


def test_page_cache_takes_one_page_and_strided_pages():
    one = _cpu_cache(K=torch.zeros(1, 2, 3, 16, 64, dtype=torch.bfloat16),
                     V=torch.zeros(1, 2, 3, 16, 64, dtype=torch.bfloat16),
                     refs=torch.zeros(1, dtype=torch.int32))
    assert one.c.page_stride == 2 * 3 * 16 * 64
    kv = torch.zeros(8, 2, 2, 3, 16, 64, dtype=torch.bfloat16)  # K and V of a page side by side
    assert _cpu_cache(K=kv[:, 0], V=kv[:, 1]).c.page_stride == 2 * 2 * 3 * 16 * 64


@pytest.mark.parametrize("pools", [
    lambda n: (lambda kv: (kv[n - 1:, 0], kv[n - 1:, 1]))(
        torch.zeros(n, 2, 3, 4, 16, 64, dtype=torch.bfloat16)),   # a page of K and V side by side
    lambda n: (lambda k: (k, k.clone().transpose(0, 1).contiguous().transpose(0, 1)))(
        torch.zeros(3, 1, 4, 16, 64, dtype=torch.bfloat16).transpose(0, 1)),  # layers first
    lambda n: (lambda k: (k[2:3], k[1:2]))(torch.zeros(n, 3, 4, 16, 64, dtype=torch.bfloat16)),
    lambda n: (lambda k: (k[::4][-1:], k[1::4][-1:]))(
        torch.zeros(n, 3, 4, 16, 64, dtype=torch.bfloat16)),      # every fourth page, the last one
])
def test_a_pool_of_one_page_has_its_page_size(pools):
    """The stride of a dimension of length one says nothing of a page's size."""
    K, V = pools(9)
    assert K.shape == V.shape == (1, 3, 4, 16, 64)
    size, stride = ops._pools(K, V, -1, "K, V")[3:]
    assert size == 3 * 4 * 16 * 64 and stride == size


# ---- the oracle itself ------------------------------------------------------

def test_oracle_keeps_its_books():
    """Every page is counted once for each table entry that names it, after any
    series of calls."""
    rng = np.random.default_rng(0)
    b = Book(6, 5, 17, 16)
    for _ in range(300):
        kind = rng.integers(4)
        if kind == 0:
            b.extend(rng.integers(-1, 40, 6) * rng.integers(0, 2, 6))
        elif kind == 1:
            b.fork(rng.integers(-1, 7, 3), rng.integers(-1, 7, 3))
        elif kind == 2:
            b.free(rng.integers(-1, 7, 2))
        else:
            n, _ = b.compact()
            assert (b.refs[:n] > 0).all() and (b.refs[n:] == 0).all()
        held = b.table[b.table >= 0]
        np.testing.assert_array_equal(np.bincount(held, minlength=17), b.refs)
        np.testing.assert_array_equal((b.table >= 0).sum(1), -(-b.n_ctx // 16))
