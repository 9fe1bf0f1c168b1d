"""GPU tests of the cache pages and of the attention that reads them."""
import numpy as np
import pytest
import torch

from c_gpt2_b200 import _lib, ops
from c_gpt2_b200.pages import PageCache
from tests import pages_oracle as po

pytestmark = pytest.mark.gpu


def i32(a, device="cuda:0"):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=device)


def make(cuda, n_pages, n_slot, max_pages, n_layer=2, n_kv=3, page=16, seed=0):
    """A cache whose pools hold random values (so that a row that should not have
    been touched shows), and its oracle."""
    c = PageCache.empty(n_pages, n_slot, max_pages, n_layer, n_kv, page, cuda)
    g = torch.Generator(device=cuda).manual_seed(seed)
    for t in (c.K, c.V):
        t.copy_(torch.randn(t.shape, generator=g, device=cuda))
    return c, po.Book(n_slot, max_pages, n_pages, page)


def same_book(c, b):
    np.testing.assert_array_equal(c.table.cpu().numpy(), b.table)
    np.testing.assert_array_equal(c.n_ctx.cpu().numpy(), b.n_ctx)
    np.testing.assert_array_equal(c.refs.cpu().numpy(), b.refs)


def apply_moves(K, V, moves):
    for f, t, rows in moves:
        K[t, :, :, :rows] = K[f, :, :, :rows]
        V[t, :, :, :rows] = V[f, :, :, :rows]


# ---- bookkeeping ------------------------------------------------------------

@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_any_series_of_calls_keeps_the_oracle_books(cuda, page):
    rng = np.random.default_rng(page)
    n_slot = 7
    c, b = make(cuda, 23, n_slot, 6, n_layer=1, n_kv=2, page=page)
    K, V = c.K.clone(), c.V.clone()
    for _ in range(60):
        kind = rng.integers(5)
        if kind <= 1:
            n_new = rng.integers(-1, 3 * page, n_slot) * rng.integers(0, 2, n_slot)
            pos0 = ops.pages_extend(c, i32(n_new))
            np.testing.assert_array_equal(pos0.cpu().numpy(), b.extend(n_new))
        elif kind == 2:
            src, dst = rng.integers(-1, n_slot + 1, 4), rng.integers(-1, n_slot + 1, 4)
            status = ops.pages_fork(c, i32(src), i32(dst))
            want, moves = b.fork(src, dst)
            np.testing.assert_array_equal(status.cpu().numpy(), want)
            apply_moves(K, V, moves)
        elif kind == 3:
            slots = rng.integers(-1, n_slot + 1, 3)
            ops.pages_free(c, i32(slots))
            b.free(slots)
        else:
            n = ops.pages_compact(c)
            want, moves = b.compact()
            assert n.item() == want
            apply_moves(K, V, moves)
        same_book(c, b)
    assert torch.equal(c.K, K) and torch.equal(c.V, V)


@pytest.mark.parametrize("n_pages,n_slot", [(1, 1), (8191, 33), (8193, 1500), (40000, 8192)])
def test_pages_over_several_rounds_of_a_scan(cuda, n_pages, n_slot):
    """More pages than one round of a scan, more slots than threads, free pages few
    and far between; then all at once until the pool runs out."""
    rng = np.random.default_rng(n_pages)
    c, b = make(cuda, n_pages, n_slot, 9, n_layer=1, n_kv=1)
    b.refs[:] = rng.random(n_pages) < 0.9
    b.refs[-1] = 0
    c.refs.copy_(i32(b.refs))
    for _ in range(3):
        n_new = rng.integers(0, 60, n_slot)
        np.testing.assert_array_equal(ops.pages_extend(c, i32(n_new)).cpu().numpy(),
                                      b.extend(n_new))
        same_book(c, b)
    if n_slot > 1:
        src, dst = rng.integers(0, n_slot, n_slot), rng.permutation(n_slot)
        gone = dst[: n_slot // 2]
        ops.pages_free(c, i32(gone))
        b.free(gone)
        same_book(c, b)
        status = ops.pages_fork(c, i32(src), i32(dst))
        np.testing.assert_array_equal(status.cpu().numpy(), b.fork(src, dst)[0])
        same_book(c, b)
    assert ops.pages_compact(c).item() == b.compact()[0]
    same_book(c, b)


def test_extend_refuses_as_a_whole(cuda):
    """The pool ends inside the first slot's second request: it and the next two get
    nothing, the fourth needs no page and is served; and a row too short."""
    c, b = make(cuda, 5, 4, 4)
    for n_new in ([16, 1, 1, 10], [20, 40, 16, 3], [1, 1, 1, 1], [0, -3, 0, 64]):
        got = ops.pages_extend(c, i32(n_new)).cpu().numpy()
        np.testing.assert_array_equal(got, b.extend(n_new))
        same_book(c, b)
    assert list(b.n_ctx) == [17, 2, 2, 14]


def test_fork_runs_out_of_pages_in_list_order(cuda):
    c, b = make(cuda, 4, 6, 4)
    ops.pages_extend(c, i32([17, 0, 0, 0, 0, 0]))
    b.extend([17, 0, 0, 0, 0, 0])
    src, dst = [0, 0, 0, 0, 9], [5, 1, 3, 1, 2]
    K, V = c.K.clone(), c.V.clone()
    status = ops.pages_fork(c, i32(src), i32(dst)).cpu().numpy()
    want, moves = b.fork(src, dst)
    np.testing.assert_array_equal(status, want)
    assert list(want) == [0, 0, 2, 1, 1]
    same_book(c, b)
    apply_moves(K, V, moves)
    assert torch.equal(c.K, K) and torch.equal(c.V, V)
    # given back, named twice and out of range: each page is counted down once
    ops.pages_free(c, i32([5, 5, -1, 6, 0]))
    b.free([5, 0])
    same_book(c, b)
    assert b.refs.sum() == 2


_FORK_FIRST = """
import sys
import torch
from c_gpt2_b200 import ops
from c_gpt2_b200.pages import PageCache
ops.init(0)
for n_slot, n in (%s):
    i32 = dict(dtype=torch.int32, device="cuda:0")
    c = PageCache.empty(n + 1, n_slot, 1, 1, 1, 16, "cuda:0")
    n_new = torch.zeros(n_slot, **i32)
    n_new[0] = 5
    ops.pages_extend(c, n_new)
    dst = torch.arange(n, **i32)
    status = ops.pages_fork(c, torch.zeros_like(dst), dst)
    assert status.tolist() == [1] + [0] * (n - 1), (n_slot, n)
    assert c.n_ctx[:n].tolist() == [5] * n and c.table[:n, 0].tolist() == list(range(n))
assert ops.device_error() == 0
"""


def test_a_first_fork_whose_lists_fill_the_default_shared_memory(cuda):
    """n_slot + 2 n words at 48 KB and just below it, where the kernel's static shared
    memory comes on top, as the first forks of a process; then smaller ones and the largest."""
    import subprocess
    import sys
    for sizes in ("(4096, 4096), (64, 9), (8192, 8192)", "(8192, 2040), (4096, 4090), (2, 2)"):
        r = subprocess.run([sys.executable, "-c", _FORK_FIRST % sizes], capture_output=True,
                           text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]


def test_bad_entries_are_skipped_and_recorded(cuda):
    """Table entries outside the pool: nothing is followed, the error word is set."""
    for bad in (-7, 5, 2 ** 31 - 1):
        c, _ = make(cuda, 5, 3, 3)
        ops.pages_extend(c, i32([40, 0, 0]))
        c.table[0, 1] = bad
        refs = c.refs.clone()
        assert ops.device_error() == 0
        ops.pages_fork(c, i32([0]), i32([1]))
        assert ops.device_error() == 0x1501
        refs[0] += 1
        refs[3] += 1  # the copied last page
        assert torch.equal(c.refs, refs)
        ops.pages_free(c, i32([0, 1]))
        assert ops.device_error() == 0x1501
        assert c.refs.tolist() == [0, 1, 0, 0, 0]
    ops.pages_copy(c.K, c.V, i32([0, 5, -1]), c.K, c.V, i32([1, 2, 3]))
    assert ops.device_error() == 0x1501
    x = torch.zeros(3, 192, dtype=torch.bfloat16, device=cuda)
    ops.pages_write(c, 0, x, x, i32([48, -1, -2]))
    assert ops.device_error() == 0x1502  # behind the table
    ops.pages_write(c, 0, x, x, i32([0, -1, -2]))
    assert ops.device_error() == 0x1501  # no page there


# ---- contents ---------------------------------------------------------------

@pytest.mark.parametrize("T,page,strided", [(1, 16, True), (5, 16, False), (70, 32, True),
                                            (200, 128, False)])
def test_write_places_the_rows(cuda, T, page, strided):
    n_seq, n_kv, n_layer = 4, 3, 3
    c, b = make(cuda, 60, 5, 14, n_layer, n_kv, page, seed=T)
    first = [0, 3, page, 2 * page - 1, 0]
    ops.pages_extend(c, i32(first))
    b.extend(first)
    n_new = [T, 1, 0, max(T - 1, 1), 0]
    pos0 = ops.pages_extend(c, i32(n_new))
    b.extend(n_new)
    same_book(c, b)
    g = torch.Generator(device=cuda).manual_seed(1)
    rows = torch.randn(n_seq * T, 3 * n_kv * 64, generator=g, device=cuda).bfloat16()
    d = n_kv * 64
    Kn, Vn = (rows[:, d:2 * d], rows[:, 2 * d:]) if strided else (rows[:, d:2 * d].contiguous(),
                                                                  rows[:, 2 * d:].contiguous())
    K, V = c.K.clone(), c.V.clone()
    ops.pages_write(c, 1, Kn, Vn, pos0[:n_seq], T=T, n_new=i32(n_new[:n_seq]))
    for s in range(n_seq):
        for t in range(n_new[s]):
            pos = first[s] + t
            p = b.table[s, pos // page]
            K[p, 1, :, pos % page] = Kn[s * T + t].view(n_kv, 64)
            V[p, 1, :, pos % page] = Vn[s * T + t].view(n_kv, 64)
    assert torch.equal(c.K, K) and torch.equal(c.V, V)


@pytest.mark.parametrize("shape", [(9, 1, 1, 16), (40, 5, 3, 32), (12, 36, 20, 32)])
def test_copy_between_pools(cuda, shape):
    """Pools of other sizes and strides; pages that are not named stay as they are."""
    n, L, G, page = shape
    g = torch.Generator(device=cuda).manual_seed(n)
    kv = torch.randn(n, 2, L, G, page, 64, generator=g, device=cuda).bfloat16()
    K2 = torch.randn(n + 3, L, G, page, 64, generator=g, device=cuda).bfloat16()
    V2 = torch.randn(n + 3, L, G, page, 64, generator=g, device=cuda).bfloat16()
    src, dst = torch.randperm(n)[: n - 1], torch.randperm(n + 3)[: n - 1]
    wk, wv = K2.clone(), V2.clone()
    wk[dst.cuda()], wv[dst.cuda()] = kv[src.cuda(), 0], kv[src.cuda(), 1]
    ops.pages_copy(kv[:, 0], kv[:, 1], i32(src), K2, V2, i32(dst))
    assert torch.equal(K2, wk) and torch.equal(V2, wv)


@pytest.mark.parametrize("which", ["source", "destination", "both", "layers first"])
def test_copy_of_one_page_pools(cuda, which):
    """One page out of a pool whose pages hold K and V side by side: its neighbours in
    both pools, which one page too many would reach, stay as they are."""
    L, G, page, n = 3, 2, 16, 6
    g = torch.Generator(device=cuda).manual_seed(3)
    a = torch.randn(n, 2, L, G, page, 64, generator=g, device=cuda).bfloat16()
    b = torch.randn(n, 2, L, G, page, 64, generator=g, device=cuda).bfloat16()
    one_src, one_dst = which in ("source", "both"), which in ("destination", "both")
    ks, vs = (a[2:3, 0], a[2:3, 1]) if one_src else (a[:, 0], a[:, 1])
    if which == "layers first":  # one page, [L, 1, ...] transposed
        a = torch.randn(L, 1, G, page, 64, generator=g, device=cuda).bfloat16()
        w = torch.randn(L, 1, G, page, 64, generator=g, device=cuda).bfloat16()
        ks, vs, one_src = a.transpose(0, 1), w.transpose(0, 1), True
    kd, vd = (b[3:4, 0], b[3:4, 1]) if one_dst else (b[:, 0], b[:, 1])
    want = b.clone()
    want[3, 0] = ks[0 if one_src else 2]
    want[3, 1] = vs[0 if one_src else 2]
    before = a.clone()
    ops.pages_copy(ks, vs, i32([0 if one_src else 2]), kd, vd, i32([0 if one_dst else 3]))
    assert torch.equal(b, want) and torch.equal(a, before)
    # and the densely packed pool
    dense = torch.zeros(1, L, G, page, 64, dtype=torch.bfloat16, device=cuda)
    k2, v2 = dense.clone(), dense.clone()
    ops.pages_copy(ks, vs, i32([0 if one_src else 2]), k2, v2, i32([0]))
    assert torch.equal(k2, want[3:4, 0]) and torch.equal(v2, want[3:4, 1])


# ---- attention --------------------------------------------------------------

def build(cuda, n_seq, T, H, G, page, n_shared, tails, n_new, seed, n_layer=2, layer=1, scale=1.5,
          junk=float("nan")):
    """A cache with these tails behind a shared prefix, its unused rows filled with
    `junk`; Q; and (O, A) of the 64-bit oracle for every sequence."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=cuda).manual_seed(seed)
    ns = n_shared // page
    per = [-(-t // page) for t in tails]
    n_pages = ns + sum(per) + 3
    order = rng.permutation(n_pages)
    table = np.full((n_seq, ns + max(per + [1])), -1, np.int32)
    at = ns
    for b in range(n_seq):
        if tails[b] >= 0:
            table[b, :ns] = order[:ns]
            table[b, ns:ns + per[b]] = order[at:at + per[b]]
            at += per[b]
    n_ctx = [n_shared + t if t >= 0 else 0 for t in tails]
    shape = (n_pages, n_layer, G, page, 64)
    K = torch.full(shape, junk, dtype=torch.bfloat16, device=cuda)
    V = torch.full(shape, junk, dtype=torch.bfloat16, device=cuda)
    for b in range(n_seq):
        for k in range(-(-n_ctx[b] // page)):
            rows = min(page, n_ctx[b] - k * page)
            if k < ns and b != next(i for i in range(n_seq) if tails[i] >= 0):
                continue
            for pool in (K, V):
                pool[table[b, k], :, :, :rows] = torch.randn(
                    n_layer, G, rows, 64, generator=g, device=cuda).bfloat16()
    Q = (torch.randn(n_seq * T, H * 64, generator=g, device=cuda) * scale).bfloat16()
    c = PageCache(K, V, i32(table), i32(n_ctx), i32(np.ones(n_pages)))
    want = []
    k64, v64 = K[:, layer].double().cpu().numpy(), V[:, layer].double().cpu().numpy()
    q64 = Q.double().cpu().numpy().reshape(n_seq, T, H, 64)
    for b in range(n_seq):
        p = table[b, :-(-n_ctx[b] // page)]
        kb = k64[p].transpose(0, 2, 1, 3).reshape(-1, G, 64)[:n_ctx[b]]
        vb = v64[p].transpose(0, 2, 1, 3).reshape(-1, G, 64)[:n_ctx[b]]
        want.append(po.attention(q64[b], kb, vb, n_new[b]))
    return c, Q, i32(order[:ns]) if ns else None, want


def check(out, want, T, H, n_new, before=7.0):
    """Against the 64-bit oracle. Roundings: the output (half a step, 2^-8 of its
    value), each weight before the product with V (2^-8 of it at most, so 2^-8 of
    A = sum w |V|), and the 32-bit scores, exponentials and sums, for which 2^-11 of
    A is ample (a score of 64 products, |s| < 100: 2^-24 * 64 * 100 = 2^-11.4)."""
    got = out.double().cpu().numpy().reshape(len(want), T, H, 64)
    for b, (O, A) in enumerate(want):
        tol = 2.0 ** -8 * np.abs(O) + (2.0 ** -8 + 2.0 ** -11) * A
        err = np.abs(got[b, :n_new[b]] - O)
        assert (err <= tol).all(), (b, float((err - tol).max()))
        assert (got[b, n_new[b]:] == before).all(), "rows behind a sequence's last were touched"


CASES = [
    # n_seq, T, H, G, page, n_shared, tails
    (1, 1, 1, 1, 16, 0, [1]),
    (1, 1, 12, 12, 16, 0, [17]),
    (2, 1, 12, 12, 16, 64, [5, 32]),
    (3, 1, 4, 2, 32, 32, [0, 1, 65]),                # a tail of zero: all in the prefix
    (5, 1, 6, 3, 16, 16, [-1, 7, -1, 130, 64]),      # empty sequences among others
    (9, 1, 7, 1, 64, 640, [3, 64, 65, 100, 1, 2, 700, 128, 127]),
    (33, 1, 4, 4, 128, 1280, list(range(1, 34))),
    (70, 1, 2, 1, 16, 304, [1 + 5 * i for i in range(70)]),
    (150, 1, 2, 2, 32, 96, [1 + i % 40 for i in range(150)]),
    (2, 1, 2, 1, 16, 8000, [1, 333]),
    (2, 2, 3, 3, 16, 48, [2, 40]),
    (3, 17, 4, 2, 32, 64, [17, 20, 90]),
    (2, 64, 2, 1, 64, 128, [64, 200]),
    (2, 150, 3, 3, 16, 208, [150, 170]),
    (1, 257, 2, 2, 128, 0, [300]),
    (1, 130, 2, 2, 32, 0, [130]),
    # prefixes long enough, times rows, for the tensor-core kernel: pairs of tiles and a single
    # one, grouped heads, packed rows of padded batches, empty sequences
    (300, 1, 8, 8, 64, 1728, [1 + i % 70 for i in range(300)]),
    (100, 1, 16, 16, 16, 2304, [i % 3 for i in range(100)]),
    (40, 1, 8, 1, 128, 13056, [3 * i - 1 for i in range(40)]),
    (5, 40, 12, 4, 32, 1760, [40, 90, -1, 41, 60]),
    (70, 5, 7, 7, 16, 2000, [5 + i % 9 if i % 7 else -1 for i in range(70)]),
    (4, 100, 6, 6, 32, 2848, [100, 101, 150, 130]),
    # short prefixes of many rows, whose last block the prefix ends inside
    (260, 7, 20, 20, 16, 80, [7 + i % 9 for i in range(260)]),
    (300, 7, 32, 32, 16, 48, [7 + i % 40 for i in range(300)]),
    (130, 8, 20, 20, 32, 320, [8 + i % 30 if i % 5 else -1 for i in range(130)]),
    (130, 8, 20, 20, 64, 384, [8 + i % 30 for i in range(130)]),
    # more keys of the sequences' own than shared, and rows enough: prefix and tail in one item
    (2, 70, 4, 2, 32, 64, [70, 2300]),
    (3, 300, 2, 1, 64, 128, [300, 1500, 400]),
]


@pytest.mark.parametrize("n_seq,T,H,G,page,n_shared,tails", CASES)
def test_attention_against_64_bits(cuda, n_seq, T, H, G, page, n_shared, tails):
    n_new = [T if t >= T else max(t, 0) for t in tails]
    n_new = [min(n, T - 2 * b % T) if T > 3 else n for b, n in enumerate(n_new)]  # padded
    uniform = T == 1 and all(t >= 1 for t in tails)
    if T == 1 and not uniform:
        n_new = [1 if t >= 0 else 0 for t in tails]
    c, Q, shared, want = build(cuda, n_seq, T, H, G, page, n_shared, tails, n_new, n_seq + T)
    out = torch.full((n_seq * T, H * 64), 7.0, dtype=torch.bfloat16, device=cuda)
    ops.attention_pages(Q, c, 1, H, T=T, n_new=None if uniform else i32(n_new),
                        max_ctx=n_shared + max(tails + [1]), shared_pages=shared,
                        n_shared=n_shared, out=out)
    check(out, want, T, H, n_new)
    # the prefix read through each table row, and the loosest bound on the lengths
    if n_shared:
        again = torch.full_like(out, 7.0)
        ops.attention_pages(Q, c, 1, H, T=T, n_new=i32(n_new), out=again)
        check(again, want, T, H, n_new)


def test_a_sequence_that_ends_inside_the_prefix(cuda):
    """n_ctx below n_shared: the row sees its own n_ctx keys of the prefix only; with
    none, or more new rows than positions, rows are zero."""
    c, Q, shared, _ = build(cuda, 4, 3, 2, 2, 16, 160, [3, 3, 3, 3], [3] * 4, 3, junk=0.0)
    lens = [163, 50, 2, 0]
    c.n_ctx.copy_(i32(lens))
    out = ops.attention_pages(Q, c, 1, 2, T=3, max_ctx=163, shared_pages=shared, n_shared=160)
    k64, v64 = c.K[:, 1].double().cpu().numpy(), c.V[:, 1].double().cpu().numpy()
    table = c.table.cpu().numpy()
    want = []
    for b, n in enumerate(lens):
        kb = k64[table[b]].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:n]
        vb = v64[table[b]].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:n]
        want.append(po.attention(Q.double().cpu().numpy().reshape(4, 3, 2, 64)[b], kb, vb, 3))
    check(out, want, 3, 2, [3] * 4)
    assert (want[3][0] == 0).all() and (want[2][0][0] == 0).all()


@pytest.mark.parametrize("n_seq,T", [(3, 1), (40, 1), (2, 70)])
def test_keys_nobody_sees_may_hold_anything(cuda, n_seq, T):
    """NaN, infinities and the lowest finite value in rows behind the sequences give
    the bits that zeros there give."""
    outs = []
    for junk in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        tails = [T + 3 * i for i in range(n_seq)]
        c, Q, shared, _ = build(cuda, n_seq, T, 4, 2, 32, 96, tails, [T] * n_seq, 5, junk=junk)
        outs.append(ops.attention_pages(Q, c, 1, 4, T=T, max_ctx=96 + max(tails),
                                        shared_pages=shared, n_shared=96))
    for o in outs[1:]:
        assert torch.equal(outs[0].view(torch.int16), o.view(torch.int16))


# the plans: whole 16-row groups, a prefix shared out to 16-row groups, tensor-core items over
# the prefix (two and, of few rows, one tile wide), and over a sequence's whole keys
PLANS = [
    # n_seq, T, H, G, page, n_shared, longest tail
    (3, 2, 4, 2, 16, 64, 40),
    (3, 2, 4, 2, 32, 320, 100),
    (150, 2, 8, 8, 64, 1728, 30),
    (60, 2, 16, 16, 16, 2304, 30),
    (2, 70, 4, 2, 32, 64, 2300),
    (2, 90, 4, 2, 64, 192, 100),
]


def sees(c, Q, T, H, lens, n_new, layer=1):
    """(O, A) of the 64-bit oracle where sequence b holds lens[b] positions, n_new[b] of them
    new, of which the first T at most have a row."""
    G, n_seq = c.n_kv_head, len(lens)
    k64, v64 = (t[:, layer].double().cpu().numpy() for t in (c.K, c.V))
    table = c.table.cpu().numpy()
    q64 = Q.double().cpu().numpy().reshape(n_seq, T, H, 64)
    want = []
    for b, (n, new) in enumerate(zip(lens, n_new)):
        n = max(n - max(new - T, 0), 0)  # what the last row sees
        p = table[b, :-(-n // c.page)]
        kb, vb = (x[p].transpose(0, 2, 1, 3).reshape(-1, G, 64)[:n] for x in (k64, v64))
        want.append(po.attention(q64[b], kb, vb, min(new, T)))
    return want


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("inside", ["page", "block", "idle", "nothing"])
@pytest.mark.parametrize("padded", [False, True])
def test_a_prefix_that_nobody_sees_the_end_of(cuda, plan, inside, padded):
    """Every sequence with a query ends inside the shared pages: what stands behind the
    longest of them, there too, may hold anything."""
    n_seq, T, H, G, page, n_shared, tail = plan
    c, Q, shared, _ = build(cuda, n_seq, T, H, G, page, n_shared, [tail] * n_seq, [T] * n_seq, 4)
    longest = {"page": n_shared - 3, "block": n_shared // 2 + 5, "idle": n_shared // 3,
               "nothing": 0}[inside]
    lens = [max(longest - 2 * b, 0) for b in range(n_seq)]
    n_new = [T] * n_seq
    if padded:
        n_new = [T - b % 2 for b in range(n_seq)]
    if inside == "idle":  # one that reaches the end, without a query
        if not padded:
            pytest.skip("n_new None: every sequence has queries")
        lens[-1], n_new[-1] = n_shared + tail, 0
    c.n_ctx.copy_(i32(lens))
    seen = torch.zeros(c.n_pages, page, dtype=torch.bool, device=cuda)
    flat = shared.long()[:, None] * page + torch.arange(page, device=cuda)
    seen.view(-1)[flat.view(-1)[:longest]] = True
    outs = []
    for junk in (0.0, float("nan"), float("inf")):
        for pool in (c.K, c.V):
            pool.permute(0, 3, 1, 2, 4)[~seen] = junk
        out = torch.full((n_seq * T, H * 64), 7.0, dtype=torch.bfloat16, device=cuda)
        ops.attention_pages(Q, c, 1, H, T=T, n_new=i32(n_new) if padded else None,
                            max_ctx=n_shared + tail, shared_pages=shared, n_shared=n_shared, out=out)
        if junk == 0.0:
            check(out, sees(c, Q, T, H, lens, n_new), T, H, n_new)
        outs.append(out.view(torch.int16))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("plan", PLANS)
def test_more_new_positions_than_rows(cuda, plan):
    """n_new[b] > T: the T rows are the first of the new positions, as pages_write places
    them, and what follows them may hold anything."""
    n_seq, T, H, G, page, n_shared, tail = plan
    tails = [tail - b % 9 for b in range(n_seq)]
    n_new = [(T, T + 1, T + 7, T - 1, T + 2 * page)[b % 5] for b in range(n_seq)]
    n_new[0] = T + 3
    lens = [n_shared + t for t in tails]
    lens[-1], n_new[-1] = n_shared + 1, T + n_shared  # rows before any position, the last at one
    c, Q, shared, _ = build(cuda, n_seq, T, H, G, page, n_shared, tails, [T] * n_seq, 6)
    c.n_ctx.copy_(i32(lens))
    for b in range(n_seq):  # positions of its own behind the last row
        for pos in range(max(lens[b] - max(n_new[b] - T, 0), n_shared), n_shared + tails[b]):
            for pool in (c.K, c.V):
                pool[c.table[b, pos // page].long(), :, :, pos % page] = float("nan")
    out = torch.full((n_seq * T, H * 64), 7.0, dtype=torch.bfloat16, device=cuda)
    ops.attention_pages(Q, c, 1, H, T=T, n_new=i32(n_new), max_ctx=n_shared + tail,
                        shared_pages=shared, n_shared=n_shared, out=out)
    check(out, sees(c, Q, T, H, lens, n_new), T, H, [min(n, T) for n in n_new])
    # lengths and counts at the ends of 32 bits
    c.n_ctx[0], c.n_ctx[1] = -2 ** 31, lens[1]
    far = i32([2 ** 31 - 1, -2 ** 31] + n_new[2:])
    out.fill_(7.0)
    ops.attention_pages(Q, c, 1, H, T=T, n_new=far, max_ctx=n_shared + tail, shared_pages=shared,
                        n_shared=n_shared, out=out)
    check(out, sees(c, Q, T, H, [0, 0] + lens[2:], [T, 0] + n_new[2:]), T, H,
          [T, 0] + [min(n, T) for n in n_new[2:]])
    c.n_ctx[0] = lens[0]
    # a bound below the lengths cuts them first
    cut = n_shared + tail // 2
    out.fill_(7.0)
    ops.attention_pages(Q, c, 1, H, T=T, n_new=i32(n_new), max_ctx=cut, shared_pages=shared,
                        n_shared=n_shared, out=out)
    want = sees(c, Q, T, H, [min(n, cut) for n in lens], n_new)
    check(out, want, T, H, [min(n, T) for n in n_new])


@pytest.mark.parametrize("T,n_shared", [(3, 0), (3, 320), (70, 32), (300, 0)])
def test_a_key_that_is_not_a_number(cuda, T, n_shared):
    """NaN in the newest position's key reaches the row that sees it and no other."""
    tails = [T + 40, T + 3]
    c, Q, shared, _ = build(cuda, 2, T, 4, 2, 32, n_shared, tails, [T] * 2, 11)
    kw = dict(T=T, max_ctx=n_shared + T + 40, shared_pages=shared, n_shared=n_shared)
    want = ops.attention_pages(Q, c, 1, 4, **kw)
    last = n_shared + tails[0] - 1
    c.K[c.table[0, last // 32].item(), 1, :, last % 32] = float("nan")
    got = ops.attention_pages(Q, c, 1, 4, **kw)
    rows = [r for r in range(2 * T) if r != T - 1]
    assert torch.equal(got[rows], want[rows]) and got[T - 1].isnan().all()


@pytest.mark.parametrize("n_seq,T,n_shared", [(2, 1, 512), (64, 1, 512), (2, 130, 512), (3, 1, 0)])
def test_large_scores(cuda, n_seq, T, n_shared):
    """Scores of some hundreds, growing along the keys and falling: the running
    maximum moves all the way. The 32-bit scores are off by 2^-24 of sums of 64
    products of up to 2^9 each; exponentials by that of a score in absolute terms,
    64 * 2^9 / 8 * 2^-24 = 2^-12 of the weight."""
    for sign in (1.0, -1.0):
        tails = [T + 40] * n_seq
        c, Q, shared, _ = build(cuda, n_seq, T, 2, 2, 16, n_shared, tails, [T] * n_seq, 9, scale=0)
        n = n_shared + T + 40
        Q.fill_(4.0)
        table = c.table.cpu().numpy()
        ramp = torch.linspace(-8, 8, n, device=cuda) * sign
        for b in range(n_seq):
            for k in range(table.shape[1]):
                if table[b, k] < 0:
                    continue
                rows = min(16, n - 16 * k)
                c.K[table[b, k], :, :, :rows] = ramp[16 * k:16 * k + rows, None].bfloat16()
        out = ops.attention_pages(Q, c, 1, 2, T=T, max_ctx=n, shared_pages=shared,
                                  n_shared=n_shared)
        k64, v64 = c.K[:, 1].double().cpu().numpy(), c.V[:, 1].double().cpu().numpy()
        want = []
        for b in range(n_seq):
            p = table[b, :-(-n // 16)]
            kb = k64[p].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:n]
            vb = v64[p].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:n]
            want.append(po.attention(np.full((T, 2, 64), 4.0), kb, vb, T))
        check(out, want, T, 2, [T] * n_seq)


def test_bad_entries_read_as_zeros_and_are_recorded(cuda):
    for bad in (-5, 10 ** 6):
        c, Q, shared, _ = build(cuda, 3, 1, 2, 2, 16, 32, [40, 40, 40], [1] * 3, 2, junk=0.0)
        good = ops.attention_pages(Q, c, 1, 2, max_ctx=72, shared_pages=shared, n_shared=32)
        assert ops.device_error() == 0
        p = int(c.table[1, 3])
        c.table[1, 3] = bad
        got = ops.attention_pages(Q, c, 1, 2, max_ctx=72, shared_pages=shared, n_shared=32)
        assert ops.device_error() == 0x1601
        assert torch.equal(got[[0, 2]], good[[0, 2]])
        c.table[1, 3] = p
        c.K[p] = 0
        c.V[p] = 0
        want = ops.attention_pages(Q, c, 1, 2, max_ctx=72, shared_pages=shared, n_shared=32)
        assert torch.equal(got, want)


def test_a_pool_behind_32_bit_offsets(cuda):
    """Pages more than 2^32 elements into the pools."""
    n_pages, L, G, page = 1100, 64, 16, 64  # 4.6e9 elements a pool, 9.2 GB
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    K = torch.empty(n_pages, L, G, page, 64, dtype=torch.bfloat16, device=cuda)
    V = torch.empty_like(K)
    c = PageCache(K, V, i32([[n_pages - 1, n_pages - 3], [n_pages - 2, -1]]), i32([100, 0]),
                  i32([0] * (n_pages - 3) + [1, 0, 1]))
    assert (n_pages - 3) * K.stride(0) > 2 ** 32
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(100, G * 64, generator=g, device=cuda).bfloat16()
    y = torch.randn(100, G * 64, generator=g, device=cuda).bfloat16()
    for layer in (0, L - 1):
        ops.pages_write(c, layer, x, y, i32([0]), T=100)
        assert torch.equal(K[n_pages - 1, layer].transpose(0, 1).reshape(64, -1), x[:64])
        assert torch.equal(V[n_pages - 3, layer, :, :36].transpose(0, 1).reshape(36, -1), y[64:])
    c.table[1, 0] = -1
    c.refs[:n_pages - 3] = 1
    assert ops.pages_fork(c, i32([0]), i32([1])).item() == 0
    assert c.table[1].tolist() == [n_pages - 1, n_pages - 2]
    assert torch.equal(V[n_pages - 2, L - 1, :, :36], V[n_pages - 3, L - 1, :, :36])
    Q = torch.randn(2, G * 64, generator=g, device=cuda).bfloat16()
    out = ops.attention_pages(Q, c, L - 1, G, max_ctx=100)
    q = Q.double().cpu().numpy().reshape(2, 1, G, 64)
    want = [po.attention(q[b], *(t.double().cpu().numpy().reshape(100, G, 64) for t in (x, y)), 1)
            for b in range(2)]
    check(out, want, 1, G, [1, 1])
    ops.pages_copy(K, V, i32([n_pages - 1]), K, V, i32([n_pages - 4]))
    assert torch.equal(K[n_pages - 4].view(torch.int16), K[n_pages - 1].view(torch.int16))
    # the pages at the end go to the front
    c.refs[:n_pages - 3] = 0
    assert ops.pages_compact(c).item() == 3
    assert c.table.tolist() == [[2, 0], [2, 1]]
    assert torch.equal(ops.attention_pages(Q, c, L - 1, G, max_ctx=100), out)


# ---- streams, graphs, refusals -----------------------------------------------

def test_another_stream_and_captured_graphs(cuda):
    """A decode step (extend, write, attend) captured once and replayed as the
    sequences grow over page ends gives what the eager steps give."""
    def steps(replay):
        c, _ = make(cuda, 40, 4, 6, n_layer=1, n_kv=2, page=16, seed=4)
        ops.pages_extend(c, i32([32, 0, 0, 0]))
        ops.pages_fork(c, i32([0, 0, 0]), i32([1, 2, 3]))
        x = torch.zeros(4, 128, dtype=torch.bfloat16, device=cuda)
        one, out = i32([1, 1, 1, 1]), torch.zeros(4, 256, dtype=torch.bfloat16, device=cuda)
        q = torch.zeros(4, 256, dtype=torch.bfloat16, device=cuda)
        shared = c.table[0, :2].clone()

        def step():
            pos0 = ops.pages_extend(c, one)
            ops.pages_write(c, 0, x, x, pos0)
            ops.attention_pages(q, c, 0, 4, max_ctx=96, shared_pages=shared, n_shared=32, out=out)

        graph = None
        got = []
        g = torch.Generator(device=cuda).manual_seed(8)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for i in range(40):
                x.copy_(torch.randn(4, 128, generator=g, device=cuda))
                q.copy_(torch.randn(4, 256, generator=g, device=cuda))
                if not replay or i == 0:
                    step()
                else:
                    if graph is None:
                        graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(graph, stream=s):
                            step()
                    graph.replay()
                got.append(out.clone())
        s.synchronize()
        assert c.n_ctx.tolist() == [72] * 4
        return torch.stack(got), c
    a, ca = steps(False)
    b, cb = steps(True)
    assert torch.equal(a, b) and torch.equal(ca.table, cb.table)
    assert torch.equal(ca.refs, cb.refs)
    assert ca.refs.sum().item() == 4 * 5 and ca.table[:, :2].unique().numel() == 2


def test_captured_steps_behind_a_long_prefix(cuda):
    """A captured step whose 16-row kernel runs behind the tensor-core kernel: lengths,
    table, rows and queries of each replay are the ones that it reads, as in eager steps
    into a cache of their own, with a wait after every call."""
    n_seq, G, H, page, ns = 100, 16, 16, 16, 144
    src, _ = make(cuda, ns + 5 * n_seq, n_seq, ns + 5, n_layer=1, n_kv=G, page=page, seed=2)
    shared = torch.arange(ns, device=cuda, dtype=torch.int32)
    src.table[:, :ns] = shared
    src.n_ctx.fill_(ns * page)
    src.refs[:ns] = n_seq
    caches = [PageCache(*(t.clone() for t in (src.K, src.V, src.table, src.n_ctx, src.refs)))
              for _ in range(2)]
    n_new, q = i32([1] * n_seq), torch.zeros(n_seq, H * 64, dtype=torch.bfloat16, device=cuda)
    x = torch.zeros(n_seq, G * 64, dtype=torch.bfloat16, device=cuda)
    outs = [torch.zeros_like(q) for _ in range(2)]

    def step(i, wait):
        c = caches[i]
        pos0 = ops.pages_extend(c, n_new)
        wait()
        ops.pages_write(c, 0, x, x, pos0)
        wait()
        ops.attention_pages(q, c, 0, H, n_new=n_new, max_ctx=(ns + 5) * page, shared_pages=shared,
                            n_shared=ns * page, out=outs[i])
        wait()

    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    before = [t.clone() for t in (src.table, src.n_ctx, src.refs)]
    with torch.cuda.graph(graph, stream=s):
        for _ in range(3):
            step(0, lambda: None)
    g = torch.Generator(device=cuda).manual_seed(8)
    for t, b in zip((caches[0].table, caches[0].n_ctx, caches[0].refs), before):
        assert torch.equal(t, b)
    for i in range(16):
        x.copy_(torch.randn(x.shape, generator=g, device=cuda))
        q.copy_(torch.randn(q.shape, generator=g, device=cuda))
        n_new.copy_((torch.rand(n_seq, generator=g, device=cuda) < 0.7).int())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for _ in range(3):
            step(1, torch.cuda.synchronize)
        assert torch.equal(outs[0], outs[1]), i
    for a, b in zip((caches[0].table, caches[0].n_ctx, caches[0].refs),
                    (caches[1].table, caches[1].n_ctx, caches[1].refs)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,n_shared", [(1, 64), (1, 0), (3, 320), (90, 32)])
def test_strided_rows_and_fewer_sequences_than_slots(cuda, T, n_shared):
    """Q in a packed [Q | K | V] row, an output with padded rows, and the first three
    of five slots: the same bits as contiguous rows, and nothing beside them written."""
    tails = [T + 5, T, T + 200, T + 1, T + 2]
    c, Q, shared, want = build(cuda, 5, T, 4, 2, 32, n_shared, tails, [T] * 5, 7)
    kw = dict(T=T, max_ctx=n_shared + max(tails), shared_pages=shared, n_shared=n_shared)
    plain = ops.attention_pages(Q[:3 * T].contiguous(), c, 1, 4, **kw)
    check(plain, want[:3], T, 4, [T] * 3)
    packed = torch.full((3 * T, 520), 3.0, dtype=torch.bfloat16, device=cuda)
    packed[:, 8:264] = Q[:3 * T]
    wide = torch.full((3 * T, 262), 7.0, dtype=torch.bfloat16, device=cuda)
    ops.attention_pages(packed[:, 8:264], c, 1, 4, out=wide[:, 2:258], **kw)
    assert torch.equal(wide[:, 2:258], plain)
    assert (wide[:, :2] == 7).all() and (wide[:, 258:] == 7).all()


def test_two_caches_on_two_streams(cuda):
    """Calls in flight together, each on its own cache, stream and workspace."""
    made = [build(cuda, n, T, 8, 8, 64, P, [T + 7 * i for i in range(n)], [T] * n, n)
            for n, T, P in ((300, 1, 1728), (3, 90, 128), (40, 1, 64))]
    args = [(c, Q, dict(T=T, max_ctx=P + T + 7 * n, shared_pages=s, n_shared=P))
            for (c, Q, s, _), (n, T, P) in zip(made, ((300, 1, 1728), (3, 90, 128), (40, 1, 64)))]
    alone = [ops.attention_pages(Q, c, 1, 8, **kw) for c, Q, kw in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    outs = [[], [], []]
    for _ in range(20):
        for i, (c, Q, kw) in enumerate(args):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ops.attention_pages(Q, c, 1, 8, **kw))
    torch.cuda.synchronize()
    for i in range(3):
        for o in outs[i]:
            assert torch.equal(o, alone[i])


def test_front_end_refusals(cuda):
    c, _ = make(cuda, 8, 2, 4)
    f = dict(device=cuda)
    Q = torch.zeros(2, 192, dtype=torch.bfloat16, **f)
    one = i32([0, 1])
    with pytest.raises(TypeError):
        ops.pages_extend(c, torch.ones(2, **f))
    with pytest.raises(ValueError):
        ops.pages_extend(c, i32([1, 1, 1]))
    with pytest.raises(ValueError):
        ops.pages_extend(c, torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.pages_fork(c, one, i32([1]))
    with pytest.raises(ValueError):
        ops.pages_free(c, i32([0, 1, 0, 1])[::2])
    with pytest.raises(ValueError):
        ops.pages_write(c, 0, Q, Q, i32([0]))            # two rows, one sequence
    with pytest.raises(ValueError):
        ops.attention_pages(Q, c, 0, 3, n_shared=16, shared_pages=i32([]))
    with pytest.raises(ValueError):
        ops.attention_pages(Q, c, 0, 3, n_shared=16)
    with pytest.raises(TypeError):
        ops.attention_pages(Q.float(), c, 0, 3)
    for n in ((1 << 30) + 1, (1 << 32) + 16):  # the second is 16 in 32 bits
        with pytest.raises(ValueError):
            ops.attention_pages(Q, c, 0, 3, max_ctx=n)
    ws = torch.empty(8, dtype=torch.uint8, **f)
    bad = [dict(layer=2), dict(layer=-1), dict(n_head=4, Q=torch.zeros(2, 256, dtype=torch.bfloat16, **f)),
           dict(max_ctx=0), dict(n_shared=8, shared_pages=one), dict(workspace=ws, max_ctx=64),
           dict(n_shared=32, max_ctx=16, shared_pages=one),
           dict(Q=torch.zeros(3, 192, dtype=torch.bfloat16, **f)),
           dict(Q=torch.zeros(2, 200, dtype=torch.bfloat16, **f)[:, 4:196]),   # 8-byte aligned
           dict(Q=torch.zeros(2, 196, dtype=torch.bfloat16, **f)[:, :192]),    # ldq % 8
           dict(out=torch.zeros(2, 193, dtype=torch.bfloat16, **f)[:, :192])]  # odd ldo
    for kw in bad:
        kw = dict(dict(Q=Q, layer=0, n_head=3), **kw)
        with pytest.raises(_lib.W8A8Error) as e:
            ops.attention_pages(kw.pop("Q"), c, kw.pop("layer"), kw.pop("n_head"), **kw)
        assert e.value.status == _lib.W8A8_ERR_INVALID, kw
    with pytest.raises(_lib.W8A8Error):
        ops.pages_write(c, 5, Q, Q, one)
    with pytest.raises(_lib.W8A8Error):
        ops.pages_write(c, 0, Q.view(-1)[4:4 + 192].view(1, 192), Q[:1], i32([0]))
    with pytest.raises(_lib.W8A8Error):
        ops.pages_compact(c, workspace=ws)
    K, V = c.K, c.V
    for bad, err in [((K.float(), V, one, K, V, one), TypeError), ((K, V.float(), one, K, V, one), TypeError),
                     ((K, V, one, K[:, :1], V[:, :1], one), ValueError),       # other pages
                     ((K, V[:4], one, K, V, one), ValueError), ((K, V, one, K, V, i32([1])), ValueError),
                     ((K[..., ::2], V[..., ::2], one, K, V, one), ValueError),  # scattered pages
                     ((K, V[::2], one, K, V, one), ValueError), ((K, V.cpu(), one, K, V, one), ValueError),
                     ((K, V, one.long(), K, V, one), TypeError)]:
        with pytest.raises(err):
            ops.pages_copy(*bad)
    assert c.n_ctx.tolist() == [0, 0]


def test_a_call_of_too_many_pieces_is_unsupported(cuda):
    c, _ = make(cuda, 8, 64, 4)
    Q = torch.zeros(64, 192, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(_lib.W8A8Error) as e:
        ops.attention_pages(Q, c, 0, 3, max_ctx=1 << 30)
    assert e.value.status == _lib.W8A8_ERR_UNSUPPORTED


def test_the_slot_cache_attention_agrees(cuda):
    """The framework's path over both caches: the packed QKV projection writes new
    rows into the slot cache and, through pages_write, into pages; decode attention
    over the two differs by the roundings of the slot cache's kernel (scores rounded
    to bf16, 2^-8 of |s| <= 8, in the weights, and its own rounded weights)."""
    d, H, n = 768, 12, 100
    g = torch.Generator(device=cuda).manual_seed(0)
    X = torch.randn(4 * n, d, generator=g, device=cuda).bfloat16()
    W = torch.randint(-127, 128, (3 * d, d), generator=g, device=cuda, dtype=torch.int8)
    sW = torch.full((3 * d,), 5e-4, device=cuda)
    bias = torch.zeros(3 * d, device=cuda).bfloat16()
    Xq, sX = ops.per_token_quant(X)
    Q = torch.empty(4 * n, d, dtype=torch.bfloat16, device=cuda)
    Kc = torch.empty(4, n, d, dtype=torch.bfloat16, device=cuda)
    Vc = torch.empty_like(Kc)
    ops.linear_qkv(Xq, sX, W, sW, bias, Q, Kc, Vc, n * d, n)
    c = PageCache.empty(40, 4, 8, 1, H, 16, cuda)
    pos0 = ops.pages_extend(c, i32([n] * 4))
    ops.pages_write(c, 0, Kc.view(4 * n, d), Vc.view(4 * n, d), pos0, T=n)
    q = Q.view(4, n, d)[:, -1].contiguous()
    slot = ops.attention_decode(q, Kc, Vc, n * d, i32([n] * 4), n, H)
    page = ops.attention_pages(q, c, 0, H)
    k64, v64 = (t.double().cpu().numpy().reshape(4, n, H, 64) for t in (Kc, Vc))
    q64 = q.double().cpu().numpy().reshape(4, 1, H, 64)
    want = [po.attention(q64[b], k64[b], v64[b], 1) for b in range(4)]
    check(page, want, 1, H, [1] * 4)
    smax = max(np.abs(np.einsum("nhd,hd->nh", k64[b], q64[b, 0])).max() / 8 for b in range(4))
    A = np.stack([w[1][0] for w in want]).reshape(4, d)
    err = (slot.double() - page.double()).abs().cpu().numpy()
    assert (err <= (2.0 ** -8 * (2 * smax + 6)) * A).all()


@pytest.mark.parametrize("blocks", [2, 60])
def test_two_prompts_in_one_batch(cuda, blocks):
    """Samples of two prompts in turn: a call for each prompt, the others' sequences left
    out by n_new, into one output. Then the slots that the prompts came in by end, and the
    pool is compacted: the rest go on behind copies of a live slot's row."""
    G, H, page, n_seq = 4, 8, 32, 12
    n_layer, lens = 1, [page * blocks + 3, page * (blocks - 1)]
    c, _ = make(cuda, 4 * blocks + 40, n_seq, blocks + 4, n_layer, G, page, seed=5)
    g = torch.Generator(device=cuda).manual_seed(6)
    held = [None] * n_seq

    def rows(n):
        return torch.randn(n, G * 64, generator=g, device=cuda).bfloat16()

    def add(n_new):
        T = max(n_new)
        K, V = rows(n_seq * T), rows(n_seq * T)
        pos0 = ops.pages_extend(c, i32(n_new))
        assert (pos0 >= -1).all()
        ops.pages_write(c, 0, K, V, pos0, T=T, n_new=i32(n_new))
        for b, n in enumerate(n_new):
            if n:
                new = [x[b * T:b * T + n].view(n, G, 64) for x in (K, V)]
                held[b] = [torch.cat(x) for x in zip(held[b], new)] if held[b] else new

    def step(live, holder):
        add(live)
        Q = torch.randn(n_seq, H * 64, generator=g, device=cuda).bfloat16()
        out = torch.full_like(Q, 7.0)
        for i in range(2):
            whole = lens[i] // page
            prefix = c.table[holder[i], :whole].clone()
            ops.attention_pages(Q, c, 0, H, n_new=i32([v * (b % 2 == i) for b, v in enumerate(live)]),
                                max_ctx=page * (blocks + 2), shared_pages=prefix,
                                n_shared=whole * page, out=out)
        q64 = Q.double().cpu().numpy().reshape(n_seq, 1, H, 64)
        want = [po.attention(q64[b], *(x.double().cpu().numpy() for x in held[b] or
                                       [torch.zeros(0, G, 64)] * 2), live[b]) for b in range(n_seq)]
        check(out, want, 1, H, live)

    add(lens + [0] * (n_seq - 2))
    src, dst = [b % 2 for b in range(2, n_seq)], list(range(2, n_seq))
    assert ops.pages_fork(c, i32(src), i32(dst)).tolist() == [0] * (n_seq - 2)
    for a, b in zip(src, dst):
        held[b] = held[a]
    step([1] * n_seq, [0, 1])
    ops.pages_free(c, i32([0, 1, 6]))
    held[0] = held[1] = held[6] = None
    live = [0, 0, 1, 1, 1, 1, 0, 1, 1, 1, 1, 1]
    step(live, [2, 3])
    ops.pages_compact(c)
    step(live, [4, 11])
    assert c.n_ctx.tolist() == [v * (lens[b % 2] + 3) for b, v in enumerate(live)]


def test_a_serving_run(cuda):
    """Two prompts of different lengths (a padded batch) through the packed QKV
    projection into pages; three samples of each, decoded step by step behind the
    first prompt's pages or their own; some given back, the pool compacted and
    halved, and the rest decoded on. Every attention output against 64 bits over the
    keys and values that the sequence has been given."""
    d, H, page, T = 768, 12, 16, 70
    g = torch.Generator(device=cuda).manual_seed(0)
    W = torch.randint(-127, 128, (3 * d, d), generator=g, device=cuda, dtype=torch.int8)
    sW = torch.full((3 * d,), 5e-4, device=cuda)
    bias = torch.randn(3 * d, generator=g, device=cuda).bfloat16()
    c = PageCache.empty(90, 8, 10, 1, H, page, cuda)
    held = [[] for _ in range(8)]  # K, V rows of every slot

    def project(rows):
        Xq, sX = ops.per_token_quant(torch.randn(rows, d, generator=g, device=cuda).bfloat16())
        Q, K, V = (torch.empty(rows, d, dtype=torch.bfloat16, device=cuda) for _ in range(3))
        ops.linear_qkv(Xq, sX, W, sW, bias, Q, K, V, rows * d, rows)
        return Q, K, V

    def attend(Q, t, n_new, **kw):
        out = torch.zeros_like(Q)
        ops.attention_pages(Q, c, 0, H, T=t, n_new=i32(n_new), out=out, **kw)
        q64 = Q.double().cpu().numpy().reshape(8, t, H, 64)
        want = []
        for s in range(8):
            kv = [np.stack(x) if n_new[s] else np.zeros((0, H, 64))
                  for x in (zip(*held[s]) if n_new[s] else ((), ()))]
            want.append(po.attention(q64[s], *kv, n_new[s]))
        check(out, want, t, H, n_new, before=0.0)

    def step(t, n_new, **kw):
        Q, K, V = project(8 * t)
        pos0 = ops.pages_extend(c, i32(n_new))
        assert (pos0.cpu().numpy() >= -1).all()
        ops.pages_write(c, 0, K, V, pos0, T=t, n_new=i32(n_new))
        k64, v64 = (x.double().cpu().numpy().reshape(8, t, H, 64) for x in (K, V))
        for s in range(8):
            held[s] += [(k64[s, i], v64[s, i]) for i in range(n_new[s])]
        attend(Q, t, n_new, **kw)

    step(T, [T, 41] + [0] * 6)
    src, dst = [0, 0, 1, 1], [2, 4, 3, 7]
    assert ops.pages_fork(c, i32(src), i32(dst)).tolist() == [0] * 4
    for a, b in zip(src, dst):
        held[b] = list(held[a])
    for i in range(12):
        step(1, [1, 1, 1, 1, 1, 0, 0, 1])
    # behind the first prompt alone: the second's samples have left
    ops.pages_free(c, i32([1, 3, 7]))
    for s in (1, 3, 7):
        held[s] = []
    n_live = ops.pages_compact(c).item()
    assert n_live == 4 + 3 * 2 and (c.refs[:4 + 6] > 0).all() and (c.refs[n_live:] == 0).all()
    small = PageCache(c.K[:45].clone(), c.V[:45].clone(), c.table, c.n_ctx, c.refs[:45].clone())
    c = small
    for i in range(8):
        step(1, [1, 0, 1, 0, 1, 0, 0, 0], shared_pages=c.table[2, :4].clone(), n_shared=64,
             max_ctx=96)
    step(30, [30, 0, 5, 0, 0, 0, 0, 0])  # two go on by more than a token
    ops.pages_free(c, i32(range(8)))
    assert c.refs.sum().item() == 0 and (c.table == -1).all() and (c.n_ctx == 0).all()
