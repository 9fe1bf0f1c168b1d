"""The cache-page operators and the attention that reads the pages: what is measured.

Sequences that go on from one prompt (several samples of a prompt, the beams
of a search, requests behind one system prompt) keep their keys and values in
pages of `page` positions. A page holds every layer's rows; the pages of the
common prompt are held once, and counted. Five operators:

  attend   attention of T new tokens a sequence over its pages, the pages of a
           shared prefix read once for the whole batch
  append   pages for the new tokens of every sequence, and one layer's new
           key and value rows written into them
  fork     sequences that go on from others' pages (whole pages are shared,
           the last, partly filled one is copied), and sequences given back
  compact  the pages in use moved to the front of the pool
  copy     pages from one pool to another (a pool that is put aside)

Pools are [n_pages, n_layer, n_kv_head, page, 64] bf16, one for the keys and
one for the values. `table` [n_slot, max_pages] lists each sequence's pages
(-1: none), `n_ctx` [n_slot] its length, `refs` [n_pages] how many sequences
hold a page (0: free). Pages are handed out lowest index first.

With `own` false each operator is computed from elementary torch operations.
"""
import math
import random

import numpy as np
import torch

own = False

HD = 64


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # two answers to one short prompt on the 12-head model: latency of the smallest call
        dict(name="attend_2x1_small", op="attend", n_seq=2, T=1, n_head=12, n_kv=12, page=16,
             n_shared=64, tail=32),
        # a decode step of the 20-head model, 64 samples of one 512-token prompt
        dict(name="attend_64x1_large", op="attend", n_seq=64, T=1, n_head=20, n_kv=20, page=16,
             n_shared=512, tail=512),
        # 96 requests behind one long document, four query heads to a key head
        dict(name="attend_96x1_long", op="attend", n_seq=96, T=1, n_head=32, n_kv=8, page=64,
             n_shared=32832, tail=1000),
        # user prompts of 1..200 tokens (a padded batch) behind a 4000-token system prompt
        dict(name="attend_8x200_prompts", op="attend", n_seq=8, T=200, n_head=20, n_kv=20,
             page=32, n_shared=4000, tail=200),
        # one decode step of 64 sequences: a page for those at a page's end, one row each
        dict(name="append_64x1", op="append", n_slot=64, T=1, n_layer=2, n_kv=20, page=16,
             held=1000, n_pages=6000),
        # 16 prompts of up to 1000 tokens arrive
        dict(name="append_16x1000", op="append", n_slot=16, T=1000, n_layer=2, n_kv=20, page=32,
             held=0, n_pages=700),
        # a second answer to a prompt of the 12-head model
        dict(name="fork_1to2_small", op="fork", n_src=1, n_dst=1, n_layer=12, n_kv=12, page=16,
             held=100, n_pages=64),
        # 63 more samples of one 512-odd-token prompt of the 20-head, 36-layer model
        dict(name="fork_1to64_large", op="fork", n_src=1, n_dst=63, n_layer=36, n_kv=20, page=32,
             held=531, n_pages=200),
        # a small pool after a few sequences ended
        dict(name="compact_64", op="compact", n_slot=4, n_layer=12, n_kv=12, page=16, held=200,
             n_pages=64),
        # a pool of 1600 pages of the 24-layer, 16-head model, half in use
        dict(name="compact_1600", op="compact", n_slot=24, n_layer=24, n_kv=16, page=16, held=900,
             n_pages=1600),
        # one sequence of the 12-head model put aside
        dict(name="copy_7_small", op="copy", n_copy=7, n_layer=12, n_kv=12, page=16, n_pages=32),
        # long sequences of the 36-layer model put aside
        dict(name="copy_301_large", op="copy", n_copy=301, n_layer=36, n_kv=20, page=32,
             n_pages=330),
    ]


def _span(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "fork", "compact", "copy"])
    page = rng.choice([16, 32, 64, 128])
    n_kv = rng.choice([4, 8, 12, 16, 20])
    if op == "attend":
        n_kv = rng.choice([2, 5, 8, 12, 16, 20])
        group = rng.choice([1, 1, 2, 4, 7, 8])
        T = 1 if rng.random() < 0.6 else _span(rng, 2, 300)
        while True:
            n_seq = _span(rng, 1, 128)
            c = dict(op=op, n_seq=n_seq, T=T, n_head=n_kv * group, n_kv=n_kv, page=page,
                     n_shared=page * (_span(rng, 1, 40000) // page), tail=max(T, _span(rng, 1, 1500)))
            keys = c["n_shared"] + c["tail"]
            # no more products than the largest listed case, no more tail bytes, and scores of
            # the plain form that fit the card
            if (n_seq * T * n_kv * group * keys <= 9.0e7 and n_seq * T * n_kv * group <= 40000
                    and n_seq * n_kv * c["tail"] <= 750000):
                return c
    if op == "append":
        n_slot = _span(rng, 1, 100)
        T = 1 if rng.random() < 0.5 else _span(rng, 2, 1000)
        while n_slot * T * n_kv > 320000:
            T = T // 2
        T = max(T, 1)
        held = rng.choice([0, _span(rng, 1, 600)])
        n_pages = n_slot * (-(-(held + T) // page) + 1)
        return dict(op=op, n_slot=n_slot, T=T, n_layer=rng.choice([1, 2]), n_kv=n_kv, page=page,
                    held=held, n_pages=n_pages)
    if op == "fork":
        n_src = rng.choice([1, 1, 2, 5])
        n_dst = _span(rng, n_src, 63)
        held = _span(rng, 1, 900)
        return dict(op=op, n_src=n_src, n_dst=n_dst, n_layer=_span(rng, 2, 36), n_kv=n_kv,
                    page=rng.choice([16, 32]), held=held,
                    n_pages=n_src * (held // 16 + 2) + n_dst + rng.randrange(9))
    page = rng.choice([16, 32])
    n_layer = _span(rng, 2, 36)
    per_page = n_layer * n_kv * page
    if op == "compact":
        n_slot = _span(rng, 1, 24)
        held = _span(rng, 1, 900)
        n_pages = 2 * n_slot * (-(-held // page)) + 1 + rng.randrange(30)
        n_layer = max(1, min(n_layer, 9000000 // (n_kv * page * n_pages)))
        return dict(op=op, n_slot=n_slot, n_layer=n_layer, n_kv=n_kv, page=page, held=held,
                    n_pages=n_pages)
    n_copy = max(1, min(_span(rng, 1, 600), 6900000 // per_page))
    return dict(op=op, n_copy=n_copy, n_layer=n_layer, n_kv=n_kv, page=page,
                n_pages=n_copy + rng.randrange(40))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def _book(table, n_ctx, refs):
    """table, n_ctx and refs as views of one int32 buffer, and its first contents."""
    first = torch.from_numpy(np.concatenate([table.ravel(), n_ctx, refs]).astype(np.int32)).cuda()
    buf = first.clone()
    a, b = table.size, table.size + n_ctx.size
    return dict(first=first, book=buf, table=buf[:a].view(*table.shape), n_ctx=buf[a:b],
                refs=buf[b:])


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    s = _prepare(case, seed)
    if own and case["op"] != "copy":
        # the handle on the cache that a program makes once and keeps
        from c_gpt2_b200.pages import PageCache
        s["cache"] = PageCache(s["K"], s["V"], s["table"], s["n_ctx"], s["refs"])
    return s


def _prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    s = dict(case=c)
    page, n_kv = c["page"], c["n_kv"]
    if c["op"] == "attend":
        n_seq, T = c["n_seq"], c["T"]
        n_new = np.full(n_seq, T)
        if T > 1:  # a padded batch: the longest fills its rows
            n_new = r.integers(1, T + 1, n_seq)
            n_new[r.integers(n_seq)] = T
        tails = np.maximum(n_new, r.integers(1, c["tail"] + 1, n_seq))
        ns = c["n_shared"] // page
        per = -(-tails // page)
        n_pages = int(ns + per.sum() + 5)
        order = r.permutation(n_pages)
        max_pages = int(ns + per.max())
        table = np.full((n_seq, max_pages), -1)
        table[:, :ns] = order[:ns]
        at = ns
        for b in range(n_seq):
            table[b, ns:ns + per[b]] = order[at:at + per[b]]
            at += per[b]
        # two layers; the call reads the second
        s.update(K=_randn(g, n_pages, 2, n_kv, page, HD), V=_randn(g, n_pages, 2, n_kv, page, HD),
                 Q=_randn(g, n_seq * T, c["n_head"] * HD) * 1.5, table=_dev(table),
                 n_ctx=_dev(c["n_shared"] + tails), n_new=_dev(n_new) if T > 1 else None,
                 refs=torch.ones(n_pages, dtype=torch.int32, device="cuda"),
                 shared=_dev(order[:ns]), max_ctx=c["n_shared"] + int(tails.max()), layer=1,
                 O=torch.zeros(n_seq * T, c["n_head"] * HD, dtype=torch.bfloat16, device="cuda"))
        return s
    if c["op"] == "copy":
        shape = (c["n_pages"], c["n_layer"], n_kv, page, HD)
        s.update(K=_randn(g, *shape), V=_randn(g, *shape),
                 K2=torch.zeros(*shape, dtype=torch.bfloat16, device="cuda"),
                 V2=torch.zeros(*shape, dtype=torch.bfloat16, device="cuda"),
                 src=_dev(r.permutation(c["n_pages"])[:c["n_copy"]]),
                 dst=_dev(r.permutation(c["n_pages"])[:c["n_copy"]]))
        return s
    n_slot = c["n_src"] + c["n_dst"] if c["op"] == "fork" else c["n_slot"]
    if c["op"] == "fork":
        held = np.zeros(n_slot, dtype=np.int64)
        held[:c["n_src"]] = np.maximum(1, c["held"] - r.integers(0, 1 + c["held"] // 8, c["n_src"]))
        held[0] = c["held"]
    elif c["op"] == "append":
        held = r.integers(c["held"] // 2, c["held"] + 1, n_slot)
    else:
        held = r.integers(1, c["held"] + 1, n_slot)
        held[0] = c["held"]
    per = -(-held // page)
    order = r.permutation(c["n_pages"])
    table = np.full((n_slot, -(-(c["held"] + c.get("T", 0)) // page)), -1)
    refs = np.zeros(c["n_pages"], dtype=np.int64)
    at = 0
    for b in range(n_slot):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
    refs[order[:at]] = 1
    shape = (c["n_pages"], c["n_layer"], n_kv, page, HD)
    s.update(_book(table, held, refs), K=_randn(g, *shape), V=_randn(g, *shape))
    if c["op"] == "append":
        T = c["T"]
        n_new = np.full(n_slot, T)
        if T > 1:
            n_new = r.integers(1, T + 1, n_slot)
            n_new[0] = T
        # the rows of a projection's output: keys and values side by side
        rows = _randn(g, n_slot * T, 2 * n_kv * HD)
        s.update(n_new=_dev(n_new), Kn=rows[:, :n_kv * HD], Vn=rows[:, n_kv * HD:],
                 layer=c["n_layer"] - 1)
    if c["op"] == "fork":
        dst = c["n_src"] + r.permutation(c["n_dst"])
        s.update(src=_dev(np.arange(c["n_dst"]) % c["n_src"]), dst=_dev(dst),
                 gone=_dev(np.concatenate([[0], dst[1::2]])))
    return s


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"attend": _attend, "append": _append, "fork": _fork, "compact": _compact,
            "copy": _copy}[op](s)


def _own(s, op):
    from c_gpt2_b200 import ops
    c = s["case"]
    if op == "copy":
        ops.pages_copy(s["K"], s["V"], s["src"], s["K2"], s["V2"], s["dst"])
        return [s["K2"], s["V2"]]
    cache = s["cache"]
    if op == "attend":
        return ops.attention_pages(s["Q"], cache, s["layer"], c["n_head"], T=c["T"],
                                   n_new=s["n_new"], max_ctx=s["max_ctx"],
                                   shared_pages=s["shared"], n_shared=c["n_shared"], out=s["O"])
    s["book"].copy_(s["first"])
    if op == "append":
        pos0 = ops.pages_extend(cache, s["n_new"])
        ops.pages_write(cache, s["layer"], s["Kn"], s["Vn"], pos0, T=c["T"], n_new=s["n_new"])
        return [s["book"], pos0, s["K"], s["V"]]
    if op == "fork":
        status = ops.pages_fork(cache, s["src"], s["dst"])
        ops.pages_free(cache, s["gone"])
        return [s["book"], status, s["K"], s["V"]]
    n_live = ops.pages_compact(cache)
    return [s["book"], n_live, s["K"], s["V"]]


def _attend(s):
    """O = softmax(q k / 8 over the keys before the row's end) v, in 32 bits."""
    c, layer = s["case"], s["layer"]
    B, T, H, G = c["n_seq"], c["T"], c["n_head"], c["n_kv"]
    P = c["n_shared"]
    ns = P // c["page"]
    S = (s["table"].shape[1] - ns) * c["page"]
    dev = s["Q"].device

    def shared(pool):  # [kv, P, 64]
        return pool[s["shared"].long(), layer].float().permute(1, 0, 2, 3).reshape(G, P, HD)

    def tails(pool):   # [b, kv, S, 64]
        t = s["table"][:, ns:].long().clamp(min=0)
        return pool[t, layer].float().permute(0, 2, 1, 3, 4).reshape(B, G, S, HD)

    q = s["Q"].float().view(B, T, G, H // G, HD)
    qp = q.permute(2, 0, 1, 3, 4).reshape(G, -1, HD)             # [kv, b t g, 64]
    qs = q.permute(0, 2, 1, 3, 4).reshape(B, G, -1, HD)          # [b, kv, t g, 64]
    sp = (qp @ shared(s["K"]).transpose(1, 2)).view(G, B, T, H // G, P).permute(1, 0, 2, 3, 4)
    ss = (qs @ tails(s["K"]).transpose(2, 3)).view(B, G, T, H // G, S)
    x = torch.cat([sp, ss], -1) * 0.125                          # [b, kv, t, g, keys]
    n_new = s["n_new"] if s["n_new"] is not None else torch.full_like(s["n_ctx"], T)
    t = torch.arange(T, device=dev)
    end = (s["n_ctx"] - n_new)[:, None] + t + 1                  # [b, t]
    seen = torch.arange(x.shape[-1], device=dev) < end[..., None]
    x = x.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = (x - torch.where(m == float("-inf"), torch.zeros_like(m), m)).exp()
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    op = p[..., :P].permute(1, 0, 2, 3, 4).reshape(G, B * T * (H // G), P) @ shared(s["V"])
    os = p[..., P:].reshape(B, G, T * (H // G), S) @ tails(s["V"])
    o = (op.view(G, B, T, H // G, HD).permute(1, 2, 0, 3, 4)
         + os.view(B, G, T, H // G, HD).permute(0, 2, 1, 3, 4)).reshape(B, T, H * HD)
    mine = t < n_new[:, None]
    return torch.where(mine[..., None], o.bfloat16(), s["O"].view(B, T, -1)).view(B * T, -1)


def _free_first(refs):
    """Page indices, the free ones first, each kind in order; and how many are free."""
    return torch.argsort((refs != 0).int(), stable=True), (refs == 0).sum()


def _append(s):
    """Whole pages for n_ctx + n_new positions, then row t of sequence b at n_ctx[b] + t."""
    c = s["case"]
    page, T = c["page"], c["T"]
    s["book"].copy_(s["first"])
    table, n_ctx, refs, n_new = s["table"], s["n_ctx"], s["refs"], s["n_new"]
    have = (n_ctx + page - 1) // page
    need = (n_ctx + n_new + page - 1) // page - have
    need = torch.where((n_new > 0) & (n_ctx + n_new <= table.shape[1] * page), need, 0 * need)
    upto = need.cumsum(0)
    order, n_free = _free_first(refs)
    ok = (n_new > 0) & (n_ctx + n_new <= table.shape[1] * page) & ((need == 0) | (upto <= n_free))
    j = torch.arange(table.shape[1], device=table.device) - have[:, None]
    mine = (j >= 0) & (j < need[:, None]) & ok[:, None]
    page_of = order[((upto - need)[:, None] + j).clamp(0, refs.numel() - 1)].int()
    table.copy_(torch.where(mine, page_of, table))
    refs.scatter_add_(0, page_of.long().reshape(-1), mine.int().reshape(-1))
    pos0 = torch.where(ok, n_ctx, torch.where(n_new > 0, -2, -1)).int()
    n_ctx.add_(torch.where(ok, n_new, 0 * n_new))
    t = torch.arange(T, device=table.device)
    rows = (t < n_new[:, None]) & ok[:, None]
    pos = pos0[:, None] + t
    pg = table.gather(1, (pos // page).clamp(0, table.shape[1] - 1).long())[rows].long()
    at = (pos % page)[rows].long()
    s["K"][pg, s["layer"], :, at] = s["Kn"].view(-1, T, c["n_kv"], HD)[rows]
    s["V"][pg, s["layer"], :, at] = s["Vn"].view(-1, T, c["n_kv"], HD)[rows]
    return [s["book"], pos0, s["K"], s["V"]]


def _fork(s):
    """dst[i] goes on from src[i]; then the sequences `gone` are given back."""
    c = s["case"]
    page = c["page"]
    s["book"].copy_(s["first"])
    table, n_ctx, refs = s["table"], s["n_ctx"], s["refs"]
    src, dst = s["src"].long(), s["dst"].long()
    n = n_ctx[src]
    part = (n % page > 0).int()
    upto = part.cumsum(0)
    order, n_free = _free_first(refs)
    ok = (n_ctx[dst] == 0) & ((part == 0) | (upto <= n_free))
    new = order[(upto - part).clamp(0, refs.numel() - 1)]
    col = torch.arange(table.shape[1], device=table.device)
    whole = (col < (n // page)[:, None]) & ok[:, None]
    last = (col == (n // page)[:, None]) & (ok & (part > 0))[:, None]
    theirs = table[src]
    rows = torch.where(whole, theirs, torch.where(last, new[:, None].int(), table[dst]))
    refs.scatter_add_(0, rows.clamp(min=0).long().reshape(-1), (whole | last).int().reshape(-1))
    table[dst] = rows
    n_ctx[dst] = torch.where(ok, n, n_ctx[dst])
    # the rows that the last page holds so far
    frm = theirs.gather(1, (n // page).clamp(max=table.shape[1] - 1).long()[:, None])[:, 0].long()
    moved = (ok & (part > 0)).nonzero()[:, 0]
    filled = (torch.arange(page, device=table.device) < (n % page)[moved][:, None])
    filled = filled[:, None, None, :, None]
    for pool in (s["K"], s["V"]):
        pool[new[moved]] = torch.where(filled, pool[frm[moved]], pool[new[moved]])
    status = torch.where(ok, 0, torch.where(n_ctx[dst] != 0, 1, 2)).int()
    # given back
    gone = s["gone"].long()
    held = table[gone]
    refs.scatter_add_(0, held.clamp(min=0).long().reshape(-1), -(held >= 0).int().reshape(-1))
    table[gone] = -1
    n_ctx[gone] = 0
    return [s["book"], status, s["K"], s["V"]]


def _compact(s):
    """The j-th page in use at n_live or above goes to the j-th free page below n_live."""
    s["book"].copy_(s["first"])
    table, refs = s["table"], s["refs"]
    live = refs > 0
    n_live = live.sum()
    p = torch.arange(refs.numel(), device=refs.device)
    frm = (live & (p >= n_live)).nonzero()[:, 0]
    to = (~live & (p < n_live)).nonzero()[:, 0]
    new = p.clone()
    new[frm] = to
    for pool in (s["K"], s["V"]):
        pool[to] = pool[frm]
    refs[to] = refs[frm]
    refs[frm] = 0
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].int(), table))
    return [s["book"], n_live.int().view(1), s["K"], s["V"]]


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["K2"][dst] = s["K"][src]
    s["V2"][dst] = s["V"][src]
    return [s["K2"], s["V2"]]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """The lengths are drawn from the seed; these are their means."""
    c = case
    row = c["n_kv"] * HD * 2                        # one position's keys of one layer, bytes
    if c["op"] == "attend":
        M = c["n_seq"] * (c["T"] + 1) / 2 if c["T"] > 1 else c["n_seq"]
        tail = max(c["tail"] / 2, (c["T"] + 1) / 2)
        keys = c["n_shared"] + c["n_seq"] * tail
        seen = c["n_shared"] + tail - (c["T"] - 1) / 4
        return {"bytes": 2 * keys * row + 2 * M * c["n_head"] * HD * 2,
                "flops": 4.0 * M * c["n_head"] * HD * seen}
    if c["op"] == "append":
        M = c["n_slot"] * ((c["T"] + 1) / 2 if c["T"] > 1 else 1)
        return {"bytes": 4 * M * row + 4 * c["n_pages"] + 16 * c["n_slot"], "flops": 0}
    page = 2 * c["n_layer"] * row * c["page"]       # a page, keys and values, bytes
    if c["op"] == "fork":
        part = (c["held"] % c["page"]) / c["page"]
        return {"bytes": (c["n_src"] + c["n_dst"]) * part * page + 4 * c["n_pages"]
                + 12 * c["n_dst"] * (c["held"] // c["page"] + 1), "flops": 0}
    if c["op"] == "compact":
        live = c["n_slot"] * (c["held"] / 2 / c["page"] + 0.5)
        return {"bytes": 2 * live * (1 - live / c["n_pages"]) * page + 8 * c["n_pages"],
                "flops": 0}
    return {"bytes": 2 * c["n_copy"] * page + 8 * c["n_copy"], "flops": 0}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """attend alone computes numbers: each sequence by itself, over its whole page list."""
    c = case
    if c["op"] != "attend":
        return None
    s = _prepare(case, seed)
    T, H, G = c["T"], c["n_head"], c["n_kv"]
    out = torch.zeros(c["n_seq"] * T, H, HD, dtype=torch.float64, device="cuda")
    lengths = s["n_ctx"].tolist()
    news = s["n_new"].tolist() if s["n_new"] is not None else [T] * c["n_seq"]
    for b, (n, new) in enumerate(zip(lengths, news)):
        pages = s["table"][b, :-(-n // c["page"])].long()
        k = s["K"][pages, 1].double().transpose(0, 1).reshape(G, -1, HD)[:, :n]
        v = s["V"][pages, 1].double().transpose(0, 1).reshape(G, -1, HD)[:, :n]
        k, v = (a.repeat_interleave(H // G, 0) for a in (k, v))
        q = s["Q"][b * T:b * T + new].double().view(new, H, HD).transpose(0, 1)
        a = torch.bmm(q, k.transpose(1, 2)) / math.sqrt(HD)
        late = torch.arange(n, device="cuda") > torch.arange(n - new, n, device="cuda")[:, None]
        a = torch.softmax(a.masked_fill(late, -math.inf), -1)
        out[b * T:b * T + new] = torch.bmm(a, v).transpose(0, 1)
    return out.view(c["n_seq"] * T, H * HD)


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(i)) for i in range(8)]:
        w = work(case)
        print(case, "%.3g MB, %.3g GFLOP" % (w["bytes"] / 1e6, w["flops"] / 1e9))
