"""The paged cache's tables, slots and rows (q4kv_paged.hip) against plain
references: whole numbers and cache bytes exactly."""
import numpy as np
import pytest

import q4kv
from gpu_util import note
from paged_util import Bufs, Pages, plan_ref, row_bytes, values

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ tables

def _plan(rt, ctx, new, page, table, free, n_free, max_tok, n_pages, optional=True, in_place=False):
    b = Bufs(rt)
    n_seq = len(ctx)
    want = plan_ref(ctx, new, page, table, free, n_free, max_tok, n_pages)
    d = dict(ctx=b.up(np.int32(ctx)), new=b.up(np.int32(new)), table=b.up(table), free=b.up(free))
    count = np.array([n_free, 77], np.int32)
    d["n_free"] = b.up(count)
    d["left"] = d["n_free"] if in_place else b.up(np.zeros(2, np.int32))
    for k in ("q_start", "kv_len", "slot", "tok_seq", "tok_pos"):
        d[k] = b.up(np.full_like(want[k], -7))
    assert rt.lib.q4_hip_paged_plan(d["ctx"], d["new"], n_seq, page, d["table"], table.shape[1],
                                    d["free"], n_pages, d["n_free"], d["left"], d["q_start"],
                                    d["kv_len"], max_tok, d["slot"], d["tok_seq"] if optional else None,
                                    d["tok_pos"] if optional else None)
    rt.sync()
    for k, w in want.items():
        if not optional and k in ("tok_seq", "tok_pos"):
            w = np.full_like(w, -7)
        got = b.get(d[k], w)
        assert np.array_equal(got, w), (k, np.flatnonzero(got.ravel() != w.ravel())[:8])
    if not in_place:
        assert np.array_equal(b.get(d["n_free"], count), count)
    assert np.array_equal(b.get(d["free"], free), free)
    b.free()
    return want


def _case(seed, n_seq, page, hi, most, spare=0, pad=0):
    """Lengths, a table with the pages held, and a stack of the others."""
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, hi, n_seq)
    new = np.where(rng.random(n_seq) < 0.3, rng.integers(0, most + 1, n_seq), 1)
    held = -(-ctx // page)
    stride = int((-(-(ctx + new) // page)).max()) + 2
    lack = int((-(-(ctx + new) // page) - held).sum())
    n_pages = int(held.sum()) + lack + max(spare, 0) + 2
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n_seq, stride), -1, np.int32)
    at = 0
    for i in range(n_seq):
        table[i, :held[i]] = perm[at:at + held[i]]
        at += held[i]
    free = np.full(n_pages, -5, np.int32)
    n_free = lack + spare
    free[:n_free] = perm[at:at + n_free]
    return ctx, new, table, free, n_free, int(new.sum()) + pad, n_pages


@pytest.mark.parametrize("n_seq,page,hi,most,spare,pad", [
    (1, 16, 3, 1, 0, 0), (1, 1, 40, 9, 5, 3), (3, 7, 100, 33, 0, 1), (64, 16, 3000, 1, 10, 0),
    (65, 24, 900, 300, 2, 70), (300, 64, 2000, 200, 0, 0), (1023, 16, 500, 20, 9, 9),
    (1025, 5, 60, 12, 1, 5), (2600, 16, 90, 3, 40, 1), (4, 100000, 300000, 5000, 1, 0),
])
def test_plan(rt, n_seq, page, hi, most, spare, pad):
    note(f"plan n_seq={n_seq} page={page}")
    ctx, new, table, free, n_free, max_tok, n_pages = _case(n_seq + page, n_seq, page, hi, most, spare, pad)
    want = _plan(rt, ctx, new, page, table, free, n_free, max(max_tok, 1), n_pages,
                 optional=n_seq % 2 == 1, in_place=n_seq % 3 == 0)
    assert want["left"][1] == 0


def test_plan_refuses_requests_past_what_there_is(rt):
    """Too few pages, a table row too short, lengths below zero, tokens past
    max_tok: those requests get nothing, the others what they need."""
    note("plan refusals")
    page = 8
    ctx = np.array([8, 0, 15, -3, 30, 8, 16, 5, 39, 7])
    new = np.array([1, 9, 1, 4, 40, -2, 17, 0, 1, 1])  # row 4 is past 5 pages a row
    table = np.arange(50, dtype=np.int32).reshape(10, 5) + 100
    table[7, 0] = 9999  # a page that does not exist, held but not read
    free = np.arange(200, 320, dtype=np.int32)
    for n_free in (0, 1, 2, 3, 4, 5, 6, 7, 8, 119, -4, 500):
        for max_tok in (1, 10, 15, 72, 90):
            want = _plan(rt, ctx, new, page, table, free, n_free, max_tok, 120)
            assert want["left"][1] >= 2 and (want["left"][0] >= 0)


def test_release(rt):
    for n, page, hi, listed in ((1, 16, 5, False), (3, 1, 9, True), (70, 24, 2000, True), (1500, 16, 100, True)):
        note(f"release n={n} page={page}")
        rng = np.random.default_rng(n)
        rows_all = n + 5
        lens = rng.integers(0, hi, rows_all).astype(np.int32)
        lens[0] = -2 if n > 3 else lens[0]
        stride = -(-hi // page) + 1
        table = rng.integers(0, 1 << 20, (rows_all, stride)).astype(np.int32)
        rows = rng.permutation(rows_all)[:n].astype(np.int32) if listed else np.arange(n, dtype=np.int32)
        if n > 3:
            rows[2] = -1
        held = [min(max(-(-int(lens[r]) // page), 0), stride) if r >= 0 else 0 for r in rows]
        for cut in (0, 4):
            n_free = 11
            n_pages = max(n_free + sum(held) - cut, n_free + 1)
            free = np.full(n_pages + 8, -9, np.int32)
            free[:n_free] = np.arange(n_free)
            want = free.copy()
            back = np.concatenate([table[r, :h] for r, h in zip(rows, held)] + [np.zeros(0, np.int32)])
            k = min(len(back), n_pages - n_free)
            want[n_free:n_free + k] = back[:k]
            b = Bufs(rt)
            df, dn, dl = b.up(free), b.up(np.array([n_free], np.int32)), b.up(np.array([-1], np.int32))
            in_place = cut == 4
            assert rt.lib.q4_hip_paged_release(b.up(table), stride, b.up(lens), b.up(rows) if listed else None,
                                               n, page, df, n_pages, dn, dn if in_place else dl)
            rt.sync()
            assert np.array_equal(b.get(df, free), want)
            left = b.get(dn if in_place else dl, np.zeros(1, np.int32))[0]
            assert left == n_free + k
            b.free()


# -------------------------------------------------------------------- rows

@pytest.mark.parametrize("kind,n,n_tok,lead,gap", [
    (2, 512, 70, 0, 0), (2, 32, 3, 0, 0), (2, 288, 41, 2, 5), (2, 1024, 130, 0, 8),
    (1, 512, 33, 0, 0), (1, 33, 19, 1, 1), (1, 1024, 5, 0, 4), (0, 512, 9, 0, 0), (0, 7, 300, 3, 2),
    (2, 512, 1, 0, 0), (1, 96, 1, 0, 0),
])
def test_rows_to_slots_and_back(rt, oracle, kind, n, n_tok, lead, gap):
    """The bytes that the oracle writes at the tokens' slots, every other byte
    of the pool as it was; tokens without a slot write nothing and read 0."""
    note(f"rows kind={kind} n={n} n_tok={n_tok}")
    rng = np.random.default_rng(n + n_tok)
    row = row_bytes(kind, n)
    bpt = row + (0 if gap % 2 else 2 * gap) * (2 if kind == 0 else 1)  # slots may be wider than a row
    n_slots = 2 * n_tok + 5
    slot = rng.permutation(n_slots)[:n_tok].astype(np.int32)
    if n_tok > 2:
        slot[1], slot[n_tok - 1] = -1, n_slots + 3
    ks, vs = n + gap, n + 2 * gap
    k = rng.standard_normal((n_tok, ks), dtype=np.float32)
    v = (rng.standard_normal((n_tok, vs)) * 300).astype(np.float32)
    pools = [rng.integers(0, 256, (n_slots, bpt)).astype(np.uint8) for _ in range(2)]
    want = [p.copy() for p in pools]
    live = [t for t in range(n_tok) if 0 <= slot[t] < n_slots]
    for p, x in zip(want, (k, v)):
        for t in live:
            p[slot[t], :row] = np.frombuffer(oracle.encode(x[t, :n], kind).tobytes(), np.uint8)
    b = Bufs(rt)
    dp = [b.up(p) for p in pools]
    dk, dv, ds = b.up(k, 4 * lead), b.up(v, 4 * lead), b.up(slot)
    assert rt.lib.q4_hip_paged_append(*dp, dk, dv, ks, vs, ds, n_tok, n, bpt, n_slots, kind)
    back = np.full((n_tok, n), 5.0, np.float32)
    do = [b.up(back, 4 * lead) for _ in range(2)]
    assert rt.lib.q4_hip_paged_read(*dp, *do, ds, n_tok, n, bpt, n_slots, kind)
    rt.sync()
    for got, w in zip(dp, want):
        assert np.array_equal(b.get(got, w), w)
    for got, w in zip(do, want):
        ref = np.zeros((n_tok, n))
        for t in live:
            ref[t] = values(kind, w[slot[t], :row])
        assert np.array_equal(b.get(got, back), ref.astype(np.float32))
    b.free()


# ------------------------------------------------------------------- lists

@pytest.mark.parametrize("page,n_list,width,in_place", [(16, 1, 2051, False), (1, 2, 5, True), (24, 2, 300, False),
                                                       (64, 3, 1, True)])
def test_lists_of_positions_become_slots(rt, page, n_list, width, in_place):
    note(f"lists page={page} n_list={n_list} width={width}")
    rng = np.random.default_rng(page + width)
    lens = [5, 700, 0, 129]
    n_pages = sum(-(-n // page) for n in lens) + 2
    stride = -(-700 // page) + 1
    table = np.full((4, stride), -1, np.int32)
    perm, at = rng.permutation(n_pages).astype(np.int32), 0
    for i, n in enumerate(lens):
        h = -(-n // page)
        table[i, :h] = perm[at:at + h]
        at += h
    table[1, 2], table[3, 0] = -1, n_pages  # pages that do not exist
    kv_len = np.array([5, 700, 0, 100000], np.int32)  # the last one is past its table row
    tok_seq = np.array([1, 0, -1, 3, 2, 1, 4, 3], np.int32)
    idx = rng.integers(-2, 720, (8 * n_list, width)).astype(np.int32)
    idx[0, 0] = 2 ** 31 - 1
    seq = np.repeat(tok_seq, n_list)[:, None]
    want = np.full_like(idx, -1)
    for r in range(idx.shape[0]):
        s = seq[r, 0]
        for j in range(width):
            p = idx[r, j]
            if 0 <= s < 4 and 0 <= p < kv_len[s] and p // page < stride and 0 <= table[s, p // page] < n_pages:
                want[r, j] = table[s, p // page] * page + p % page
    b = Bufs(rt)
    di = b.up(idx)
    do = di if in_place else b.up(np.full_like(idx, 7))
    batch = q4kv.PagedBatch(b.up(table), None, b.up(kv_len), 4, stride, page, n_pages)
    assert rt.lib.q4_hip_paged_slots(di, do, b.up(tok_seq), 8, n_list, width, batch)
    rt.sync()
    assert np.array_equal(b.get(do, idx), want)
    b.free()


# ---------------------------------------------------------------- refusals

def test_calls_refuse_what_they_cannot_do(rt):
    """Null pointers, zero and too large sizes, widths and alignments that
    rows cannot have; nothing is launched."""
    note("paged refusals")
    p = rt.alloc(1 << 16)
    L = rt.lib
    batch = q4kv.PagedBatch

    def each(fn, good, bad):
        for at, value in bad:
            args = list(good)
            args[at] = value
            assert not fn(*args), (fn.__name__, at, value)

    big = 1 << 30
    each(L.q4_hip_paged_release, [p, 4, p, None, 2, 16, p, 8, p, p],
         [(0, None), (1, 0), (2, None), (4, 0), (4, 65537), (5, 0), (6, None), (7, 0), (8, None), (9, None),
          (5, big), (7, big)])
    each(L.q4_hip_paged_plan, [p, p, 2, 16, p, 4, p, 8, p, p, p, p, 4, p, None, None],
         [(0, None), (1, None), (2, 0), (2, 65537), (3, 0), (4, None), (5, 0), (6, None), (7, 0), (8, None),
          (9, None), (10, None), (11, None), (12, 0), (13, None), (3, big), (5, big), (7, big), (12, 1 << 31)])
    for fn, tail in ((L.q4_hip_paged_append, [64, 64, p, 2, 64]), (L.q4_hip_paged_read, [p, 2, 64])):
        good = [p, p, p, p] + tail + [68, 10, 2]
        n = len(good)
        bad = [(i, None) for i in range(4)] + [(n - 6, None) if fn is L.q4_hip_paged_read else (6, None)]
        bad += [(n - 5, 0), (n - 4, 0), (n - 4, 63), (n - 3, 0), (n - 3, 66), (n - 2, 0), (n - 2, 1 << 31),
                (n - 1, 3), (n - 1, -1), (0, p + 1), (1, p + 1), (n - 3, 69)]
        if fn is L.q4_hip_paged_append:
            bad += [(4, 63), (5, 63)]
        each(fn, good, bad)
        f32 = list(good)
        f32[n - 1], f32[n - 3] = 0, 256
        each(fn, f32, [(0, p + 2), (n - 3, 258), (n - 3, 252)])
    ok = batch(p, p, p, 2, 4, 16, 8)
    bads = [batch(None, p, p, 2, 4, 16, 8), batch(p, p, None, 2, 4, 16, 8), batch(p, p, p, 0, 4, 16, 8),
            batch(p, p, p, 65537, 4, 16, 8), batch(p, p, p, 2, 0, 16, 8), batch(p, p, p, 2, 4, 0, 8),
            batch(p, p, p, 2, 4, 16, 0), batch(p, p, p, 2, big, 2, 8), batch(p, p, p, 2, 4, 2, big), None]
    each(L.q4_hip_paged_slots, [p, p, p, 2, 1, 4, ok],
         [(0, None), (1, None), (2, None), (3, 0), (4, 0), (5, 0)] + [(6, x) for x in bads])
    each(L.q4_hip_qsa_paged_attend, [p, p, p, None, p, ok, 2, 1, 8, 2, 64, 0.125, 2],
         [(0, None), (1, None), (2, None), (4, None), (6, 0), (7, 0), (8, 0), (8, 7), (9, 0), (10, 0), (10, 257),
          (10, 48), (12, 3), (12, -1), (1, p + 1), (6, 1 << 31)]
         + [(5, x) for x in bads + [batch(p, None, p, 2, 4, 16, 8)]])
    each(L.q4_hip_qsa_paged_attend, [p, p, p, None, p, ok, 2, 1, 8, 2, 64, 0.125, 0], [(1, p + 2), (2, p + 2)])
    rt.sync()
    rt.free(p)
