"""The paged cache's calls as a serving loop makes them: pages given back and
handed out, rows written, attention, step after step, launched and replayed
from a graph; selections read through a pool; other streams, a held append,
sizes past 32 bits."""
import ctypes as C

import numpy as np
import pytest

import q4kv
from gpu_util import note
from paged_util import Bufs, Pages, attend_ref, row_bytes
from test_gpu_paged_attn import Call, _close, _inputs

pytestmark = pytest.mark.gpu

F32, F16, Q8 = 0, 1, 2
ROWS, PAGE, STRIDE, MAX_TOK, MAX_Q = 6, 16, 24, 150, 70


class Mirror:
    """The same caches, one long page per request, for the reference."""

    def __init__(self, kind, n_kvh, hd):
        self.kind, self.n_kvh, self.hd = kind, n_kvh, hd
        self.page, self.stride, self.n_pages = STRIDE * PAGE, 1, ROWS
        self.table = np.arange(ROWS, dtype=np.int32)[:, None]
        rb = row_bytes(kind, hd)
        self.pools = [np.zeros((ROWS * self.page, n_kvh, rb), np.uint8) for _ in range(2)]


class Loop:
    """Two layers' pools and the device arrays of a step."""

    def __init__(self, rt, oracle, kind, n_head, n_kvh, hd, n_pages):
        self.rt, self.oracle, self.kind, self.n_head, self.n_kvh, self.hd = rt, oracle, kind, n_head, n_kvh, hd
        self.n_pages, self.bpt = n_pages, n_kvh * row_bytes(kind, hd)
        self.b = Bufs(rt)
        self.layers = []
        for _ in range(2):
            pools = [self.b.up(np.full((n_pages * PAGE, self.bpt), 0x7F, np.uint8)) for _ in range(2)]
            io = {x: self.b.up(np.zeros((MAX_TOK, h, hd), np.float32))
                  for x, h in (("q", n_head), ("g", n_head), ("k", n_kvh), ("v", n_kvh), ("o", n_head), ("o2", n_head))}
            self.layers.append((pools, io, Mirror(kind, n_kvh, hd)))
        ints = dict(ctx=ROWS, new=ROWS, lens=ROWS, rows=2, q_start=ROWS + 1, kv_len=ROWS, slot=MAX_TOK,
                    tok_seq=MAX_TOK, tok_pos=MAX_TOK)
        self.d = {k: self.b.up(np.full(n, -1, np.int32)) for k, n in ints.items()}
        self.d["table"] = self.b.up(np.full((ROWS, STRIDE), -1, np.int32))
        self.d["free"] = self.b.up(np.arange(n_pages, dtype=np.int32))
        self.d["left"] = self.b.up(np.array([n_pages, 0], np.int32))
        self.batch = q4kv.PagedBatch(self.d["table"], self.d["q_start"], self.d["kv_len"], ROWS, STRIDE, PAGE, n_pages)

    def attend(self, layer, out):
        pools, io, _ = self.layers[layer]
        return self.rt.lib.q4_hip_qsa_paged_attend(io["q"], *pools, io["g"], io[out], self.batch, MAX_TOK, MAX_Q,
                                                   self.n_head, self.n_kvh, self.hd, self.hd ** -0.5, self.kind)

    def launch(self):
        L, d = self.rt.lib, self.d
        ok = L.q4_hip_paged_release(d["table"], STRIDE, d["lens"], d["rows"], 2, PAGE, d["free"], self.n_pages,
                                    d["left"], d["left"])
        ok &= L.q4_hip_paged_plan(d["ctx"], d["new"], ROWS, PAGE, d["table"], STRIDE, d["free"], self.n_pages,
                                  d["left"], d["left"], d["q_start"], d["kv_len"], MAX_TOK, d["slot"],
                                  d["tok_seq"], d["tok_pos"])
        n = self.n_kvh * self.hd
        for i, (pools, io, _) in enumerate(self.layers):
            ok &= L.q4_hip_paged_append(*pools, io["k"], io["v"], n, n, d["slot"], MAX_TOK, n, self.bpt,
                                        self.n_pages * PAGE, self.kind)
            ok &= self.attend(i, "o")
        return ok


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("kind,n_head,n_kvh,hd", [(Q8, 16, 2, 256), (F16, 8, 4, 128), (F32, 4, 2, 64), (F16, 4, 1, 36)])
def test_serving_steps(rt, oracle, kind, n_head, n_kvh, hd, graph):
    """Requests come in chunks, decode, end and hand their pages to others;
    once the pages run out for one of them. Every step's outputs against the
    formula over caches that no page moves, rows behind the last request left
    as they were, and the attention run again, eagerly, to the same bits."""
    note(f"serving kind={kind} hd={hd} graph={graph}")
    rng = np.random.default_rng(hd + kind)
    loop = Loop(rt, oracle, kind, n_head, n_kvh, hd, n_pages=30)
    ctx = np.zeros(ROWS, np.int32)
    # per step: new tokens of each row, rows that ended before it
    steps = [([33, 0, 70, 5, 0, 1], []), ([1, 60, 1, 1, 0, 1], []), ([1, 1, 1, 17, 40, 1], [0, 5]),
             ([64, 1, 1, 1, 1, 0], [3]), ([70, 0, 4, 0, 70, 2], [2]), ([1, 1, 1, 90, 1, 1], [4]),
             ([1, 70, 0, 1, 70, 3], []), ([1, 1, 0, 1, 1, 1], [])]
    g = None
    if graph:
        assert rt.lib.q4_hip_graph_begin() == 1
        ok = loop.launch()
        g = rt.lib.q4_hip_graph_end()
        assert ok and g
    refused_once = False
    for at, (new, ended) in enumerate(steps):
        note(f"serving step {at}")
        lens = np.zeros(ROWS, np.int32)
        rows = np.full(2, -1, np.int32)
        for j, r in enumerate(ended):
            rows[j], lens[r] = r, ctx[r]
        ctx[ended] = 0
        new = np.int32(new)
        for k, x in (("ctx", ctx), ("new", new), ("lens", lens), ("rows", rows)):
            rt.h2d(loop.d[k], x)
        data = []
        for pools, io, _ in loop.layers:
            x = {"k": rng.standard_normal((MAX_TOK, n_kvh, hd), dtype=np.float32),
                 "v": rng.standard_normal((MAX_TOK, n_kvh, hd), dtype=np.float32)}
            x["q"], x["g"] = _inputs(rng, MAX_TOK, n_head, hd)
            x["o"] = x["o2"] = np.full((MAX_TOK, n_head, hd), 123.0, np.float32)
            for k, a in x.items():
                rt.h2d(io[k], a)
            data.append(x)
        assert rt.lib.q4_hip_graph_launch(g) if graph else loop.launch()
        rt.sync()
        start = np.minimum(np.concatenate([[0], np.cumsum(new)]), MAX_TOK).astype(np.int32)
        assert np.array_equal(loop.b.get(loop.d["q_start"], start), start)
        kv_len = loop.b.get(loop.d["kv_len"], ctx)
        granted = kv_len > 0
        assert np.array_equal(kv_len[granted], (ctx + new)[granted])
        refused_once |= bool((~granted & (new > 0)).any())
        ctx[granted] = kv_len[granted]
        for (pools, io, mirror), x in zip(loop.layers, data):
            for i in np.flatnonzero(granted & (new > 0)):
                s = slice(int(start[i]), int(start[i]) + int(new[i]))
                to = i * mirror.page + int(ctx[i] - new[i]) + np.arange(new[i])
                for p, a in zip(mirror.pools, (x["k"], x["v"])):
                    p[to] = oracle.encode(a[s], kind).reshape(len(to), n_kvh, -1)
            got = loop.b.get(io["o"], x["q"])
            took = np.diff(start)
            _close(got, mirror, took, x["q"], x["g"], hd ** -0.5, f"step {at}", lens=kv_len, start=start)
            x["first"] = got
        for i, x in enumerate(data):  # eager work between the replays
            assert loop.attend(i, "o2")
            rt.sync()
            assert np.array_equal(loop.b.get(loop.layers[i][1]["o2"], x["q"]), x["first"])
    assert refused_once
    if graph:
        rt.lib.q4_hip_graph_free(g)
    loop.b.free()


def test_two_graphs_share_the_scratch(rt, oracle):
    """Two captured attentions of different batches, replayed in turn."""
    note("paged two graphs")
    rng = np.random.default_rng(9)
    made = []
    for kind, new, lens in ((Q8, [1, 200, 1], [3000, 300, 9]), (F16, [4, 4], [2500, 77])):
        pages = Pages(rng, kind, 2, 128, 16, lens, oracle)
        q, gate = _inputs(rng, sum(new), 16, 128)
        call = Call(rt, pages, new, q, gate)
        first = call.run(0.1)
        _close(first, pages, new, q, gate, 0.1, "eager")
        assert rt.lib.q4_hip_graph_begin() == 1
        ok = rt.lib.q4_hip_qsa_paged_attend(call.dq, *call.dp, call.dg, call.do, call.batch, call.n_tok, call.max_q,
                                            16, 2, 128, 0.1, kind)
        g = rt.lib.q4_hip_graph_end()
        assert ok and g
        made.append((g, call, first))
    for _ in range(4):
        for _, call, first in made:
            rt.h2d(call.do, np.zeros_like(first))
        for g, _, _ in made:
            assert rt.lib.q4_hip_graph_launch(g)
        rt.sync()
        for _, call, first in made:
            assert np.array_equal(call.b.get(call.do, first), first)
            assert np.array_equal(call.run(0.1), first)  # eager, between the replays
    for g, call, _ in made:
        rt.lib.q4_hip_graph_free(g)
        call.b.free()


@pytest.mark.parametrize("kind,page", [(Q8, 16), (F16, 24)])
def test_selections_read_through_a_pool(rt, oracle, kind, page):
    """Lists of the indexer's positions as lists of slots (in place), and the
    sparse attention over the pool: the bits of the same attention over a
    cache without pages. Chunks' lists and, per KV head, decodes'."""
    note(f"selections kind={kind} page={page}")
    rng = np.random.default_rng(page)
    lens, n_head, n_kvh, hd, ratio, k_blk = [700, 1500], 16, 2, 256, 4, 64
    pages = Pages(rng, kind, n_kvh, hd, page, lens, oracle)
    new = [5, 9]
    n_tok, bpt, n_slots = sum(new), n_kvh * row_bytes(kind, hd), pages.n_pages * page
    width = k_blk * ratio + ratio
    q, gate = _inputs(rng, n_tok, n_head, hd)
    b = Bufs(rt)
    dp = [b.up(p) for p in pages.pools]
    tok_seq = np.repeat(np.arange(2, dtype=np.int32), new)
    batch = q4kv.PagedBatch(b.up(pages.table), None, b.up(np.int32(lens)), 2, pages.stride, page, pages.n_pages)
    # the selections of the indexer's scores
    sel = []
    for i, n in enumerate(new):
        blocks = lens[i] // ratio + 1
        score = rng.standard_normal((n, blocks)).astype(np.float32)
        ds, dsel = b.up(score), b.up(np.full((n, width), -1, np.int32))
        assert rt.lib.q4_hip_qsa_topk(ds, dsel, n, blocks, blocks, k_blk, ratio, lens[i] - n, width)
        rt.sync()
        sel.append(b.get(dsel, np.zeros((n, width), np.int32)))
        assert (sel[-1] >= 0).any() and sel[-1].max() < lens[i]
    sel = np.concatenate(sel)
    dq, dg, dsel = b.up(q), b.up(gate), b.up(sel)
    assert rt.lib.q4_hip_paged_slots(dsel, dsel, b.up(tok_seq), n_tok, 1, width, batch)
    do = b.up(np.zeros_like(q))
    assert rt.lib.q4_hip_qsa_decode_idx(dq, *dp, dg, do, dsel, width, n_head, n_kvh, hd, n_tok, n_slots, 0.1, kind)
    rt.sync()
    got = b.get(do, q)
    at = 0
    for i, n in enumerate(new):
        flat = [np.zeros((n_slots, bpt), np.uint8) for _ in range(2)]
        for f, p in zip(flat, pages.pools):
            f[:lens[i]] = p[pages.slots(i, lens[i])].reshape(lens[i], bpt)
        df, dlist = [b.up(f) for f in flat], b.up(sel[at:at + n])
        dw = b.up(np.zeros_like(q))
        off = at * n_head * hd * 4
        assert rt.lib.q4_hip_qsa_decode_idx(dq + off, *df, dg + off, dw, dlist, width, n_head, n_kvh, hd, n, n_slots,
                                            0.1, kind)
        rt.sync()
        want = b.get(dw, q)[:n]
        scale = np.abs(want).max()
        # launches of other sizes cut the lists elsewhere: fp32 sums in another order
        assert np.abs(got[at:at + n] - want).max() <= 2e-5 * scale
        at += n
    # a list per KV head, one token each
    two = np.stack([np.sort(rng.choice(lens[i], 300, replace=False)) for i in (0, 0, 1, 1)]).astype(np.int32)
    dl = b.up(two)
    assert rt.lib.q4_hip_paged_slots(dl, dl, b.up(np.arange(2, dtype=np.int32)), 2, 2, 300, batch)
    assert rt.lib.q4_hip_qsa_decode_idx_kv(dq, *dp, None, do, dl, 300, 600, 300, n_head, n_kvh, hd, 2, n_slots, 0.1, kind)
    rt.sync()
    got = b.get(do, q)[:2]
    for i in range(2):
        for h in range(n_kvh):
            few = Pages.__new__(Pages)
            few.__dict__.update(kind=kind, n_kvh=1, hd=hd, page=300, stride=1, n_pages=1, table=np.zeros((1, 1), np.int32))
            few.pools = [p[pages.slots(i, lens[i])[two[2 * i + h]], h:h + 1] for p in pages.pools]
            ref, bound = attend_ref(few, 0, q[i:i + 1, 8 * h:8 * h + 8], None, 299, 0.1)
            assert (np.abs(got[i, 8 * h:8 * h + 8] - ref[0]) <= bound[0]).all()
    b.free()


def test_another_stream(rt, oracle):
    """All of a step on the caller's stream."""
    note("paged another stream")
    rng = np.random.default_rng(12)
    pages = Pages(rng, Q8, 2, 128, 16, [900, 40], oracle)
    new = [130, 1]
    q, gate = _inputs(rng, sum(new), 16, 128)
    call = Call(rt, pages, new, q, gate)
    want = call.run(0.1)
    _close(want, pages, new, q, gate, 0.1, "own stream")
    hip = rt.lib  # with the libraries that it was linked with
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    try:
        assert rt.lib.q4kv_use_stream(stream)
        rt.h2d(call.do, np.zeros_like(q))
        assert np.array_equal(call.run(0.1), want)
    finally:
        assert rt.lib.q4kv_use_stream(None)
    assert hip.hipStreamDestroy(stream) == 0
    assert np.array_equal(call.run(0.1), want)
    call.b.free()


@pytest.mark.parametrize("call_kind", ["attend", "read", "slots"])
def test_a_held_append_comes_first(rt, oracle, call_kind):
    """An append that the library holds for its next call is done before a
    paged call reads the pool."""
    note(f"held append before paged {call_kind}")
    rng = np.random.default_rng(13)
    n_kvh, hd = 2, 256
    bpt = n_kvh * row_bytes(Q8, hd)
    k, v = (rng.standard_normal((1, n_kvh, hd), dtype=np.float32) for _ in range(2))
    pages = Pages(rng, Q8, n_kvh, hd, 16, [16], oracle, spare=0)
    pages.table[0, 0] = 0
    pools = [p.copy() for p in pages.pools]
    q, _ = _inputs(rng, 1, 8, hd, gated=False)
    call = Call(rt, pages, [1], q, None)
    slot = call.b.up(np.array([9], np.int32))
    outs = [call.b.up(np.zeros((1, n_kvh * hd), np.float32)) for _ in range(2)]
    dk, dv = call.b.up(k), call.b.up(v)
    rt.lib.q4_hip_pos_push(9)
    assert rt.lib.q4_hip_kv_append_d(*call.dp, dk, dv, n_kvh * hd, bpt, Q8)
    for p, x in zip(pools, (k, v)):
        p[9] = oracle.encode(x, Q8).reshape(n_kvh, -1)
    if call_kind == "attend":
        got = call.run(0.1)
        pages.pools = pools
        _close(got, pages, [1], q, None, 0.1, "held")
    elif call_kind == "read":
        assert rt.lib.q4_hip_paged_read(*call.dp, *outs, slot, 1, n_kvh * hd, bpt, 16, Q8)
    else:
        assert rt.lib.q4_hip_paged_slots(slot, slot, call.b.up(np.zeros(1, np.int32)), 1, 1, 1, call.batch)
    rt.sync()
    for dev, w in zip(call.dp, pools):
        assert np.array_equal(call.b.get(dev, w), w)
    call.b.free()


@pytest.mark.parametrize("kind,n_head,n_kvh,hd,new", [
    (F16, 32, 32, 64, [1, 3]), (F16, 66, 33, 64, [1, 3]), (Q8, 40, 40, 32, [20]), (Q8, 64, 32, 32, [70, 1]),
])
def test_many_kv_heads(rt, oracle, kind, n_head, n_kvh, hd, new):
    note(f"paged attend {n_kvh} KV heads")
    rng = np.random.default_rng(n_kvh)
    lens = [300 + 20 * i for i in range(len(new))]
    pages = Pages(rng, kind, n_kvh, hd, 16, lens, oracle)
    q, gate = _inputs(rng, sum(new), n_head, hd)
    call = Call(rt, pages, new, q, gate)
    _close(call.run(0.125), pages, new, q, gate, 0.125, "many heads")
    call.b.free()


@pytest.mark.parametrize("kind,new", [(Q8, [1, 1, 1]), (F16, [130, 1, 4]), (F32, [1, 30, 0])])
def test_table_rows_of_nearly_all_positions(rt, oracle, kind, new):
    """Rows that could hold 2e9 positions: a run's costs are then counted in
    units of several positions."""
    note(f"paged attend wide tables kind={kind}")
    rng = np.random.default_rng(31)
    pages = Pages(rng, kind, 1, 32, 100000, [120000, 5, 60000], oracle, spare=1)
    wide = np.full((3, 20000), -1, np.int32)
    wide[:, :pages.stride] = pages.table
    pages.table, pages.stride = wide, 20000
    q, gate = _inputs(rng, sum(new), 16, 32)
    call = Call(rt, pages, new, q, gate)
    _close(call.run(0.2), pages, new, q, gate, 0.2, "wide tables")
    call.b.free()


@pytest.mark.parametrize("kind,n_kvh,n_slots,new", [(F32, 4, 1100000, [1, 2]), (F16, 8, 1100000, [150, 1]),
                                                    (Q8, 8, 2050000, [1, 40]), (Q8, 8, 2050000, [3, 1])])
def test_pools_past_4_gib(rt, oracle, kind, n_kvh, n_slots, new):
    """Rows written to, read from and attended at byte offsets past 2^32."""
    note(f"paged pool of {n_slots} slots kind={kind}")
    rng = np.random.default_rng(77)
    hd, page, lens = 256, 50, [400, 330]
    row = row_bytes(kind, hd)
    bpt, n_pages = n_kvh * row, n_slots // page
    assert n_slots * bpt > 1 << 32
    pages = Pages(rng, kind, n_kvh, hd, page, lens, oracle, spare=0)
    few = pages.table.copy()
    real = n_pages - 1 - np.arange(pages.n_pages) * 3  # the pool's last pages
    real[: pages.n_pages // 2] = np.arange(pages.n_pages // 2)[::-1]  # and its first
    q, gate = _inputs(rng, sum(new), 2 * n_kvh, hd)
    b = Bufs(rt)
    big = [rt.alloc(n_slots * bpt) for _ in range(2)]
    try:
        n = n_kvh * hd
        slot = np.concatenate([real[few[i, np.arange(m) // page]] * page + np.arange(m) % page
                               for i, m in enumerate(lens)]).astype(np.int32)
        k, v = (rng.standard_normal((len(slot), n), dtype=np.float32) for _ in range(2))
        ds = b.up(slot)
        assert rt.lib.q4_hip_paged_append(*big, b.up(k), b.up(v), n, n, ds, len(slot), n, bpt, n_slots, kind)
        outs = [b.up(np.zeros_like(k)) for _ in range(2)]
        assert rt.lib.q4_hip_paged_read(*big, *outs, ds, len(slot), n, bpt, n_slots, kind)
        rt.sync()
        at = 0
        for i, m in enumerate(lens):
            for p, x in zip(pages.pools, (k, v)):
                p[pages.slots(i, m)] = oracle.encode(x[at:at + m], kind).reshape(m, n_kvh, row)
            at += m
        from paged_util import values
        for o, p in zip(outs, pages.pools):
            held = np.concatenate([pages.slots(i, m) for i, m in enumerate(lens)])
            assert np.array_equal(b.get(o, k), values(kind, p[held]).reshape(k.shape).astype(np.float32))
        table = np.where(few >= 0, real[np.maximum(few, 0)], -1).astype(np.int32)
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        batch = q4kv.PagedBatch(b.up(table), b.up(start), b.up(np.int32(lens)), 2, pages.stride, page, n_pages)
        do = b.up(np.full_like(q, 123.0))
        assert rt.lib.q4_hip_qsa_paged_attend(b.up(q), *big, b.up(gate), do, batch, sum(new), max(new), 2 * n_kvh,
                                              n_kvh, hd, 0.1, kind)
        rt.sync()
        _close(b.get(do, q), pages, new, q, gate, 0.1, "past 4 GiB")
    finally:
        for p in big:
            rt.free(p)
        b.free()


@pytest.mark.parametrize("kind,n_head,n_kvh,hd,new", [
    (Q8, 16, 2, 256, [64]), (Q8, 16, 2, 256, [65]), (F16, 16, 2, 256, [60, 4]), (F16, 16, 2, 256, [60, 5]),
    (Q8, 32, 8, 128, [24]), (Q8, 32, 8, 128, [25]), (F16, 24, 4, 64, [8, 8, 16]), (F16, 24, 4, 64, [8, 9, 16]),
    (Q8, 16, 2, 160, [1, 1, 60, 1, 1]), (Q8, 16, 2, 160, [1, 1, 61, 1, 1]), (Q8, 5, 5, 256, [220]), (Q8, 16, 2, 96, [3, 33, 1]),
])
def test_short_chunks_either_way(rt, oracle, kind, n_head, n_kvh, hd, new):
    """Launches whose columns are just few enough for the rows kernel alone,
    and one token more."""
    note(f"paged attend short chunks kind={kind} hd={hd} new={new}")
    rng = np.random.default_rng(sum(new) + hd)
    lens = [n + 37 * i for i, n in enumerate(new)]
    lens[-1] += 900
    pages = Pages(rng, kind, n_kvh, hd, 16, lens, oracle)
    q, gate = _inputs(rng, sum(new), n_head, hd)
    call = Call(rt, pages, new, q, gate)
    _close(call.run(hd ** -0.5), pages, new, q, gate, hd ** -0.5, "short chunks")
    call.b.free()


@pytest.mark.parametrize("hd,new", [(256, 150), (96, 160)])
def test_large_scales_on_the_tiles(rt, oracle, hd, new):
    """q8_0 rows with block scales past 512 that a tile meets late."""
    note(f"paged attend large scales hd={hd}")
    rng = np.random.default_rng(hd)
    pages = Pages(rng, Q8, 2, hd, 16, [700, 300], oracle)
    for i, at in ((0, 650), (1, 70)):
        big = rng.standard_normal((1, 2, hd)).astype(np.float32) * np.float32(1.5e5)
        pages.pools[1][pages.slots(i, 300 if i else 700)[at]] = oracle.encode(big, Q8).reshape(2, row_bytes(Q8, hd))
    q, gate = _inputs(rng, 2 * new, 8, hd)
    call = Call(rt, pages, [new, new], q, gate)
    _close(call.run(0.1), pages, [new, new], q, gate, 0.1, "large scales")
    call.b.free()


@pytest.mark.parametrize("kind,n_head,hd,new", [(Q8, 16, 256, [1, 4]), (Q8, 24, 256, [100, 1]), (F16, 16, 128, [130, 2]),
                                                (F32, 16, 256, [2, 3]), (F16, 4, 40, [3, 1])])
def test_queries_and_scales_at_the_edges(rt, oracle, kind, n_head, hd, new):
    """Scales of zero and below it; queries of zeros; a query that is not
    finite makes its own row so and no other."""
    note(f"paged attend edge queries kind={kind} hd={hd}")
    rng = np.random.default_rng(hd + kind)
    pages = Pages(rng, kind, 2, hd, 16, [500, 160], oracle)
    q, gate = _inputs(rng, sum(new), n_head, hd)
    q[0, 1] = 0.0
    call = Call(rt, pages, new, q, gate)
    for scale in (0.0, -0.07):
        _close(call.run(scale), pages, new, q, gate, scale, f"scale {scale}")
    first = call.run(0.1)
    call.b.free()
    bad = q.copy()
    bad[0, 2, 5], bad[-1, n_head - 1, 0] = np.nan, np.inf
    call = Call(rt, pages, new, bad, gate)
    got = call.run(0.1)
    hit = np.zeros(q.shape[:2], bool)
    hit[0, 2] = hit[-1, n_head - 1] = True
    assert np.isnan(got[hit]).all()
    # the others' bits may follow another running maximum: fp32 sums in another order
    assert np.abs(got[~hit] - first[~hit]).max() <= 1e-5 * np.abs(first).max()
    call.b.free()


@pytest.mark.parametrize("kind,hd", [(Q8, 128), (F16, 256), (F32, 64)])
def test_sizes_told_that_are_not_those_of_the_batch(rt, oracle, kind, hd):
    """n_tok = n_seq * max_q looks like requests that are alike; these are not."""
    note(f"paged attend told sizes kind={kind} hd={hd}")
    rng = np.random.default_rng(hd)
    new = [1, 200, 0, 15]
    pages = Pages(rng, kind, 2, hd, 16, [900, 333, 40, 15], oracle)
    q, gate = _inputs(rng, 216, 8, hd)
    call = Call(rt, pages, new, q, gate)
    for told in (54, 1, 1 << 30):  # 216 = 4 * 54
        _close(call.run(0.1, max_q=told), pages, new, q, gate, 0.1, f"told {told}")
    call.b.free()


def test_the_same_bits_again(rt, oracle):
    """No result depends on an order that changes from run to run."""
    note("paged attend repeated")
    rng = np.random.default_rng(14)
    for kind, new in ((Q8, [1, 200, 1, 64, 1]), (F16, [1, 1, 1, 1, 1]), (F32, [3, 3, 3, 3, 3])):
        pages = Pages(rng, kind, 2, 128, 16, [5000, 900, 77, 1300, 2], oracle)
        q, gate = _inputs(rng, sum(new), 16, 128)
        call = Call(rt, pages, new, q, gate)
        first = call.run(0.1)
        for _ in range(3):
            assert np.array_equal(call.run(0.1), first)
        call.b.free()


BIG = 1 << 30


def test_plan_refuses(rt):
    """One wrong argument at a time, lengths out that are lengths in among
    them; every pointer its own memory."""
    note("plan refusals, pointers apart")
    p, ctx, new = (rt.alloc(1 << 12) for _ in range(3))
    good = [ctx, new, 2, 16, p, 4, p, 8, p, p, p, p, 4, p, None, None]
    bad = [(0, None), (1, None), (2, 0), (2, 65537), (3, 0), (4, None), (5, 0), (6, None), (7, 0), (8, None),
           (9, None), (10, None), (11, None), (12, 0), (13, None), (3, BIG), (5, BIG), (7, BIG), (12, 1 << 31),
           (11, ctx), (11, new), (10, ctx), (10, new)]
    for at, v in bad:
        args = list(good)
        args[at] = v
        assert not rt.lib.q4_hip_paged_plan(*args), (at, v)
    rt.sync()
    for x in (p, ctx, new):
        rt.free(x)


def test_attend_refuses(rt):
    """The same for the attention, outputs over its inputs among them."""
    note("paged attend refusals, pointers apart")
    p, q, out, gate = (rt.alloc(1 << 14) for _ in range(4))
    batch = q4kv.PagedBatch
    ok = batch(p, p, p, 2, 4, 16, 8)
    bads = [None, batch(None, p, p, 2, 4, 16, 8), batch(p, None, p, 2, 4, 16, 8), batch(p, p, None, 2, 4, 16, 8),
            batch(p, p, p, 0, 4, 16, 8), batch(p, p, p, 65537, 4, 16, 8), batch(p, p, p, 2, 0, 16, 8),
            batch(p, p, p, 2, 4, 0, 8), batch(p, p, p, 2, 4, 16, 0), batch(p, p, p, 2, BIG, 2, 8),
            batch(p, p, p, 2, 4, 2, BIG)]
    good = [q, p, p, gate, out, ok, 2, 1, 8, 2, 64, 0.125, Q8]
    bad = [(0, None), (1, None), (2, None), (4, None), (4, q), (4, gate), (6, 0), (7, 0), (8, 0), (8, 7), (9, 0),
           (10, 0), (10, 257), (10, 48), (12, 3), (12, -1), (1, p + 1), (2, p + 1), (6, 1 << 31)]
    for at, v in bad + [(5, x) for x in bads]:
        args = list(good)
        args[at] = v
        assert not rt.lib.q4_hip_qsa_paged_attend(*args), (at, v)
    rt.sync()
    for x in (p, q, out, gate):
        rt.free(x)
