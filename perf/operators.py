"""The paged KV cache's operators as measured cases: what a serving engine calls
for a ragged batch of requests whose cache rows lie in pages.

  tables   the requests that ended give their pages back, then the block
           tables, slot maps and query ranges of the next step are built from
           the requests' lengths
  rows     the new tokens' K and V rows are written to their slots and read
           back as the values that the cache holds
  lists    the indexer's position lists become lists of slots
  attend   causal attention of each request's new tokens over its pages, from
           one token per request (decode) to chunks of a prompt

A pool is [slot][kv head][row]; slot = page number * page size + offset. Values:
K, V and queries are N(0, 1) with four outlier channels x8 per head, gates
N(0, 1). Head layouts: 24 or 16 query heads over 2 KV heads of 256 dims (the
layouts of the other cases), others as generic sizes. Lengths follow from the
case alone (log-spaced between two bounds); pages are in random order.
"""
from __future__ import annotations

import math

import torch

own = False

F32, F16, Q8 = 0, 1, 2
WIDTH = 2051
OUTLIERS = (3, 77, 150, 201)
DEV = "cuda"


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a decode step of a small server: a token per request, few new pages
        dict(name="tables_decode_64", family="tables", n_seq=64, n_done=3, page=16, lo=200, hi=9000,
             chunk=1, n_chunk=0, spare=2048),
        # prompts arriving in chunks beside a large decode batch
        dict(name="tables_prefill_16k", family="tables", n_seq=384, n_done=40, page=16, lo=100,
             hi=12000, chunk=1000, n_chunk=16, spare=6000),
        # a prompt chunk's rows of one layer
        dict(name="rows_q8_8192", family="rows", kind=Q8, n_tok=8192, n_kvh=2, hd=256, page=64,
             spare=100000),
        # a decode batch's rows of one layer
        dict(name="rows_f16_48", family="rows", kind=F16, n_tok=48, n_kvh=8, hd=128, page=16,
             spare=60000),
        # the selections of a 512-token slice, one list per token
        dict(name="lists_slice_512", family="lists", n_seq=4, per_seq=128, n_list=1, page=64,
             lo=4000, hi=60000),
        # the selections of a decode batch, one list per KV head
        dict(name="lists_decode_32", family="lists", n_seq=32, per_seq=1, n_list=2, page=16,
             lo=8192, hi=131072),
        # one chat, one token: the smallest call
        dict(name="attend_one_q8", family="attend", kind=Q8, n_head=24, n_kvh=2, hd=256, page=16,
             n_seq=1, lo=1500, hi=1500, chunk=1, n_chunk=0),
        # a decode batch of long documents
        dict(name="attend_decode_q8_32", family="attend", kind=Q8, n_head=24, n_kvh=2, hd=256,
             page=64, n_seq=32, lo=8192, hi=131072, chunk=1, n_chunk=0),
        # a larger decode batch of 128-dim heads in f16
        dict(name="attend_decode_f16_64", family="attend", kind=F16, n_head=32, n_kvh=8, hd=128,
             page=16, n_seq=64, lo=1000, hi=16000, chunk=1, n_chunk=0),
        # drafts of four tokens verified at once, f32 cache
        dict(name="attend_verify_f32_8", family="attend", kind=F32, n_head=16, n_kvh=2, hd=256,
             page=32, n_seq=8, lo=2000, hi=30000, chunk=4, n_chunk=8),
        # three prompt chunks of odd length beside 40 decode tokens
        dict(name="attend_mixed_q8_43", family="attend", kind=Q8, n_head=24, n_kvh=2, hd=256,
             page=64, n_seq=43, lo=700, hi=16000, chunk=701, n_chunk=3),
        # a long prompt's chunk over what came before
        dict(name="attend_chunk_f16_4096", family="attend", kind=F16, n_head=16, n_kvh=2, hd=256,
             page=16, n_seq=1, lo=12288, hi=12288, chunk=4096, n_chunk=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _layout(rng, kind):
    """(n_head, n_kvh, hd): the layouts of the cases above and generic ones."""
    hd = rng.choice((256, 256, 256, 128, 128, 64, 96))
    if hd == 256:
        return rng.choice(((24, 2), (24, 2), (16, 2), (16, 4), (8, 2))) + (hd,)
    return rng.choice(((32, 8), (16, 2), (16, 4), (32, 4), (24, 2))) + (hd,)


def draw(rng):
    family = rng.choice(("tables", "rows", "lists", "attend", "attend", "attend", "attend", "attend"))
    page = rng.choice((16, 16, 32, 64, 128, 24))
    if family == "tables":
        n_seq = _log(rng, 1, 700)
        n_chunk = rng.randint(0, min(n_seq, 8))
        return dict(family=family, n_seq=n_seq, n_done=rng.randint(1, 40), page=page,
                    lo=_log(rng, 20, 500), hi=_log(rng, 600, 12000), chunk=_log(rng, 1, 2000) if n_chunk else 1,
                    n_chunk=n_chunk, spare=_log(rng, 500, 8000))
    if family == "rows":
        _, n_kvh, hd = _layout(rng, Q8)
        return dict(family=family, kind=rng.choice((Q8, Q8, F16, F32)), n_tok=_log(rng, 1, 6000 if hd * n_kvh <= 512 else 3000),
                    n_kvh=n_kvh, hd=hd, page=page, spare=_log(rng, 10, 100000))
    if family == "lists":
        n_seq = _log(rng, 1, 40)
        return dict(family=family, n_seq=n_seq, per_seq=_log(rng, 1, max(1, 500 // n_seq)),
                    n_list=rng.choice((1, 2)), page=page, lo=_log(rng, 50, 6000), hi=_log(rng, 7000, 100000))
    kind = rng.choice((Q8, Q8, Q8, F16, F16, F32))
    n_head, n_kvh, hd = _layout(rng, kind)
    form = rng.choice(("decode", "decode", "verify", "mixed", "chunk"))
    case = dict(family="attend", kind=kind, n_head=n_head, n_kvh=n_kvh, hd=hd, page=page)
    if form in ("decode", "verify"):
        n_seq = _log(rng, 1, 64)
        lo = _log(rng, 16, 8000)
        hi = _log(rng, lo, min(130000, 600000 // n_seq + lo))
        chunk = 1 if form == "decode" else rng.randint(2, 8)
        return dict(case, n_seq=n_seq, lo=max(lo, chunk), hi=max(hi, chunk), chunk=chunk,
                    n_chunk=n_seq if chunk > 1 else 0)
    if form == "mixed":
        n_seq = _log(rng, 2, 40)
        n_chunk = rng.randint(1, min(3, n_seq))
        chunk = _log(rng, 20, 500)
        return dict(case, n_seq=n_seq, lo=_log(rng, 500, 1500), hi=_log(rng, 1600, 9000), chunk=chunk,
                    n_chunk=n_chunk)
    chunk = _log(rng, 17, 2500 if kind != F32 else 700)
    ctx = chunk + rng.choice((0, _log(rng, 1, 9000)))
    return dict(case, n_seq=1, lo=ctx, hi=ctx, chunk=chunk, n_chunk=1)


def _lengths(case):
    """(positions held, the new tokens' included; new tokens) of every request."""
    n, lo, hi = case["n_seq"], case["lo"], case["hi"]
    kv = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    # the chunks lie spread over the lengths
    new = [1] * n
    for j in range(case["n_chunk"]):
        i = j * n // case["n_chunk"]
        new[i] = case["chunk"]
        kv[i] = max(kv[i], case["chunk"])
    return kv, new


# ----------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _vectors(g, *shape):
    """N(0, 1) rows [..., hd] with the outlier channels."""
    x = torch.randn(shape, generator=g, device=DEV)
    for c in OUTLIERS:
        if c < shape[-1]:
            x[..., c] *= 8.0
    return x


def _encode(kind, x):
    """Cache bytes [..., row] of fp32 rows [..., hd]. q8_0: blocks of 32, scale
    amax / 127 in fp16, values rint(x * (1 / scale)), every step rounded to
    binary32 (formed in 64 bits, where a quotient's second rounding is none)."""
    if kind != Q8:
        return (x.half() if kind == F16 else x.contiguous()).view(torch.uint8)
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = (b.abs().amax(-1, keepdim=True).double() / 127.0).float()
    inv = torch.where(d > 0, (1.0 / d.double()).float(), torch.zeros_like(d))
    q = (b * inv).round().clamp(-127, 127).to(torch.int8)
    return torch.cat([d.half().view(torch.uint8), q.view(torch.uint8)], -1).reshape(*x.shape[:-1], -1)


def _decode(kind, rows, to=torch.float32):
    """The values [..., hd] of cache bytes [..., row]."""
    if kind != Q8:
        return rows.contiguous().view(torch.float16 if kind == F16 else torch.float32).to(to)
    b = rows.reshape(*rows.shape[:-1], -1, 34)
    d = b[..., :2].contiguous().view(torch.float16).to(to)
    return (b[..., 2:].contiguous().view(torch.int8).to(to) * d).reshape(*rows.shape[:-1], -1)


def _rows_at(kind, pool, at):
    """Rows [n, kv head, row] of a pool's bytes, gathered in the widest unit that every row has."""
    unit = (torch.float32, torch.float16, torch.int16)[kind]
    return pool.view(unit)[at].view(torch.uint8)


def _row_bytes(kind, hd):
    return hd // 32 * 34 if kind == Q8 else hd * (2 if kind == F16 else 4)


def _pool(g, kind, n_slots, n_kvh, hd):
    """A pool [slot][kv head][row]: 16384 distinct rows, then those repeated
    (what a larger pool adds are addresses)."""
    some = min(n_slots, 16384)
    rows = _encode(kind, _vectors(g, some, n_kvh, hd))
    out = torch.empty(n_slots, n_kvh, rows.shape[-1], dtype=torch.uint8, device=DEV)
    for at in range(0, n_slots, some):
        out[at:at + some] = rows[:min(some, n_slots - at)]
    return out


def _pages(n, page):
    return -(-n // page)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _shuffled(g, values):
    """The lengths of a case in an order of the seed's."""
    order = torch.randperm(len(values[0]), generator=g, device=DEV).tolist()
    return [[v[i] for i in order] for v in values]


def _tables(g, lens, page, spare=0):
    """Block tables [request][most pages] of requests of these lengths, -1
    behind a request's pages, and how many pages there are; random order."""
    held = [_pages(n, page) for n in lens]
    n_pages = sum(held) + spare
    perm = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((len(lens), max(1, max(held))), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = perm[at:at + h]
        at += h
    return table, n_pages, perm[at:]


# ------------------------------------------------------- prepare, run, work

def prepare(case, seed):
    return globals()["_prepare_" + case["family"]](case, _gen(seed))


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["family"]](state)


def work(case):
    return globals()["_work_" + case["family"]](case)


def exact(case, seed):
    if case["family"] == "rows":
        return _exact_rows(prepare(case, seed))
    if case["family"] == "attend":
        return _exact_attend(prepare(case, seed))
    return None


_bound = None


def _lib():
    """The library's binding (q4kv.Runtime starts the library)."""
    global _bound
    if _bound is None:
        import sys
        from pathlib import Path

        pkg = str(Path(__file__).resolve().parent.parent / "suzuqu-engine-4exp_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import q4kv

        _bound = q4kv, q4kv.Runtime().lib
    return _bound


def _done(ok, name):
    if not ok:
        raise RuntimeError(name + " failed")


# tables: requests 0..n_seq-1 go on, rows n_seq.. of the table have ended

def _prepare_tables(case, g):
    page, n_seq, n_done = case["page"], case["n_seq"], case["n_done"]
    kv, new = _shuffled(g, _lengths(case))
    ctx = [a - b for a, b in zip(kv, new)]
    done = [max(1, case["hi"] * (j + 1) // (2 * n_done)) for j in range(n_done)]
    most = max(_pages(n, page) for n in kv + done)
    table, n_pages, free = _tables(g, ctx + done, page, case["spare"])
    wide = torch.full((n_seq + n_done, most + 3), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    stack = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    stack[:free.numel()] = free
    n_tok = sum(new) + 5  # a padded batch: the tokens behind the last request
    rows = torch.randperm(n_done, generator=g, device=DEV).int() + n_seq
    lens = _ints(ctx + done)
    return dict(family="tables", n_seq=n_seq, n_done=n_done, page=page, n_pages=n_pages, n_tok=n_tok,
                table=wide, ctx=lens[:n_seq].clone(), new=_ints(new), lens=lens, rows=rows, stack=stack,
                n_free=_ints([free.numel()]), mid=_ints([0]), left=_ints([0, 0]),
                q_start=_ints([0] * (n_seq + 1)), kv_len=_ints([0] * n_seq),
                slot=_ints([0] * n_tok), tok_seq=_ints([0] * n_tok), tok_pos=_ints([0] * n_tok))


def _plain_tables(s):
    page, n_seq, n_tok = s["page"], s["n_seq"], s["n_tok"]
    col = torch.arange(s["table"].shape[1], device=DEV)
    # the pages of the requests that ended, behind those that are free
    rows = s["rows"].long()
    held = (s["lens"][rows].long() + page - 1) // page
    at = s["n_free"].long() + held.cumsum(0) - held
    n_pages = s["n_pages"]
    put = torch.where(col < held[:, None], at[:, None] + col, n_pages)
    stack = torch.cat([s["stack"], s["stack"][:1]])
    stack[put.flatten()] = s["table"][rows].flatten()
    stack = stack[:n_pages]
    avail = s["n_free"].long() + held.sum()
    # pages that each request still needs, in the requests' order
    ctx, new = s["ctx"].long(), s["new"].long()
    held = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - held
    upto = need.cumsum(0)
    granted = (need == 0) | (upto <= avail)
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None]) & granted[:, None]
    nth = (upto - need)[:, None] + col - held[:, None]
    page_of = stack[(avail - 1 - nth).clamp(0, n_pages - 1)]
    table = s["table"].clone()
    table[:n_seq] = torch.where(fresh, page_of, table[:n_seq])
    left = avail - torch.where(granted & (need > 0), upto, 0).max()
    # token ranges, slots
    q_start = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    t = torch.arange(n_tok, device=DEV)
    seq = torch.searchsorted(q_start[1:].contiguous(), t, right=True)
    live = seq < n_seq
    i = seq.clamp(max=n_seq - 1)
    pos = ctx[i] + t - q_start[i]
    fits = live & granted[i]
    col_of = (pos // page).clamp(0, table.shape[1] - 1)
    slot = torch.where(fits, table[i, col_of].long() * page + pos % page, -1)
    return [table, stack, torch.cat([left, (~granted).sum(0, keepdim=True)]).int(), q_start.int(),
            torch.where(granted, ctx + new, 0).int(), slot.int(), torch.where(live, seq, -1).int(),
            torch.where(live, pos, -1).int()]


def _own_tables(s):
    _, lib = _lib()
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    stride = s["table"].shape[1]
    _done(lib.q4_hip_paged_release(p["table"], stride, p["lens"], p["rows"], s["n_done"], s["page"],
                                   p["stack"], s["n_pages"], p["n_free"], p["mid"]), "paged_release")
    _done(lib.q4_hip_paged_plan(p["ctx"], p["new"], s["n_seq"], s["page"], p["table"], stride, p["stack"],
                                s["n_pages"], p["mid"], p["left"], p["q_start"], p["kv_len"], s["n_tok"],
                                p["slot"], p["tok_seq"], p["tok_pos"]), "paged_plan")
    return [s[k] for k in ("table", "stack", "left", "q_start", "kv_len", "slot", "tok_seq", "tok_pos")]


def _work_tables(case):
    kv, new = _lengths(case)
    done = sum(_pages(max(1, case["hi"] * (j + 1) // (2 * case["n_done"])), case["page"])
               for j in range(case["n_done"]))
    fresh = sum(_pages(a, case["page"]) - _pages(a - b, case["page"]) for a, b in zip(kv, new))
    return {"bytes": 16 * len(kv) + 8 * case["n_done"] + 8 * (done + fresh) + 12 * sum(new), "flops": 0}


# rows: slots anywhere in the pool, the last token a padding row without a slot

def _prepare_rows(case, g):
    kind, n_tok, n_kvh, hd, page = (case[k] for k in ("kind", "n_tok", "n_kvh", "hd", "page"))
    n_slots = _pages(n_tok + case["spare"], page) * page
    first = torch.randperm(n_slots // page, generator=g, device=DEV)[:_pages(n_tok, page)]
    slot = (first[:, None] * page + torch.arange(page, device=DEV)).flatten()[:n_tok].int()
    if n_tok > 1:
        slot[-1] = -1
    n = n_kvh * hd
    return dict(family="rows", kind=kind, n_tok=n_tok, n_kvh=n_kvh, hd=hd, n_slots=n_slots,
                bpt=n_kvh * _row_bytes(kind, hd), k=_vectors(g, n_tok, n_kvh, hd), v=_vectors(g, n_tok, n_kvh, hd),
                slot=slot, kp=_pool(g, kind, n_slots, n_kvh, hd), vp=_pool(g, kind, n_slots, n_kvh, hd),
                ko=torch.empty(n_tok, n, device=DEV), vo=torch.empty(n_tok, n, device=DEV))


def _plain_rows(s):
    keep = s["slot"] >= 0
    # a row without a slot repeats the first one's write, so the pool keeps its other rows
    at = torch.where(keep, s["slot"], s["slot"][0]).long()
    got = []
    for pool, x in ((s["kp"], s["k"]), (s["vp"], s["v"])):
        rows = _encode(s["kind"], x)
        pool[at] = torch.where(keep[:, None, None], rows, rows[:1])
        back = _decode(s["kind"], _rows_at(s["kind"], pool, at)).reshape(s["n_tok"], -1)
        got.append(torch.where(keep[:, None], back, 0.0))
    return got


def _own_rows(s):
    _, lib = _lib()
    n = s["n_kvh"] * s["hd"]
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    _done(lib.q4_hip_paged_append(p["kp"], p["vp"], p["k"], p["v"], n, n, p["slot"], s["n_tok"], n, s["bpt"],
                                  s["n_slots"], s["kind"]), "paged_append")
    _done(lib.q4_hip_paged_read(p["kp"], p["vp"], p["ko"], p["vo"], p["slot"], s["n_tok"], n, s["bpt"],
                                s["n_slots"], s["kind"]), "paged_read")
    return [s["ko"], s["vo"]]


def _exact_rows(s):
    got = []
    for x in (s["k"], s["v"]):
        if s["kind"] == F32:
            y = x.double()
        elif s["kind"] == F16:
            y = x.double().to(torch.float16).double()
        else:
            b = x.double().reshape(s["n_tok"], -1, 32)
            top = b.abs().amax(-1, keepdim=True)
            d = (top / 127).float().double()
            inv = torch.where(d > 0, 1 / d, 0).float().double()
            y = (b * inv).float().double().round().clamp(-127, 127) * d.half().double()
        got.append(torch.where(s["slot"][:, None] >= 0, y.reshape(s["n_tok"], -1), 0.0))
    return got


def _work_rows(case):
    n = case["n_kvh"] * case["hd"]
    row = case["n_kvh"] * _row_bytes(case["kind"], case["hd"])
    return {"bytes": case["n_tok"] * (2 * (4 * n + row) + 2 * (row + 4 * n) + 8), "flops": 0}


# lists: `per_seq` tokens of each request, n_list lists of WIDTH positions each

def _prepare_lists(case, g):
    kv, = _shuffled(g, [_lengths(dict(case, chunk=1, n_chunk=0))[0]])
    table, n_pages, _ = _tables(g, kv, case["page"], 100)
    n_tok = case["n_seq"] * case["per_seq"]
    seq = torch.arange(case["n_seq"], device=DEV).repeat_interleave(case["per_seq"]).int()
    n = torch.tensor(kv, device=DEV)[seq.long()]
    u = torch.rand((n_tok * case["n_list"], WIDTH), generator=g, device=DEV)
    idx = (u.sort(-1).values * n.repeat_interleave(case["n_list"])[:, None]).int()
    idx[:, -3:] = -1  # a list's padding
    return dict(family="lists", idx=idx, out=torch.empty_like(idx), table=table, kv_len=_ints(kv), tok_seq=seq,
                n_tok=n_tok, n_list=case["n_list"], page=case["page"], n_pages=n_pages, n_seq=case["n_seq"])


def _plain_lists(s):
    idx = s["idx"].long()
    seq = s["tok_seq"].long().repeat_interleave(s["n_list"], output_size=idx.shape[0])[:, None]
    ok = (idx >= 0) & (idx < s["kv_len"].long()[seq])
    at = torch.where(ok, idx, 0)
    number = s["table"][seq, at // s["page"]].long()
    ok = ok & (number >= 0) & (number < s["n_pages"])
    return torch.where(ok, number * s["page"] + at % s["page"], -1).int()


def _own_lists(s):
    q4kv, lib = _lib()
    if "batch" not in s:
        s["batch"] = q4kv.PagedBatch(s["table"].data_ptr(), None, s["kv_len"].data_ptr(), s["n_seq"],
                                     s["table"].shape[1], s["page"], s["n_pages"])
    _done(lib.q4_hip_paged_slots(s["idx"].data_ptr(), s["out"].data_ptr(), s["tok_seq"].data_ptr(), s["n_tok"],
                                 s["n_list"], WIDTH, s["batch"]), "paged_slots")
    return s["out"]


def _work_lists(case):
    kv, _ = _lengths(dict(case, chunk=1, n_chunk=0))
    entries = case["n_seq"] * case["per_seq"] * case["n_list"] * WIDTH
    return {"bytes": 8 * entries + 4 * sum(_pages(n, case["page"]) for n in kv), "flops": 0}


# attend: the new tokens are the last ones of each request's positions

def _prepare_attend(case, g):
    kind, n_head, n_kvh, hd, page = (case[k] for k in ("kind", "n_head", "n_kvh", "hd", "page"))
    kv, new = _shuffled(g, _lengths(case))
    table, n_pages, _ = _tables(g, kv, page, 7)
    n_tok = sum(new)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return dict(family="attend", kind=kind, n_head=n_head, n_kvh=n_kvh, hd=hd, page=page, n_pages=n_pages,
                n_seq=len(kv), n_tok=n_tok, max_q=max(new), scale=1.0 / math.sqrt(hd), kv=kv, start=start,
                table=table, q_start=_ints(start), kv_len=_ints(kv),
                kp=_pool(g, kind, n_pages * page, n_kvh, hd), vp=_pool(g, kind, n_pages * page, n_kvh, hd),
                q=_vectors(g, n_tok, n_head, hd), gate=torch.randn((n_tok, n_head, hd), generator=g, device=DEV),
                out=torch.empty(n_tok, n_head, hd, device=DEV))


def _slots_of(s, i):
    """The slots of request i's positions."""
    n, page = s["kv"][i], s["page"]
    pages = s["table"][i, :_pages(n, page)].long()
    return (pages[:, None] * page + torch.arange(page, device=DEV)).flatten()[:n]


def _plain_attend(s):
    nk, hd = s["n_kvh"], s["hd"]
    gqa = s["n_head"] // nk
    out = torch.empty_like(s["q"])
    for i in range(s["n_seq"]):  # requests differ in both lengths
        a, b, n = s["start"][i], s["start"][i + 1], s["kv"][i]
        at = _slots_of(s, i)
        k = _decode(s["kind"], _rows_at(s["kind"], s["kp"], at)).permute(1, 2, 0).contiguous()
        v = _decode(s["kind"], _rows_at(s["kind"], s["vp"], at)).permute(1, 0, 2).contiguous()
        q = (s["q"][a:b] * s["scale"]).reshape(b - a, nk, gqa, hd).permute(1, 0, 2, 3).reshape(nk, -1, hd)
        w = torch.matmul(q, k)
        if b - a > 1:
            seen = torch.arange(n, device=DEV) <= torch.arange(n - (b - a), n, device=DEV)[:, None]
            w.view(nk, b - a, gqa, n).masked_fill_(~seen[None, :, None, :], -math.inf)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
        o = o.reshape(nk, b - a, gqa, hd).permute(1, 0, 2, 3).reshape(b - a, s["n_head"], hd)
        out[a:b] = o / (1.0 + torch.exp(-s["gate"][a:b]))
    return out


def _own_attend(s):
    q4kv, lib = _lib()
    if "batch" not in s:
        s["batch"] = q4kv.PagedBatch(s["table"].data_ptr(), s["q_start"].data_ptr(), s["kv_len"].data_ptr(),
                                     s["n_seq"], s["table"].shape[1], s["page"], s["n_pages"])
    _done(lib.q4_hip_qsa_paged_attend(s["q"].data_ptr(), s["kp"].data_ptr(), s["vp"].data_ptr(),
                                      s["gate"].data_ptr(), s["out"].data_ptr(), s["batch"], s["n_tok"],
                                      s["max_q"], s["n_head"], s["n_kvh"], s["hd"], s["scale"], s["kind"]),
          "qsa_paged_attend")
    return s["out"]


def _exact_attend(s):
    gqa, hd = s["n_head"] // s["n_kvh"], s["hd"]
    out = torch.zeros(s["n_tok"], s["n_head"], hd, dtype=torch.float64, device=DEV)
    for i in range(s["n_seq"]):
        a, b, n = s["start"][i], s["start"][i + 1], s["kv"][i]
        at = _slots_of(s, i)
        first = torch.arange(n - (b - a), n, device=DEV)
        for kh in range(s["n_kvh"]):
            k = _decode(s["kind"], s["kp"][at, kh], torch.float64)
            v = _decode(s["kind"], s["vp"][at, kh], torch.float64)
            kt = k.t().contiguous()
            for t0 in range(0, b - a, 512):  # 512 tokens' weights at a time
                t1 = min(b - a, t0 + 512)
                for h in range(kh * gqa, (kh + 1) * gqa):
                    x = torch.mm(s["q"][a + t0:a + t1, h].double(), kt) * s["scale"]
                    x[torch.arange(n, device=DEV)[None, :] > first[t0:t1, None]] = -math.inf
                    y = torch.mm(torch.softmax(x, -1), v)
                    out[a + t0:a + t1, h] = y * torch.sigmoid(s["gate"][a + t0:a + t1, h].double())
    return out


def _work_attend(case):
    kv, new = _lengths(case)
    row = case["n_kvh"] * _row_bytes(case["kind"], case["hd"])
    n_tok = sum(new)
    seen = sum(b * n - b * (b - 1) // 2 for n, b in zip(kv, new))
    return {"bytes": 2 * row * sum(kv) + 12 * n_tok * case["n_head"] * case["hd"]
            + 4 * sum(_pages(n, case["page"]) for n in kv),
            "flops": 4 * case["hd"] * case["n_head"] * seen}
