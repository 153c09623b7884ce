"""Plain references of the paged cache's operators, in 64 bits and whole
numbers, and the buffers that the tests hand to the library."""
from __future__ import annotations

import numpy as np

import q4kv


def row_bytes(kind: int, hd: int) -> int:
    return hd // 32 * 34 if kind == q4kv.KV_Q8 else hd * (2 if kind == q4kv.KV_F16 else 4)


def values(kind: int, rows: np.ndarray) -> np.ndarray:
    """Cache bytes [..., row] -> the values that they hold, float64 [..., hd]."""
    rows = np.ascontiguousarray(rows)
    if kind == q4kv.KV_F16:
        return rows.view(np.float16).astype(np.float64)
    if kind == q4kv.KV_F32:
        return rows.view(np.float32).astype(np.float64)
    b = rows.reshape(*rows.shape[:-1], rows.shape[-1] // 34, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    q = np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64)
    return (q * d).reshape(*rows.shape[:-1], rows.shape[-1] // 34 * 32)


class Pages:
    """A pool of n_pages pages for one layer and block tables over it. Rows
    that no request holds are filled with values that are not finite."""

    def __init__(self, rng, kind, n_kvh, hd, page, lens, oracle, spare=3, scale_v=1.0, heads=None):
        self.kind, self.n_kvh, self.hd, self.page = kind, n_kvh, hd, page
        self.lens = list(lens)
        held = [-(-n // page) for n in lens]
        self.n_pages = sum(held) + spare
        self.stride = max(held + [1]) + 1
        perm = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        at = 0
        for i, h in enumerate(held):
            self.table[i, :h] = perm[at:at + h]
            at += h
        n_slots = self.n_pages * page
        rb = row_bytes(kind, hd)
        self.pools = []
        used = np.zeros(n_slots, bool)
        for i, n in enumerate(lens):
            used[self.slots(i, n)] = True
        for s in (1.0, scale_v):
            x = rng.standard_normal((n_slots, n_kvh, hd), dtype=np.float32) * np.float32(s)
            for c in (3, 77, 150, 201):
                if c < hd:
                    x[..., c] *= 8.0
            pool = oracle.encode(x, kind).reshape(n_slots, n_kvh, rb).copy()
            if kind == q4kv.KV_F32:
                pool[~used] = np.frombuffer(np.float32(np.nan).tobytes() * (rb // 4), np.uint8)
            elif kind == q4kv.KV_F16:
                pool[~used] = np.frombuffer(np.float16(np.inf).tobytes() * (rb // 2), np.uint8)
            else:
                pool[~used] = np.frombuffer((np.float16(np.nan).tobytes() + b"\x7f" * 32) * (rb // 34), np.uint8)
            self.pools.append(pool)

    def slots(self, i, n):
        p = np.arange(n)
        return self.table[i, p // self.page].astype(np.int64) * self.page + p % self.page


def attend_ref(pages, i, q, gate, pos0, scale):
    """Request i's outputs [n_q][n_head][hd] in 64 bits and the bound that an
    fp32 result keeps. Token t sees positions <= pos0 + t on pages that exist.

    The bound: a score is a sum of hd products in fp32, off by at most hd *
    2^-24 of the sum of their magnitudes A whatever its order (two-part
    operands keep 2^-22 of them beside that), so a weight by twice that, and
    the weighted sum and its parts by 2^-16 of the weighted magnitudes (fp32
    sums over runs of a few thousand positions, rounded to nearest). A weight
    in two fp16 parts, beside a largest one of at least 1, is off by at most
    2^-23 of itself or, where the second part is below fp16's normal numbers,
    by their step 2^-24 (fp32 weights below 2^-126 by less than that): 2^-24
    of the magnitudes that are seen, over the weights' sum."""
    n_q, n_head, hd = q.shape
    gqa = n_head // pages.n_kvh
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    n_all = max(0, min(pos0 + n_q, pages.stride * pages.page))
    p = np.arange(n_all)
    number = pages.table[i, p // pages.page].astype(np.int64)
    ok = (number >= 0) & (number < pages.n_pages)
    slot = np.where(ok, number * pages.page + p % pages.page, 0)
    k = values(pages.kind, pages.pools[0][slot])
    v = values(pages.kind, pages.pools[1][slot])
    seen = ok[None, :] & (p[None, :] <= pos0 + np.arange(n_q)[:, None])
    g = np.ones(q.shape) if gate is None else 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
    with np.errstate(invalid="ignore", over="ignore"):
        for h in range(n_head):
            kk, vv = k[:, h // gqa], v[:, h // gqa]
            qq = q[:, h].astype(np.float64) * scale
            s = np.where(seen, qq @ kk.T, -np.inf)
            a = np.where(seen, np.abs(qq) @ np.abs(kk).T, 0.0).max(1, initial=0.0)
            m = s.max(1, initial=-np.inf, keepdims=True)
            w = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0.0)), 0.0)
            total = w.sum(1, keepdims=True)
            w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
            step = np.divide(2.0 ** -24, total, out=np.zeros_like(total), where=total > 0)
            vz = np.where(seen.any(0)[:, None], vv, 0.0)  # rows that nobody sees
            out[:, h] = _seen_product(w, vz, seen) * g[:, h]
            mag = _seen_product(w, np.abs(vz), seen)
            bound[:, h] = (((2.0 * hd * 2.0 ** -24) * a[:, None] + 2.0 ** -16) * mag
                           + step * _seen_product(seen.astype(np.float64), np.abs(vz), seen)) * np.abs(g[:, h])
    return out, bound


def _seen_product(w, v, seen):
    """w @ v where a weight of zero on a row that the token does not see takes
    nothing from it, whatever it holds."""
    if np.isfinite(v).all():
        return w @ v
    out = np.empty((w.shape[0], v.shape[1]))
    for t in range(w.shape[0]):
        out[t] = w[t, seen[t]] @ v[seen[t]]
    return out


def plan_ref(ctx, new, page, table, free, n_free, max_tok, n_pages):
    """q4_hip_paged_plan, request by request."""
    n_seq, stride = len(ctx), table.shape[1]
    table = table.copy()
    n_free = max(0, min(n_free, n_pages))
    q_start, kv_len = np.zeros(n_seq + 1, np.int32), np.zeros(n_seq, np.int32)
    slot, seq, pos = (np.full(max_tok, -1, np.int32) for _ in range(3))
    tok = lacked = taken = refused = 0
    for i in range(n_seq):
        add = max(int(new[i]), 0)
        first, tok = tok, tok + add
        q_start[i], q_start[i + 1] = min(first, max_tok), min(tok, max_tok)
        fits = ctx[i] >= 0 and ctx[i] + add <= stride * page and (add == 0 or tok <= max_tok)
        held = -(-int(ctx[i]) // page) if fits else 0
        need = -(-(int(ctx[i]) + add) // page) - held if fits else 0
        top = n_free - lacked
        lacked += need
        granted = fits and (need == 0 or lacked <= n_free)
        if granted:
            if need:
                taken = lacked
            for j in range(need):
                table[i, held + j] = free[top - 1 - j]
            kv_len[i] = ctx[i] + add
        else:
            refused += 1
        for t in range(first, min(tok, max_tok)):
            p = int(ctx[i]) + t - first
            seq[t], pos[t] = i, p
            if granted and 0 <= table[i, p // page] < n_pages:
                slot[t] = table[i, p // page] * page + p % page
    return dict(table=table, left=np.array([n_free - taken, refused], np.int32), q_start=q_start,
                kv_len=kv_len, slot=slot, tok_seq=seq, tok_pos=pos)


class Bufs:
    """Device copies that are freed together."""

    def __init__(self, rt):
        self.rt, self.owned = rt, []

    def up(self, x, shift=0):
        x = np.ascontiguousarray(x)
        p = self.rt.alloc(x.nbytes + 64)
        self.owned.append(p)
        self.rt.h2d(p + shift, x)
        return p + shift

    def get(self, p, like):
        return self.rt.download(p, like.nbytes, like.dtype).reshape(like.shape)

    def free(self):
        for p in self.owned:
            self.rt.free(p)
        self.owned = []
