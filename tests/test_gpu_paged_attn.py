"""Paged attention (q4kv_paged_attn.hip) against the formula in 64 bits: every
width, head layouts, head dims and page sizes, one token to chunks, ragged and
mixed batches, rows that see nothing, pages that do not exist, rows behind the
last request, values that are not finite where nobody looks."""
import numpy as np
import pytest

import q4kv
from gpu_util import note
from paged_util import Bufs, Pages, attend_ref, row_bytes

pytestmark = pytest.mark.gpu

F32, F16, Q8 = 0, 1, 2


class Call:
    """A batch on the device and one attend call."""

    def __init__(self, rt, pages, new, q, gate, shift=0, n_tok=None, lens=None, starts=None):
        self.rt, self.pages, self.q = rt, pages, q
        self.b = Bufs(rt)
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if starts is None else np.int32(starts)
        self.n_tok = q.shape[0] if n_tok is None else n_tok
        self.dq, self.dg = self.b.up(q, shift), None if gate is None else self.b.up(gate, shift)
        self.shift = shift
        self.do = self.b.up(np.full_like(q, 123.0), shift)
        self.dp = [self.b.up(p) for p in pages.pools]
        self.batch = q4kv.PagedBatch(self.b.up(pages.table), self.b.up(self.start),
                                     self.b.up(np.int32(pages.lens if lens is None else lens)),
                                     len(pages.lens), pages.stride, pages.page, pages.n_pages)
        self.max_q = int(max(max(new), 1))

    def run(self, scale, max_q=None):
        n_head, hd = self.q.shape[1:]
        assert self.rt.lib.q4_hip_qsa_paged_attend(self.dq, *self.dp, self.dg, self.do, self.batch, self.n_tok,
                                                   max_q or self.max_q, n_head, self.pages.n_kvh, hd, scale,
                                                   self.pages.kind)
        self.rt.sync()
        return self.b.get(self.do, self.q)


def _close(got, pages, new, q, gate, scale, what, lens=None, start=None):
    """Every request's rows against the formula; rows of nobody untouched.
    Beside the bound of each element, the whole is within 2e-5 in norm."""
    start = np.concatenate([[0], np.cumsum(new)]) if start is None else start
    lens = pages.lens if lens is None else lens
    mine = np.zeros(q.shape[0], bool)
    err = norm = 0.0
    for i, n in enumerate(new):
        a = int(start[i])
        if n == 0:
            continue
        ref, bound = attend_ref(pages, i, q[a:a + n], None if gate is None else gate[a:a + n],
                                int(lens[i]) - n, scale)
        mine[a:a + n] = True
        fine = np.isfinite(ref)  # values that the cache's width cannot hold are inf
        assert (np.isfinite(got[a:a + n]) == fine).all(), f"{what}: request {i}: not finite"
        ref, bound = np.where(fine, ref, 0.0), np.where(fine, bound, 0.0)
        d = np.abs(np.where(fine, got[a:a + n], 0.0).astype(np.float64) - ref)
        bad = d > bound
        assert not bad.any(), (f"{what}: request {i}: {bad.sum()} of {bad.size} past the bound, "
                               f"worst {np.max(d - bound):.3e} over at {np.argwhere(bad)[0]}, err {d.max():.3e}")
        err, norm = err + (d ** 2).sum(), norm + (ref ** 2).sum()
    assert (got[~mine] == 123.0).all(), f"{what}: rows of no request were written"
    assert err <= (2e-5) ** 2 * norm or norm == 0, f"{what}: off by {np.sqrt(err / norm):.2e} in norm"
    return np.sqrt(err / max(norm, 1e-300))


def _inputs(rng, n_tok, n_head, hd, gated=True):
    q = rng.standard_normal((n_tok, n_head, hd), dtype=np.float32)
    for c in (3, 77, 150, 201):
        if c < hd:
            q[..., c] *= 8.0
    return q, rng.standard_normal(q.shape).astype(np.float32) if gated else None


# kind, n_head, n_kvh, hd, page, (length, new tokens) of each request
CASES = [
    # one token each
    (Q8, 24, 2, 256, 16, [(1500, 1)]),
    (Q8, 16, 2, 256, 64, [(1, 1), (63, 1), (64, 1), (65, 1), (4001, 1)]),
    (Q8, 8, 8, 256, 7, [(333, 1), (20, 1)]),
    (F16, 32, 8, 128, 16, [(1000, 1), (17, 1), (129, 1), (5000, 1)]),
    (F16, 24, 2, 256, 32, [(3000, 1), (31, 1)]),
    (F32, 16, 2, 256, 16, [(700, 1), (15, 1), (2500, 1)]),
    (F32, 32, 4, 128, 1, [(257, 1), (2, 1)]),
    (Q8, 40, 2, 128, 24, [(999, 1), (48, 1)]),     # 20 heads per KV head
    (Q8, 4, 1, 32, 5, [(100, 1), (1, 1)]),
    (F16, 14, 2, 64, 128, [(1300, 1), (128, 1)]),
    # drafts of a few tokens
    (Q8, 24, 2, 256, 16, [(800, 4), (4, 4), (77, 3), (2100, 5)]),
    (F32, 16, 2, 256, 32, [(1200, 4), (600, 2)]),
    (F16, 16, 4, 96, 16, [(500, 3), (3, 3), (999, 8)]),
    (Q8, 16, 4, 96, 16, [(500, 3), (33, 8)]),      # rows of 102 bytes
    # chunks
    (Q8, 24, 2, 256, 64, [(900, 300)]),
    (Q8, 24, 2, 256, 16, [(301, 301), (64, 64), (65, 65)]),
    (F16, 16, 2, 256, 16, [(1500, 257)]),
    (F16, 32, 8, 128, 48, [(700, 133), (129, 129)]),
    (Q8, 32, 8, 128, 16, [(515, 200)]),
    (Q8, 16, 2, 64, 16, [(1027, 150), (31, 17)]),
    (F16, 6, 3, 64, 9, [(400, 399)]),              # 2 heads per KV head
    (Q8, 12, 1, 160, 16, [(333, 200)]),
    (F16, 8, 1, 192, 64, [(640, 130), (5, 5)]),
    (F32, 16, 2, 128, 16, [(400, 140), (3, 2)]),
    (F32, 8, 2, 256, 64, [(300, 77)]),
    (Q8, 3, 3, 256, 16, [(260, 260)]),             # one head per KV head
    (Q8, 72, 2, 64, 16, [(90, 40), (300, 1)]),     # 36 heads per KV head
    # mixed
    (Q8, 24, 2, 256, 64, [(700, 1), (450, 200), (90, 1), (1, 1), (1300, 64), (2000, 1), (8, 8)]),
    (F16, 16, 2, 256, 16, [(129, 128), (900, 1), (555, 11), (16, 1)]),
    (Q8, 32, 8, 128, 16, [(300, 1)] * 9 + [(200, 90)] + [(64, 2)] * 5),
    # shapes of the plain kernel
    (F16, 4, 2, 33, 16, [(200, 1), (90, 20)]),
    (F32, 3, 1, 7, 3, [(50, 50), (1, 1)]),
    (F16, 2, 2, 250, 16, [(130, 2)]),
]


@pytest.mark.parametrize("kind,n_head,n_kvh,hd,page,reqs", CASES)
def test_paged_attention(rt, oracle, kind, n_head, n_kvh, hd, page, reqs):
    note(f"paged attend kind={kind} heads={n_head}/{n_kvh} hd={hd} page={page} reqs={reqs[:4]}")
    rng = np.random.default_rng(hd + page + 7 * n_head + kind)
    lens, new = [r[0] for r in reqs], [r[1] for r in reqs]
    pages = Pages(rng, kind, n_kvh, hd, page, lens, oracle)
    q, gate = _inputs(rng, sum(new) + 3, n_head, hd)  # three rows that nobody has
    call = Call(rt, pages, new, q, gate)
    scale = 1.0 / np.sqrt(hd)
    _close(call.run(scale), pages, new, q, gate, scale, f"hd={hd}")
    call.b.free()


@pytest.mark.parametrize("kind,hd", [(Q8, 256), (F16, 256), (F32, 128), (Q8, 64), (F16, 40)])
def test_rows_that_see_nothing(rt, oracle, kind, hd):
    """Requests without tokens, without positions, with more tokens than
    positions (the first ones see nothing: 0), negative lengths; no gate;
    unaligned queries; a length past the table row; max_q too small."""
    note(f"paged attend empty rows kind={kind} hd={hd}")
    rng = np.random.default_rng(hd)
    lens = [100, 0, 3, 60, 0, 1, 200]
    new = [2, 5, 40, 0, 0, 1, 30]
    pages = Pages(rng, kind, 2, hd, 16, lens, oracle)
    q, _ = _inputs(rng, sum(new) + 2, 16, hd, gated=False)
    told = [100, -4, 3, 60, 0, 1, 200]
    call = Call(rt, pages, new, q, None, shift=4, lens=told)
    got = call.run(0.3, max_q=1)
    _close(got, pages, new, q, None, 0.3, "empty", lens=told)
    assert (got[2:7] == 0).all() and (got[7:7 + 37] == 0).all()
    call.b.free()
    # the same rows whatever the launches are sized for
    other = Call(rt, pages, new, q, None, shift=4, lens=told)
    _close(other.run(0.3), pages, new, q, None, 0.3, "empty, sized", lens=told)
    # a length past what the table row holds: the tokens see all of the row
    pages.table[6, :] = pages.table[6, 0]
    far = told[:6] + [pages.stride * 16 + 50]
    pages.lens = lens
    third = Call(rt, pages, new, q, None, lens=far)
    _close(third.run(0.3), pages, new, q, None, 0.3, "past the row", lens=far)
    for c in (other, third):
        c.b.free()


@pytest.mark.parametrize("kind,hd,new", [(Q8, 256, [1, 1]), (Q8, 128, [150, 1]), (F16, 256, [140, 3]), (F32, 64, [4, 1]),
                                         (F16, 33, [3, 1])])
def test_pages_that_do_not_exist(rt, oracle, kind, hd, new):
    """Table entries < 0 or past the pool: their positions are passed over,
    also where they are all of a request."""
    note(f"paged attend bad pages kind={kind} hd={hd}")
    rng = np.random.default_rng(3 * hd)
    pages = Pages(rng, kind, 2, hd, 16, [700, 40], oracle)
    pages.table[0, [0, 5, 6, 20]] = [-1, pages.n_pages, 2 ** 31 - 1, -2 ** 31]
    pages.table[0, 30:38] = -1
    q, gate = _inputs(rng, sum(new), 8, hd)
    call = Call(rt, pages, new, q, gate)
    _close(call.run(0.1), pages, new, q, gate, 0.1, "bad pages")
    call.b.free()
    pages.table[1, :] = -1
    call = Call(rt, pages, new, q, gate)
    got = call.run(0.1)
    _close(got, pages, new, q, gate, 0.1, "no page")
    assert (got[new[0]:] == 0).all()
    call.b.free()


@pytest.mark.parametrize("kind,hd,n_head,new", [(Q8, 256, 16, 4), (F16, 256, 16, 8), (F32, 256, 16, 3), (Q8, 256, 24, 200),
                                                (F16, 128, 32, 150), (Q8, 64, 16, 170), (F32, 128, 8, 60),
                                                (F16, 128, 4, 2), (F16, 33, 4, 9)])
def test_values_not_finite_ahead_of_a_token(rt, oracle, kind, hd, n_head, new):
    """inf or NaN in a K or V row takes nothing from tokens that do not see
    it; the others are not finite where the row holds them."""
    note(f"paged attend not finite kind={kind} hd={hd} new={new}")
    rng = np.random.default_rng(hd + new)
    n = 300 + new
    pages = Pages(rng, kind, 2, hd, 16, [n, 50], oracle)
    q, gate = _inputs(rng, new + 1, n_head, hd)
    gqa = n_head // 2
    clean = Call(rt, pages, [new, 1], q, gate)
    first = clean.run(0.1)
    clean.b.free()
    at = n - max(1, new // 2)  # the tokens from new - new // 2 on see it
    t = at - (n - new)
    slot = int(pages.slots(0, n)[at])
    row = pages.pools[1][slot, 1]
    if kind == Q8:
        row.view(np.uint16)[17 * (hd // 64)] = 0x7C00
        dims = np.arange(32 * (hd // 64), 32 * (hd // 64) + 32)
    elif kind == F16:
        row.view(np.uint16)[[3, hd - 1]] = (0x7E00, 0xFC00)
        dims = np.array([3, hd - 1])
    else:
        row.view(np.float32)[[5, hd - 2]] = (np.inf, np.nan)
        dims = np.array([5, hd - 2])
    call = Call(rt, pages, [new, 1], q, gate)
    got = call.run(0.1)
    hit = np.zeros(q.shape, bool)
    hit[t:new, gqa:, dims] = True
    assert not np.isfinite(got[hit]).any()
    assert np.isfinite(got[~hit]).all()
    tol = 1e-5 * np.abs(first).max()
    assert np.abs(got[~hit] - first[~hit]).max() <= tol
    call.b.free()
    # a key: the rows of its KV head that see it are NaN
    pages.pools[1][slot, 1] = pages.pools[1][slot, 0]
    pages.pools[0][slot, 1].view(np.uint16)[1 if kind == F32 else 0] = 0x7FC0 if kind == F32 else 0x7E00
    call = Call(rt, pages, [new, 1], q, gate)
    got = call.run(0.1)
    hit[:] = False
    hit[t:new, gqa:] = True
    assert np.isnan(got[hit]).all()
    assert np.isfinite(got[~hit]).all()
    call.b.free()


@pytest.mark.parametrize("kind,hd,new", [(Q8, 256, 1), (Q8, 128, 120), (F16, 256, 2), (F32, 256, 1), (Q8, 256, 60)])
def test_magnitudes(rt, oracle, kind, hd, new):
    """Queries and values from 1e-4 to 1e4 keep the bound, and q8_0 block
    scales past 512 beside small ones."""
    rng = np.random.default_rng(hd * new)
    for mq, mv in ((1e-4, 1.0), (1e3, 1e-4), (1.0, 3e3), (1.0, 3e4)):
        note(f"paged attend magnitudes kind={kind} hd={hd} q x {mq} v x {mv}")
        if kind == F16 and mv > 5e3:
            continue
        pages = Pages(rng, kind, 2, hd, 16, [500, 130], oracle, scale_v=mv if mv < 1e4 else 1.0)
        if mv >= 1e4:  # one row whose blocks' scales are large
            from paged_util import values
            big = rng.standard_normal((1, 2, hd)).astype(np.float32) * np.float32(mv * 6)
            pages.pools[1][pages.slots(0, 500)[77]] = oracle.encode(big, kind).reshape(2, row_bytes(kind, hd))
            assert np.isfinite(values(kind, pages.pools[1][pages.slots(0, 500)])).all()
        q, gate = _inputs(rng, 2 * new, 8, hd)
        q *= np.float32(mq)
        scale = min(0.1, 0.05 / mq)
        call = Call(rt, pages, [new, new], q, gate)
        _close(call.run(scale), pages, [new, new], q, gate, scale, f"q x {mq} v x {mv}")
        call.b.free()


def test_many_requests(rt, oracle):
    """More requests than a workgroup has threads, chunks among them."""
    note("paged attend many requests")
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 60, 1300).tolist()
    new = [min(n, 1) for n in lens]
    for i in range(0, 1300, 100):
        lens[i] = 90
        new[i] = 33
    pages = Pages(rng, F16, 2, 64, 16, lens, oracle)
    q, gate = _inputs(rng, sum(new) + 1, 8, 64)
    call = Call(rt, pages, new, q, gate)
    _close(call.run(0.125), pages, new, q, gate, 0.125, "many")
    call.b.free()


def test_a_long_request_beside_short_ones(rt, oracle):
    """One cache far longer than the rest is cut into many pieces."""
    note("paged attend long request")
    rng = np.random.default_rng(6)
    for kind, new in ((Q8, [1, 1, 1]), (F16, [20, 1, 2])):
        pages = Pages(rng, kind, 1, 128, 64, [60000, 5, 300], oracle)
        q, gate = _inputs(rng, sum(new), 8, 128)
        call = Call(rt, pages, new, q, gate)
        _close(call.run(0.1), pages, new, q, gate, 0.1, "long")
        call.b.free()
