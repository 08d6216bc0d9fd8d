"""GPU: attention of a batch of sequences over paged caches (nmx_attn_batch) against its definition in 64 bits,
and its prep (nmx_attn_batch_prep) against nmx_attn_prep bit for bit.

Tolerance of o, relative to the largest |v| in sight. A score's operands are held to 2^-22 of their rows'
largest element at worst (two binary16 parts; the vector product holds all of them and adds fewer terms in a
row), products are added in 32 bits over hd / 32 chained instructions and rounded a few times more, so a
score is off by at most ds = |q| |k| scale (4 2^-22 + (hd / 32 + 8) 2^-24), and a softmax mean by 2 ds. The
sums of weighted values round once a position that a lane adds (of L positions a share spreads at least
`lanes` neighbours over its lanes), a part and a rescale, half a step of a partial sum that is at most the largest value: (L / lanes +
AB_WGS / 8 + 16) 2^-24; exponentials, parts of the weights, quotient and gate add less than 2^-18."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nibblemac_amd.nmx import A8, AttnArgs, AttnBatchArgs, Device, Pages
from tests.batch_refuse import refuses
from tests.test_gpu_q4k import assert_bits_equal

KV_F32, KV_F16, KV_I8 = 0, 1, 2


def block_bytes(kv, nkv, page, hd):
    return nkv * page * (hd * (4, 2, 1)[kv] + (4 if kv == KV_I8 else 0))


def encode(rows, kv):
    """(bytes of each page, the values that they stand for in 64 bits) of rows [npages][nkv][page][hd]."""
    m = len(rows)
    if kv == KV_F32:
        return rows.reshape(m, -1).view(np.uint8).copy(), rows.astype(np.float64)
    if kv == KV_F16:
        h = rows.astype(np.float16)
        return h.reshape(m, -1).view(np.uint8).copy(), h.astype(np.float64)
    amax = np.abs(rows).max(3)
    codes = np.rint(rows * np.where(amax > 0, 127 / np.where(amax > 0, amax, 1), 0)[..., None]).astype(np.int8)
    scale = (amax / np.float32(127)).astype(np.float32)
    return (np.concatenate([codes.reshape(m, -1).view(np.uint8), scale.reshape(m, -1).view(np.uint8)], 1),
            codes.astype(np.float64) * scale.astype(np.float64)[..., None])


class Case:
    """A batch: rows and positions before them of each sequence, tables of random pages, groups (first
    sequence, shared rows). Pages are shared where a group's rows are, a partly shared page has copies."""

    def __init__(self, rng, rows, ctx, nh, nkv, hd, page, kv, groups=(), pad=0, std=1.0, spread=0.0, extra=3):
        self.rows, self.ctx = np.asarray(rows), np.asarray(ctx)
        self.nh, self.nkv, self.hd, self.page, self.kv, self.groups = nh, nkv, hd, page, kv, list(groups)
        S, self.n = len(rows), int(sum(rows)) + pad
        self.len = self.rows + self.ctx
        self.row0 = np.concatenate([[0], np.cumsum(rows)])
        counts = -(-self.len // page)
        self.first = [g[0] for g in self.groups] + [S]
        self.shared = [g[1] for g in self.groups]
        wide = int(counts.max()) + 1
        self.table = np.full((S, wide), -1, np.int32)
        need = int(counts.sum()) + extra
        ids, at = rng.permutation(need), 0
        f = (rng.standard_normal((need, nkv, page, hd)) * std).astype(np.float32), \
            (rng.standard_normal((need, nkv, page, hd)) * std).astype(np.float32)
        if spread:
            for x in f:
                x *= np.exp(rng.uniform(-spread, spread, x.shape[:3])).astype(np.float32)[..., None]
        for s in range(S):
            for i in range(counts[s]):
                g = next((j for j in range(len(self.groups)) if self.first[j] <= s < self.first[j + 1]), None)
                lead = s if g is None else self.first[g]
                left = 0 if g is None else min(self.shared[g], int(self.len[lead])) - i * page
                if s != lead and left >= page:
                    self.table[s, i] = self.table[lead, i]
                    continue
                self.table[s, i] = ids[at]
                if s != lead and left > 0:      # the shared rows of a page of its own
                    for x in f:
                        x[ids[at], :, :left] = x[self.table[lead, i], :, :left]
                at += 1
        self.npages = need
        self.used = np.zeros((need, page), bool)
        for s in range(S):
            for p in range(self.len[s]):
                self.used[self.table[s, p // page], p % page] = True
        (self.kb, self.K), (self.vb, self.V) = (encode(x, kv) for x in f)
        self.q = rng.standard_normal((self.n, nh, 2 * hd)).astype(np.float32)

    def poison(self):
        """Rows that no sequence sees hold NaN (int8: their scales)."""
        hide = ~self.used
        for b in (self.kb, self.vb):
            if self.kv == KV_I8:
                scale = b[:, self.nkv * self.page * self.hd:].view(np.float32).reshape(-1, self.nkv, self.page)
                scale[np.broadcast_to(hide[:, None], scale.shape)] = np.nan
            else:
                t = (np.float32, np.float16)[self.kv]
                rows = b.view(t).reshape(-1, self.nkv, self.page, self.hd)
                rows[np.broadcast_to(hide[:, None], rows.shape[:3])] = np.nan

    def reference(self):
        """(o, the tolerance of each row)"""
        nh, hd, o, tol = self.nh, self.hd, np.full((self.n, self.nh, self.hd), 7.0), np.zeros(self.n)
        scale, rep = float(np.float32(1 / np.sqrt(hd))), nh // self.nkv
        for s in range(len(self.rows)):
            at = np.arange(self.len[s])
            pg, off = self.table[s, at // self.page], at % self.page
            for i in range(self.rows[s]):
                t, see = self.row0[s] + i, max(0, self.ctx[s] + i + 1)
                for h in range(nh):
                    k, v = (x[pg[:see], h // rep, off[:see]] for x in (self.K, self.V))
                    o[t, h] = 0
                    if not see:
                        continue
                    q = self.q[t, h, :hd].astype(np.float64)
                    e = k @ q * scale
                    p = np.exp(e - e.max())
                    o[t, h] = p @ v / p.sum() / (1 + np.exp(-self.q[t, h, hd:].astype(np.float64)))
                    ds = np.linalg.norm(q) * np.linalg.norm(k, axis=1).max() * scale * (4 * 2.0 ** -22 + (hd / 32 + 8) * 2.0 ** -24)
                    lanes = 2 if hd > 256 else 8
                    adds = (see / lanes + 32 + 16) * 2.0 ** -24
                    tol[t] = max(tol[t], (2 * ds + adds + 2.0 ** -18) * np.abs(v).max())
        return o.reshape(self.n, -1), tol

    def upload(self, dev):
        i32 = lambda x: dev.to_device(np.asarray(x, np.int32))  # noqa: E731
        return dict(table=i32(self.table), len=i32(self.len), row0=i32(self.row0), kc=dev.to_device(self.kb),
                    vc=dev.to_device(self.vb), q=dev.to_device(self.q), group0=i32(self.first), shared=i32(self.shared or [0]),
                    o=dev.to_device(np.full((self.n + 1, self.nh * self.hd), 7, np.float32)))

    def args(self, d, a8=(None, None, None), **more):
        pages = Pages(seqs=len(self.rows), npages=self.npages, page=self.page, max_pages=self.table.shape[1],
                      table=d["table"].ptr, len=d["len"].ptr, nkv=self.nkv, hd=self.hd, kv_dtype=self.kv)
        return AttnBatchArgs(pages=pages, n=self.n, row0=d["row0"].ptr, nh=self.nh, q=d["q"].ptr, kc=d["kc"].ptr,
                             vc=d["vc"].ptr, scale=np.float32(1 / np.sqrt(self.hd)), groups=len(self.groups),
                             group0=d["group0"].ptr, shared=d["shared"].ptr, o=d["o"].ptr, a8=A8(*a8), **more)

    def work(self, dev):
        return dev.alloc(dev.attn_batch_work_bytes(self.n, len(self.rows), len(self.groups), self.nh, self.nkv, self.hd))


def attend(dev, c, times=2, a8=False, fill=None):
    d, w = c.upload(dev), c.work(dev)
    if fill is not None:
        dev.upload(w, np.full(w.nbytes // 4, fill, np.float32))
    nb = c.nh * c.hd // 32
    aq = (dev.zeros((nb, c.n, 32), np.int8), dev.zeros((nb, c.n), np.float32), dev.zeros((nb, c.n), np.float32)) if a8 else ()
    args = c.args(d, [x.ptr for x in aq] if a8 else (None,) * 3)
    for _ in range(times):
        dev.attn_batch(args, w)
    dev.sync()
    o = d["o"].numpy()
    assert (o[c.n] == 7).all()
    codes = [x.numpy() for x in aq]
    for x in (*d.values(), w, *aq):
        x.free()
    return (o[:c.n], *codes) if a8 else o[:c.n]


def check(dev, c):
    want, tol = c.reference()
    c.poison()
    got = attend(dev, c, fill=np.nan)
    live = int(c.row0[-1])
    assert (got[live:] == 7).all()
    err = np.abs(got - want).max(1)
    bad = np.flatnonzero(~(err <= tol))
    assert not len(bad), (bad[:8], err[bad[:8]], tol[bad[:8]])


CASES = [
    # rows of each sequence, positions before them, nh, nkv, hd, page, kv, groups
    ([1], [0], 8, 2, 256, 16, KV_F32, ()),                    # the first token of all
    ([1], [600], 8, 2, 256, 64, KV_F16, ()),
    ([1, 1, 1], [15, 16, 17], 8, 2, 256, 16, KV_I8, ()),      # about a page's end
    ([1, 0, 1, 1], [31, 50, 0, 64], 1, 1, 64, 32, KV_F16, ()),
    ([1] * 9, range(0, 900, 100), 8, 2, 256, 64, KV_F32, ()),
    ([1] * 40, range(1, 401, 10), 8, 2, 256, 16, KV_F16, ()),
    ([1, 2, 3, 4], [100, 200, 0, 31], 6, 2, 128, 32, KV_I8, ()),    # 3 heads a group: 3 to 12 query rows
    ([2, 1], [300, 77], 8, 1, 512, 16, KV_F32, ()),           # 16 query rows, then 8
    ([2, 1], [300, 77], 8, 1, 512, 128, KV_I8, ()),
    ([1] * 4, [500, 3, 64, 129], 16, 2, 256, 64, KV_I8, ()),  # 8 heads a group
    ([1] * 5, [40, 80, 120, 160, 200], 16, 1, 192, 64, KV_F32, ()),
    ([5, 1, 33], [0, 200, 70], 8, 2, 256, 64, KV_F16, ()),    # prompts: 20 and 132 query rows
    ([5, 1, 33], [0, 200, 70], 8, 2, 256, 64, KV_F32, ()),
    ([70], [0], 4, 4, 64, 16, KV_I8, ()),                     # a prompt from its beginning
    ([70, 9], [1, 300], 8, 1, 512, 32, KV_F16, ()),
    ([9, 70], [1, 300], 8, 1, 320, 32, KV_F32, ()),
    ([70, 9], [10, 300], 8, 1, 448, 32, KV_I8, ()),
    ([40], [100], 4, 2, 384, 256, KV_F16, ()),
    ([1, 1], [300, 10], 32, 1, 64, 16, KV_F16, ()),           # 32 heads on one: a single row in the matrix product
    ([1] * 6, [300, 301, 340, 299, 400, 303], 8, 2, 256, 16, KV_F16, [(0, 290)]),     # a prefix that ends in a page
    ([1] * 6, [300, 301, 340, 299, 400, 303], 8, 2, 256, 32, KV_F32, [(0, 256)]),
    ([1] * 3, [70, 64, 90], 8, 2, 256, 64, KV_I8, [(0, 64)]),                         # 12 query rows share
    ([1] * 7, [64, 200, 64, 100, 128, 300, 5], 6, 2, 128, 32, KV_I8, [(0, 64), (3, 96), (6, 5)]),  # three groups
    ([1, 0, 2, 30, 1], [100, 120, 96, 100, 400], 8, 2, 256, 16, KV_F16, [(0, 96), (4, 380)]),
    ([1] * 5, [40, 33, 50, 60, 70], 4, 4, 64, 16, KV_F32, [(1, 33)]),                 # the first one is in no group
    ([1] * 5, [40, 33, 50, 60, 70], 4, 4, 64, 16, KV_F32, [(0, 1000)]),               # all that comes before the rows
    ([3] * 30, [200] * 30, 4, 2, 192, 64, KV_F16, [(0, 190)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{c[2]}on{c[3]}x{c[4]}_p{c[5]}_kv{c[6]}_g{len(c[7])}")
def test_definition(dev, case):
    rows, ctx, nh, nkv, hd, page, kv, groups = case
    if groups and groups[0][1] == 1000:    # declared longer than any context: as far as the shortest one
        c = Case(np.random.default_rng(7), rows, list(ctx), nh, nkv, hd, page, kv, [(0, 33)])
        c.shared = [1000]
    else:
        c = Case(np.random.default_rng(len(rows) * 31 + hd + kv), rows, list(ctx), nh, nkv, hd, page, kv, groups, pad=2)
    check(dev, c)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("std,spread", [(4.0, 0.0), (1e-3, 2.0), (0.3, 3.0)])
def test_values_of_other_sizes(dev, kv, std, spread):
    """Sharp and flat softmax rows, rows of magnitudes far apart, by both products."""
    c = Case(np.random.default_rng(5), [1, 1, 9, 1], [700, 33, 300, 128], 8, 2, 256, 32, kv, [(0, 33)], std=std, spread=spread)
    check(dev, c)


@pytest.mark.gpu
def test_long_sequences(dev):
    """Several turns of every wave, parts by the hundred, both products, a prefix by matrix instructions."""
    c = Case(np.random.default_rng(6), [1] * 6, [9000, 12000, 8200, 8192, 8193, 20000], 8, 2, 256, 64, KV_F16, [(0, 8192)])
    check(dev, c)
    c = Case(np.random.default_rng(7), [1, 1], [40000, 100], 4, 4, 64, 128, KV_I8)
    check(dev, c)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 64), (8, 1, 64), (6, 2, 128), (4, 1, 192), (8, 2, 256), (8, 1, 256), (4, 1, 320), (8, 1, 512)])
def test_shares_of_waves_and_workgroups(dev, nh, nkv, hd, kv):
    """Short sequences that single waves take beside long ones whose parts whole workgroups take, several turns each,
    with 3 to 8 query rows."""
    rng = np.random.default_rng(hd + kv)
    ctx = [6000, 10, 40, 300, 1, 0, 700, 33, 15, 2000, 64, 100, 31, 32, 129, 5, 5, 900]
    check(dev, Case(rng, [1] * len(ctx), ctx, nh, nkv, hd, 16, kv, [(4, 0), (6, 10)] if hd == 128 else ()))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kv", [(256, KV_F16), (64, KV_F32), (320, KV_I8)])
def test_many_rows(dev, hd, kv):
    """Joins by waves: 300 rows of 8 heads, padded, and their A8."""
    c = Case(np.random.default_rng(hd), [1] * 100 + [0, 150, 49, 1], [7] * 90 + [100] * 14, 8, 2, hd, 32, kv, [(0, 5)], pad=3)
    check(dev, c)
    o, q, d, fs = attend(dev, c, a8=True)
    live, nb = int(c.row0[-1]), c.nh * c.hd // 32
    x = dev.to_device(o[:live])
    a = (dev.zeros((nb, live, 32), np.int8), dev.zeros((nb, live), np.float32), dev.zeros((nb, live), np.float32))
    dev.quant_a8(x, live, c.nh * c.hd, *a)
    dev.sync()
    for got, want in zip((q, d, fs), a):
        assert_bits_equal(got[:, :live], want.numpy(), "A8")
        assert not got[:, live:].any()
    for b in (x, *a):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
def test_queries_of_different_sizes(dev, kv):
    """Rows and heads that share a wave or a tile: near-uniform weights beside a single position that takes all, and zeros."""
    rng = np.random.default_rng(8 + kv)
    c = Case(rng, [1, 1, 2, 20], [400, 90, 33, 300], 8, 2, 128, 16, kv)
    c.q[..., :128] *= np.exp(rng.uniform(-8, 3, c.q.shape[:2])).astype(np.float32)[..., None]
    c.q[0, 3, :128] = c.q[7, 2, :128] = 0
    check(dev, c)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
def test_what_one_row_holds_stays_in_it(dev, kv):
    """NaN and infinities in a row's query, in its gate and in a sequence's cache: all other rows' bits are as without them."""
    c = Case(np.random.default_rng(5), [1, 1, 30, 1, 3, 1], [200, 300, 64, 70, 20, 500], 8, 2, 128, 16, kv, [(0, 48), (3, 0)])
    want = attend(dev, c)
    t = int(c.row0[2]) + 7
    c.q[t, 3, 5], c.q[t, 4, 128 + 9], c.q[0, 1, :128] = np.nan, np.nan, np.inf
    for p in range(c.len[4]):    # a sequence of its own pages
        for b in (c.kb, c.vb):
            page, off = c.table[4, p // 16], p % 16
            if kv == KV_I8:
                b[page, 2 * 16 * 128:].view(np.float32).reshape(2, 16)[:, off] = np.nan
            else:
                b[page].view((np.float32, np.float16)[kv]).reshape(2, 16, 128)[:, off] = np.nan
    got = attend(dev, c)
    same = np.ones((c.n, 8), bool)
    same[t, [3, 4]] = same[0, 1] = False
    same[c.row0[4]:c.row0[5]] = False
    heads = lambda x: x.reshape(c.n, 8, 128)  # noqa: E731
    assert (heads(got)[same].view(np.uint32) == heads(want)[same].view(np.uint32)).all()
    assert np.isnan(heads(got)[t, 3]).all() and np.isnan(heads(got)[t, 4, 9]) and np.isnan(heads(got)[0, 1]).all()
    assert np.isnan(heads(got)[c.row0[4]:c.row0[5]]).all()


@pytest.mark.gpu
def test_most_sequences(dev):
    """256 sequences and groups."""
    rng = np.random.default_rng(15)
    ctx = rng.integers(0, 60, 256)
    check(dev, Case(rng, [1] * 255 + [0], ctx, 4, 2, 64, 16, KV_F16, [(s, int(ctx[s])) for s in range(256)]))
    check(dev, Case(rng, [1] * 256, [40] * 256, 4, 2, 64, 16, KV_I8, [(0, 33), (100, 20)]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,ctx,nh,nkv,hd,page,kv,groups", [
    ([1, 1], [70, 5], 1024, 1, 64, 16, KV_F16, ()),           # most heads, on one KV head
    ([2], [40], 1024, 1024, 64, 256, KV_I8, ()),              # and each on its own
    ([512], [0], 16, 2, 64, 32, KV_F32, ()),                  # a chunk of a prompt, nothing before it
    ([511, 1], [33, 600], 4, 1, 384, 64, KV_F16, ()),
    ([200, 1, 1, 100], [100, 64, 31, 32], 4, 2, 448, 16, KV_I8, [(0, 31)]),
    ([1] * 9, [3000] * 9, 8, 1, 256, 64, KV_F32, [(0, 2999), (5, 17)]),
])
def test_largest_shapes(dev, rows, ctx, nh, nkv, hd, page, kv, groups):
    check(dev, Case(np.random.default_rng(nh + hd), rows, ctx, nh, nkv, hd, page, kv, groups))


@pytest.mark.gpu
def test_caches_past_4_gib(dev):
    """Pages whose bytes lie past 2^32 in the cache."""
    page, nkv, hd = 256, 4, 512
    c = Case(np.random.default_rng(8), [1, 20], [700, 40], 4, nkv, hd, page, KV_F32)
    npages = (5 << 30) // block_bytes(KV_F32, nkv, page, hd)
    want, tol = c.reference()
    d, w = c.upload(dev), c.work(dev)
    block, far = block_bytes(KV_F32, nkv, page, hd), npages - c.npages
    for k in ("kc", "vc"):
        big = dev.alloc(npages * block)
        dev.copy(big.ptr + far * block, d[k].ptr, c.npages * block)
        dev.sync()
        d[k].free()
        d[k] = big
    dev.upload(d["table"], np.where(c.table >= 0, c.table + far, -1).astype(np.int32))
    c.npages = npages
    dev.attn_batch(c.args(d), w)
    dev.sync()
    err = np.abs(d["o"].numpy()[:c.n] - want).max(1)
    for x in (*d.values(), w):
        x.free()
    assert (err <= tol).all(), (err, tol)


@pytest.mark.gpu
def test_a8_of_the_rows(dev):
    c = Case(np.random.default_rng(9), [1, 3, 1], [40, 100, 3], 8, 2, 256, 32, KV_F16)
    o, q, d, fs = attend(dev, c, a8=True)
    x = dev.to_device(o)
    nb = c.nh * c.hd // 32
    a = (dev.zeros((nb, c.n, 32), np.int8), dev.zeros((nb, c.n), np.float32), dev.zeros((nb, c.n), np.float32))
    dev.quant_a8(x, c.n, c.nh * c.hd, *a)
    dev.sync()
    for got, want in zip((q, d, fs), a):
        assert_bits_equal(got, want.numpy(), "A8")
    for b in (x, *a):
        b.free()


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_batch_within_rounding(dev):
    """A sequence alone and in a batch, where its positions are cut at other places."""
    rng = np.random.default_rng(10)
    c = Case(rng, [1] * 8, [500, 10, 700, 20, 30, 900, 64, 1], 8, 2, 256, 16, KV_F32)
    all_, (want, tol) = attend(dev, c), c.reference()
    for s in (0, 5):
        one = Case(np.random.default_rng(1), [1], [int(c.ctx[s])], 8, 2, 256, 16, KV_F32)
        one.table, one.npages, one.kb, one.vb, one.q = c.table[s:s + 1], c.npages, c.kb, c.vb, c.q[s:s + 1]
        assert np.abs(attend(dev, one) - all_[s:s + 1]).max() <= 2 * tol[s]


@pytest.mark.gpu
def test_replayed_with_other_lengths(dev):
    """Lengths, rows and tables are the device's: one graph serves steps that differ in all of them, with
    eager calls in between; the largest workspace of the shape is enough for each."""
    rng = np.random.default_rng(11)
    shape = dict(nh=8, nkv=2, hd=256, page=16, kv=KV_F16)
    steps = [Case(rng, [1, 1, 1, 1], [30, 500, 2, 64], groups=[(0, 0)], **shape), Case(rng, [0, 2, 1, 1], [30, 700, 20, 64], groups=[(1, 20)], **shape),
             Case(rng, [1, 0, 0, 1], [900, 5, 5, 64], groups=[(0, 60)], pad=2, **shape)]
    npages, wide = max(c.npages for c in steps), max(c.table.shape[1] for c in steps)
    for c in steps:
        c.table = np.pad(c.table, ((0, 0), (0, wide - c.table.shape[1])), constant_values=-1)
        extra = ((0, npages - c.npages), (0, 0))
        c.kb, c.vb, c.npages = np.pad(c.kb, extra), np.pad(c.vb, extra), npages
    d, w = steps[0].upload(dev), steps[0].work(dev)
    args = steps[0].args(d)
    dev.attn_batch(args, w)
    dev.sync()
    dev.graph_begin()
    dev.attn_batch(args, w)
    g = dev.graph_end()
    for c in steps + steps[:1]:
        want, tol = c.reference()
        for k, v in (("table", c.table), ("len", c.len), ("row0", c.row0), ("q", c.q), ("kc", c.kb), ("vc", c.vb), ("group0", c.first),
                     ("shared", c.shared), ("o", np.full((c.n + 1, c.nh * c.hd), 7))):
            dev.upload(d[k], np.asarray(v, d[k].dtype))
        dev.graph_launch(g)
        dev.sync()
        got = d["o"].numpy()[:c.n]
        live = int(c.row0[-1])
        assert (np.abs(got - want).max(1)[:live] <= tol[:live]).all() and (got[live:] == 7).all()
        dev.attn_batch(args, w)
        dev.sync()
        assert_bits_equal(d["o"].numpy()[:c.n], got, "eager and replayed")
    dev.graph_destroy(g)
    for x in (*d.values(), w):
        x.free()


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Two contexts with workspaces of their own."""
    rng = np.random.default_rng(12)
    cs = [Case(rng, [1] * 5, [900, 30, 400, 2, 1200], 8, 2, 256, 64, KV_F16), Case(rng, [20, 1], [300, 800], 8, 2, 256, 16, KV_F32)]
    with Device(0) as other:
        devs = [dev, other]
        d = [c.upload(x) for c, x in zip(cs, devs)]
        w = [c.work(x) for c, x in zip(cs, devs)]
        for _ in range(20):
            for i in range(2):
                devs[i].attn_batch(cs[i].args(d[i]), w[i])
        for x in devs:
            x.sync()
        for i, c in enumerate(cs):
            want, tol = c.reference()
            assert (np.abs(d[i]["o"].numpy()[:c.n] - want).max(1) <= tol).all()
        for x in (*d[0].values(), w[0]):
            x.free()


@pytest.mark.gpu
def test_lists_that_mean_nothing_stay_in_bounds(dev):
    """Lengths, rows and tables that contradict each other: no fault and no write outside o. The checks in the
    kernels that this relies on: seq_rows and seq_len clamp, falling lists have no rows, entries that are
    no pages read page 0, a row without positions gives 0."""
    rng = np.random.default_rng(13)
    c = Case(rng, [1, 2, 1], [40, 50, 3], 8, 2, 256, 16, KV_F16, [(0, 16)])
    for change in (dict(len=[-5, 10 ** 9, 2]), dict(row0=[3, 1, 4, 0]), dict(row0=[-9, 2, 2, 900]), dict(group0=[9, -3]),
                   dict(group0=[-1, 2]), dict(shared=[-7]), dict(shared=[2 ** 31 - 1]), dict(len=[0, 1, 0]),
                   dict(table=np.full(c.table.shape, -1)), dict(table=np.full(c.table.shape, 2 ** 31 - 1))):
        d, w = c.upload(dev), c.work(dev)
        for k, v in change.items():
            dev.upload(d[k], np.asarray(v, np.int32))
        dev.attn_batch(c.args(d), w)
        dev.sync()
        o = d["o"].numpy()
        assert (o[c.n] == 7).all() and np.isfinite(o).all(), change
        if "len" in change and change["len"][0] == 0:      # rows before the sequence's beginning see nothing
            assert (o[0] == 0).all() and (o[1] == 0).all() and (o[3] == 0).all()
        for x in (*d.values(), w):
            x.free()


# ---- the prep ------------------------------------------------------------------------------------
PREP = [
    # rows, positions before them, nh, nkv, hd, rot, page, kv, axes (None: a row's position)
    ([1], [0], 8, 2, 256, 64, 16, KV_F32, None),
    ([1, 1, 1], [15, 16, 700], 8, 2, 256, 64, 16, KV_F16, 3),
    ([3, 0, 40, 1], [0, 9, 100, 31], 8, 2, 256, 64, 32, KV_I8, 3),
    ([2, 2], [10, 0], 6, 2, 128, 128, 64, KV_F16, 1),
    ([1, 7], [3, 250], 4, 4, 64, 32, 256, KV_I8, 4),
    ([4], [60], 4, 1, 512, 512, 64, KV_F32, 2),
    ([2], [5], 2, 1, 192, 0, 16, KV_F16, None),      # no rotary columns
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PREP, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{c[2]}on{c[3]}x{c[4]}_rot{c[5]}_kv{c[7]}_axes{c[8]}")
def test_prep_equals_attn_prep(dev, case):
    """Rows as nmx_attn_prep makes them from tables whose row t holds each frequency's own angle of row t."""
    rows, ctx, nh, nkv, hd, rot, page, kv, axes = case
    rng = np.random.default_rng(sum(rows) + hd + kv)
    c = Case(rng, rows, ctx, nh, nkv, hd, page, kv, pad=1)
    n, h2, span = c.n, rot // 2, int(c.len.max()) + 50
    live = int(c.row0[-1])
    cos, sin = rng.uniform(-1, 1, (2, span, max(h2, 1))).astype(np.float32)
    axis = rng.integers(0, axes or 1, max(h2, 1)).astype(np.uint8)
    where = rng.integers(0, span, (n, axes or 1)).astype(np.int32)
    if axes:        # outside the tables: the nearer end
        where[0, 0], where[live - 1, -1] = -3, span + 9
    pos = np.concatenate([c.ctx[s] + np.arange(rows[s]) for s in range(len(rows))] + [[0]]).astype(int)
    at = where.clip(0, span - 1) if axes else pos[:, None]
    mixed = [np.stack([t[at[r, axis[:h2]], np.arange(h2)] for r in range(n)]).astype(np.float32) if h2 else np.zeros((n, 1), np.float32)
             for t in (cos, sin)]
    k_in, v_in = rng.standard_normal((2, n, nkv * hd)).astype(np.float32)
    qn, kn = rng.uniform(0.5, 1.5, (2, hd)).astype(np.float32)
    # the chain's call: row t at position t of a plain cache
    up = {k: dev.to_device(v) for k, v in dict(k=k_in, v=v_in, qn=qn, kn=kn, cos=cos, sin=sin, mc=mixed[0], ms=mixed[1], where=where,
                                               q=c.q, pos=np.array([0], np.int32)).items()}
    flat = [dev.zeros((block_bytes(kv, nkv, n, hd),), np.uint8) for _ in range(2)]
    dev.attn_prep(AttnArgs(n=n, nh=nh, nkv=nkv, hd=hd, rot=rot, max_ctx=n, q=up["q"].ptr, k_in=up["k"].ptr, v_in=up["v"].ptr,
                           q_norm=up["qn"].ptr, k_norm=up["kn"].ptr, eps=1e-6, rope_cos=up["mc"].ptr, rope_sin=up["ms"].ptr,
                           kc=flat[0].ptr, vc=flat[1].ptr, pos=up["pos"].ptr, o=up["k"].ptr, kv_dtype=kv))
    d = c.upload(dev)
    dev.attn_batch_prep(c.args(d, rot=rot, k_in=up["k"].ptr, v_in=up["v"].ptr, q_norm=up["qn"].ptr, k_norm=up["kn"].ptr, eps=1e-6,
                               rope_cos=up["cos"].ptr, rope_sin=up["sin"].ptr, rope_rows=span, axes=axes or 1,
                               axis=axis.ctypes.data if axes else None, rope_pos=up["where"].ptr if axes else None))
    dev.sync()
    got_q, want_q = d["q"].numpy(), up["q"].numpy()
    want_q[live:] = c.q[live:]          # a row of no sequence is left as it was
    assert_bits_equal(got_q, want_q, "q")
    size = nkv * hd * (4, 2, 1)[kv]
    for name, was, chain in (("kc", c.kb, flat[0]), ("vc", c.vb, flat[1])):
        want, src = was.copy(), chain.numpy()
        rows_of = src[:n * size].reshape(nkv, n, -1)
        for s in range(len(rows)):
            for i in range(rows[s]):
                t, p = c.row0[s] + i, c.ctx[s] + i
                pg, off = c.table[s, p // page], p % page
                want[pg, :page * size].reshape(nkv, page, -1)[:, off] = rows_of[:, t]
                if kv == KV_I8:
                    want[pg, page * size:].reshape(nkv, page, 4)[:, off] = src[n * size:].reshape(nkv, n, 4)[:, t]
        assert_bits_equal(d[name].numpy(), want, name)
    for x in (*d.values(), *up.values(), *flat):
        x.free()


@pytest.mark.gpu
def test_prep_rows_without_a_place(dev):
    """Negative positions, tables that end or name no page: turned, nothing stored."""
    rng = np.random.default_rng(14)
    c = Case(rng, [2, 1, 1], [0, 5, 40], 4, 2, 64, 16, KV_F16)
    d = c.upload(dev)
    table, ln = c.table.copy(), c.len.copy()
    ln[0], table[1, 0], table[2, 2] = 1, -1, c.npages   # row 0 at -1, a missing page, a page outside
    dev.upload(d["table"], table)
    dev.upload(d["len"], ln.astype(np.int32))
    up = [dev.to_device(x) for x in (*rng.standard_normal((2, 4, 128)).astype(np.float32), np.ones(64, np.float32))]
    dev.attn_batch_prep(c.args(d, rot=0, k_in=up[0].ptr, v_in=up[1].ptr, q_norm=up[2].ptr, k_norm=up[2].ptr, eps=1e-6, axes=1))
    dev.sync()
    want = c.kb.copy().view(np.float16).reshape(c.npages, 2, 16, 64)
    got = d["kc"].numpy().view(np.float16).reshape(want.shape)
    changed = np.argwhere((got != want).any(3).any(1))
    assert changed.tolist() == [[c.table[0, 0], 0]]     # row 1 of the first sequence alone
    assert (d["q"].numpy()[..., :64] != c.q[..., :64]).any((1, 2)).all()
    for x in (*d.values(), *up):
        x.free()


def test_refusals():
    at = iter(range(1 << 30, 1 << 45, 1 << 30))
    names = ("table", "len", "row0", "q", "kc", "vc", "o", "work", "k_in", "v_in", "q_norm", "k_norm", "rope_cos", "rope_sin", "rope_pos",
             "group0", "shared", "x")
    P = {k: next(at) for k in names}
    axis = (ctypes.c_uint8 * 32)(*[i % 3 for i in range(32)])

    def args(pages={}, **more):
        pg = dict(seqs=3, npages=10, page=16, max_pages=4, table=P["table"], len=P["len"], nkv=2, hd=128, kv_dtype=KV_I8)
        pg.update(pages)
        a = dict(n=3, nh=8, rot=64, rope_rows=100, axes=3, axis=ctypes.addressof(axis), groups=1, eps=1e-6, scale=1.0,
                 **{k: P[k] for k in names if k not in ("table", "len", "work", "x")})
        a.update(more)
        return AttnBatchArgs(pages=Pages(**pg), **a)

    both = [args(pages={k: v}) for k, v in (("seqs", 0), ("seqs", 257), ("npages", 0), ("npages", (1 << 20) + 1), ("page", 8), ("page", 48),
                                            ("page", 512), ("page", 0), ("max_pages", 0), ("max_pages", 65537), ("nkv", 0), ("nkv", 3), ("hd", 96),
                                            ("hd", 0), ("hd", 576), ("kv_dtype", 3), ("kv_dtype", -1), ("table", None), ("len", None))]
    both += [args(**{k: v}) for k, v in (("n", 0), ("n", 513), ("nh", 7), ("nh", 1), ("nh", 2048), ("row0", None), ("q", None), ("kc", None),
                                         ("vc", None), ("q", P["q"] + 4), ("kc", P["kc"] + 8), ("vc", P["vc"] + 1), ("vc", P["kc"]),
                                         ("q", P["kc"] + 16))]
    for i, a in enumerate(both):
        refuses("nmx_attn_batch_prep", i, a)
        refuses("nmx_attn_batch", i, a, P["work"])
    for i, a in enumerate([args(**{k: v}) for k, v in (
            ("k_in", None), ("v_in", None), ("q_norm", None), ("k_norm", None), ("rot", 63), ("rot", -2), ("rot", 130), ("rope_cos", None),
            ("rope_rows", 0), ("axes", 0), ("axes", 5), ("axes", 2), ("k_in", P["q"]), ("rope_cos", P["vc"]), ("row0", P["q"] + 32),
            ("rope_pos", P["kc"]), ("q", P["table"]), ("kc", P["len"]))]):
        refuses("nmx_attn_batch_prep", i, a)
    for i, a in enumerate([args(**{k: v}) for k, v in (
            ("o", None), ("o", P["o"] + 4), ("groups", -1), ("groups", 4), ("group0", None), ("shared", None), ("o", P["q"]), ("o", P["kc"]),
            ("o", P["table"]), ("o", P["work"]), ("o", P["group0"]), ("a8", A8(P["x"], None, P["x"] + 8)), ("a8", A8(P["x"], P["x"] + 16, P["x"])),
            ("a8", A8(P["o"], P["x"], P["x"] + (1 << 20))), ("o", P["row0"]))]):
        refuses("nmx_attn_batch", i, a, P["work"])
    refuses("nmx_attn_batch", "no work", args(), None)
    refuses("nmx_attn_batch", "odd work", args(), P["work"] + 8)
    refuses("nmx_attn_batch", "work over q", args(), P["q"])


def test_work_bytes():
    from nibblemac_amd.nmx import load_library
    lib = load_library()
    for bad in ((0, 1, 0, 1, 1, 64), (513, 1, 0, 1, 1, 64), (1, 0, 0, 1, 1, 64), (1, 257, 0, 1, 1, 64), (1, 2, 3, 1, 1, 64), (1, 1, -1, 1, 1, 64),
                (1, 1, 0, 3, 2, 64), (1, 1, 0, 1, 2, 64), (1, 1, 0, 1025, 1, 64), (1, 1, 0, 1, 1, 32), (1, 1, 0, 1, 1, 65), (1, 1, 0, 1, 1, 576)):
        assert lib.nmx_attn_batch_work_bytes(*bad) == 0, bad
    assert 0 < lib.nmx_attn_batch_work_bytes(1, 1, 0, 1, 1, 64) < 4 << 20
