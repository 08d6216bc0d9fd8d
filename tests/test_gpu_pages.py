"""GPU: the pages of a step (nmx_pages_update) against a model in Python lists, number by number, and the
rows that sequences see in every cache byte by byte."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import Device, Pages, load_library, pages_args
from tests.batch_refuse import refuses
from tests.test_gpu_q4k import assert_bits_equal

KV_F32, KV_F16, KV_I8 = 0, 1, 2


class Model:
    """Tables, lengths, page counts and caches on the host; step() as the header describes it."""

    def __init__(self, rng, seqs, page, npages, wide, caches=2, nkv=2, hd=64, kv=KV_F16):
        self.seqs, self.page, self.npages, self.wide, self.nkv, self.hd, self.kv = seqs, page, npages, wide, nkv, hd, kv
        self.row = hd * (4, 2, 1)[kv]
        self.block = nkv * page * (self.row + (4 if kv == KV_I8 else 0))
        self.kvs = [rng.integers(0, 256, (npages, self.block)).astype(np.uint8) for _ in range(caches)]
        self.table = [[] for _ in range(seqs)]
        self.len, self.had = [0] * seqs, [0] * seqs

    def rows_of(self, cache, page, n):
        """Views of the first n rows and scales of a page."""
        size = self.nkv * self.page * self.row
        b = self.kvs[cache][page]
        out = [b[:size].reshape(self.nkv, self.page, self.row)[:, :n]]
        if self.kv == KV_I8:
            out.append(b[size:].reshape(self.nkv, self.page, 4)[:, :n])
        return out

    def step(self, src, keep, add, pack=0):
        """The out words; with an error nothing changes."""
        S, page = self.seqs, self.page
        src = [f if 0 <= f < S else -1 for f in src]
        keep = [0 if src[s] < 0 else max(0, min(keep[s], self.len[src[s]])) for s in range(S)]
        add = [max(0, a) for a in add]
        for s in range(S):
            if -(-(keep[s] + add[s]) // page) > self.wide:
                return [-1 - s, 0, 0, 0]
        new = [[] if src[s] < 0 else self.table[src[s]][:-(-keep[s] // page)] for s in range(S)]
        writes = [add[s] > 0 and keep[s] % page > 0 for s in range(S)]
        holders = {}
        for s in range(S):
            for i, p in enumerate(new[s]):
                holders.setdefault(p, []).append((s, writes[s] and i == len(new[s]) - 1))
        used = {p for x in new for p in x}
        free = [p for p in range(self.npages) if p not in used]
        copies, taken = [], []
        for s in range(S):
            if writes[s]:
                who = holders[new[s][-1]]
                if len(who) > 1 and not (all(w for _, w in who) and who[0][0] == s):
                    copies.append((new[s].pop(), len(taken), keep[s] % page))
            while len(new[s]) < -(-(keep[s] + add[s]) // page):
                taken.append((s, len(new[s])))
                new[s].append(free[len(taken) - 1] if len(taken) <= len(free) else None)
        if len(taken) > len(free):
            return [len(taken) - len(free), 0, 0, 0]
        for c in range(len(self.kvs)):
            for p, i, n in copies:
                for to, at in zip(self.rows_of(c, free[i], n), self.rows_of(c, p, n)):
                    to[:] = at
        self.had = [max(h, len(t)) for h, t in zip(self.had, self.table)]
        self.table, self.len = new, [k + a for k, a in zip(keep, add)]
        used = sorted({p for x in new for p in x})
        out = [0, len(taken), 0, 0]
        if pack:
            holes = [p for p in range(len(used)) if p not in set(used)]
            to = dict(zip([p for p in used if p >= len(used)], holes))
            for b in self.kvs:
                for p, h in to.items():
                    b[h] = b[p]
            self.table = [[to.get(p, p) for p in x] for x in new]
            out[2:] = [len(used), len(to)]
        return out

    def refs(self):
        r = np.zeros(self.npages, np.int32)
        for x in self.table:
            for p in x:
                r[p] += 1
        return r


class Box:
    """The same on the device."""

    def __init__(self, dev, m):
        self.dev, self.m = dev, m
        i32 = lambda *s: np.zeros(s, np.int32)  # noqa: E731
        self.b = {k: dev.to_device(v) for k, v in dict(table=i32(m.seqs, m.wide) - 9, len=i32(m.seqs), refs=i32(m.npages),
                                                       src=i32(m.seqs), keep=i32(m.seqs), add=i32(m.seqs), out=i32(4)).items()}
        self.kv = [dev.to_device(x) for x in m.kvs]
        self.work = dev.alloc(dev.pages_work_bytes(m.npages, m.seqs, m.wide))
        dev.upload(self.work, np.full(self.work.nbytes, 0xAB, np.uint8))

    def args(self, pack=0):
        m, b = self.m, self.b
        pages = Pages(seqs=m.seqs, npages=m.npages, page=m.page, max_pages=m.wide, table=b["table"].ptr, len=b["len"].ptr,
                      nkv=m.nkv, hd=m.hd, kv_dtype=m.kv)
        return pages_args(pages, b["refs"], b["src"], b["keep"], b["add"], self.kv, b["out"], pack=pack)

    def put(self, src, keep, add):
        for k, v in (("src", src), ("keep", keep), ("add", add)):
            self.dev.upload(self.b[k], np.asarray(v, np.int32))

    def step(self, src, keep, add, pack=0):
        self.put(src, keep, add)
        self.dev.pages_update(self.args(pack), self.work)
        self.dev.sync()
        return self.b["out"].numpy().tolist()

    def check(self, what=""):
        m = self.m
        table = self.b["table"].numpy()
        for s in range(m.seqs):
            got, n = table[s].tolist(), len(m.table[s])
            assert got[:n] == m.table[s], (what, s, got[:n], m.table[s])
            behind = m.had[s]
            assert got[n:] == [-1] * max(0, behind - n) + [-9] * (m.wide - max(n, behind)) or set(got[n:]) <= {-1, -9}, (what, s)
        assert self.b["len"].numpy().tolist() == m.len, what
        assert (self.b["refs"].numpy() == m.refs()).all(), what
        for got, want in zip(self.kv, m.kvs):
            assert_bits_equal(got.numpy(), want, what)

    def free(self):
        for x in (*self.b.values(), *self.kv, self.work):
            x.free()


def both(m, box, src, keep, add, pack=0, what=""):
    want = m.step(src, keep, add, pack)
    got = box.step(src, keep, add, pack)
    assert got == want, (what, got, want)
    box.check(what)


@pytest.mark.gpu
@pytest.mark.parametrize("page,kv,hd", [(16, KV_F16, 64), (64, KV_I8, 128), (256, KV_F32, 64), (32, KV_I8, 192)])
def test_a_conversation_of_many(dev, page, kv, hd):
    """Prompts, tokens, forks, exchanges, drafts taken back, ends, packing; no page is lost or held twice."""
    rng = np.random.default_rng(page + kv)
    S = 5
    m = Model(rng, S, page, 60, 12, hd=hd, kv=kv)
    box = Box(dev, m)
    go = list(range(S))
    p = page
    both(m, box, [-1] * S, [0] * S, [3 * p + 5, p, 1, 0, p - 1], what="prompts")
    both(m, box, go, [999] * S, [1, 1, 1, 0, 1], what="a token each")
    both(m, box, go, [999] * S, [1, 1, 1, 0, 1], what="another: one begins a page")
    both(m, box, [0, 1, 0, 0, 4], [999] * S, [0, 1, 0, 0, 1], what="forks of the first, nobody writes")
    both(m, box, go, [999] * S, [1, 0, 1, 0, 0], what="two of three write: both copy, the third keeps")
    both(m, box, [0, 1, 0, 0, 0], [999, 9, 999, 999, 999], [1] * S, what="all of them write: the first keeps")
    both(m, box, [1, 0, 3, 2, 4], [999] * S, [0] * S, what="exchanges")
    both(m, box, [1, 0, 3, 2, 4], [999, 999, p + 3, 2 * p, 1], [2, 2, p, 1, 0], what="exchanges that write")
    both(m, box, go, [m.len[0] - 2, p, 0, 5, m.len[4]], [0, 1, 1, 0, 0], what="cut back: in a page, to its end, to nothing")
    both(m, box, [0, 0, 0, 0, 0], [p, p + 1, 2 * p, 0, 3], [0, 0, 0, 7, 1], what="prefixes of the first")
    both(m, box, [0, -1, 99, -3, 4], [999] * S, [0, 0, 3, 0, 0], what="ends")
    both(m, box, go, [999] * S, [1] * S, pack=1, what="pack")
    both(m, box, go, [999] * S, [0] * S, pack=1, what="packed already")
    both(m, box, [4, 4, -1, 0, 4], [-5, 999, 999, 999, 2], [-7, 3, 0, 1, 1], pack=1, what="forks, ends and packing in one")
    both(m, box, [-1] * S, [0] * S, [0] * S, what="all end")
    assert not m.refs().any()
    box.free()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_random_steps(dev, seed):
    rng = np.random.default_rng(100 + seed)
    S, page = int(rng.choice([1, 3, 17, 64])), int(rng.choice([16, 32]))
    m = Model(rng, S, page, int(S * 4 + rng.integers(0, 20)), 9, caches=1, nkv=1, kv=int(rng.integers(0, 3)))
    box = Box(dev, m)
    for i in range(25):
        stay = rng.random(S) < 0.7
        src = np.where(stay, np.arange(S), rng.integers(-1, S, S))
        keep = np.where(rng.random(S) < 0.8, 10 ** 6, rng.integers(-2, 9 * page, S))
        add = np.where(rng.random(S) < 0.2, rng.integers(0, 3 * page, S), rng.integers(0, 3, S))
        both(m, box, src.tolist(), keep.tolist(), add.tolist(), pack=int(rng.random() < 0.3), what=(seed, i))
    box.free()


@pytest.mark.gpu
def test_steps_that_do_not_fit_change_nothing(dev):
    rng = np.random.default_rng(7)
    m = Model(rng, 4, 16, 10, 5)
    box = Box(dev, m)
    both(m, box, [-1] * 4, [0] * 4, [40, 33, 16, 5])
    both(m, box, [0, 1, 2, 3], [99] * 4, [1, 0, 33, 1], what="three pages too few")
    assert box.b["out"].numpy()[0] == 1 and m.len == [40, 33, 16, 5]
    both(m, box, [1, 0, 0, 1], [99] * 4, [16, 16, 16, 16], what="forks that do not fit")
    both(m, box, [0, 1, 2, 3], [99] * 4, [0, 48, 0, 99], what="too long, the first of two")
    assert box.b["out"].numpy()[0] == -2
    both(m, box, [0, 1, 2, 3], [99] * 4, [2 ** 31 - 1] * 4, what="lengths past 32 bits")
    assert box.b["out"].numpy()[0] == -1
    both(m, box, [1, 0, 0, 1], [99] * 4, [0, 0, 1, 0], pack=1, what="goes on after")
    box.free()


@pytest.mark.gpu
def test_many_pages(dev):
    """Page counts searched in several turns, long tables, forks of them, thousands of moves."""
    rng = np.random.default_rng(8)
    m = Model(rng, 256, 16, 70001, 5000, caches=1, nkv=1, hd=64, kv=KV_I8)
    box = Box(dev, m)
    S = m.seqs
    go = list(range(S))
    both(m, box, [-1] * S, [0] * S, [16 * 260 - s for s in range(S)], what="66000 pages")
    both(m, box, [s if s % 3 else -1 for s in range(S)], [10 ** 6] * S, [0] * S, what="a third ends")
    both(m, box, go, [10 ** 6] * S, [0] * S, pack=1, what="pack")
    both(m, box, [1] * S, [10 ** 6] * S, [20] * S, what="all fork from one")
    both(m, box, go, [10 ** 6] * S, [16] * S, pack=1, what="and pack")
    box.free()


@pytest.mark.gpu
def test_without_caches_and_with_many(dev):
    rng = np.random.default_rng(9)
    for caches in (0, 64):
        m = Model(rng, 3, 16, 12, 4, caches=caches, nkv=1)
        box = Box(dev, m)
        both(m, box, [-1] * 3, [0] * 3, [20, 5, 0])
        both(m, box, [0, 0, 0], [99] * 3, [1, 1, 1], pack=1)
        box.free()


@pytest.mark.gpu
def test_caches_past_4_gib(dev):
    """Copies and moves whose bytes lie past 2^32."""
    page, nkv, hd = 256, 4, 512
    npages = (5 << 30) // (page * nkv * hd * 4)
    block = page * nkv * hd * 4
    kv = dev.alloc(npages * block)
    i32 = lambda x: dev.to_device(np.asarray(x, np.int32))  # noqa: E731
    last = npages - 1
    rows = np.random.default_rng(1).integers(0, 256, block).astype(np.uint8)
    b = dict(table=i32([[last, -1], [last, -1]]), len=i32([100, 100]), refs=i32([0] * last + [2]), src=i32([0, 1]), keep=i32([100, 100]),
             add=i32([0, 1]), out=i32([0] * 4))
    at = dev.to_device(rows)
    dev.copy(kv.ptr + last * block, at.ptr, block)
    pages = Pages(seqs=2, npages=npages, page=page, max_pages=2, table=b["table"].ptr, len=b["len"].ptr, nkv=nkv, hd=hd, kv_dtype=KV_F32)
    work = dev.alloc(dev.pages_work_bytes(npages, 2, 2))
    dev.pages_update(pages_args(pages, b["refs"], b["src"], b["keep"], b["add"], [kv], b["out"], pack=1), work)
    dev.sync()
    assert b["out"].numpy().tolist() == [0, 1, 2, 1] and b["table"].numpy()[:, 0].tolist() == [1, 0]
    want = rows.reshape(nkv, page, -1)
    assert_bits_equal(dev.download(kv, np.uint8, (block,)).reshape(want.shape)[:, :100], want[:, :100], "copied")
    dev.copy(at.ptr, kv.ptr + block, block)
    dev.sync()
    assert_bits_equal(at.numpy(), rows, "moved")
    for x in (kv, at, work, *b.values()):
        x.free()


@pytest.mark.gpu
def test_replayed(dev):
    """One graph for steps that differ, eager steps in between; a second context at the same time."""
    rng = np.random.default_rng(10)
    with Device(0) as other:
        ms = [Model(rng, 4, 16, 40, 8) for _ in range(2)]
        boxes = [Box(d, m) for d, m in zip((dev, other), ms)]
        both(ms[0], boxes[0], [-1] * 4, [0] * 4, [30, 20, 10, 0])
        both(ms[1], boxes[1], [-1] * 4, [0] * 4, [9, 40, 17, 16])
        graphs = []
        for box in boxes:
            box.dev.graph_begin()
            box.dev.pages_update(box.args(1), box.work)
            graphs.append(box.dev.graph_end())
        steps = [([0, 1, 2, 3], [99] * 4, [1] * 4), ([0, 0, 0, 3], [99] * 4, [1, 1, 1, 0]), ([3, -1, 2, 1], [99, 0, 5, 99], [9, 0, 20, 1])]
        for st in steps + steps:
            for m, box, g in zip(ms, boxes, graphs):
                box.put(*st)
                box.dev.graph_launch(g)
            for m, box in zip(ms, boxes):
                box.dev.sync()
                assert box.b["out"].numpy().tolist() == m.step(*st, 1)
                box.check(st)
            both(ms[0], boxes[0], [0, 1, 2, 3], [99] * 4, [1, 0, 1, 0], what="eager")
        for box, g in zip(boxes, graphs):
            box.dev.graph_destroy(g)
        boxes[0].free()


def test_refusals():
    at = iter(range(1 << 36, 1 << 45, 1 << 36))
    names = ("table", "len", "refs", "src", "keep", "add", "out", "work", "kv0", "kv1")
    P = {k: next(at) for k in names}

    def args(pages={}, kvs=None, **more):
        pg = dict(seqs=3, npages=10, page=16, max_pages=4, table=P["table"], len=P["len"], nkv=2, hd=128, kv_dtype=KV_I8)
        pg.update(pages)
        a = pages_args(Pages(**pg), P["refs"], P["src"], P["keep"], P["add"], [P["kv0"], P["kv1"]] if kvs is None else kvs, P["out"])
        for k, v in more.items():
            setattr(a, k, v)
        return a

    bad = [args(pages={k: v}) for k, v in (("seqs", 0), ("seqs", 257), ("npages", 0), ("npages", (1 << 20) + 1), ("page", 8), ("page", 48),
                                           ("page", 512), ("max_pages", 0), ("max_pages", 65537), ("nkv", 0), ("nkv", 1025), ("hd", 96),
                                           ("hd", 576), ("kv_dtype", 3), ("kv_dtype", -1), ("table", None), ("len", None),
                                           ("table", P["refs"]), ("len", P["table"] + 44), ("table", P["src"]))]
    bad += [args(**{k: v}) for k, v in (("refs", None), ("src", None), ("keep", None), ("add", None), ("out", None), ("caches", -1), ("caches", 65),
                                        ("kv", None), ("refs", P["kv0"] + 64), ("out", P["len"]), ("out", P["keep"]), ("add", P["refs"] + 36),
                                        ("src", P["work"] + 64))]
    bad += [args(kvs=c) for c in ([P["kv0"], None], [P["kv0"] + 4], [P["kv0"], P["kv0"]], [P["kv0"], P["kv0"] + 16], [P["work"]], [P["table"]])]
    for i, a in enumerate(bad):
        refuses("nmx_pages_update", i, a, P["work"])
    refuses("nmx_pages_update", "no work", args(), None)
    refuses("nmx_pages_update", "odd work", args(), P["work"] + 4)
    lib = load_library()
    for x in ((0, 1, 1), ((1 << 20) + 1, 1, 1), (1, 0, 1), (1, 257, 1), (1, 1, 0), (1, 1, 65537)):
        assert lib.nmx_pages_work_bytes(*x) == 0
    assert lib.nmx_pages_work_bytes(1, 1, 1) > 0
