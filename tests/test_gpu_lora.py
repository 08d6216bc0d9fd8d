"""GPU: low-rank adapters of many requests (nmx_lora) against their definition in 64 bits.

Tolerance of each element, half a step of 32 bits (2^-24) an addition, of sums that are at most those of the
absolute values. A rank's sum has a chain of cols / 16 additions in a wave's two accumulators (its columns are
shared out over 8), the accumulators, and 8 waves: cols / 16 + 16 (at least 32 for a wave's own step); B's has rank,
rounded up to 32, the scale and y itself two more."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import Device, load_library, lora_args
from tests.batch_refuse import refuses

H = 2.0 ** -24


def bf16(x):
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + (u >> 16 & 1)) >> 16).astype(np.uint16)


def weights(x, w):
    """(as stored, the values that they stand for in 64 bits)"""
    if w == 0:
        return x.astype(np.float32), x.astype(np.float32).astype(np.float64)
    if w == 1:
        return x.astype(np.float16), x.astype(np.float16).astype(np.float64)
    b = bf16(x)
    return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Case:
    def __init__(self, rng, n, cols, rows, adapters, rank, w, ids=None, ranks=None, stride=0, ystride=0, spread=1.0):
        self.n, self.cols, self.rows, self.adapters, self.rank, self.w = n, cols, rows, adapters, rank, w
        self.xs, self.ys = cols + stride, [r + ystride for r in rows]
        self.x = (rng.standard_normal((n, self.xs)) * np.exp(rng.uniform(-spread, spread, (n, 1)))).astype(np.float32)
        self.ids = np.asarray(rng.integers(0, adapters, n) if ids is None else ids, np.int32)
        self.ranks = None if ranks is None else np.asarray(ranks, np.int32)
        self.scale = rng.uniform(-2, 2, adapters).astype(np.float32)
        A, B = zip(*[(weights(rng.standard_normal((adapters, rank, cols)) * cols ** -0.5, w), weights(rng.standard_normal((adapters, r, rank)), w))
                     for r in rows])
        self.A, self.A64 = zip(*A)
        self.B, self.B64 = zip(*B)
        self.y = [rng.standard_normal((n, s)).astype(np.float32) for s in self.ys]

    def poison(self):
        """What lies behind an adapter's own rank, and adapters that no row has, hold NaN."""
        nan = {0: np.float32(np.nan), 1: np.float16(np.nan), 2: np.uint16(0x7fc0)}[self.w]
        for m in range(self.adapters):
            rk = self.rank if self.ranks is None else max(0, min(self.rank, int(self.ranks[m])))
            for A, B in zip(self.A, self.B):
                if m not in self.ids:
                    A[m], B[m] = nan, nan
                A[m, rk:], B[m, :, rk:] = nan, nan

    def reference(self):
        ys, tols = [], []
        c1, c2 = max(self.cols / 16, 32) + 16, -(-self.rank // 32) * 32 + 2
        for A, B, y, r in zip(self.A64, self.B64, self.y, self.rows):
            want, tol = y.astype(np.float64), np.zeros(y.shape)
            for t in range(self.n):
                m = self.ids[t]
                if not 0 <= m < self.adapters:
                    continue
                rk = self.rank if self.ranks is None else max(0, min(self.rank, int(self.ranks[m])))
                x, a, b, s = self.x[t, :self.cols].astype(np.float64), A[m, :rk], B[m][:, :rk], float(self.scale[m])
                low, alow = a @ x, np.abs(a) @ np.abs(x)
                want[t, :r] += s * (b @ low)
                tol[t, :r] = H * (abs(s) * (np.abs(b) @ (c1 * alow + c2 * np.abs(low))) + 2 * np.abs(want[t, :r]) + abs(s) * np.abs(b @ low))
            ys.append(want), tols.append(tol)
        return ys, tols

    def upload(self, dev):
        return dict(x=dev.to_device(self.x), ids=dev.to_device(self.ids), ranks=None if self.ranks is None else dev.to_device(self.ranks),
                    scale=dev.to_device(self.scale), A=[dev.to_device(a) for a in self.A], B=[dev.to_device(b) for b in self.B],
                    y=[dev.to_device(y) for y in self.y], work=dev.alloc(dev.lora_work_bytes(self.n, len(self.rows), self.rank)))

    def args(self, d):
        return lora_args(self.n, self.cols, d["x"], self.xs, self.adapters, self.rank, self.w, d["ids"], d["scale"],
                         list(zip(self.rows, d["A"], d["B"], d["y"], self.ys)), ranks=d["ranks"])


def free(d):
    for v in d.values():
        for x in v if isinstance(v, list) else [v]:
            if x is not None:
                x.free()


def run(dev, c):
    d = c.upload(dev)
    dev.upload(d["work"], np.full(d["work"].nbytes // 4, np.nan, np.float32))
    dev.lora(c.args(d), d["work"])
    dev.sync()
    got = [y.numpy() for y in d["y"]]
    free(d)
    return got


def check(dev, c):
    want, tol = c.reference()
    c.poison()
    for g, w, t, y, r in zip(run(dev, c), want, tol, c.y, c.rows):
        assert (g[:, r:] == y[:, r:]).all()
        none = (c.ids < 0) | (c.ids >= c.adapters)
        assert (g[none].view(np.uint32) == y[none].view(np.uint32)).all()
        bad = ~(np.abs(g - w) <= t)
        assert not bad.any(), (np.argwhere(bad)[:5], np.abs(g - w).max(), t.max())


CASES = [
    # n, cols, rows, adapters, rank, w, ids, ranks, strides of x and y beyond the row
    (1, 1024, [512], 1, 16, 1, None, None, 0, 0),
    (1, 32, [1], 1, 1, 0, None, None, 4, 1),
    (3, 64, [5, 16, 100], 4, 3, 2, [2, 2, 0], None, 0, 3),
    (8, 1024, [4096, 512, 512], 5, 16, 1, None, None, 0, 0),
    (16, 256, [64], 2, 8, 2, [1] * 16, None, 0, 0),                # a whole tile
    (17, 256, [64], 2, 8, 0, [1] * 17, None, 0, 0),                # and a row more
    (64, 1024, [3584, 3584], 40, 64, 2, None, "ragged", 0, 0),
    (64, 3584, [1024], 64, 32, 1, list(range(64)), None, 0, 0),    # each its own
    (65, 288, [33], 3, 25, 1, None, "ragged", 12, 7),              # odd everything
    (130, 96, [48, 1000], 3, 40, 2, [0, 1, 2, -1, 7] * 26, [0, 40, 99], 0, 0),   # none, an empty one, ids outside
    (300, 1024, [512], 2, 96, 0, None, None, 0, 0),
    (512, 512, [256], 1, 256, 1, None, None, 0, 0),
    (512, 32, [64] * 6, 512, 8, 2, list(range(512)), None, 0, 0),
    (5, 32768, [16], 2, 5, 0, None, None, 0, 0),
    (64, 1024, [3584, 3584], 40, 16, 1, None, None, 0, 0),         # small ranks, many workgroups: two launches
    (200, 64, [512, 40], 9, 12, 2, None, "ragged", 0, 0),          # in one
    (200, 64, [4096, 4096], 9, 12, 2, None, "ragged", 0, 0),       # in two
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"n{c[0]}_{c[1]}to{'+'.join(map(str, c[2]))}_a{c[3]}r{c[4]}w{c[5]}")
def test_definition(dev, case):
    n, cols, rows, adapters, rank, w, ids, ranks, xs, ys = case
    rng = np.random.default_rng(n + cols + rank)
    if ranks == "ragged":
        ranks = rng.integers(0, rank + 1, adapters)
    check(dev, Case(rng, n, cols, rows, adapters, rank, w, ids, ranks, xs, ys))


@pytest.mark.gpu
def test_no_adapter_at_all(dev):
    check(dev, Case(np.random.default_rng(1), 9, 64, [40], 3, 8, 1, ids=[-1, 3, 99, -2 ** 31, 2 ** 31 - 1, 3, 3, 3, 3]))


@pytest.mark.gpu
def test_rows_do_not_depend_on_each_other(dev):
    """The same row alone, among others of its adapter and among others: the same bits."""
    rng = np.random.default_rng(2)
    c = Case(rng, 40, 512, [96], 4, 24, 2, ids=[2] * 20 + [0, 1, 2, 3] * 5)
    all_ = run(dev, c)[0]
    for t in (0, 19, 22, 39):
        one = Case(np.random.default_rng(3), 1, 512, [96], 4, 24, 2, ids=[c.ids[t]])
        one.x, one.A, one.B, one.scale, one.y = c.x[t:t + 1], c.A, c.B, c.scale, [c.y[0][t:t + 1]]
        assert (run(dev, one)[0].view(np.uint32) == all_[t:t + 1].view(np.uint32)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,rank", [(1, 256), (2, 200), (3, 32), (7, 256)])
def test_few_rows_of_large_ranks(dev, n, rank):
    """Tiles that are mostly empty, the workspace's rows longer than its list of tiles."""
    check(dev, Case(np.random.default_rng(n + rank), n, 128, [100, 24], 2, rank, 1, ids=[1] * n))


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 48])
def test_what_one_row_holds_stays_in_it(dev, rank):
    """NaN and infinities in a row, in its adapter and in rows without one: the others' bits are as without them."""
    rng = np.random.default_rng(rank)
    c = Case(rng, 24, 96, [80, 33], 4, rank, 0, ids=[0, 1, 2, -1] * 6)
    want = run(dev, c)
    c.x[4], c.x[8, 5], c.x[3::4] = np.nan, np.inf, np.nan
    for B in c.B:
        B[2] = np.inf
    got = run(dev, c)
    for g, w in zip(got, want):
        for t in range(24):
            if t in (4, 8):
                assert not np.isfinite(g[t]).any()
            elif c.ids[t] != 2:
                assert (g[t].view(np.uint32) == w[t].view(np.uint32)).all()


@pytest.mark.gpu
def test_replayed_with_other_adapters(dev):
    """Adapters, ranks and scales are the device's; a replay adds to y again. Two contexts at once."""
    rng = np.random.default_rng(4)
    with Device(0) as other:
        cs = [Case(rng, 20, 256, [128, 32], 5, 16, 1, ranks=[16, 3, 0, 9, 16]) for _ in range(2)]
        devs, ds = (dev, other), []
        for x, c in zip(devs, cs):
            d = c.upload(x)
            ds.append(d)
            x.graph_begin()
            x.lora(c.args(d), d["work"])
            d["g"] = x.graph_end()
        for k in range(3):
            for x, c, d in zip(devs, cs, ds):
                c.ids = rng.integers(-1, 5, 20).astype(np.int32)
                x.upload(d["ids"], c.ids)
                x.graph_launch(d["g"])
            for x, c, d in zip(devs, cs, ds):
                want, tol = c.reference()
                x.sync()
                c.y = [y.numpy() for y in d["y"]]
                assert all((np.abs(g - w) <= t).all() for g, w, t in zip(c.y, want, tol))
        for x, d in zip(devs, ds):
            x.graph_destroy(d.pop("g"))
        free(ds[0])


@pytest.mark.gpu
def test_matrices_side_by_side(dev):
    """Outputs that are columns of the same rows."""
    rng = np.random.default_rng(5)
    c = Case(rng, 11, 128, [40, 24, 30], 3, 12, 1)
    d, Y = c.upload(dev), dev.to_device(np.concatenate([y for y in c.y] + [c.y[0][:, :2]], 1))
    wide, at = 40 + 24 + 30 + 2, 0
    segs = []
    for r, A, B in zip(c.rows, d["A"], d["B"]):
        segs.append((r, A, B, Y.ptr + 4 * at, wide))
        at += r
    dev.lora(lora_args(11, 128, d["x"], c.xs, 3, 12, 1, d["ids"], d["scale"], segs[::-1]), d["work"])
    dev.sync()
    want, tol = c.reference()
    got = Y.numpy()
    assert (np.abs(got[:, :94] - np.concatenate(want, 1)) <= np.concatenate(tol, 1)).all() and (got[:, 94:] == c.y[0][:, :2]).all()
    Y.free()
    free(d)


def test_refusals():
    at = iter(range(1 << 36, 1 << 45, 1 << 36))
    P = {k: next(at) for k in ("x", "ids", "ranks", "scale", "A", "B", "Y", "A2", "B2", "Y2", "work")}

    def args(segs=None, **more):
        a = lora_args(4, 64, P["x"], 64, 3, 8, 1, P["ids"], P["scale"],
                      segs or [(32, P["A"], P["B"], P["Y"], 32), (16, P["A2"], P["B2"], P["Y2"], 20)], ranks=P["ranks"])
        for k, v in more.items():
            setattr(a, k, v)
        return a

    bad = [args(**{k: v}) for k, v in (("n", 0), ("n", 513), ("cols", 0), ("cols", 48), ("cols", 32800), ("x_stride", 60), ("x_stride", 66),
                                       ("count", 0), ("count", 7), ("adapters", 0), ("rank", 0), ("rank", 257), ("w_dtype", 3), ("w_dtype", -1),
                                       ("x", None), ("adapter", None), ("scale", None), ("x", P["x"] + 4))]
    one = lambda **k: [tuple({**dict(r=32, A=P["A"], B=P["B"], Y=P["Y"], s=32), **k}.values())]  # noqa: E731
    bad += [args(one(**k)) for k in (dict(r=0), dict(r=(1 << 20) + 1, s=1 << 21), dict(s=31), dict(A=None), dict(B=None), dict(Y=None),
                                     dict(A=P["A"] + 8), dict(B=P["B"] + 2), dict(Y=P["Y"] + 2), dict(Y=P["x"]), dict(Y=P["A"] + 64),
                                     dict(Y=P["B"]), dict(Y=P["ids"]), dict(Y=P["ranks"] + 8), dict(Y=P["scale"]), dict(Y=P["work"]))]
    bad += [args([(32, P["A"], P["B"], P["Y"], s), (16, P["A2"], P["B2"], P["Y"] + 4 * at, t)])
            for s, t, at in ((32, 32, 16), (48, 48, 31), (48, 48, 33), (48, 64, 32), (47, 47, 32), (48, 48, 48 + 31), (48, 48, 0))]
    for i, a in enumerate(bad):
        refuses("nmx_lora", i, a, P["work"])
    refuses("nmx_lora", "no work", args(), None)
    refuses("nmx_lora", "odd work", args(), P["work"] + 4)
    refuses("nmx_lora", "work over A", args(), P["A"])
    lib = load_library()
    for x in ((0, 1, 1), (513, 1, 1), (1, 0, 1), (1, 7, 1), (1, 1, 0), (1, 1, 257)):
        assert lib.nmx_lora_work_bytes(*x) == 0
