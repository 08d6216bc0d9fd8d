"""GPU: the DeltaNet mixer over a tree of drafts (nmx_lin_mix_tree).

The conv outputs, gates and raw copies of a node equal, bit for bit, those that nmx_lin_pre gives the
last token of the node's path; the state after the pending rows equals nmx_lin_apply's, and y and its
A8 equal nmx_lin_post of o. o and delta are held to the recurrence in 64 bits over the device's own
conv outputs.

Tolerance of o and delta, with M the largest of |v|, the state's column norms and |delta|: k and q
have norm at most 1, so a product of a row with the state is off by at most (dk / 4 + 4) 2^-24 M
(chained instructions of 4 terms), each of a node's at most L ancestors adds a product of the same
kind ((dk / 4 + 4) 2^-24 M), its decay factor (6 products of at most 2^-23) and one rounding, and a delta's
own error enters its descendants' sums, where the triangular system's inverse (|k . k'| <= 1, beta <=
1) multiplies it by at most 1 + L for the trees below: tol = (1 + L) (L + 1) (dk / 4 + 16) 2^-24 M."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import A8, LinArgs, LinMixArgs, LinPreArgs, NmxError
from tests.test_gpu_attn_tree import ancestors, tree
from tests.test_gpu_q4k import assert_bits_equal

EPS = 1e-6


def at_index(heads, dk, dv):
    """nmx_state_index of every (head, column, key)."""
    h, j, i = np.meshgrid(np.arange(heads), np.arange(dv), np.arange(dk), indexing="ij")
    return (h * dv + j // 16 * 16) * dk + ((i % (dk // 4)) // 4 * 64 + 4 * (j % 16) + i // (dk // 4)) * 4 + i % 4


def make(rng, n, heads, rep, dk, dv, K, keep, pad=0):
    kd = heads // rep * dk
    C, vd = 2 * kd + heads * dv, heads * dv
    pend = (rng.standard_normal((max(keep, 1), heads, dk + dv + 1)) * 0.1).astype(np.float32)
    pend[:, :, -1] = rng.uniform(0.9, 0.99, pend.shape[:2])
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return dict(raw=f(n, C + pad), z=f(n, vd + pad), b=f(n, heads + pad), a=f(n, heads + pad), conv=f(max(K - 1, 1), C),
                conv_w=rng.uniform(-0.5, 0.5, (C, K)).astype(np.float32), A_log=rng.uniform(-1.6, -0.9, heads).astype(np.float32),
                dt=rng.uniform(-4.5, -1, heads).astype(np.float32), norm=rng.uniform(0.8, 1.2, dv).astype(np.float32),
                rec=(rng.standard_normal(heads * dv * dk) * 0.1).astype(np.float32), pend=pend)


class Run:
    """The buffers and arguments of one call."""

    def __init__(self, dev, host, n, heads, rep, dk, dv, K, keep, pad=0, keep_dev=None, a8=True, xin=True, cap=0):
        kd = heads // rep * dk
        C, vd = 2 * kd + heads * dv, heads * dv
        self.dev, self.shape = dev, (n, heads, rep, dk, dv, K, C)
        self.b = b = {k: dev.to_device(v) for k, v in host.items()}
        for k, s in (("cv", (n, C)), ("beta", (n, heads)), ("decay", (n, heads)), ("o", (n, vd + pad)), ("y", (n, vd + pad)),
                     ("log", (n + 1, heads, dk + dv + 1)), ("xin", (n + 1, C)), ("ad", (vd // 32, n)), ("afs", (vd // 32, n))):
            b[k] = dev.to_device(np.full(s, 7, np.float32))
        b["aq"] = dev.zeros((vd // 32, n, 32), np.int8)
        if keep_dev is not None:
            b["keep_dev"] = dev.to_device(np.array([keep_dev], np.int32))
        p = lambda k: b[k].ptr  # noqa: E731
        self.pre = LinPreArgs(n, C, K, dk, kd, p("raw"), C + pad, p("cv"), p("conv"), p("conv_w"), p("xin") if xin else None,
                              np.float32(dk ** -0.5), 1e-6, p("b"), p("a"), heads + pad, heads, p("A_log"), None, p("dt"),
                              p("beta"), p("decay"))
        self.rule = LinArgs(n, heads, rep, dk, dv, 0, vd + pad, None, None, None, p("rec"), p("o"), p("log"), p("pend"), keep,
                            0, p("keep_dev") if keep_dev is not None else None)
        self.args = LinMixArgs(self.pre, self.rule, p("z"), vd + pad, p("norm"), EPS, p("y"), vd + pad,
                               A8(p("aq"), p("ad"), p("afs")) if a8 else A8(None, None, None))

    def __call__(self, parent):
        par = self.dev.to_device(parent)
        self.dev.lin_mix_tree(self.args, par)
        self.dev.sync()
        par.free()
        return {k: v.numpy() for k, v in self.b.items()}

    def free(self):
        for x in self.b.values():
            x.free()


def recurrence(cv, beta, decay, S0, parent, heads, rep, dk, dv, kd):
    """o, delta [n][heads][dv] in 64 bits, every node from its parent's state; and M."""
    n = len(parent)
    q = cv[:, :kd].reshape(n, -1, dk).astype(np.float64).repeat(rep, 1)
    k = cv[:, kd:2 * kd].reshape(n, -1, dk).astype(np.float64).repeat(rep, 1)
    v = cv[:, 2 * kd:].reshape(n, heads, dv).astype(np.float64)
    S, o, d = [], np.zeros((n, heads, dv)), np.zeros((n, heads, dv))
    for t in range(n):
        p = parent[t] if 0 <= parent[t] < t else -1
        R = (S[p] if p >= 0 else S0) * decay[t].astype(np.float64)[:, None, None]
        d[t] = (v[t] - (R @ k[t][:, :, None])[..., 0]) * beta[t].astype(np.float64)[:, None]
        R = R + d[t][:, :, None] * k[t][:, None, :]
        o[t] = (R @ q[t][:, :, None])[..., 0]
        S.append(R)
    return o, d, max(np.abs(v).max(), np.sqrt((S0 ** 2).sum(2)).max(), np.abs(d).max())


SHAPES = [
    # n, heads, rep, dk, dv, conv taps, keep, stride padding
    (1, 2, 1, 128, 128, 4, 0, 0), (2, 16, 1, 128, 128, 4, 1, 0), (9, 16, 1, 128, 128, 4, 3, 8), (16, 2, 1, 64, 64, 4, 0, 0),
    (17, 4, 2, 128, 128, 4, 9, 3), (33, 2, 1, 32, 32, 2, 2, 0), (40, 4, 4, 64, 96, 3, 0, 1), (64, 3, 1, 128, 128, 4, 5, 0),
    (64, 2, 1, 256, 64, 8, 64, 0), (48, 2, 2, 256, 512, 4, 1, 0), (64, 2, 1, 32, 160, 1, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "n%d_h%d_r%d_%dx%d_K%d_keep%d_pad%d" % s)
def test_against_recurrence(dev, shape, kind):
    n, heads, rep, dk, dv, K, keep, pad = shape
    print(f"[case] lin tree {shape} {kind}", flush=True)
    rng = np.random.default_rng(sum(shape))
    parent = tree(rng, n, kind)
    host = make(rng, n, heads, rep, dk, dv, K, keep, pad)
    r = Run(dev, host, n, heads, rep, dk, dv, K, keep, pad)
    got = r(parent)
    C, vd, kd = r.shape[6], heads * dv, heads // rep * dk

    # conv, gates: the last token of each node's path
    for t in range(n):
        path = np.flatnonzero(ancestors(parent)[t])
        h1 = {k: (v[path] if k in ("raw", "b", "a") else v) for k, v in host.items()}
        one = Run(dev, {**h1, "z": host["z"][:1]}, len(path), heads, rep, dk, dv, K, 0, pad, xin=False)
        dev.lin_pre(one.pre)
        dev.sync()
        for k in ("cv", "beta", "decay"):
            assert_bits_equal(got[k][t], one.b[k].numpy()[-1], f"{k} of node {t}")
        one.free()
        if t >= 12:
            break
    assert_bits_equal(got["xin"][:n], host["raw"][:, :C], "xin")
    assert_bits_equal(got["conv"], host["conv"], "conv state")

    # the state, then the recurrence from it
    S = dev.to_device(host["rec"])
    if keep:
        dev.lin_apply(S, r.b["pend"], keep, heads, dk, dv)
    dev.sync()
    assert_bits_equal(got["rec"], S.numpy(), "state")
    S.free()
    o, d, M = recurrence(got["cv"], got["beta"], got["decay"], got["rec"].astype(np.float64)[at_index(heads, dk, dv)], parent,
                         heads, rep, dk, dv, kd)
    L = ancestors(parent).sum(1).max()
    tol = (1 + L) * (L + 1) * (dk / 4 + 16) * 2.0 ** -24 * M
    assert np.abs(got["o"][:, :vd].reshape(o.shape) - o).max() <= tol, (np.abs(got["o"][:, :vd].reshape(o.shape) - o).max(), tol)
    log = got["log"][:n]
    assert np.abs(log[:, :, dk:dk + dv] - d).max() <= tol
    assert_bits_equal(log[:, :, :dk], got["cv"][:, kd:2 * kd].reshape(n, -1, dk).repeat(rep, 1), "log k")
    assert_bits_equal(log[:, :, -1], got["decay"], "log decay")
    assert (got["log"][n] == 7).all() and (got["xin"][n] == 7).all()
    if pad:
        assert (got["o"][:, vd:] == 7).all() and (got["y"][:, vd:] == 7).all()

    # y and its A8
    y, aq, ad, afs = (dev.zeros((n, vd), np.float32), dev.zeros(got["aq"].shape, np.int8), dev.zeros(got["ad"].shape, np.float32),
                      dev.zeros(got["ad"].shape, np.float32))
    dev.lin_post(r.b["o"], vd + pad, r.b["z"], vd + pad, r.b["norm"], n, heads, dv, EPS, y, vd, (aq, ad, afs))
    dev.sync()
    for k, x in (("aq", aq), ("ad", ad), ("afs", afs)):
        assert_bits_equal(got[k], x.numpy(), k)
    assert_bits_equal(got["y"][:, :vd], y.numpy(), "y")
    for x in (y, aq, ad, afs):
        x.free()
    r.free()


@pytest.mark.gpu
def test_other_branches_do_not_reach_a_node(dev):
    """NaN and infinities in a branch's inputs and gates leave every node outside it as it was."""
    print("[case] lin tree poison", flush=True)
    rng = np.random.default_rng(3)
    n, heads, dk, dv = 20, 2, 128, 128
    parent = tree(rng, n, "random")
    host = make(rng, n, heads, 1, dk, dv, 4, 0)
    r = Run(dev, host, n, heads, 1, dk, dv, 4, 0)
    clean = r(parent)
    r.free()
    seen = ancestors(parent)
    for bad in (np.nan, np.inf):
        h2 = {k: v.copy() for k, v in host.items()}
        for k in ("raw", "z", "b", "a"):
            h2[k][4] = bad
        r = Run(dev, h2, n, heads, 1, dk, dv, 4, 0)
        got = r(parent)
        r.free()
        out = ~seen[:, 4]
        for k in ("y", "o", "cv"):
            assert_bits_equal(got[k][out], clean[k][out], k)
        assert_bits_equal(got["log"][:n][out], clean["log"][:n][out], "log")


@pytest.mark.gpu
@pytest.mark.parametrize("keep_dev,kept", [(2, 2), (9, 5), (0, 0), (-3, 0)])
def test_keep_from_the_device(dev, keep_dev, kept):
    print(f"[case] lin tree keep_dev={keep_dev}", flush=True)
    rng = np.random.default_rng(4)
    n, heads, dk, dv = 6, 2, 64, 64
    host = make(rng, n, heads, 1, dk, dv, 4, 5)
    parent = tree(rng, n, "random")
    a, b = Run(dev, host, n, heads, 1, dk, dv, 4, 5, keep_dev=keep_dev), Run(dev, host, n, heads, 1, dk, dv, 4, kept)
    x, y = a(parent), b(parent)
    for k in ("rec", "y", "o", "log"):
        assert_bits_equal(x[k], y[k], k)
    a.free()
    b.free()


@pytest.mark.gpu
def test_zero_decay_and_beta(dev):
    """Decays of 0 (a long gap of the gates) and of 1, betas of 0: no division, no logarithm."""
    print("[case] lin tree gates", flush=True)
    rng = np.random.default_rng(5)
    n, heads, dk, dv = 30, 2, 64, 64
    host = make(rng, n, heads, 1, dk, dv, 4, 0)
    host["a"][::5] = 1e30       # decay 0
    host["a"][1::5] = -1e30     # decay 1
    host["b"][2::5] = -1e30     # beta 0
    parent = tree(rng, n, "chain")
    r = Run(dev, host, n, heads, 1, dk, dv, 4, 0)
    got = r(parent)
    assert (got["decay"] == 0).any() and (got["decay"] == 1).any() and (got["beta"] == 0).any()
    o, d, M = recurrence(got["cv"], got["beta"], got["decay"], got["rec"].astype(np.float64)[at_index(heads, dk, dv)], parent,
                         heads, 1, dk, dv, heads * dk)
    tol = (1 + n) * (n + 1) * (dk / 4 + 16) * 2.0 ** -24 * M
    assert np.abs(got["o"].reshape(o.shape) - o).max() <= tol and np.abs(got["log"][:n, :, dk:dk + dv] - d).max() <= tol
    r.free()


@pytest.mark.gpu
def test_captured_call(dev):
    """A captured call, replayed with other trees and inputs (no pending rows: the state stays)."""
    print("[case] lin tree graph", flush=True)
    rng = np.random.default_rng(6)
    n, heads, dk, dv = 21, 2, 128, 128
    host = make(rng, n, heads, 1, dk, dv, 4, 0)
    r = Run(dev, host, n, heads, 1, dk, dv, 4, 0)
    par = dev.empty(n, np.int32)
    dev.graph_begin()
    dev.lin_mix_tree(r.args, par)
    g = dev.graph_end()
    for kind in ("chain", "random", "star", "forest"):
        h2 = {**host, "raw": rng.standard_normal(host["raw"].shape).astype(np.float32)}
        parent = tree(rng, n, kind)
        dev.upload(par, parent)
        dev.upload(r.b["raw"], h2["raw"])
        dev.graph_launch(g)
        dev.sync()
        e = Run(dev, h2, n, heads, 1, dk, dv, 4, 0)
        want = e(parent)
        for k in ("y", "o", "log", "xin", "rec", "aq"):
            assert_bits_equal(r.b[k].numpy(), want[k], f"{kind} {k}")
        e.free()
    dev.graph_destroy(g)


@pytest.mark.gpu
def test_refusals(dev):
    print("[case] lin tree refusals", flush=True)
    rng = np.random.default_rng(7)
    n, heads, dk, dv = 4, 2, 64, 64
    r = Run(dev, make(rng, n, heads, 1, dk, dv, 4, 2), n, heads, 1, dk, dv, 4, 2)
    par = dev.to_device(tree(rng, n, "chain"))
    before = {k: v.numpy() for k, v in r.b.items()}

    def call(pre=None, rule=None, mix=None, parent=par):
        a = LinMixArgs(LinPreArgs.from_buffer_copy(r.pre), LinArgs.from_buffer_copy(r.rule), r.args.z, r.args.z_stride,
                       r.args.norm_w, r.args.eps, r.args.y, r.args.y_stride, r.args.a8)
        for part, ch in ((a.pre, pre), (a.rule, rule), (a, mix)):
            for k, v in (ch or {}).items():
                setattr(part, k, v)
        dev.lin_mix_tree(a, parent)

    p = {k: v.ptr for k, v in r.b.items()}
    bad = [dict(pre=dict(n=0), rule=dict(n=0)), dict(pre=dict(n=65), rule=dict(n=65)), dict(pre=dict(n=3)), dict(pre=dict(dk=128)),
           dict(pre=dict(heads=1)), dict(rule=dict(rep=0)), dict(rule=dict(rep=3)), dict(rule=dict(dv=48)), dict(rule=dict(dv=544)),
           dict(pre=dict(conv_k=0)), dict(pre=dict(conv_k=9)), dict(pre=dict(kd=64)), dict(pre=dict(C=1)), dict(pre=dict(raw_stride=10)),
           dict(pre=dict(g_stride=1)), dict(rule=dict(o_stride=10)), dict(mix=dict(z_stride=10)), dict(mix=dict(y_stride=10)),
           dict(rule=dict(keep=-1)), dict(rule=dict(keep=65)), dict(rule=dict(pend=None)), dict(rule=dict(log=None)),
           dict(rule=dict(S=None)), dict(rule=dict(o=None)), dict(pre=dict(raw=None)), dict(pre=dict(out=None)),
           dict(pre=dict(state=None)), dict(pre=dict(conv_w=None)), dict(pre=dict(b_in=None)), dict(pre=dict(a_in=None)),
           dict(pre=dict(beta=None)), dict(pre=dict(decay=None)), dict(pre=dict(dt_bias=None)), dict(pre=dict(A_log=None)),
           dict(mix=dict(z=None)), dict(mix=dict(norm_w=None)), dict(mix=dict(y=None, a8=A8(None, None, None))),
           dict(mix=dict(a8=A8(p["aq"], None, None))), dict(pre=dict(out=p["cv"] + 4)), dict(rule=dict(S=p["rec"] + 4)),
           dict(rule=dict(o=p["raw"])), dict(rule=dict(log=p["pend"])), dict(pre=dict(out=p["raw"])), dict(rule=dict(o=p["cv"])),
           dict(pre=dict(xin=p["raw"])), dict(mix=dict(y=p["z"])), dict(mix=dict(y=p["o"])), dict(parent=None)]
    for b in bad:
        with pytest.raises(NmxError, match="nmx_lin_mix_tree"):
            call(**b)
    assert dev.lib.nmx_lin_mix_tree(dev.ctx, None, par.ptr) == -1
    dev.sync()
    for k, v in r.b.items():
        assert_bits_equal(v.numpy(), before[k], k)
    r.free()


def bounded(cv, beta, decay, S0, parent, heads, rep, dk, dv, kd, rests=True):
    """o and delta [n][heads][dv] in 64 bits, as sums over a node's ancestors, and what each element may be
    off by. u = 2^-24. A product of a row with the state is dk / 8 chained instructions of 4 terms in each of
    two chains, each off by at most two roundings of its sum: (dk / 4 + 2) u of the sum of magnitudes. A
    product of nodes: rows scaled to a norm of at least 2^11 (q 2^11.5), an element as a whole number of 11
    bits and a rest of at most 1/2 + 2^-11 of the element in 11 bits, so with s = sqrt(dk) / 2 the rests
    have a norm of at most s + 1 for every 2^11 of the row's and are themselves off by 2^-11 of that: the
    product is off by (2 (s + 1) + 2) 2^-22 of the norms' product, its sums counted as one such unit. A factor of
    decays has one rounding a level; every product and sum one more. rests False: the same sums with the rests left out
    (a mistake to be noticed)."""
    n, u = len(parent), 2.0 ** -24
    q = cv[:, :kd].reshape(n, -1, dk).astype(np.float64).repeat(rep, 1)
    k = cv[:, kd:2 * kd].reshape(n, -1, dk).astype(np.float64).repeat(rep, 1)
    v = cv[:, 2 * kd:].reshape(n, heads, dv).astype(np.float64)
    nq, nk = np.linalg.norm(q, axis=2), np.linalg.norm(k, axis=2)
    qq, kk = q, k
    if not rests:
        up = lambda x, nx: 2.0 ** (11 - np.floor(np.log2(np.maximum(nx, 1e-300))))[..., None]  # noqa: E731
        qq, kk = (np.rint(x * up(x, nx)) / up(x, nx) for x, nx in ((q, nq), (k, nk)))
    KK, QK = (np.einsum("thd,ahd->tah", x, kk) for x in (kk, qq))
    s = np.sqrt(dk) / 2
    eta = (2 * (s + 1) + 2) * 2.0 ** -22
    o, d, eo, ed = (np.zeros((n, heads, dv)) for _ in range(4))
    for t in range(n):
        g, D, a, path = np.ones(heads), {}, t, []
        while a >= 0:
            D[a] = g
            path.append(a)
            g = g * decay[a]
            a = parent[a] if 0 <= parent[a] < a else -1
        L = len(path)
        state = ((dk / 4 + 2) + (L + 2)) * u
        for x, out, err, prod, nx in ((k, d, ed, KK, nk), (q, o, eo, QK, nq)):
            first = x is k
            S = g[:, None] * (S0 @ x[t][:, :, None])[..., 0]
            val, mag = (v[t] - S, np.abs(v[t]) + np.abs(S)) if first else (S, np.abs(S))
            e = state * g[:, None] * (np.abs(S0) @ np.abs(x[t])[:, :, None])[..., 0]
            for b in (path[1:] if first else path):
                c = (D[b] * prod[t, b])[:, None]
                val = val + (-c if first else c) * d[b]
                mag = mag + np.abs(c * d[b])
                e = e + (D[b] * (eta * nx[t] * nk[b] + (L + 4) * u * np.abs(prod[t, b])))[:, None] * np.abs(d[b]) + np.abs(c) * ed[b]
            e = e + (L + 1) * u * mag
            w = beta[t].astype(np.float64)[:, None] if first else 1.0
            out[t], err[t] = val * w, (e * w + u * np.abs(val * w)) * 1.001 + 1e-40
    return o, d, eo, ed


def bushes(rng, n):
    """Roots at nodes 0, 16, 32, 48, every other node below one of those before it: pairs in every block
    of 16 x 16 nodes, no depth to hide in."""
    return np.array([-1 if t % 16 == 0 else 16 * rng.integers(0, t // 16 + 1) for t in range(n)], np.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "bushes"])
@pytest.mark.parametrize("scale", [1.0, 1e-3, 1e-4, 1e-5, 1e-6, 1e-8, 1e-12])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_small_keys_and_queries(dev, dk, scale, kind):
    """Conv rows of q and k small against the norm's epsilon keep norms far below 1 (1e-6 normalises to
    1e-3): products of nodes are right relative to their rows, whatever those measure. The state is zero,
    so o is nothing but such products."""
    print(f"[case] lin tree small rows dk={dk} scale={scale} {kind}", flush=True)
    rng = np.random.default_rng(dk)
    n, heads, dv = (9, 2, 64) if kind == "chain" else (64, 2, 64)
    parent = tree(rng, n, "chain") if kind == "chain" else bushes(rng, n)
    host = make(rng, n, heads, 1, dk, dv, 4, 0)
    kd = heads * dk
    host["rec"][:] = 0
    host["b"][:] = 2
    for x in (host["raw"], host["conv"]):
        x[:, :2 * kd] *= np.float32(scale)
    host["raw"][n // 2, :kd] *= np.float32(1e-3)     # one query and one key smaller than the others
    host["raw"][n // 3, kd:2 * kd] *= np.float32(1e-2)
    r = Run(dev, host, n, heads, 1, dk, dv, 4, 0)
    got = r(parent)
    r.free()
    args = (got["cv"], got["beta"], got["decay"], np.zeros((heads, dv, dk)), parent, heads, 1, dk, dv, kd)
    o, d, eo, ed = bounded(*args)
    assert eo.max() <= 1e-3 * np.abs(o).max() and ed.max() <= 1e-3 * np.abs(d).max()
    off = bounded(*args, rests=False)
    assert (np.abs(off[0] - o) > eo).any()      # the bound would notice the rests
    err, errd = np.abs(got["o"].reshape(o.shape) - o), np.abs(got["log"][:n, :, dk:dk + dv] - d)
    assert (err <= eo).all(), (err.max(), (err / eo).max(), np.abs(o).max())
    assert (errd <= ed).all(), (errd.max(), (errd / ed).max())


@pytest.mark.gpu
def test_outputs_inside_other_inputs_are_refused(dev):
    """Every written range against the tree, the weights, the gates' vectors, the device's keep and the A8."""
    print("[case] lin tree overlaps", flush=True)
    rng = np.random.default_rng(8)
    n, heads, dk, dv = 4, 2, 64, 64
    r = Run(dev, make(rng, n, heads, 1, dk, dv, 4, 2), n, heads, 1, dk, dv, 4, 2, keep_dev=1)
    r.b["parent"] = par = dev.to_device(tree(rng, n, "chain"))
    p = {k: v.ptr for k, v in r.b.items()}
    before = {k: v.numpy() for k, v in r.b.items()}
    a8 = r.args.a8

    def call(pre=None, rule=None, mix=None, parent=par.ptr):
        a = LinMixArgs(LinPreArgs.from_buffer_copy(r.pre), LinArgs.from_buffer_copy(r.rule), r.args.z, r.args.z_stride,
                       r.args.norm_w, r.args.eps, r.args.y, r.args.y_stride, r.args.a8)
        for part, ch in ((a.pre, pre), (a.rule, rule), (a, mix)):
            for k, v in (ch or {}).items():
                setattr(part, k, v)
        dev.lin_mix_tree(a, parent)

    bad = [dict(parent=p[k]) for k in ("beta", "decay", "log", "cv", "o", "y", "rec", "xin", "aq", "ad", "afs")]
    bad += [dict(rule=dict(keep_dev=p[k])) for k in ("beta", "decay", "log", "cv", "o", "y", "rec", "xin", "aq")]
    bad += [dict(pre={f: p[k]}) for f in ("conv_w", "A_log", "dt_bias", "A") for k in ("cv", "beta", "log", "y", "aq")]
    bad += [dict(mix=dict(norm_w=p[k])) for k in ("cv", "o", "log", "y", "aq")]
    bad += [dict(mix=dict(a8=A8(p[k], a8.d, a8.fs))) for k in ("o", "y", "log", "cv", "rec", "z", "raw", "pend", "norm", "parent", "ad")]
    bad += [dict(mix=dict(a8=A8(a8.q, p[k], a8.fs))) for k in ("o", "y", "log", "norm", "keep_dev", "afs")]
    bad += [dict(mix=dict(a8=A8(a8.q, a8.d, p[k]))) for k in ("o", "y", "log", "norm", "conv_w", "aq")]
    for b in bad:
        with pytest.raises(NmxError, match="nmx_lin_mix_tree"):
            call(**b)
    dev.sync()
    for k, v in r.b.items():
        assert_bits_equal(v.numpy(), before[k], k)
    call()      # and as it is: accepted
    dev.sync()
    r.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dk,rep,keep", [(32, 1, 0), (64, 2, 3), (128, 1, 5), (256, 1, 1)])
def test_bushes_within_element_bounds(dev, dk, rep, keep):
    """o and delta of shallow trees of 64 nodes from a state, element by element; products of nodes without
    their rests would be noticed."""
    print(f"[case] lin tree bounds dk={dk}", flush=True)
    rng = np.random.default_rng(dk + 1)
    n, heads, dv = 64, 2, 96
    parent, kd = bushes(rng, n), heads // rep * dk
    host = make(rng, n, heads, rep, dk, dv, 4, keep)
    host["rec"] *= np.float32(0.05)
    host["pend"][:, :, dk:dk + dv] *= np.float32(0.05)
    host["b"][:] = 2
    r = Run(dev, host, n, heads, rep, dk, dv, 4, keep)
    got = r(parent)
    r.free()
    args = (got["cv"], got["beta"], got["decay"], got["rec"].astype(np.float64)[at_index(heads, dk, dv)], parent, heads, rep, dk, dv, kd)
    o, d, eo, ed = bounded(*args)
    off = bounded(*args, rests=False)
    assert eo.max() <= 1e-3 * np.abs(o).max() and (np.abs(off[0] - o) > 2 * eo).any() and (np.abs(off[1] - d) > ed).any()
    err, errd = np.abs(got["o"].reshape(o.shape) - o), np.abs(got["log"][:n, :, dk:dk + dv] - d)
    assert (err <= eo).all() and (errd <= ed).all(), ((err / eo).max(), (errd / ed).max())


def plain32(cv, beta, decay, S0, parent, heads, rep, dk, dv, kd):
    """The recurrence node by node in 32 bits."""
    n = len(parent)
    q, k = (cv[:, a:a + kd].reshape(n, -1, dk).repeat(rep, 1) for a in (0, kd))
    v = cv[:, 2 * kd:].reshape(n, heads, dv)
    S, o, d = [], np.zeros((n, heads, dv), np.float32), np.zeros((n, heads, dv), np.float32)
    for t in range(n):
        R = (S[parent[t]] if 0 <= parent[t] < t else S0) * decay[t][:, None, None]
        d[t] = (v[t] - (R @ k[t][:, :, None])[..., 0]) * beta[t][:, None]
        R = R + d[t][:, :, None] * k[t][:, None, :]
        o[t] = (R @ q[t][:, :, None])[..., 0]
        S.append(R)
    return o, d


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "random", "forest"])
@pytest.mark.parametrize("dk,dv", [(32, 64), (64, 128), (128, 128), (256, 64)])
def test_deep_trees_beside_plain_32_bits(dev, dk, dv, kind):
    """Errors of o and delta over 64 nodes, root mean square and largest, against those of the plain
    recurrence in 32 bits on the same inputs. A product of nodes is off by about 2^-24 of its rows' norms, and
    its sums over a node's ancestors are rounded as often as these are many; the plain form rounds its
    state's elements at each node, about one such unit a level of a product, and its sums. So the two are of one
    size: at most 8 times the plain one's passes (16 for the largest), a product without rests, 2^-13.3 of the
    norms, is 1000 times it."""
    print(f"[case] lin tree 32 bits dk={dk} {kind}", flush=True)
    rng = np.random.default_rng(dk + 2)
    n, heads = 64, 2
    parent, kd = tree(rng, n, kind), heads * dk
    host = make(rng, n, heads, 1, dk, dv, 4, 2)
    r = Run(dev, host, n, heads, 1, dk, dv, 4, 2)
    got = r(parent)
    r.free()
    S0 = got["rec"][at_index(heads, dk, dv)]
    args = (got["cv"], got["beta"], got["decay"], S0, parent, heads, 1, dk, dv, kd)
    o, d, _ = recurrence(*args[:3], S0.astype(np.float64), *args[4:])
    for name, x, want, plain in zip("od", (got["o"].reshape(o.shape), got["log"][:n, :, dk:dk + dv]), (o, d), plain32(*args)):
        err, ref = x - want, plain - want
        rms, rms32 = (float(np.sqrt((e * e).mean())) for e in (err, ref))
        print(f"[case]   {name}: rms {rms:.2e} ({rms32:.2e} plain), largest {np.abs(err).max():.2e} ({np.abs(ref).max():.2e})", flush=True)
        assert rms <= 8 * rms32 and np.abs(err).max() <= 16 * np.abs(ref).max()


@pytest.mark.gpu
def test_optional_arguments(dev):
    """y alone, the A8 alone, no xin, A in place of A_log: what is given equals the full call's, bit for bit."""
    print("[case] lin tree optional arguments", flush=True)
    rng = np.random.default_rng(13)
    n, heads, dk, dv = 21, 2, 64, 64
    host = make(rng, n, heads, 1, dk, dv, 4, 2)
    host["A"] = -np.exp(host["A_log"].astype(np.float64)).astype(np.float32)
    parent = tree(rng, n, "random")

    def call(change=lambda a: None):
        r = Run(dev, host, n, heads, 1, dk, dv, 4, 2)
        change(r)
        got = r(parent)
        r.free()
        return got

    full = call()
    outs = ("y", "aq", "ad", "afs", "o", "log", "rec", "xin", "cv")

    def same(got, but):
        for k in outs:
            if k not in but:
                assert_bits_equal(got[k], full[k], k)

    def no_a8(r):
        r.args.a8 = A8(None, None, None)

    def no_y(r):
        r.args.y = None

    def no_xin(r):
        r.args.pre.xin = None

    got = call(no_a8)
    same(got, ("aq", "ad", "afs"))
    assert not got["aq"].any() and (got["ad"] == 7).all()
    got = call(no_y)
    same(got, ("y",))
    assert (got["y"] == 7).all()
    got = call(no_xin)
    same(got, ("xin",))
    assert (got["xin"] == 7).all()

    def given_A(r):
        r.args.pre.A, r.args.pre.A_log = r.b["A"].ptr, None

    got = call(given_A)     # A may differ from the device's -exp(A_log) in the last place: an exponent of at most 1
    assert np.abs(got["decay"] - full["decay"]).max() <= 2.0 ** -22
    same(got, outs[:7])


@pytest.mark.gpu
def test_replays_that_advance_the_state(dev):
    """A captured call with pending rows folds them in at every replay, as eager calls do."""
    print("[case] lin tree replays", flush=True)
    rng = np.random.default_rng(14)
    n, heads, dk, dv = 40, 2, 128, 64
    host = make(rng, n, heads, 1, dk, dv, 4, 9)
    parent = tree(rng, n, "random")
    a, b = (Run(dev, host, n, heads, 1, dk, dv, 4, 9, keep_dev=9) for _ in range(2))
    par = dev.to_device(parent)
    dev.graph_begin()
    dev.lin_mix_tree(a.args, par)
    g = dev.graph_end()
    for keep in (3, 0, 9, 5):
        for r in (a, b):
            dev.upload(r.b["keep_dev"], np.array([keep], np.int32))
        dev.graph_launch(g)
        dev.lin_mix_tree(b.args, par)
        dev.sync()
        for k in ("y", "o", "log", "rec"):
            assert_bits_equal(a.b[k].numpy(), b.b[k].numpy(), f"keep {keep} {k}")
    dev.graph_destroy(g)
    for x in (a, b):
        x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("decay", [0.999, 0.5])
def test_one_key_for_every_node(dev, decay):
    """A chain of 64 tokens alike: every product of keys is that of a row with itself, which the deltas'
    triangular system is hardest on; held as in the deep trees above."""
    print(f"[case] lin tree one key decay={decay}", flush=True)
    rng = np.random.default_rng(15)
    n, heads, dk, dv = 64, 2, 128, 64
    parent, kd = tree(rng, n, "chain"), heads * dk
    host = make(rng, n, heads, 1, dk, dv, 4, 0)
    host["raw"][:, :2 * kd] = host["raw"][:1, :2 * kd]
    host["b"][:] = 3
    host["a"][:] = np.log(np.expm1(-np.log(decay) / np.exp(host["A_log"]))) - host["dt"]
    r = Run(dev, host, n, heads, 1, dk, dv, 4, 0)
    got = r(parent)
    r.free()
    S0 = got["rec"][at_index(heads, dk, dv)]
    args = (got["cv"], got["beta"], got["decay"], S0, parent, heads, 1, dk, dv, kd)
    o, d, _ = recurrence(*args[:3], S0.astype(np.float64), *args[4:])
    for name, x, want, plain in zip("od", (got["o"].reshape(o.shape), got["log"][:n, :, dk:dk + dv]), (o, d), plain32(*args)):
        err, ref = x - want, plain - want
        rms, rms32 = (float(np.sqrt((e * e).mean())) for e in (err, ref))
        print(f"[case]   {name}: rms {rms:.2e} ({rms32:.2e} plain), largest {np.abs(err).max():.2e} ({np.abs(ref).max():.2e})", flush=True)
        assert rms <= 8 * rms32 and np.abs(err).max() <= 16 * np.abs(ref).max()
