"""GPU: attention of a tree of drafts (nmx_attn_tree, nmx_attn_tree_prep) against its definition in 64
bits, and the prep against nmx_attn_prep bit for bit.

Tolerance of o, relative to the largest |v| in sight: a score's operands are held to 2^-22 of their
rows' largest element (two binary16 parts), products are added in 32 bits over hd / 32 chained
instructions of 32 terms and rounded a few times more, so a score is off by at most
    ds = |q| |k| scale (4 2^-22 + (hd / 32 + 8) 2^-24)
(norms of the longest rows; the 2^-22 of the largest element is at most that of the norm); a
softmax mean moves by at most 2 ds times the largest value, and the exponentials, the weights' two
parts, the running rescales (one rounding a tile, and a tile a part on average) and the last quotient
and gate add less than 2^-18."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import A8, AttnArgs, Device, NmxError, tree_commit_args
from tests.test_gpu_q4k import assert_bits_equal

KV_F32, KV_F16, KV_I8 = 0, 1, 2


def tree(rng, n, kind):
    if kind == "chain":
        return np.arange(-1, n - 1, dtype=np.int32)
    if kind == "star":
        return np.array([-1] + [0] * (n - 1), np.int32)
    if kind == "forest":   # several nodes after the context
        return np.array([-1 if t % 3 == 0 else rng.integers(0, t) for t in range(n)], np.int32)
    return np.array([-1] + [rng.integers(max(0, t - 8), t) for t in range(1, n)], np.int32)


def ancestors(parent):
    seen = np.zeros((len(parent), len(parent)), bool)
    for t, p in enumerate(parent):
        if 0 <= p < t:
            seen[t] = seen[p]
        seen[t, t] = True
    return seen


def make_cache(rng, kv, nkv, ctx, hd, std=1.0, spread=0.0):
    """(bytes in the cache's format, the values that they stand for in 64 bits). spread: rows of
    magnitudes e^(+-spread)."""
    rows = rng.standard_normal((nkv, ctx, hd)).astype(np.float32) * np.float32(std)
    rows *= np.exp(rng.uniform(-spread, spread, (nkv, ctx, 1))).astype(np.float32)
    return encode(rows, kv)


def encode(rows, kv):
    if kv == KV_F32:
        return rows.copy(), rows.astype(np.float64)
    if kv == KV_F16:
        h = rows.astype(np.float16)
        return h, h.astype(np.float64)
    amax = np.abs(rows).max(2)
    codes = np.rint(rows * np.where(amax > 0, 127 / np.where(amax > 0, amax, 1), 0)[..., None]).astype(np.int8)
    scale = (amax / np.float32(127)).astype(np.float32)
    return (np.concatenate([codes.ravel().view(np.uint8), scale.ravel().view(np.uint8)]),
            codes.astype(np.float64) * scale.astype(np.float64)[..., None])


def run(dev, q, kc, vc, parent, pos, shape, kv, a8=False, work=None, pos_off=-2, times=1):
    n, nh, nkv, hd, ctx = shape
    b = dict(q=dev.to_device(q), kc=dev.to_device(kc), vc=dev.to_device(vc), parent=dev.to_device(parent),
             pos=dev.to_device(np.array([pos - pos_off], np.int32)), o=dev.to_device(np.full((n + 1, nh * hd), 7, np.float32)))
    w = work or dev.alloc(dev.attn_tree_work_bytes(n, nh, nkv, hd))
    nb = nh * hd // 32
    aq = (dev.zeros((nb, n, 32), np.int8), dev.zeros((nb, n), np.float32), dev.zeros((nb, n), np.float32)) if a8 else ()
    a = AttnArgs(n=n, nh=nh, nkv=nkv, hd=hd, max_ctx=ctx, q=b["q"].ptr, scale=np.float32(1 / np.sqrt(hd)),
                 kc=b["kc"].ptr, vc=b["vc"].ptr, pos=b["pos"].ptr, pos_off=pos_off, o=b["o"].ptr,
                 a8=A8(*([x.ptr for x in aq] or [None] * 3)), kv_dtype=kv)
    for _ in range(times):
        dev.attn_tree(a, b["parent"].ptr, w.ptr)
    dev.sync()
    o = b["o"].numpy()
    assert (o[n] == 7).all()
    codes = [x.numpy() for x in aq]
    for x in (*b.values(), *aq, *([] if work else [w])):
        x.free()
    return (o[:n], *codes) if a8 else o[:n]


def reference(q, K, V, parent, pos, shape):
    """(o, the tolerance): 64-bit attention of the nodes whose rows are in the cache."""
    n, nh, nkv, hd, ctx = shape
    pos0 = max(pos, 0)
    seen = ancestors(parent)
    slots = pos + np.arange(n)
    inside = (slots >= 0) & (slots < ctx)
    o, scale, tol = np.zeros((n, nh, hd)), float(np.float32(1 / np.sqrt(hd))), 0.0
    for h in range(nh):
        g = h // (nh // nkv)
        for t in range(n):
            at = np.concatenate([np.arange(min(pos0, ctx)), slots[seen[t] & inside]]).astype(int)
            if not len(at):
                continue
            qt, k, v = q[t, h, :hd].astype(np.float64), K[g, at], V[g, at]
            s = k @ qt * scale
            p = np.exp(s - s.max())
            o[t, h] = p @ v / p.sum() / (1 + np.exp(-q[t, h, hd:].astype(np.float64)))
            ds = np.linalg.norm(qt) * np.linalg.norm(k, axis=1).max() * scale * (4 * 2.0 ** -22 + (hd / 32 + 8) * 2.0 ** -24)
            tol = max(tol, (2 * ds + 2.0 ** -18) * np.abs(v).max())
    return o.reshape(n, nh * hd), tol


def check(dev, rng, case, kind="random", std=1.0, spread=0.0, poison=True):
    n, nh, nkv, hd, ctx, kv, pos = case
    shape = (n, nh, nkv, hd, ctx)
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    parent = tree(rng, n, kind)
    (kc, K), (vc, V) = (make_cache(rng, kv, nkv, ctx, hd, std, spread) for _ in range(2))
    want, tol = reference(q, K, V, parent, pos, shape)
    if poison and pos + n < ctx:    # rows past the tree hold anything
        for c in (kc, vc):
            rows = c if kv != KV_I8 else c[nkv * ctx * hd:].view(np.float32).reshape(nkv, ctx)
            rows[:, pos + n:] = np.nan
    got = run(dev, q, kc, vc, parent, pos, shape, kv, times=2)
    assert np.abs(got - want).max() <= tol, (np.abs(got - want).max(), tol)


CASES = [
    # n, query heads, KV heads, head size, max_ctx, kv dtype, position of node 0
    (1, 8, 2, 256, 64, 0, 0),          # the first token of a conversation
    (1, 8, 2, 256, 64, 1, 1),
    (1, 8, 2, 256, 3000, 2, 2999),     # the last slot
    (2, 1, 1, 64, 40, 1, 31),
    (5, 8, 2, 256, 700, 0, 600),
    (9, 8, 2, 256, 700, 1, 33),
    (9, 6, 2, 128, 300, 2, 64),        # three heads per group
    (4, 4, 4, 64, 257, 0, 250),
    (17, 8, 1, 512, 200, 0, 95),
    (17, 8, 1, 512, 200, 1, 127),
    (16, 8, 1, 512, 200, 2, 129),
    (33, 4, 2, 192, 500, 0, 300),
    (33, 4, 2, 320, 500, 1, 300),
    (21, 4, 2, 448, 500, 2, 300),
    (64, 8, 2, 256, 1100, 1, 1000),
    (64, 8, 2, 256, 1100, 0, 1036),    # the tree ends with the cache
    (64, 16, 2, 256, 600, 2, 0),       # no context at all
    (64, 2, 1, 128, 9000, 1, 8900),    # more than one tile of positions a part
    (3, 12, 1, 64, 5000, 2, 4900),
    (8, 4, 2, 128, 20000, 0, 19990),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "n%d_h%d_%d_hd%d_ctx%d_kv%d_pos%d" % c)
def test_against_definition(dev, case):
    print(f"[case] attn tree {case}", flush=True)
    check(dev, np.random.default_rng(sum(case)), case)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "star", "forest"])
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
def test_tree_shapes(dev, kind, kv):
    print(f"[case] attn tree {kind} kv={kv}", flush=True)
    check(dev, np.random.default_rng(kv), (64, 4, 2, 64, 300, kv, 130), kind=kind)
    check(dev, np.random.default_rng(kv), (13, 4, 2, 128, 300, kv, 31), kind=kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
def test_rows_of_many_magnitudes(dev, kv):
    """Value rows from e^-8 to e^8 of each other, keys alike; fp32 and int8 rows far outside
    binary16's range."""
    print(f"[case] attn tree magnitudes kv={kv}", flush=True)
    rng = np.random.default_rng(11 + kv)
    n, nh, nkv, hd, ctx, pos = 6, 4, 2, 128, 400, 380
    parent = tree(rng, n, "random")
    for vstd, spread in ((1.0, 8.0), (1e30, 3.0), (1e-30, 3.0), (0.0, 0.0)) if kv != KV_F16 else ((1.0, 5.0), (2e3, 2.0), (1e-6, 1.0)):
        q = (rng.standard_normal((n, nh, 2 * hd)) * 1e3).astype(np.float32)
        q[..., hd:] *= 1e-3
        kc, K = make_cache(rng, kv, nkv, ctx, hd, 1e-3, 1.0)
        vc, V = make_cache(rng, kv, nkv, ctx, hd, vstd, spread)
        want, tol = reference(q, K, V, parent, pos, (n, nh, nkv, hd, ctx))
        got = run(dev, q, kc, vc, parent, pos, (n, nh, nkv, hd, ctx), kv)
        assert np.abs(got - want).max() <= tol, (vstd, np.abs(got - want).max(), tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_unseen_nodes_may_hold_anything(dev, kv, bad):
    """NaN and infinities in the rows of nodes that a node does not descend from, and behind them."""
    print(f"[case] attn tree poison {bad} kv={kv}", flush=True)
    rng = np.random.default_rng(5)
    n, nh, nkv, hd, ctx, pos = 9, 8, 2, 256, 80, 45
    parent = np.array([-1, 0, 0, 1, 1, 2, 2, 3, 5], np.int32)
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    (kc, K), (vc, V) = (make_cache(rng, kv, nkv, ctx, hd) for _ in range(2))
    want, tol = reference(q, K, V, parent, pos, (n, nh, nkv, hd, ctx))
    for c in (kc, vc):
        c[:, pos + 2] = bad      # nodes 2, 5, 6, 8 see it
        c[:, pos + n:] = bad
    got = run(dev, q, kc, vc, parent, pos, (n, nh, nkv, hd, ctx), kv)
    clean = [0, 1, 3, 4, 7]
    assert np.abs(got[clean] - want[clean]).max() <= tol
    assert not np.isfinite(got[[2, 5, 6, 8]]).any()


@pytest.mark.gpu
def test_parents_outside_the_tree(dev):
    """Parents that are not -1 .. t - 1 count as -1: equal bits."""
    print("[case] attn tree bad parents", flush=True)
    rng = np.random.default_rng(6)
    n, nh, nkv, hd, ctx, pos = 8, 4, 2, 64, 100, 50
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    (kc, _), (vc, _) = (make_cache(rng, KV_F16, nkv, ctx, hd) for _ in range(2))
    a = run(dev, q, kc, vc, np.array([-1, 0, -1, 2, -1, 4, -1, -1], np.int32), pos, (n, nh, nkv, hd, ctx), KV_F16)
    b = run(dev, q, kc, vc, np.array([5, 0, 2, 2, 99, 4, -7, -2 ** 31], np.int32), pos, (n, nh, nkv, hd, ctx), KV_F16)
    assert_bits_equal(a, b, "o")


@pytest.mark.gpu
@pytest.mark.parametrize("pos", [-3, -100, 95, 100, 500, 2 ** 31 - 3, -2 ** 31 + 3])
def test_nodes_outside_the_cache(dev, pos):
    """Slots before the cache or past its end: those nodes have no row, none is read or written."""
    print(f"[case] attn tree pos={pos}", flush=True)
    rng = np.random.default_rng(7)
    n, nh, nkv, hd, ctx = 8, 4, 2, 64, 100
    parent = tree(rng, n, "random")
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    (kc, K), (vc, V) = (make_cache(rng, KV_F32, nkv, ctx, hd) for _ in range(2))
    got = run(dev, q, kc, vc, parent, pos, (n, nh, nkv, hd, ctx), KV_F32, pos_off=0)
    want, tol = reference(q, K, V, parent, min(max(pos, -200), 300), (n, nh, nkv, hd, ctx))
    assert np.abs(got - want).max() <= max(tol, 1e-30)


@pytest.mark.gpu
def test_a8_and_graph(dev):
    """The A8 of the rows is what nmx_quant_a8 makes of them; a captured call, replayed at other
    positions with other trees, gives what plain calls give."""
    print("[case] attn tree a8, graph", flush=True)
    rng = np.random.default_rng(8)
    n, nh, nkv, hd, ctx = 12, 8, 2, 256, 500
    shape = (n, nh, nkv, hd, ctx)
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    (kc, _), (vc, _) = (make_cache(rng, KV_I8, nkv, ctx, hd) for _ in range(2))
    o, aq, ad, afs = run(dev, q, kc, vc, tree(rng, n, "random"), 300, shape, KV_I8, a8=True)
    x = dev.to_device(o)
    eq, ed, efs = dev.zeros(aq.shape, np.int8), dev.zeros(ad.shape, np.float32), dev.zeros(ad.shape, np.float32)
    dev.quant_a8(x, n, nh * hd, eq, ed, efs)
    dev.sync()
    for got, want, k in ((aq, eq, "q"), (ad, ed, "d"), (afs, efs, "fsum")):
        assert_bits_equal(got, want.numpy(), k)
    b = dict(q=dev.to_device(q), kc=dev.to_device(kc), vc=dev.to_device(vc), parent=dev.empty(n, np.int32),
             pos=dev.empty(1, np.int32), o=dev.empty((n, nh * hd), np.float32))
    work = dev.alloc(dev.attn_tree_work_bytes(n, nh, nkv, hd))
    a = AttnArgs(n=n, nh=nh, nkv=nkv, hd=hd, max_ctx=ctx, q=b["q"].ptr, scale=np.float32(1 / np.sqrt(hd)),
                 kc=b["kc"].ptr, vc=b["vc"].ptr, pos=b["pos"].ptr, o=b["o"].ptr, kv_dtype=KV_I8)
    dev.graph_begin()
    dev.attn_tree(a, b["parent"].ptr, work.ptr)
    g = dev.graph_end()
    for pos, kind in ((0, "chain"), (488, "star"), (100, "random"), (31, "forest"), (0, "random")):
        parent = tree(rng, n, kind)
        dev.upload(b["parent"], parent)
        dev.upload(b["pos"], np.array([pos], np.int32))
        dev.graph_launch(g)
        dev.sync()
        assert_bits_equal(b["o"].numpy(), run(dev, q, kc, vc, parent, pos, shape, KV_I8), f"replay {pos}")
    dev.graph_destroy(g)


def prep_args(dev, host, n, nh, nkv, hd, rot, ctx, kv, pos):
    b = {k: dev.to_device(v) for k, v in host.items()}
    b["pos"] = dev.to_device(np.array([pos], np.int32))
    return b, AttnArgs(n, nh, nkv, hd, rot, ctx, b["q"].ptr, b["k_in"].ptr, b["v_in"].ptr, b["q_norm"].ptr,
                       b["k_norm"].ptr, 1e-6, np.float32(1 / np.sqrt(hd)), b["cos"].ptr, b["sin"].ptr, b["kc"].ptr,
                       b["vc"].ptr, b["pos"].ptr, 0, b["kc"].ptr, A8(None, None, None), None, kv)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("n,nh,nkv,hd,rot,pos", [(1, 8, 2, 256, 64, 0), (13, 6, 2, 128, 32, 40), (64, 4, 2, 64, 64, 130),
                                                 (5, 2, 1, 512, 128, 190), (20, 4, 1, 320, 64, 5)])
def test_prep_equals_the_chains(dev, kv, n, nh, nkv, hd, rot, pos):
    """Each node's query and cache rows equal those that nmx_attn_prep gives a token at the node's
    position, moved to the node's slot; the cache is untouched elsewhere, also where slots end."""
    print(f"[case] attn tree prep n={n} hd={hd} kv={kv}", flush=True)
    rng = np.random.default_rng(n + hd + kv)
    ctx = 200
    parent = tree(rng, n, "random")
    depth = ancestors(parent).sum(1) - 1
    ang = rng.uniform(0, 2 * np.pi, (ctx, rot // 2))
    zero, _ = encode(np.zeros((nkv, ctx, hd), np.float32), kv)
    host = dict(q=rng.standard_normal((n, nh, 2 * hd)).astype(np.float32),
                k_in=rng.standard_normal((n, nkv * hd)).astype(np.float32),
                v_in=rng.standard_normal((n, nkv * hd)).astype(np.float32),
                q_norm=rng.uniform(0.5, 1.5, hd).astype(np.float32), k_norm=rng.uniform(0.5, 1.5, hd).astype(np.float32),
                cos=np.cos(ang).astype(np.float32), sin=np.sin(ang).astype(np.float32), kc=zero, vc=zero)
    b, a = prep_args(dev, host, n, nh, nkv, hd, rot, ctx, kv, pos)
    par = dev.to_device(parent)
    dev.attn_tree_prep(a, par)
    dev.sync()
    got = {k: b[k].numpy() for k in ("q", "kc", "vc")}

    def rows(c):
        return c if kv != KV_I8 else c[:nkv * ctx * hd].reshape(nkv, ctx, hd)

    def scales(c):
        return c[nkv * ctx * hd:].view(np.float32).reshape(nkv, ctx)

    want = {k: host[k].copy() for k in ("q", "kc", "vc")}
    for t in range(n):   # one token at its own position
        one = dict(host, q=host["q"][t:t + 1], k_in=host["k_in"][t:t + 1], v_in=host["v_in"][t:t + 1])
        p = min(pos + depth[t], ctx - 1)
        ob, oa = prep_args(dev, one, 1, nh, nkv, hd, rot, ctx, kv, p)
        dev.attn_prep(oa)
        dev.sync()
        want["q"][t] = ob["q"].numpy()[0]
        if pos + t < ctx:
            for c in ("kc", "vc"):
                rows(want[c])[:, pos + t] = rows(ob[c].numpy())[:, p]
                if kv == KV_I8:
                    scales(want[c])[:, pos + t] = scales(ob[c].numpy())[:, p]
        for x in ob.values():
            x.free()
    for k in want:
        assert_bits_equal(got[k], want[k], k)
    for x in (*b.values(), par):
        x.free()


def test_work_bytes():
    from nibblemac_amd.nmx import load_library

    f = load_library().nmx_attn_tree_work_bytes
    for bad in ((0, 8, 2, 256), (65, 8, 2, 256), (1, 0, 1, 64), (1, 2, 0, 64), (1, 3, 2, 64), (1, 2, 4, 64), (1, 2, 2, 32),
                (1, 2, 2, 96), (1, 2, 2, 576), (1, 1025, 1, 64)):
        assert f(*bad) == 0, bad
    assert all(0 < f(n, 8, 2, 256) <= 160 << 20 for n in range(1, 65))


@pytest.mark.gpu
def test_refusals(dev):
    print("[case] attn tree refusals", flush=True)
    n, nh, nkv, hd, ctx = 4, 2, 1, 64, 32
    b = dict(q=dev.zeros((n, nh, 2 * hd), np.float32), kc=dev.zeros((nkv, ctx, hd), np.float32),
             vc=dev.zeros((nkv, ctx, hd), np.float32), o=dev.zeros((n, nh * hd), np.float32), pos=dev.zeros(1, np.int32),
             x=dev.zeros(n * nkv * hd, np.float32))
    par = dev.to_device(np.array([-1, 0, 0, 1], np.int32))
    work = dev.zeros(dev.attn_tree_work_bytes(n, nh, nkv, hd), np.uint8)
    good = dict(n=n, nh=nh, nkv=nkv, hd=hd, rot=0, max_ctx=ctx, q=b["q"].ptr, k_in=b["x"].ptr, v_in=b["x"].ptr,
                q_norm=b["x"].ptr, k_norm=b["x"].ptr, kc=b["kc"].ptr, vc=b["vc"].ptr, pos=b["pos"].ptr, o=b["o"].ptr)
    both = [dict(n=0), dict(n=65), dict(nh=0), dict(nkv=0), dict(nh=3, nkv=2), dict(hd=32), dict(hd=96), dict(hd=576),
            dict(max_ctx=0), dict(max_ctx=(1 << 20) + 1), dict(q=None), dict(kc=None), dict(vc=None), dict(pos=None),
            dict(kv_dtype=3), dict(kv_dtype=-1), dict(q=b["q"].ptr + 4), dict(kc=b["kc"].ptr + 8), dict(vc=b["kc"].ptr),
            dict(q=b["kc"].ptr)]
    for bad in both + [dict(o=None), dict(o=b["q"].ptr), dict(o=b["vc"].ptr), dict(a8=A8(b["x"].ptr, None, None))]:
        with pytest.raises(NmxError, match="nmx_attn_tree"):
            dev.attn_tree(AttnArgs(**{**good, **bad}), par, work)
    for w in (None, work.ptr + 8, b["q"].ptr, b["kc"].ptr, b["o"].ptr):
        with pytest.raises(NmxError, match="nmx_attn_tree"):
            dev.attn_tree(AttnArgs(**good), par, w)
    with pytest.raises(NmxError, match="nmx_attn_tree"):
        dev.attn_tree(AttnArgs(**good), None, work)
    for bad in both + [dict(rot=3), dict(rot=128), dict(rot=-2), dict(rot=32), dict(k_in=None), dict(v_in=None),
                       dict(q_norm=None), dict(k_norm=None)]:
        with pytest.raises(NmxError, match="nmx_attn_tree_prep"):
            dev.attn_tree_prep(AttnArgs(**{**good, **bad}), par)
    with pytest.raises(NmxError, match="nmx_attn_tree_prep"):
        dev.attn_tree_prep(AttnArgs(**good), None)
    assert dev.lib.nmx_attn_tree(dev.ctx, None, par.ptr, work.ptr) == -1
    assert dev.lib.nmx_attn_tree_prep(dev.ctx, None, par.ptr) == -1
    dev.sync()
    assert not b["o"].numpy().any() and not b["kc"].numpy().any()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("n,nh,nkv,hd,pos", [(1, 8, 1, 512, 9001), (23, 4, 1, 448, 12300), (1, 4, 2, 64, 20011), (3, 4, 2, 192, 20000),
                                             (20, 8, 2, 320, 5000), (2, 16, 2, 256, 13000)])
def test_several_tiles_to_a_part(dev, n, nh, nkv, hd, pos, kv):
    print(f"[case] attn tree tiles n={n} hd={hd} pos={pos} kv={kv}", flush=True)
    check(dev, np.random.default_rng(n + hd + kv), (n, nh, nkv, hd, pos + n + 3, kv, pos), poison=False)


@pytest.mark.gpu
def test_two_contexts_at_once(dev):
    """Two devices' streams with workspaces of their own, calls queued in turn without a wait."""
    print("[case] attn tree two streams", flush=True)
    rng = np.random.default_rng(31)
    n, nh, nkv, hd, ctx, pos = 19, 4, 2, 128, 2100, 2000
    shape = (n, nh, nkv, hd, ctx)
    other = Device(0)
    jobs = []
    for d, kv in ((dev, KV_F16), (other, KV_F32)):
        q, parent = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32), tree(rng, n, "random")
        (kc, _), (vc, _) = (make_cache(rng, kv, nkv, ctx, hd) for _ in range(2))
        want = run(d, q, kc, vc, parent, pos, shape, kv)
        b = [d.to_device(x) for x in (q, kc, vc, parent, np.array([pos], np.int32))]
        outs = [d.zeros((n, nh * hd), np.float32) for _ in range(6)]
        w = d.alloc(d.attn_tree_work_bytes(n, nh, nkv, hd))
        d.sync()
        jobs.append((d, kv, b, outs, w, want))
    for r in range(6):
        for d, kv, b, outs, w, _ in jobs:
            a = AttnArgs(n=n, nh=nh, nkv=nkv, hd=hd, max_ctx=ctx, q=b[0].ptr, scale=np.float32(1 / np.sqrt(hd)), kc=b[1].ptr,
                         vc=b[2].ptr, pos=b[4].ptr, o=outs[r].ptr, a8=A8(None, None, None), kv_dtype=kv)
            d.attn_tree(a, b[3].ptr, w.ptr)
    for d, _, _, outs, _, want in jobs:
        d.sync()
        for o in outs:
            assert_bits_equal(o.numpy(), want, "beside another stream's calls")
    other.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kv,nkv,hd", [(KV_F32, 5, 256), (KV_F16, 5, 512), (KV_I8, 9, 512)])
def test_offsets_past_32_bits(dev, kv, nkv, hd):
    """Caches of more than 4 GiB: zeros but for a few rows of each head, which hold their query's
    direction at scores near the logarithm of the positions; then the commit's move in the same caches."""
    print(f"[case] attn tree long caches kv={kv}", flush=True)
    rng = np.random.default_rng(41 + kv)
    ctx, n = 1 << 20, 3
    pos, parent = ctx - 7, np.array([-1, 0, 0], np.int32)
    size = {KV_F32: 4, KV_F16: 2, KV_I8: 1}[kv]
    total = nkv * ctx * hd * size + (nkv * ctx * 4 if kv == KV_I8 else 0)
    assert nkv * ctx * hd * size > 1 << 32
    caches = [dev.zeros(total, np.uint8) for _ in range(2)]

    def move(b, g, slot, codes, scale, up):
        """a row to (up) or from the cache"""
        f = dev.lib.nmx_upload if up else dev.lib.nmx_download
        for arr, off in ((codes, ((g * ctx) + slot) * hd * size), (scale, nkv * ctx * hd + (g * ctx + slot) * 4)):
            if arr is not None:
                dev.check(f(dev.ctx, *((b.ptr + off, arr.ctypes.data) if up else (arr.ctypes.data, b.ptr + off)), arr.nbytes))

    def parts(enc):
        return (enc[:hd].copy(), enc[hd:].copy()) if kv == KV_I8 else (enc.ravel().copy(), None)

    q = rng.standard_normal((n, nkv, 2 * hd)).astype(np.float32)
    scale = float(np.float32(1 / np.sqrt(hd)))
    slots = [3, 777777, pos - 1, pos, pos + 1, pos + 2]
    want, tol, rows = np.zeros((n, nkv, hd)), 0.0, {}
    for g in range(nkv):
        K, V = [], []
        for i, s in enumerate(slots):
            toward = q[i % n, g, :hd].astype(np.float64)
            k = (toward * rng.uniform(12, 15) / (toward @ toward * scale)).astype(np.float32)
            for b, x, out in ((caches[0], k, K), (caches[1], rng.standard_normal(hd).astype(np.float32), V)):
                enc, val = encode(x[None, None], kv)
                codes, sc = parts(enc)
                move(b, g, s, codes, sc, True)
                out.append(val[0, 0])
                rows[b.ptr, g, s] = codes, sc
        K, V = np.array(K), np.array(V)
        for t in range(n):
            at = [0, 1, 2] + [3 + a for a in range(n) if a == t or a == 0]
            qt = q[t, g, :hd].astype(np.float64)
            s = K[at] @ qt * scale
            w = np.exp(s)
            want[t, g] = w @ V[at] / (w.sum() + pos - 3) / (1 + np.exp(-q[t, g, hd:].astype(np.float64)))
            ds = np.linalg.norm(qt) * np.linalg.norm(K, axis=1).max() * scale * (4 * 2.0 ** -22 + (hd / 32 + 8) * 2.0 ** -24)
            tol = max(tol, (2 * ds + 2.0 ** -18) * np.abs(V).max())
    i = dict(parent=dev.to_device(parent), pos=dev.to_device(np.array([pos], np.int32)), q=dev.to_device(q), o=dev.zeros((n, nkv * hd), np.float32),
             tok=dev.to_device(np.array([5, 6, 7], np.int32)), choice=dev.to_device(np.array([7, 0, 8], np.int32)), out=dev.zeros(n + 2, np.int32))
    work = dev.alloc(dev.attn_tree_work_bytes(n, nkv, nkv, hd))
    dev.attn_tree(AttnArgs(n=n, nh=nkv, nkv=nkv, hd=hd, max_ctx=ctx, q=i["q"].ptr, scale=np.float32(scale), kc=caches[0].ptr,
                           vc=caches[1].ptr, pos=i["pos"].ptr, o=i["o"].ptr, a8=A8(None, None, None), kv_dtype=kv), i["parent"], work)
    dev.sync()
    got = i["o"].numpy().reshape(n, nkv, hd)
    assert np.abs(got - want).max() <= tol, (np.abs(got - want).max(), tol)
    dev.tree_commit(tree_commit_args(n, i["parent"], i["tok"], i["choice"], i["out"],
                                     kv=dict(caches=caches, nkv=nkv, max_ctx=ctx, hd=hd, kv_dtype=kv, pos=i["pos"])))
    dev.sync()
    assert i["out"].numpy().tolist() == [1, 8, 0, 2, -1]
    for b in caches:
        for g in range(nkv):
            for s in (*slots[:4], pos + 1, pos + 2):
                codes, sc = (x if x is None else np.empty_like(x) for x in rows[b.ptr, g, s])
                move(b, g, s, codes, sc, False)
                for x, y in zip((codes, sc), rows[b.ptr, g, pos + 2 if s == pos + 1 else s]):
                    assert x is None or np.array_equal(x, y), (g, s)
    for b in (*caches, work, *i.values()):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_I8])
@pytest.mark.parametrize("n,nh,nkv,hd,pos", [(1, 2, 1, 64, 400), (6, 4, 2, 128, 400), (40, 4, 1, 256, 70), (5, 2, 1, 512, 9000)])
def test_zero_value_rows_beside_small_ones(dev, kv, n, nh, nkv, hd, pos):
    """Value rows of zeros (an int8 row's scale is 0) at the highest scores, the others small: a row of
    zeros says nothing about the magnitude of the rest."""
    print(f"[case] attn tree zero values n={n} hd={hd} kv={kv}", flush=True)
    for vstd in (1e-2, 1e-4, 1e-8, 1e-16, 1e-30):
        rng = np.random.default_rng(n + hd)
        shape = (n, nh, nkv, hd, pos + n)
        q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
        parent = tree(rng, n, "random")
        kc, K = make_cache(rng, kv, nkv, pos + n, hd)
        rows = (rng.standard_normal((nkv, pos + n, hd)) * vstd).astype(np.float32)
        for g in range(nkv):    # a third of the rows, the highest score of every query row among them
            s = q[:, g * (nh // nkv):(g + 1) * (nh // nkv), :hd].reshape(-1, hd) @ K[g].T.astype(np.float32)
            rows[g, s.argmax(1)] = 0
            rows[g, rng.random(pos + n) < 0.3] = 0
        vc, V = encode(rows, kv)
        want, tol = reference(q, K, V, parent, pos, shape)
        assert tol < 1e-3 * np.abs(V).max()
        got = run(dev, q, kc, vc, parent, pos, shape, kv)
        assert np.abs(got - want).max() <= tol, (vstd, np.abs(got - want).max(), tol)


@pytest.mark.gpu
def test_outputs_inside_inputs_are_refused(dev):
    """The position, the tree, the A8 and the prep's inputs against everything that is written."""
    print("[case] attn tree overlaps", flush=True)
    n, nh, nkv, hd, ctx, rot = 4, 2, 1, 64, 32, 32
    f = dict(q=(n, nh, 2 * hd), kc=(nkv, ctx, hd), vc=(nkv, ctx, hd), o=(n, nh * hd), ki=(n, hd), vi=(n, hd), qn=hd, kn=hd, cos=(ctx, rot // 2),
             sin=(ctx, rot // 2), ad=n * nh * hd // 32, afs=n * nh * hd // 32, aq=n * nh * hd // 4)
    b = {k: dev.zeros(s, np.float32) for k, s in f.items()}
    b["pos"], b["par"] = dev.zeros(1, np.int32), dev.to_device(np.array([-1, 0, 0, 1], np.int32))
    b["work"] = dev.zeros(dev.attn_tree_work_bytes(n, nh, nkv, hd), np.uint8)
    p = {k: v.ptr for k, v in b.items()}
    good = dict(n=n, nh=nh, nkv=nkv, hd=hd, rot=rot, max_ctx=ctx, q=p["q"], k_in=p["ki"], v_in=p["vi"], q_norm=p["qn"], k_norm=p["kn"],
                rope_cos=p["cos"], rope_sin=p["sin"], kc=p["kc"], vc=p["vc"], pos=p["pos"], o=p["o"], a8=A8(p["aq"], p["ad"], p["afs"]))

    def refused(call, name, par=p["par"], **bad):
        with pytest.raises(NmxError, match=name):
            call(AttnArgs(**{**good, **bad}), par, *([p["work"]] if call == dev.attn_tree else []))

    for k in ("o", "aq", "ad", "afs", "work"):
        refused(dev.attn_tree, "nmx_attn_tree", par=p[k])
        refused(dev.attn_tree, "nmx_attn_tree", pos=p[k])
    for k in ("q", "kc", "vc", "o", "work", "pos", "par"):
        refused(dev.attn_tree, "nmx_attn_tree", a8=A8(p[k], p["ad"], p["afs"]))
        refused(dev.attn_tree, "nmx_attn_tree", a8=A8(p["aq"], p[k], p["afs"]))
        refused(dev.attn_tree, "nmx_attn_tree", a8=A8(p["aq"], p["ad"], p[k]))
    refused(dev.attn_tree, "nmx_attn_tree", a8=A8(p["aq"], p["afs"], p["afs"]))
    refused(dev.attn_tree, "nmx_attn_tree", a8=A8(p["aq"], p["aq"], p["afs"]))
    for k in ("q", "kc", "vc"):
        refused(dev.attn_tree_prep, "nmx_attn_tree_prep", par=p[k])
        for what in ("pos", "k_in", "v_in", "q_norm", "k_norm", "rope_cos", "rope_sin"):
            refused(dev.attn_tree_prep, "nmx_attn_tree_prep", **{what: p[k]})
    dev.sync()
    assert not any(b[k].numpy().any() for k in b if k != "par")
    dev.attn_tree_prep(AttnArgs(**good), p["par"])      # and as they are: accepted
    dev.attn_tree(AttnArgs(**good), p["par"], p["work"])
    dev.sync()
    for x in b.values():
        x.free()


def held(x):
    """What is left of rows of x without the low halves: 11 bits of each element."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 2048), e - 11)


def off_grid(rng, shape):
    """Values in [1, 2) that lie 0.45 of a step above what 11 bits hold."""
    return (1 + (rng.integers(0, 1023, shape) + 0.45) / 1024).astype(np.float32)


def on_grid(rng, shape):
    return (1 + rng.integers(0, 1023, shape) / 1024).astype(np.float32)


def attend(q, K, V, parent, pos, shape, kv, less=""):
    """64-bit attention of every node and what each element may be off by. less: the context's part with the
    low halves of q, k, w (the weights) or v left out, mistakes to be noticed.

    Per context position: q's and an fp32 row's elements are two binary16 parts, the low one rounded (2^-22
    of the element), low times low left out (2^-22 more); a matrix instruction adds 32 products
    and drops from each what lies below 2^-26 of the sum, then rounds (2^-23): 1.25 2^-21 of the sum of
    magnitudes for each of the hd / 32 times 2 (fp32 rows 3) chained ones. The score is rounded 5 times on its
    way to the exponential, which adds 2^-23 and 2^-24 of its distance to the maximum. These errors move o by p |v -
    o|. The weights have 21 bits (the first part towards zero) and their low part times fp32 values' low part
    is left out: 2^-21, fp32 values 2^-22 + 2^-21 more; a tile adds 2 (3) instructions' 1.25 2^-21 and a
    rescale of 2^-23, the join at most 64 roundings, quotient and gate 2^-21: these move o by p |v|. What is
    below 2^-24 of the largest scaled part is lost: 2^-36 of the row's, or tile's, largest for each term."""
    n, nh, nkv, hd, ctx = shape
    u22 = 2.0 ** -22
    f32, hp = kv == KV_F32, 64 if hd <= 64 else 128 if hd <= 128 else 256 if hd <= 256 else 512
    mfma = 1.25 * 2.0 ** -21
    tiles = -(-pos // 32)
    halves, mt = (2, 4) if hp == 512 else (1, 8)
    splits = max(1, min(256, 256 // (nkv * (-(-(-(-n * (nh // nkv) // 16)) // mt)) * halves)))
    T = -(-tiles // splits)
    seen, scale = ancestors(parent), float(np.float32(1 / np.sqrt(hd)))
    o, tol = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    for t in range(n):
        at = np.concatenate([np.arange(pos), pos + np.flatnonzero(seen[t])])
        c = np.arange(len(at)) < pos
        for h in range(nh):
            g = h // (nh // nkv)
            x, k, v = q[t, h, :hd].astype(np.float64), K[g, at], V[g, at]
            s = np.where(c, (held(k) if "k" in less else k) @ (held(x) if "q" in less else x), k @ x) * scale
            w = np.exp(s - s.max())
            wv = w
            if "w" in less:     # towards zero, of the weight times an int8 row's scale
                f = np.abs(v).max(1) / 127 if kv == KV_I8 else np.ones(len(at))
                m, e = np.frexp(w * f)
                wv = np.where(c, np.ldexp(np.floor(m * 2048), e - 11) / f, w)
            y = np.where(c[:, None], held(v), v) if "v" in less else v
            out = wv @ y / w.sum()
            gate = 1 / (1 + np.exp(-q[t, h, hd:].astype(np.float64)))
            o[t, h] = out * gate
            mag = np.abs(k) @ np.abs(x)
            ds = scale * (mag * ((3 if f32 else 1) * u22 + hp / 32 * (3 if f32 else 2) * mfma) +
                          2.0 ** -36 * (np.abs(x).max() * np.abs(k).sum(1) + np.abs(x).sum() * np.abs(k).max(1)))
            p = w / w.sum()
            e1 = ds + 5 * 2.0 ** -24 * np.abs(s) + 2.0 ** -23 + 2.0 ** -24 * np.abs(s - s.max())
            e2 = 2 * u22 + (3 * u22 if f32 else 0) + T * ((3 if f32 else 2) * mfma + 2.0 ** -23) + 64 * 2.0 ** -24 + 2 * u22
            lost = len(at) * 2.0 ** -36 * (p * np.abs(v).max(1)).max()
            tol[t, h] = ((p * e1) @ np.abs(v - out) + e2 * (p @ np.abs(v)) + lost) * gate
    return o.reshape(n, nh * hd), tol.reshape(n, nh * hd)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("n,nh,nkv,hd,pos", [(1, 2, 1, 64, 150), (9, 4, 2, 128, 333), (5, 4, 1, 192, 95), (1, 8, 2, 256, 3000), (64, 4, 1, 256, 200),
                                             (7, 4, 2, 320, 130), (6, 4, 1, 512, 250), (33, 2, 1, 512, 64)])
def test_every_operand_is_held_to_22_bits(dev, n, nh, nkv, hd, pos, kv):
    """Inputs whose 11-bit halves are all off to the same side: leaving out the low half of the queries, of
    fp32 keys, of the weights or of fp32 values moves o by far more than what it may be off by."""
    print(f"[case] attn tree parts n={n} hd={hd} kv={kv}", flush=True)
    rng = np.random.default_rng(n + hd + kv)
    ctx, shape, rep = pos + n, (n, nh, nkv, hd, pos + n), nh // nkv
    parent, half, scale = tree(rng, n, "random"), hd // 2, 1 / np.sqrt(hd)
    sign = np.where(rng.random((nkv, hd)) < 0.5, -1, 1).astype(np.float32)
    q = np.empty((n, nh, 2 * hd), np.float32)
    q[..., :half], q[..., half:hd] = off_grid(rng, (n, nh, half)), on_grid(rng, (n, nh, hd - half))
    q[..., :hd] *= sign.repeat(rep, 0)
    q[..., hd:] = rng.standard_normal((n, nh, hd))

    def device_and_bounds(k, v, *less):
        (kc, K), (vc, V) = encode(k, kv), encode(v, kv)
        want, tol = attend(q, K, V, parent, pos, shape, kv)
        for part in less:
            off = np.abs(attend(q, K, V, parent, pos, shape, kv, part)[0] - want)
            assert (off > 2 * tol).any(), (part, (off / tol).max())
        got = run(dev, q, kc, vc, parent, pos, shape, kv)
        assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()

    # scores about 12: of one half of the positions from the columns where q is off the grid, of the other from
    # those where (fp32) k is; values of +-1 by half
    first = rng.random((nkv, ctx)) < 0.5
    cols = np.where(first[..., None], np.arange(hd) < half, np.arange(hd) >= half)
    size = np.float32(12 / (scale * 1.5 * half))
    top = np.float32(2.0 ** np.floor(np.log2(size)))    # a power of two: the grid's steps stay where they are
    lift = (1 + rng.integers(0, 64, (nkv, ctx, 1)) / 1024).astype(np.float32)
    k = np.where(first[..., None], lift, lift + np.float32(0.45 / 1024) if kv == KV_F32 else lift) * top * cols * sign[:, None]
    v = np.where(first, 1, -1)[..., None] * on_grid(rng, (nkv, ctx, hd))
    device_and_bounds(k.astype(np.float32), v.astype(np.float32), *("qk" if kv == KV_F32 else "q"))
    # weights of all sizes, values above 0
    k = rng.standard_normal((nkv, ctx, hd)).astype(np.float32) * np.float32(0.25)
    v = (off_grid if kv == KV_F32 else on_grid)(rng, (nkv, ctx, hd)) * np.float32(0.5)
    device_and_bounds(k, v, *("wv" if kv == KV_F32 else "w"))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("zero", ["queries", "keys", "values", "some_of_each"])
def test_rows_of_zeros(dev, kv, zero):
    """Zero queries or keys weigh every position alike; zero values give zeros."""
    print(f"[case] attn tree zeros {zero} kv={kv}", flush=True)
    rng = np.random.default_rng(17 + kv)
    n, nh, nkv, hd, ctx, pos = 10, 4, 2, 128, 300, 280
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    k, v = (rng.standard_normal((nkv, ctx, hd)).astype(np.float32) for _ in range(2))
    some = lambda x: x[..., 0] * 0 + (rng.random(x.shape[:-1]) < 0.5)  # noqa: E731
    if zero in ("queries", "some_of_each"):
        q[..., :hd] *= 0 if zero == "queries" else some(q)[..., None]
    if zero in ("keys", "some_of_each"):
        k *= 0 if zero == "keys" else some(k)[..., None]
    if zero in ("values", "some_of_each"):
        v *= 0 if zero == "values" else some(v)[..., None]
    parent = tree(rng, n, "random")
    (kc, K), (vc, V) = encode(k.astype(np.float32), kv), encode(v.astype(np.float32), kv)
    want, tol = reference(q, K, V, parent, pos, (n, nh, nkv, hd, ctx))
    got = run(dev, q, kc, vc, parent, pos, (n, nh, nkv, hd, ctx), kv)
    assert np.abs(got - want).max() <= tol
    if zero == "values":
        assert not got.any()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_I8])
@pytest.mark.parametrize("big", [1e18, 1e30, 1e-18, 1e-30])
def test_queries_and_keys_of_opposite_magnitudes(dev, kv, big):
    """Queries of 1e30 against keys of 1e-30 and the other way round: scores are ordinary."""
    print(f"[case] attn tree magnitudes {big} kv={kv}", flush=True)
    rng = np.random.default_rng(18 + kv)
    n, nh, nkv, hd, ctx, pos = 10, 4, 2, 128, 300, 280
    q = rng.standard_normal((n, nh, 2 * hd)).astype(np.float32)
    q[..., :hd] *= np.float32(big)
    kc, K = make_cache(rng, kv, nkv, ctx, hd, 1 / big)
    vc, V = make_cache(rng, kv, nkv, ctx, hd)
    parent = tree(rng, n, "random")
    want, tol = reference(q, K, V, parent, pos, (n, nh, nkv, hd, ctx))
    got = run(dev, q, kc, vc, parent, pos, (n, nh, nkv, hd, ctx), kv)
    assert np.abs(got - want).max() <= tol, (np.abs(got - want).max(), tol)
