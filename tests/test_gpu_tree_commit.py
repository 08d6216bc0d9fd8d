"""GPU: the commit of a verified tree (nmx_tree_commit) against a plain walk and copies, bit for bit;
and whole tree rounds against the chain calls that the accepted tokens would have taken."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import A8, AttnArgs, LinArgs, LinMixArgs, LinPreArgs, NmxError, SAMPLE_PARAMS, tree_commit_args
from tests.test_gpu_attn_tree import KV_F16, KV_F32, KV_I8, encode, tree
from tests.test_gpu_q4k import assert_bits_equal


def walk(parent, tok, choice):
    path = [0]
    while True:
        nxt = [t for t in range(len(tok)) if 0 <= parent[t] < t and parent[t] == path[-1] and tok[t] == choice[path[-1]]
               and choice[path[-1]] >= 0]
        if not nxt:
            return path
        path.append(nxt[0])


def rows_of(c, kv, nkv, ctx, hd):
    """Views of a cache's rows and scales."""
    if kv != KV_I8:
        return [c]
    return [c[:nkv * ctx * hd].reshape(nkv, ctx, hd), c[nkv * ctx * hd:].view(np.float32).reshape(nkv, ctx)]


def check(dev, rng, n, parent, tok, choice, kv, pos, ctx, layers=3, C=320, K=4, row=131, cap=None, caches=5, nkv=2, hd=64,
          pos_off=0, vt_is_tok=False):
    cap = cap or n
    host = dict(state=rng.standard_normal((layers, max(K - 1, 1), C)).astype(np.float32), xin=rng.standard_normal((layers, cap, C)).astype(np.float32),
                log=rng.standard_normal((layers, cap, row)).astype(np.float32), pend=rng.standard_normal((layers, cap, row)).astype(np.float32))
    kvh = [encode(rng.standard_normal((nkv, ctx, hd)).astype(np.float32), kv)[0] for _ in range(caches)]
    b = {k: dev.to_device(v) for k, v in host.items()}
    kvd = [dev.to_device(c) for c in kvh]
    ints = {k: dev.to_device(np.asarray(v, np.int32)) for k, v in (("parent", parent), ("tok", tok), ("choice", choice), ("out", [-9] * (3 + n)),
                                                                  ("ctl", [pos - pos_off] + [-9] * 15), ("vt", [-9, -9]))}
    vt = ints["tok"] if vt_is_tok else ints["vt"]
    lin = dict(layers=layers, C=C, conv_k=K, cap=cap, row=row, **b) if layers else None
    kvs = dict(caches=kvd, nkv=nkv, max_ctx=ctx, hd=hd, kv_dtype=kv, pos=ints["ctl"], pos_off=pos_off) if caches else None
    dev.tree_commit(tree_commit_args(n, ints["parent"], ints["tok"], ints["choice"], ints["out"], ctl=ints["ctl"], vt=vt, lin=lin, kv=kvs))
    dev.sync()
    path = walk(parent, tok, choice)
    e = len(path)
    out = ints["out"].numpy()
    assert out.tolist() == [e - 1, choice[path[-1]]] + path + [-1] * (n - e) + [-9], (out, path)
    ctl = ints["ctl"].numpy()
    assert ctl[0] == pos - pos_off and ctl[1] == ctl[2] == e and (ctl[3:] == -9).all()
    assert vt.numpy()[0] == choice[path[-1]] and (vt_is_tok or vt.numpy()[1] == -9)
    if layers:
        if K > 1:
            full = np.concatenate([host["state"], host["xin"][:, path]], 1)
            assert_bits_equal(b["state"].numpy(), np.ascontiguousarray(full[:, -(K - 1):]), "state")
        pend = host["pend"].copy()
        pend[:, :e] = host["log"][:, path]
        assert_bits_equal(b["pend"].numpy(), pend, "pend")
        for k in ("xin", "log"):
            assert_bits_equal(b[k].numpy(), host[k], k)
    for c, d in zip(kvh, kvd):
        want = c.copy()
        for x, y in zip(rows_of(c, kv, nkv, ctx, hd), rows_of(want, kv, nkv, ctx, hd)):
            for i, node in enumerate(path):
                if 0 <= pos + i and pos + node < ctx:
                    y[:, pos + i] = x[:, pos + node]
        assert_bits_equal(d.numpy(), want, "cache")
    for x in (*b.values(), *kvd, *ints.values()):
        x.free()
    return e


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("n", [1, 2, 9, 33, 64])
def test_against_plain_walk(dev, n, kv):
    print(f"[case] tree commit n={n} kv={kv}", flush=True)
    rng = np.random.default_rng(n + 100 * kv)
    longest = 0
    for kind in ("random", "chain", "star", "forest"):
        for few in (2, 3, 1000):     # few tokens: long paths and siblings of one token
            parent = tree(rng, n, kind)
            tok, choice = rng.integers(0, few, n).tolist(), rng.integers(0, few, n).tolist()
            longest = max(longest, check(dev, rng, n, parent, tok, choice, kv, int(rng.integers(0, 60)), 130, cap=n + n % 3))
    assert n < 9 or longest > 1
    # the whole chain, nothing at all
    assert check(dev, rng, n, tree(rng, n, "chain"), [5] * n, [5] * n, kv, 3, 70, hd=256, row=4112) == n
    assert check(dev, rng, n, tree(rng, n, "chain"), [5] * n, [6] * n, kv, 3, 70) == 1


@pytest.mark.gpu
def test_odd_calls(dev):
    print("[case] tree commit odd calls", flush=True)
    rng = np.random.default_rng(1)
    n = 12
    parent = tree(rng, n, "random")
    tok, choice = rng.integers(0, 2, n).tolist(), rng.integers(0, 2, n).tolist()
    args = (dev, rng, n, parent, tok, choice, KV_I8, 20, 64)
    check(*args, layers=0)
    check(*args, caches=0)
    check(*args, layers=0, caches=0, vt_is_tok=True)
    check(*args, K=1)
    check(*args, K=8, C=33, row=1, caches=64, nkv=1)
    check(*args, pos_off=-4)
    for pos in (-5, 55, 64, 100):    # nodes without a slot
        check(dev, rng, n, parent, tok, choice, KV_F32, pos, 64)
    check(dev, rng, n, parent, [-1] * n, [-1] * n, KV_F32, 5, 64)            # negative choices accept nothing
    check(dev, rng, 6, [3, 0, 2, -1, 99, 4], [1] * 6, [1] * 6, KV_F32, 5, 64)  # parents outside their range


@pytest.mark.gpu
def test_refusals(dev):
    print("[case] tree commit refusals", flush=True)
    n = 4
    i = {k: dev.zeros(32, np.int32) for k in ("parent", "tok", "choice", "out", "ctl", "vt")}
    f = {k: dev.zeros(4096, np.float32) for k in ("state", "xin", "log", "pend")}
    kv = [dev.zeros((1, 16, 64), np.float32) for _ in range(2)]
    lin = dict(layers=1, C=32, conv_k=4, cap=4, row=33, **f)
    kvs = dict(caches=kv, nkv=1, max_ctx=16, hd=64, kv_dtype=0, pos=i["ctl"])

    def call(lin_=None, kv_=None, **ch):
        g = {**dict(n=n, parent=i["parent"], tok=i["tok"], choice=i["choice"], out=i["out"], ctl=i["ctl"], vt=i["vt"]), **ch}
        dev.tree_commit(tree_commit_args(g["n"], g["parent"], g["tok"], g["choice"], g["out"], ctl=g["ctl"], vt=g["vt"],
                                         lin={**lin, **(lin_ or {})}, kv={**kvs, **(kv_ or {})}))

    bad = [dict(n=0), dict(n=65), dict(parent=None), dict(tok=None), dict(choice=None), dict(out=None), dict(out=i["tok"]),
           dict(out=i["ctl"]), dict(vt=i["choice"]), dict(vt=i["tok"].ptr + 4), dict(vt=i["out"]), dict(ctl=i["parent"])]
    bad += [dict(lin_=x) for x in (dict(layers=-1), dict(layers=1025), dict(C=0), dict(conv_k=0), dict(conv_k=9), dict(cap=3),
                                   dict(row=0), dict(log=None), dict(pend=None), dict(state=None), dict(xin=None),
                                   dict(pend=f["log"]), dict(state=f["xin"]), dict(state=f["pend"]))]
    bad += [dict(kv_=x) for x in (dict(caches=kv * 33), dict(nkv=0), dict(max_ctx=0), dict(hd=32), dict(hd=96), dict(hd=1024),
                                  dict(kv_dtype=3), dict(pos=None), dict(caches=[kv[0], None]), dict(caches=[kv[0], kv[0]]),
                                  dict(caches=[kv[0].ptr + 2]))]
    for b in bad:
        with pytest.raises(NmxError, match="nmx_tree_commit"):
            call(**b)
    a = tree_commit_args(n, i["parent"], i["tok"], i["choice"], i["out"], kv=kvs)
    a.kv = None
    with pytest.raises(NmxError, match="nmx_tree_commit"):
        dev.tree_commit(a)
    assert dev.lib.nmx_tree_commit(dev.ctx, None) == -1
    dev.sync()
    assert not any(x.numpy().any() for x in (*i.values(), *f.values(), *kv))


# ---- whole rounds --------------------------------------------------------------------------
class Layer:
    """One DeltaNet layer and one attention layer behind fixed projections of token embeddings, and a
    head: every piece of a tree round, with the products in numpy (they are not what is tested)."""

    def __init__(self, dev, rng, kv):
        self.dev, self.kv = dev, kv
        self.heads, self.dk, self.dv, self.K, self.nh, self.nkv, self.hd, self.rot, self.ctx, self.vocab = 2, 64, 64, 4, 4, 2, 64, 32, 160, 40
        self.C = 2 * self.heads * self.dk + self.heads * self.dv
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        h, V = self.heads, self.vocab
        self.emb = dict(raw=f(V, self.C), z=f(V, h * self.dv), b=f(V, h), a=f(V, h) - 2, q=f(V, self.nh * 2 * self.hd),
                        k=f(V, self.nkv * self.hd), v=f(V, self.nkv * self.hd))
        self.head = f(h * self.dv + self.nh * self.hd, V)
        ang = rng.uniform(0, 2 * np.pi, (self.ctx, self.rot // 2))
        one = {k: dev.to_device(v) for k, v in dict(
            conv_w=rng.uniform(-0.5, 0.5, (self.C, 4)).astype(np.float32), A_log=np.full(h, -1.2, np.float32), dt=np.full(h, -2, np.float32),
            norm=np.ones(self.dv, np.float32), qn=np.ones(self.hd, np.float32), kn=np.ones(self.hd, np.float32),
            cos=np.cos(ang).astype(np.float32), sin=np.sin(ang).astype(np.float32)).items()}
        self.w = one

    def state(self):
        d, zero = self.dev, encode(np.zeros((self.nkv, self.ctx, self.hd), np.float32), self.kv)[0]
        row = self.heads * (self.dk + self.dv + 1)
        return dict(conv=d.zeros((3, self.C), np.float32), rec=d.zeros(self.heads * self.dv * self.dk, np.float32), pend=d.zeros((16, row), np.float32),
                    kc=d.to_device(zero), vc=d.to_device(zero), ctl=d.zeros(16, np.int32), log=d.zeros((16, row), np.float32), xin=d.zeros((16, self.C), np.float32))

    def forward(self, s, tok, parent=None, keep_dev=True):
        """The rows [n] of (DeltaNet y | attention o) of a pass over tok at the state's position: a tree
        pass (parent), else a plain chain pass that advances the conv and recurrent states."""
        d, w, n = self.dev, self.w, len(tok)
        e = {k: d.to_device(np.ascontiguousarray(v[tok])) for k, v in self.emb.items()}
        t = {k: d.zeros(x, np.float32) for k, x in dict(cv=(n, self.C), beta=(n, self.heads), decay=(n, self.heads), o=(n, self.heads * self.dv),
                                                        y=(n, self.heads * self.dv), ao=(n, self.nh * self.hd), sc=(n, self.nh, self.ctx)).items()}
        vd = self.heads * self.dv
        tree_ = parent is not None
        pre = LinPreArgs(n, self.C, 4, self.dk, self.heads * self.dk, e["raw"].ptr, self.C, t["cv"].ptr, s["conv"].ptr, w["conv_w"].ptr,
                         s["xin"].ptr if tree_ else None, np.float32(self.dk ** -0.5), 1e-6, e["b"].ptr, e["a"].ptr, self.heads, self.heads,
                         w["A_log"].ptr, None, w["dt"].ptr, t["beta"].ptr, t["decay"].ptr)
        rule = LinArgs(n, self.heads, 1, self.dk, self.dv, self.C, vd, t["cv"].ptr, t["decay"].ptr, t["beta"].ptr, s["rec"].ptr, t["o"].ptr,
                       s["log"].ptr if tree_ else None, s["pend"].ptr, 16 if tree_ else 0, 0, s["ctl"].ptr + 8 if tree_ else None)
        mix = LinMixArgs(pre, rule, e["z"].ptr, vd, w["norm"].ptr, 1e-6, t["y"].ptr, vd, A8(None, None, None))
        at = AttnArgs(n, self.nh, self.nkv, self.hd, self.rot, self.ctx, e["q"].ptr, e["k"].ptr, e["v"].ptr, w["qn"].ptr, w["kn"].ptr, 1e-6,
                      np.float32(self.hd ** -0.5), w["cos"].ptr, w["sin"].ptr, s["kc"].ptr, s["vc"].ptr, s["ctl"].ptr, 0, t["ao"].ptr,
                      A8(None, None, None), t["sc"].ptr, self.kv)
        if tree_:
            par, work = d.to_device(parent), d.alloc(d.attn_tree_work_bytes(n, self.nh, self.nkv, self.hd))
            d.lin_mix_tree(mix, par)
            d.attn_tree_prep(at, par)
            d.attn_tree(at, par, work)
            self.par = par
        else:
            d.lin_mix(mix)
            d.attn_prep(at)
            d.attn(at)
        d.sync()
        out = np.concatenate([t["y"].numpy(), t["ao"].numpy()], 1)
        for x in (*e.values(), *t.values(), *([work] if tree_ else [])):
            x.free()
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
def test_rounds_equal_the_accepted_chain(dev, kv):
    """Eight rounds of tree drafts, verified by sampled tokens and committed, against the plain chain
    calls over the same tokens: the rows of every accepted node, the caches and the states. Rows agree
    to the two paths' 32-bit rounding; a cache row differs by no bit (the same prep), and the sampled
    tokens of a round equal those drawn from the chain's rows with the same uniform numbers."""
    print(f"[case] tree rounds kv={kv}", flush=True)
    rng = np.random.default_rng(20 + kv)
    L = Layer(dev, rng, kv)
    ts, cs = L.state(), L.state()
    cur, accepted = 3, 0
    for rnd in range(8):
        n = int(rng.integers(2, 16))
        parent = tree(rng, n, "random")
        tok = np.concatenate([[cur], rng.integers(0, L.vocab, n - 1)]).astype(np.int32)
        rows = L.forward(ts, tok, parent)
        # tokens sampled from each node's logits; one uniform number per depth, so a chain draws alike
        depth = np.array([0] * n)
        for t in range(1, n):
            depth[t] = depth[parent[t]] + 1
        u_depth = rng.random(n, np.float32)
        logits = (rows @ L.head).astype(np.float32)
        par = np.zeros(1, SAMPLE_PARAMS)
        par["temperature"], par["top_p"], par["top_k"] = 0.8, 0.95, 30
        b = [dev.to_device(x) for x in (logits, par, u_depth[depth], tok)]
        choice, work, out = dev.zeros(n, np.int32), dev.alloc(dev.sample_work_bytes(n, L.vocab)), dev.zeros(2 + n, np.int32)
        dev.sample(b[0], L.vocab, L.vocab, n, b[1], b[2], work, choice, per_row=False)
        dev.sync()
        # drafts as a good drafter would have made them, now that the choices are known: some children match
        ch = choice.numpy()
        if rnd % 2 == 0:
            for t in range(1, n):
                if t == np.flatnonzero(parent == parent[t])[0] and t < 9:
                    tok[t] = ch[parent[t]]
            # other tokens, other rows: the pass again over the tree with these drafts (the pending rows were
            # folded in already: keep is 0 now)
            dev.upload(ts["ctl"], np.array([ts["ctl"].numpy()[0], 0, 0] + [0] * 13, np.int32))
            rows = L.forward(ts, tok, parent)
            dev.upload(b[0], (rows @ L.head).astype(np.float32))
            dev.upload(b[3], tok)
            dev.sample(b[0], L.vocab, L.vocab, n, b[1], b[2], work, choice, per_row=False)
            dev.sync()
            ch = choice.numpy()
        dev.tree_commit(tree_commit_args(n, L.par, b[3], choice, out, ctl=ts["ctl"],
                                         lin=dict(layers=1, C=L.C, conv_k=4, state=ts["conv"], xin=ts["xin"], log=ts["log"], pend=ts["pend"], cap=16,
                                                  row=L.heads * (L.dk + L.dv + 1)),
                                         kv=dict(caches=[ts["kc"], ts["vc"]], nkv=L.nkv, max_ctx=L.ctx, hd=L.hd, kv_dtype=kv, pos=ts["ctl"])))
        dev.sync()
        path = walk(parent.tolist(), tok.tolist(), ch.tolist())
        e = len(path)
        accepted += e - 1
        assert out.numpy()[:2 + e].tolist() == [e - 1, ch[path[-1]]] + path
        # the chain: the accepted tokens through the plain calls
        want = L.forward(cs, tok[path])
        scale = np.abs(want).max()
        assert np.abs(rows[path] - want).max() <= 2e-4 * scale, np.abs(rows[path] - want).max()
        for i, node in enumerate(path):     # the draws
            lg = dev.to_device((want[i:i + 1] @ L.head).astype(np.float32))
            ud, tk = dev.to_device(u_depth[i:i + 1]), dev.zeros(1, np.int32)
            dev.sample(lg, L.vocab, L.vocab, 1, b[1], ud, work, tk)
            dev.sync()
            assert tk.numpy()[0] == ch[node]
            for x in (lg, ud, tk):
                x.free()
        pos = ts["ctl"].numpy()
        assert pos[1] == pos[2] == e
        dev.upload(ts["ctl"], np.array([pos[0] + e, 0, e] + [0] * 13, np.int32))
        dev.upload(cs["ctl"], np.array([pos[0] + e] + [0] * 15, np.int32))
        for k in ("kc", "vc"):
            for x, y in zip(*(rows_of(s[k].numpy(), kv, L.nkv, L.ctx, L.hd) for s in (ts, cs))):
                assert_bits_equal(np.ascontiguousarray(x[:, :pos[0] + e]), np.ascontiguousarray(y[:, :pos[0] + e]), f"{k} after round {rnd}")
        assert_bits_equal(ts["conv"].numpy(), cs["conv"].numpy(), "conv state")
        S = dev.to_device(ts["rec"].numpy())    # the tree's state with its pending rows folded in
        dev.lin_apply(S, ts["pend"], e, L.heads, L.dk, L.dv)
        dev.sync()
        ref = cs["rec"].numpy()
        assert np.abs(S.numpy() - ref).max() <= 2e-4 * max(np.abs(ref).max(), 1e-3)
        cur = int(ch[path[-1]])
        for x in (*b, choice, work, out, S, L.par):
            x.free()
    assert accepted >= 4


@pytest.mark.gpu
def test_position_among_the_outputs_is_refused(dev):
    print("[case] tree commit pos refusals", flush=True)
    n = 4
    i = {k: dev.zeros(32, np.int32) for k in ("parent", "tok", "choice", "out", "ctl", "vt")}
    kv = dev.zeros((1, 16, 64), np.float32)
    for pos in (i["out"].ptr, i["out"].ptr + 4 * (n + 1), i["vt"].ptr, i["ctl"].ptr + 4, i["ctl"].ptr + 8):
        with pytest.raises(NmxError, match="nmx_tree_commit"):
            dev.tree_commit(tree_commit_args(n, i["parent"], i["tok"], i["choice"], i["out"], ctl=i["ctl"], vt=i["vt"],
                                             kv=dict(caches=[kv], nkv=1, max_ctx=16, hd=64, kv_dtype=0, pos=pos)))
    dev.sync()
    assert not any(x.numpy().any() for x in (*i.values(), kv))


@pytest.mark.gpu
def test_captured_call(dev):
    """One captured commit, replayed over other choices and positions, against the eager call's check."""
    print("[case] tree commit graph", flush=True)
    rng = np.random.default_rng(21)
    n, ctx, nkv, hd, cap, C, row = 12, 64, 2, 64, 16, 96, 70
    parent = np.array([-1] + [int(rng.integers(0, t)) for t in range(1, n)], np.int32)
    i = dict(parent=dev.to_device(parent), tok=dev.zeros(n, np.int32), choice=dev.zeros(n, np.int32), out=dev.zeros(n + 2, np.int32),
             ctl=dev.zeros(16, np.int32))
    f = dict(state=dev.zeros((2, 3, C), np.float32), xin=dev.zeros((2, cap, C), np.float32), log=dev.zeros((2, cap, row), np.float32),
             pend=dev.zeros((2, cap, row), np.float32))
    kv = dev.zeros((nkv, ctx, hd), np.float32)
    a = tree_commit_args(n, i["parent"], i["tok"], i["choice"], i["out"], ctl=i["ctl"],
                         lin=dict(layers=2, C=C, conv_k=4, cap=cap, row=row, **f),
                         kv=dict(caches=[kv], nkv=nkv, max_ctx=ctx, hd=hd, kv_dtype=0, pos=i["ctl"]))

    def fill():
        tok = rng.integers(0, 3, n).astype(np.int32)
        x = {k: rng.standard_normal(b.numpy().shape).astype(np.float32) for k, b in (*f.items(), ("kv", kv))}
        new = dict(tok=tok, choice=rng.integers(0, 3, n).astype(np.int32), ctl=np.array([int(rng.integers(0, 40))] + [0] * 15, np.int32), **x)
        return new

    def put(new):
        for k, v in new.items():
            dev.upload(kv if k == "kv" else f[k] if k in f else i[k], v)

    def outputs():
        dev.sync()
        return [x.numpy() for x in (i["out"], i["ctl"], f["state"], f["pend"], kv)]

    dev.graph_begin()
    dev.tree_commit(a)
    g = dev.graph_end()
    for _ in range(4):
        new = fill()
        put(new)
        dev.graph_launch(g)
        got = outputs()
        put(new)
        dev.tree_commit(a)
        for x, y in zip(got, outputs()):
            assert_bits_equal(x, y, "replay")
    dev.graph_destroy(g)


@pytest.mark.gpu
def test_overlaps_are_refused(dev):
    """Everything that is written (out, ctl, vt, states, pending rows, caches) against everything else."""
    print("[case] tree commit overlaps", flush=True)
    n = 4
    i = {k: dev.zeros(32, np.int32) for k in ("parent", "tok", "choice", "out", "ctl", "vt")}
    f = {k: dev.zeros(4096, np.float32) for k in ("state", "xin", "log", "pend")}
    kv = [dev.zeros((1, 16, 64), np.float32) for _ in range(2)]
    lin = dict(layers=1, C=32, conv_k=4, cap=4, row=33, **f)
    kvs = dict(caches=kv, nkv=1, max_ctx=16, hd=64, kv_dtype=0, pos=i["ctl"])

    def call(lin_=None, kv_=None, **ch):
        g = {**dict(n=n, **i), **ch}
        dev.tree_commit(tree_commit_args(g["n"], g["parent"], g["tok"], g["choice"], g["out"], ctl=g["ctl"], vt=g["vt"],
                                         lin={**lin, **(lin_ or {})}, kv={**kvs, **(kv_ or {})}))

    p = {k: v.ptr for k, v in {**i, **f, "kv0": kv[0], "kv1": kv[1]}.items()}
    arrays = ("state", "xin", "log", "pend", "kv0", "kv1")
    bad = [{k: p[a]} for k in ("out", "vt", "ctl") for a in arrays]
    bad += [{k: p[a]} for k in ("parent", "tok", "choice") for a in ("state", "pend", "kv0", "kv1")]
    bad += [dict(vt=p["ctl"] + 4), dict(vt=p["ctl"] + 8), dict(vt=p["ctl"]), dict(ctl=p["vt"] - 4), dict(vt=p["out"] + 4)]
    bad += [dict(kv_=dict(pos=p[a])) for a in ("state", "pend", "kv0", "kv1")]
    bad += [dict(lin_={k: p[a]}) for k in ("state", "pend", "log", "xin") for a in ("kv0", "kv1")]
    bad += [dict(lin_={k: p[a]}) for k in ("state", "pend") for a in ("parent", "tok", "choice", "out", "vt", "ctl")]
    bad += [dict(lin_=dict(xin=p["pend"])), dict(kv_=dict(caches=[kv[0], kv[0]])), dict(kv_=dict(caches=[kv[0], f["pend"]])),
            dict(kv_=dict(caches=[i["out"]])), dict(kv_=dict(caches=[f["log"]]))]
    for b in bad:
        with pytest.raises(NmxError, match="nmx_tree_commit"):
            call(**b)
    dev.sync()
    assert not any(x.numpy().any() for x in (*i.values(), *f.values(), *kv))
    call()                                  # as they are, the tokens' own first as vt, no layers or caches
    call(vt=i["tok"])
    dev.tree_commit(tree_commit_args(n, i["parent"], i["tok"], i["choice"], i["out"], ctl=i["ctl"], vt=i["tok"]))
    dev.sync()
    for x in (*i.values(), *f.values(), *kv):
        x.free()
