"""GPU: steps of many requests as a program makes them, tables, DeltaNet states, caches, attention, a projection and its
adapters in one captured graph, against each sequence's own history: nmx_lin_mix on a state of its own (bit for bit),
nmx_attn_prep and nmx_attn over a contiguous cache of its own (within the batch form's rounding), the projection's
rows by nmx_q4k_matmul one at a time (bit for bit) and the adapters in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from nibblemac_amd.nmx import A8, AttnArgs, AttnBatchArgs, LinArgs, LinBatch, LinMixArgs, LinPreArgs, Pages, lora_args, pages_args
from tests.test_gpu_q4k import assert_bits_equal

S, MOST, N = 5, 4, 12                      # sequences, rows of one, rows of a step (a padded batch)
NH, NKV, HD, ROT, PAGE, CTX = 8, 2, 64, 32, 16, 96
H, DK, DV, K = 4, 64, 64, 4                # the DeltaNet layer
C = H * (2 * DK + DV)
OUT, RANK, ADAPTERS = 256, 8, 3
EPS = 1e-6
KV_F32 = 0

STEPS = [  # (sources, rows kept, rows of each): prompts, tokens, forks and an exchange, cut back drafts and an end, new ones
    ([-1] * 5, [0] * 5, [4, 3, 1, 0, 2]),
    ([0, 1, 2, 3, 4], [99] * 5, [1, 1, 4, 0, 1]),
    ([0, 0, 1, 0, 4], [99, 99, 99, 3, 99], [1, 1, 1, 1, 1]),
    ([1, 0, -1, 3, 4], [99, 99, 0, 2, 99], [2, 1, 0, 3, 1]),
    ([0, 1, 0, 3, -1], [99] * 5, [1, 1, 4, 2, 4]),
    ([0, 1, 2, 3, 4], [99] * 5, [1, 0, 3, 1, 1]),
]


def attn_chain(dev, hist, q, k, v, qn, kn, cos, sin, m):
    """The last m rows of a history of (k, v) rows through nmx_attn_prep and nmx_attn: (o, rotated q)."""
    n0 = len(hist) - m
    b = {x: dev.to_device(y) for x, y in dict(q=q, qn=qn, kn=kn, cos=cos, sin=sin).items()}
    kc, vc = (dev.zeros((NKV, CTX, HD), np.float32) for _ in range(2))
    sc, o = dev.zeros((64, NH, CTX), np.float32), dev.zeros((64, NH * HD), np.float32)
    dummy = dev.to_device(np.zeros((64, NH, 2 * HD), np.float32))

    def call(n, pos, qb, rows):
        kb, vb, pb = dev.to_device(rows[0]), dev.to_device(rows[1]), dev.to_device(np.array([pos], np.int32))
        a = AttnArgs(n=n, nh=NH, nkv=NKV, hd=HD, rot=ROT, max_ctx=CTX, q=qb.ptr, k_in=kb.ptr, v_in=vb.ptr, q_norm=b["qn"].ptr,
                     k_norm=b["kn"].ptr, eps=EPS, scale=np.float32(1 / np.sqrt(HD)), rope_cos=b["cos"].ptr, rope_sin=b["sin"].ptr,
                     kc=kc.ptr, vc=vc.ptr, pos=pb.ptr, o=o.ptr, a8=A8(None, None, None), scores=sc.ptr, kv_dtype=KV_F32)
        dev.attn_prep(a)
        return a, [kb, vb, pb]

    stack = lambda rows: [np.stack([r[i] for r in rows]).astype(np.float32) for i in (0, 1)]  # noqa: E731
    tmp = []
    if n0:
        tmp += call(n0, 0, dummy, stack(hist[:n0]))[1]
    a, t = call(m, n0, b["q"], stack(hist[n0:]))
    dev.attn(a)
    dev.sync()
    out = o.numpy()[:m]
    for x in (*b.values(), kc, vc, sc, o, dummy, *tmp, *t):
        x.free()
    return out


def lin_chain(dev, state, Sx, raw, z, g, a, w):
    """nmx_lin_mix over the rows from a conv state and a recurrent state: (y, state, S)."""
    m = len(raw)
    if not m:
        return np.zeros((0, H * DV), np.float32), state, Sx
    b = {x: dev.to_device(np.ascontiguousarray(y)) for x, y in dict(raw=raw, z=z, b=g, a=a, state=state, S=Sx, **w).items()}
    y = dev.zeros((m, H * DV), np.float32)
    pre = LinPreArgs(n=m, C=C, conv_k=K, dk=DK, kd=H * DK, raw=b["raw"].ptr, raw_stride=C, state=b["state"].ptr, conv_w=b["conv_w"].ptr,
                     qscale=np.float32(1 / np.sqrt(DK)), l2eps=EPS, b_in=b["b"].ptr, a_in=b["a"].ptr, g_stride=H, heads=H,
                     A_log=b["A_log"].ptr, dt_bias=b["dt_bias"].ptr)
    rule = LinArgs(n=m, heads=H, rep=1, dk=DK, dv=DV, S=b["S"].ptr)
    dev.lin_mix(LinMixArgs(pre, rule, b["z"].ptr, H * DV, b["norm_w"].ptr, EPS, y.ptr, H * DV, A8(None, None, None)))
    dev.sync()
    out = y.numpy(), b["state"].numpy(), b["S"].numpy()
    for x in (*b.values(), y):
        x.free()
    return out


@pytest.mark.gpu
def test_steps_of_many_requests(dev):
    rng = np.random.default_rng(3)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    lw = dict(conv_w=rng.uniform(-0.5, 0.5, (C, K)).astype(np.float32), A_log=rng.uniform(-1.5, -0.9, H).astype(np.float32),
              dt_bias=rng.uniform(-4.5, -3.5, H).astype(np.float32), norm_w=rng.uniform(0.5, 1.5, DV).astype(np.float32))
    angle = np.outer(np.arange(CTX), 1e4 ** (-np.arange(ROT // 2) / (ROT // 2)))
    aw = dict(qn=rng.uniform(0.5, 1.5, HD).astype(np.float32), kn=rng.uniform(0.5, 1.5, HD).astype(np.float32),
              cos=np.cos(angle).astype(np.float32), sin=np.sin(angle).astype(np.float32))
    W = oracle.q4k_quantize(f(OUT, NH * HD) * np.float32(0.02))
    A, B, scale = f(ADAPTERS, RANK, NH * HD) * np.float32(0.05), f(ADAPTERS, OUT, RANK), rng.uniform(0.5, 2, ADAPTERS).astype(np.float32)
    npages, wide, nb = S * CTX // PAGE, CTX // PAGE, NH * HD // 32
    i32 = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    d = {k: dev.to_device(v) for k, v in dict(
        table=i32(S, wide), len=i32(S), refs=i32(npages), src=i32(S), keep=i32(S), add=i32(S), out=i32(4), row0=i32(S + 1), ids=i32(N),
        q=f(N, NH, 2 * HD), k=f(N, NKV * HD), v=f(N, NKV * HD), kc=np.full((npages, NKV, PAGE, HD), np.nan, np.float32),
        vc=np.full((npages, NKV, PAGE, HD), np.nan, np.float32), o=f(N, NH * HD), aq=np.zeros((nb, N, 32), np.int8),
        ad=f(nb, N), afs=f(nb, N), W=W, A=A, B=B, scale=scale, Y=f(N, OUT), Y0=f(N, OUT), raw=f(N, C), z=f(N, H * DV), b=f(N, H), a=f(N, H),
        y=f(N, H * DV), state0=np.zeros((S, K - 1, C), np.float32), state1=np.zeros((S, K - 1, C), np.float32),
        S0=np.zeros((S, H * DV * DK), np.float32), S1=np.zeros((S, H * DV * DK), np.float32), **lw, **aw).items()}
    work = [dev.alloc(x) for x in (dev.pages_work_bytes(npages, S, wide), dev.attn_batch_work_bytes(N, S, 0, NH, NKV, HD),
                                   dev.lora_work_bytes(N, 1, RANK))]
    pages = Pages(seqs=S, npages=npages, page=PAGE, max_pages=wide, table=d["table"].ptr, len=d["len"].ptr, nkv=NKV, hd=HD, kv_dtype=KV_F32)
    pa = pages_args(pages, d["refs"], d["src"], d["keep"], d["add"], [d["kc"], d["vc"]], d["out"])
    aa = AttnBatchArgs(pages=pages, n=N, row0=d["row0"].ptr, nh=NH, rot=ROT, q=d["q"].ptr, k_in=d["k"].ptr, v_in=d["v"].ptr, q_norm=d["qn"].ptr,
                       k_norm=d["kn"].ptr, eps=EPS, scale=np.float32(1 / np.sqrt(HD)), rope_cos=d["cos"].ptr, rope_sin=d["sin"].ptr,
                       rope_rows=CTX, axes=1, kc=d["kc"].ptr, vc=d["vc"].ptr, o=d["o"].ptr, a8=A8(d["aq"].ptr, d["ad"].ptr, d["afs"].ptr))
    la = lora_args(N, NH * HD, d["o"], NH * HD, ADAPTERS, RANK, 0, d["ids"], d["scale"], [(OUT, d["A"], d["B"], d["Y"], OUT)])
    graphs = []
    for k in (0, 1):   # the states change hands from one buffer to the other
        pre = LinPreArgs(n=N, C=C, conv_k=K, dk=DK, kd=H * DK, raw=d["raw"].ptr, raw_stride=C, state=d[f"state{k}"].ptr,
                         conv_w=d["conv_w"].ptr, qscale=np.float32(1 / np.sqrt(DK)), l2eps=EPS, b_in=d["b"].ptr, a_in=d["a"].ptr, g_stride=H,
                         heads=H, A_log=d["A_log"].ptr, dt_bias=d["dt_bias"].ptr)
        mix = LinMixArgs(pre, LinArgs(n=N, heads=H, rep=1, dk=DK, dv=DV, S=d[f"S{k}"].ptr), d["z"].ptr, H * DV, d["norm_w"].ptr, EPS,
                         d["y"].ptr, H * DV, A8(None, None, None))
        bt = LinBatch(seqs=S, most=MOST, row0=d["row0"].ptr, src=d["src"].ptr, state_out=d[f"state{1 - k}"].ptr, S_out=d[f"S{1 - k}"].ptr)
        dev.graph_begin()
        dev.pages_update(pa, work[0])
        dev.lin_mix_batch(mix, bt)
        dev.attn_batch_prep(aa)
        dev.attn_batch(aa, work[1])
        dev.q4k_matmul(d["W"], OUT, NH * HD, N, d["aq"], d["ad"], d["afs"], d["Y"])
        dev.copy(d["Y0"], d["Y"], N * OUT * 4)
        dev.lora(la, work[2])
        graphs.append(dev.graph_end())
    hist, states = [[] for _ in range(S)], [(np.zeros((K - 1, C), np.float32), np.zeros(H * DV * DK, np.float32)) for _ in range(S)]
    for step, (src, keep, rows) in enumerate(STEPS):
        row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        x = dict(q=f(N, NH, 2 * HD), k=f(N, NKV * HD), v=f(N, NKV * HD), raw=f(N, C), z=f(N, H * DV), b=f(N, H), a=f(N, H),
                 ids=rng.integers(-1, ADAPTERS, N).astype(np.int32), src=np.array(src, np.int32), keep=np.array(keep, np.int32),
                 add=np.array(rows, np.int32), row0=row0, y=np.full((N, H * DV), 7, np.float32), o=np.full((N, NH * HD), 7, np.float32))
        for k, v in x.items():
            dev.upload(d[k], v)
        dev.graph_launch(graphs[step % 2])
        dev.sync()
        assert d["out"].numpy()[0] == 0
        old = hist
        hist = [list(old[s][:kp]) if s >= 0 else [] for s, kp in zip(src, keep)]
        # a sequence that keeps fewer rows than its source goes on from the source's state all the same: its program's to roll back
        states = [states[s] if s >= 0 else (np.zeros((K - 1, C), np.float32), np.zeros(H * DV * DK, np.float32)) for s in src]
        got = {k: d[k].numpy() for k in ("y", "o", "Y", "Y0", "aq", "ad", "afs")}
        live = int(row0[-1])
        assert (got["y"][live:] == 7).all() and (got["o"][live:] == 7).all()
        st, Sx = d[f"state{1 - step % 2}"].numpy(), d[f"S{1 - step % 2}"].numpy()
        for s in range(S):
            r = slice(int(row0[s]), int(row0[s + 1]))
            y, *states[s] = lin_chain(dev, *states[s], x["raw"][r], x["z"][r], x["b"][r], x["a"][r], lw)
            assert_bits_equal(got["y"][r], y, f"y of {s} at step {step}")
            assert_bits_equal(st[s], states[s][0], f"conv state of {s} at step {step}")
            assert_bits_equal(Sx[s], states[s][1], f"state of {s} at step {step}")
            hist[s] += list(zip(x["k"][r], x["v"][r]))
            if not rows[s]:
                continue
            want = attn_chain(dev, hist[s], x["q"][r], None, None, aw["qn"], aw["kn"], aw["cos"], aw["sin"], rows[s])
            # normed rows of 64: |q| |k| scale is at most 1.5^2 8; both sides are off by (16 + 10 + 64) 2^-24 of it at most, twice
            # that of the largest value (below 5), and 2^-18
            tol = (2 * 18 * 90 * 2.0 ** -24 + 2.0 ** -18) * 5 * 2
            assert np.abs(got["o"][r] - want).max() <= tol, (step, s)
        assert d["len"].numpy().tolist() == [len(h) for h in hist]
        dO, dq = dev.to_device(got["o"]), [dev.to_device(got[k]) for k in ("aq", "ad", "afs")]
        one = [dev.zeros((nb, 1, 32), np.int8), dev.zeros((nb, 1), np.float32), dev.zeros((nb, 1), np.float32)]
        Yr = dev.zeros((1, OUT), np.float32)
        for t in range(live):
            dev.quant_a8(dO.ptr + 4 * t * NH * HD, 1, NH * HD, *one)
            dev.q4k_matmul(d["W"], OUT, NH * HD, 1, *one, Yr)
            dev.sync()
            assert_bits_equal(got["Y0"][t], Yr.numpy()[0], f"projection of row {t}")
            m = x["ids"][t]
            if m < 0:
                assert_bits_equal(got["Y"][t], got["Y0"][t], "no adapter")
                continue
            o64, a64, b64 = got["o"][t].astype(np.float64), A[m].astype(np.float64), B[m].astype(np.float64)
            want = got["Y0"][t] + float(scale[m]) * (b64 @ (a64 @ o64))
            bound = 2.0 ** -24 * (scale[m] * (np.abs(b64) @ ((NH * HD / 16 + 48) * (np.abs(a64) @ np.abs(o64)))) + 4 * np.abs(want) + 4 * np.abs(got["Y0"][t]))
            assert (np.abs(got["Y"][t] - want) <= bound).all()
        for b in (dO, *dq, *one, Yr):
            b.free()
    for g in graphs:
        dev.graph_destroy(g)
    for b in (*d.values(), *work):
        b.free()
