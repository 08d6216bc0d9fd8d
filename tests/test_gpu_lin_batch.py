"""GPU: the DeltaNet mixer over a batch of sequences (nmx_lin_mix_batch) against nmx_lin_mix on each sequence
alone: outputs, A8, conv states and recurrent states bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import A8, LinArgs, LinBatch, LinMixArgs, LinPreArgs, NmxError
from tests.batch_refuse import refuses
from tests.test_gpu_q4k import assert_bits_equal

K = 4
EPS = 1e-6


def make(rng, rows, heads, rep, dk, dv, pad=0):
    kd = heads // rep * dk
    C, n, S = 2 * kd + heads * dv, int(sum(rows)) + pad, len(rows)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return dict(rows=rows, n=n, heads=heads, rep=rep, dk=dk, dv=dv, kd=kd, C=C,
                t=dict(raw=f(n, C), z=f(n, heads * dv), b=f(n, heads), a=2 * f(n, heads), state=f(S, K - 1, C),
                       S=f(S, heads * dv * dk) * np.float32(0.05), conv_w=rng.uniform(-0.5, 0.5, (C, K)).astype(np.float32),
                       A_log=rng.uniform(np.log(0.2), np.log(0.4), heads).astype(np.float32),
                       dt_bias=rng.uniform(-4.5, -3.5, heads).astype(np.float32),
                       norm_w=rng.uniform(0.5, 1.5, dv).astype(np.float32)))


def structs(c, d, n, y, aq, state, S, raw=0, z=0, g=0):
    """LinMixArgs on rows from byte offsets raw, z, g on."""
    H, dk, dv, C = c["heads"], c["dk"], c["dv"], c["C"]
    pre = LinPreArgs(n=n, C=C, conv_k=K, dk=dk, kd=c["kd"], raw=d["raw"].ptr + raw, raw_stride=C, state=state,
                     conv_w=d["conv_w"].ptr, qscale=np.float32(1 / np.sqrt(dk)), l2eps=EPS, b_in=d["b"].ptr + g,
                     a_in=d["a"].ptr + g, g_stride=H, heads=H, A_log=d["A_log"].ptr, dt_bias=d["dt_bias"].ptr)
    rule = LinArgs(n=n, heads=H, rep=c["rep"], dk=dk, dv=dv, S=S)
    return LinMixArgs(pre, rule, d["z"].ptr + z, H * dv, d["norm_w"].ptr, EPS, y, H * dv,
                      A8(*[x.ptr for x in aq]) if aq else A8(None, None, None))


def batch(dev, c, src=None, a8=True, row0=None, most=None, graph=False):
    """The batch call's (y, A8 arrays, state, S); in place where src is None."""
    d = {k: dev.to_device(v) for k, v in c["t"].items()}
    n, S, H, dv = c["n"], len(c["rows"]), c["heads"], c["dv"]
    row0 = np.concatenate([[0], np.cumsum(c["rows"])]) if row0 is None else row0
    r0 = dev.to_device(np.asarray(row0, np.int32))
    y = dev.to_device(np.full((n, H * dv), 7, np.float32))
    nb = H * dv // 32
    aq = (dev.zeros((nb, n, 32), np.int8), dev.zeros((nb, n), np.float32), dev.zeros((nb, n), np.float32)) if a8 else ()
    out = [d["state"], d["S"]]
    sb = None
    if src is not None:
        sb = dev.to_device(np.asarray(src, np.int32))
        out = [dev.to_device(np.full(c["t"][k].shape, 9, np.float32)) for k in ("state", "S")]
    a = structs(c, d, n, y.ptr, aq, d["state"].ptr, d["S"].ptr)
    b = LinBatch(seqs=S, most=most or max(max(c["rows"]), 1), row0=r0.ptr, src=sb.ptr if sb else None,
                 state_out=out[0].ptr, S_out=out[1].ptr)
    dev.lin_mix_batch(a, b)
    dev.sync()
    got = dict(y=y.numpy(), state=out[0].numpy(), S=out[1].numpy(), aq=[x.numpy() for x in aq])
    for x in {id(v): v for v in [*d.values(), r0, y, *aq, *out] + ([sb] if sb else [])}.values():
        x.free()
    return got


def alone(dev, c, src=None, row0=None):
    """Each sequence by nmx_lin_mix."""
    H, dk, dv, C, n = c["heads"], c["dk"], c["dv"], c["C"], c["n"]
    row0 = np.concatenate([[0], np.cumsum(c["rows"])]) if row0 is None else row0
    y, nb = np.full((n, H * dv), 7, np.float32), H * dv // 32
    aq = [np.zeros((nb, n, 32), np.int8), np.zeros((nb, n), np.float32), np.zeros((nb, n), np.float32)]
    state, Sx = np.zeros_like(c["t"]["state"]), np.zeros_like(c["t"]["S"])
    d = {k: dev.to_device(v) for k, v in c["t"].items() if k not in ("state", "S")}
    for s in range(len(c["rows"])):
        f = s if src is None else src[s]
        ok = 0 <= f < len(c["rows"])
        st0 = c["t"]["state"][f] if ok else np.zeros_like(state[0])
        S0 = c["t"]["S"][f] if ok else np.zeros_like(Sx[0])
        m, r = c["rows"][s], int(row0[s])
        if m == 0:
            state[s], Sx[s] = st0, S0
            continue
        st, Sd, yd = dev.to_device(st0), dev.to_device(S0), dev.zeros((m, H * dv), np.float32)
        q = (dev.zeros((nb, m, 32), np.int8), dev.zeros((nb, m), np.float32), dev.zeros((nb, m), np.float32))
        tmp = [dev.zeros((m, C), np.float32), dev.zeros((m, H), np.float32), dev.zeros((m, H), np.float32),
               dev.zeros((m, H * dv), np.float32)]
        a = structs(c, d, m, yd.ptr, q, st.ptr, Sd.ptr, raw=4 * r * C, z=4 * r * H * dv, g=4 * r * H)
        a.pre.out, a.pre.beta, a.pre.decay = tmp[0].ptr, tmp[1].ptr, tmp[2].ptr
        a.rule.qkv, a.rule.qkv_stride, a.rule.beta, a.rule.decay = tmp[0].ptr, C, tmp[1].ptr, tmp[2].ptr
        a.rule.o, a.rule.o_stride = tmp[3].ptr, H * dv
        dev.lin_mix(a)
        dev.sync()
        state[s], Sx[s], y[r:r + m] = st.numpy(), Sd.numpy(), yd.numpy()
        for i, x in enumerate(q):
            aq[i][:, r:r + m] = x.numpy()
        for x in (st, Sd, yd, *q, *tmp):
            x.free()
    for x in d.values():
        x.free()
    return dict(y=y, state=state, S=Sx, aq=aq)


def same(got, want, rows=None):
    for k in ("y", "state", "S"):
        assert_bits_equal(got[k], want[k], k)
    for g, w, k in zip(got["aq"], want["aq"], ("codes", "d", "fs")):
        assert_bits_equal(g, w, k)


CASES = [
    # rows of each sequence, heads, rep, dk, dv, sources, rows past the last sequence
    ([1], 16, 1, 128, 128, None, 0),
    ([1] * 5, 16, 1, 128, 128, None, 0),
    ([1, 3, 0, 1, 9], 4, 1, 128, 128, None, 2),          # ragged, one waits, a padded batch
    ([1] * 7, 4, 1, 64, 64, [1, 0, 2, -1, 99, 0, 0], 0),  # two change places, two start, forks
    ([2, 0, 64, 5], 4, 1, 128, 128, [3, 2, 2, -1], 1),    # one that waits is forked too
    ([1, 2, 1], 4, 2, 64, 96, [2, 1, 0], 0),              # shared key heads
    ([17] * 3, 2, 1, 64, 128, [0, 0, 0], 0),
    ([1] * 256, 2, 1, 64, 64, None, 3),
    ([0], 1, 1, 64, 64, [-1], 1),                         # a new sequence that waits
    ([64] * 8, 1, 1, 128, 128, [7] * 8, 0),
    ([1, 2], 6, 3, 128, 128, [1, -1], 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_h{c[1]}r{c[2]}_{c[3]}_{c[4]}_{'fork' if c[5] else 'own'}")
def test_equals_each_sequence_alone(dev, case):
    rows, heads, rep, dk, dv, src, pad = case
    c = make(np.random.default_rng(len(rows) * 7 + heads + dk), rows, heads, rep, dk, dv, pad)
    same(batch(dev, c, src), alone(dev, c, src))


@pytest.mark.gpu
def test_y_alone_and_codes_alone(dev):
    c = make(np.random.default_rng(3), [1, 2, 1], 4, 1, 64, 64)
    want, got = alone(dev, c), batch(dev, c, a8=False)
    assert_bits_equal(got["y"], want["y"], "y")
    assert_bits_equal(got["S"], want["S"], "S")


@pytest.mark.gpu
def test_most_bounds_the_rows_of_a_sequence(dev):
    """A sequence with more rows than `most` is taken up to them; row0 outside [0, n] is the nearer end."""
    c = make(np.random.default_rng(4), [3, 1, 2], 4, 1, 64, 64)
    got = batch(dev, c, most=2, row0=[-5, 3, 4, 99])
    short = dict(c, rows=[2, 1, 2])
    want = alone(dev, short, row0=[0, 3, 4])
    assert (got["y"][2] == 7).all()
    same(got, want)


def test_refusals():
    H, dk, dv = 2, 64, 64
    C = H * (2 * dk + dv)
    p = iter(range(1 << 20, 1 << 30, 1 << 20))
    q = {k: next(p) for k in ("raw", "state", "conv_w", "b", "a", "A_log", "dt", "S", "z", "w", "y", "row0", "so", "So", "src")}

    def args(mix={}, pre={}, rule={}, bt={}, a8=()):
        pr = dict(n=3, C=C, conv_k=4, dk=dk, kd=H * dk, raw=q["raw"], raw_stride=C, state=q["state"], conv_w=q["conv_w"],
                  b_in=q["b"], a_in=q["a"], g_stride=H, heads=H, A_log=q["A_log"], dt_bias=q["dt"])
        ru = dict(n=3, heads=H, rep=1, dk=dk, dv=dv, S=q["S"])
        m = dict(z=q["z"], z_stride=H * dv, norm_w=q["w"], eps=EPS, y=q["y"], y_stride=H * dv)
        b = dict(seqs=3, most=1, row0=q["row0"], state_out=q["so"], S_out=q["So"])
        pr.update(pre), ru.update(rule), m.update(mix), b.update(bt)
        x = LinMixArgs(pre=LinPreArgs(**pr), rule=LinArgs(**ru), **m)
        x.a8 = A8(*a8) if a8 else A8(None, None, None)
        return x, LinBatch(**b)

    bad = [
        args(pre=dict(n=0), rule=dict(n=0)), args(pre=dict(n=513), rule=dict(n=513)), args(rule=dict(n=2)),
        args(bt=dict(seqs=0)), args(bt=dict(seqs=257)), args(bt=dict(most=0)), args(bt=dict(most=65)),
        args(pre=dict(conv_k=3)), args(pre=dict(dk=32), rule=dict(dk=32)), args(rule=dict(dv=48)), args(rule=dict(dv=160)),
        args(rule=dict(rep=0)), args(pre=dict(C=C + 32)), args(pre=dict(kd=64)), args(pre=dict(heads=3)),
        args(pre=dict(xin=q["src"])), args(rule=dict(log=q["src"])), args(rule=dict(keep=1)), args(rule=dict(log0=1)),
        args(pre=dict(raw_stride=C - 1)), args(pre=dict(g_stride=1)), args(mix=dict(z_stride=H * dv - 4)),
        args(mix=dict(z_stride=H * dv + 2)), args(mix=dict(y_stride=H * dv - 1)),
        args(mix=dict(z=q["z"] + 4)), args(mix=dict(norm_w=q["w"] + 4)), args(pre=dict(conv_w=q["conv_w"] + 8)),
        args(rule=dict(S=q["S"] + 4)), args(bt=dict(S_out=q["So"] + 4)),
        args(mix=dict(y=None)), args(a8=(q["src"], None, q["src"])),
        *[args(pre={k: None}) for k in ("raw", "state", "conv_w", "b_in", "a_in", "A_log", "dt_bias")],
        args(rule=dict(S=None)), args(mix=dict(z=None)), args(mix=dict(norm_w=None)),
        *[args(bt={k: None}) for k in ("row0", "state_out", "S_out")],
        # in place with sources; half in place; outputs over inputs and over each other
        args(bt=dict(state_out=q["state"], S_out=q["S"], src=q["src"])), args(bt=dict(S_out=q["S"])),
        args(bt=dict(S_out=q["S"] + 3 * H * dv * dk * 4 - 16)), args(mix=dict(y=q["z"])), args(mix=dict(y=q["So"])),
        args(mix=dict(y=q["row0"])), args(bt=dict(src=q["y"])),
        args(a8=(q["y"], q["src"], q["src"] + 4096)),
    ]
    for i, (m, b) in enumerate(bad):
        refuses("nmx_lin_mix_batch", i, m, b)
    shared = dict(rule=dict(heads=H, rep=2), pre=dict(kd=dk, C=2 * dk + H * dv, raw_stride=C))
    refuses("nmx_lin_mix_batch", "rep in place", *args(**shared, bt=dict(state_out=q["state"], S_out=q["S"])))
