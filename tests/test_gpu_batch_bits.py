"""Attention of a batch holds its operands to 22 bits of their rows' largest: queries, keys, values and weights whose
high parts (11 bits) leave rests of one sign, so that a part that is left out moves the result by 2^-12 of it, many times
the tolerance of the definition's test. That it would is shown on the CPU, by a model of the products of parts."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_attn_batch import KV_F16, KV_F32, KV_I8, Case, attend, encode

OVER = 1 + 2.0 ** -12 - 2.0 ** -19     # nearest binary16: 1; the rest nearly half a step


def case(hd, kv, rows=(1, 7), ctx=(90, 70), nh=8, nkv=2):
    """Keys along one direction or against it, values of 1 with the key's sign in every other column, queries along it
    with scores from about -2 to 2, gates open."""
    rng = np.random.default_rng(hd + kv)
    c = Case(rng, list(rows), list(ctx), nh, nkv, hd, 16, kv)
    u = rng.choice([-1.0, 1.0], hd)
    shape = c.npages, nkv, c.page
    sign, size = rng.choice([-1.0, 1.0], shape), rng.choice([0.5, 1.0], shape)
    part = OVER if kv == KV_F32 else 1.0
    K = (sign * size)[..., None] * u * part
    V = np.where(np.arange(hd) % 2, sign[..., None], 1.0) * part
    (c.kb, c.K), (c.vb, c.V) = encode(K.astype(np.float32), kv), encode(V.astype(np.float32), kv)
    s = 2.0 ** np.round(np.log2(rng.uniform(0.5, 2, (c.n, nh, 1)) / np.sqrt(hd)))
    c.q[..., :hd] = s * u * OVER
    c.q[..., hd:] = 20 + rng.uniform(0, 1, (c.n, nh, hd))
    return c


KINDS = [(hd, kv) for hd in (64, 128, 192, 256, 320, 448, 512) for kv in (KV_F32, KV_F16, KV_I8)]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kv", KINDS)
def test_operands(dev, hd, kv):
    c = case(hd, kv)
    want, tol = c.reference()
    c.poison()
    err = np.abs(attend(dev, c, fill=np.nan) - want).max(1)
    assert (err <= tol).all(), (err, tol)


def parts(x, toward_zero=False):
    """(high, low) binary16 parts of numbers, scaled to a row's largest element below 2^12."""
    e = np.ceil(np.log2(np.abs(x).max(-1, keepdims=True) * (1 + 2.0 ** -30)))
    up = x * 2.0 ** (12 - e)
    hi = up.astype(np.float16).astype(np.float64)
    if toward_zero:
        over = np.abs(hi) > np.abs(up)
        hi = np.where(over, np.nextafter(hi.astype(np.float16), np.float16(0)).astype(np.float64), hi)
    lo = (up - hi).astype(np.float16).astype(np.float64)
    return hi * 2.0 ** (e - 12), lo * 2.0 ** (e - 12)


def model(c, without, few):
    """o from the products of parts, in 64 bits else; few: the product of few rows, which has weights and values in 32 bits."""
    o, scale = np.zeros((c.n, c.nh, c.hd)), float(np.float32(1 / np.sqrt(c.hd)))
    for s in range(len(c.rows)):
        at = np.arange(c.len[s])
        pg, off = c.table[s, at // c.page], at % c.page
        for i in range(c.rows[s]):
            see, t = c.ctx[s] + i + 1, c.row0[s] + i
            for h in range(c.nh):
                k, v = (x[pg[:see], h * c.nkv // c.nh, off[:see]] for x in (c.K, c.V))
                qh, ql = parts(c.q[t, h, :c.hd].astype(np.float64)[None])
                kh, kl = parts(k) if c.kv == KV_F32 else (k, 0 * k)
                vh, vl = parts(v) if c.kv == KV_F32 else (v, 0 * v)
                qh, ql = qh[0], ql[0]
                e = (kh @ qh + (0 if "query" in without else kh @ ql) + (0 if "keys" in without else kl @ qh)) * scale
                w = np.exp(e - e.max())
                wh, wl = (w, 0 * w) if few else (x[:, 0] for x in parts(w[:, None], True))
                y = wh @ vh + (0 if "weights" in without else wl @ vh) + (0 if "values" in without else wh @ vl)
                o[t, h] = y / w.sum() / (1 + np.exp(-c.q[t, h, c.hd:].astype(np.float64)))
    return o.reshape(c.n, -1)


@pytest.mark.parametrize("hd,kv", KINDS)
def test_a_part_left_out_would_show(hd, kv):
    """By all but the product of few fp32 rows, whose operands have no parts."""
    c = case(hd, kv)
    want, tol = c.reference()
    few = np.arange(c.n) < 1           # the first sequence's row
    off = lambda x, f: (np.abs(model(c, x, f) - want).max(1) / tol)  # noqa: E731
    for f in (True, False):
        assert (off((), f) <= 0.5).all()
    for part in ("query",) + (("keys", "values") if kv == KV_F32 else ()):
        assert (off((part,), False) > 3).all(), part
    assert (off(("weights",), False)[~few] > 3).all()
    if kv != KV_F32:
        assert (off(("query",), True)[few] > 3).all()
