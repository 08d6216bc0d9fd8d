"""GPU: sequences that are longer than their tables (nmx_attn_batch_prep, nmx_attn_batch). A row past the table is
turned at its own position and not stored, the rows before it stay as they are, and attention sees the positions that
the table holds."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import AttnArgs
from tests.test_gpu_attn_batch import KV_F16, KV_F32, KV_I8, Case, attend, block_bytes
from tests.test_gpu_q4k import assert_bits_equal

MOST = 2 ** 31 - 1


def shorten(c, lens):
    """The case with tables that end at the last page in use, and lengths of its own for the device."""
    c.table = np.ascontiguousarray(c.table[:, :-1])
    c.room = c.table.shape[1] * c.page
    c.ctx = np.minimum(np.asarray(lens, np.int64) - c.rows, c.room)
    c.len = np.minimum(lens, c.room)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
def test_prep(dev, kv):
    """Rows that the table's end divides, lengths one past it and as long as a length can be."""
    rows, ctx, lens = [4, 1, 3, 2, 2], [60, 63, 61, 62, 10], [66, 65, 64, MOST, 12]
    nh, nkv, hd, rot, page, span = 4, 2, 128, 64, 16, 100
    rng = np.random.default_rng(kv)
    c = shorten(Case(rng, rows, ctx, nh, nkv, hd, page, kv), lens)
    assert c.room == 64
    n, h2 = c.n, rot // 2
    pos = np.concatenate([lens[s] - rows[s] + np.arange(rows[s]) for s in range(len(rows))])
    cos, sin = rng.uniform(-1, 1, (2, span, h2)).astype(np.float32)
    mixed = [t[np.minimum(pos, span - 1)] for t in (cos, sin)]
    k_in, v_in = rng.standard_normal((2, n, nkv * hd)).astype(np.float32)
    qn, kn = rng.uniform(0.5, 1.5, (2, hd)).astype(np.float32)
    up = {k: dev.to_device(v) for k, v in dict(k=k_in, v=v_in, qn=qn, kn=kn, cos=cos, sin=sin, mc=mixed[0], ms=mixed[1], q=c.q,
                                               pos=np.array([0], np.int32)).items()}
    flat = [dev.zeros((block_bytes(kv, nkv, n, hd),), np.uint8) for _ in range(2)]
    dev.attn_prep(AttnArgs(n=n, nh=nh, nkv=nkv, hd=hd, rot=rot, max_ctx=n, q=up["q"].ptr, k_in=up["k"].ptr, v_in=up["v"].ptr,
                           q_norm=up["qn"].ptr, k_norm=up["kn"].ptr, eps=1e-6, rope_cos=up["mc"].ptr, rope_sin=up["ms"].ptr,
                           kc=flat[0].ptr, vc=flat[1].ptr, pos=up["pos"].ptr, o=up["k"].ptr, kv_dtype=kv))
    d = c.upload(dev)
    dev.upload(d["len"], np.asarray(lens, np.int32))
    dev.attn_batch_prep(c.args(d, rot=rot, k_in=up["k"].ptr, v_in=up["v"].ptr, q_norm=up["qn"].ptr, k_norm=up["kn"].ptr, eps=1e-6,
                               rope_cos=up["cos"].ptr, rope_sin=up["sin"].ptr, rope_rows=span, axes=1))
    dev.sync()
    size = nkv * hd * (4, 2, 1)[kv]
    caches = []
    for name, was, chain in (("kc", c.kb, flat[0]), ("vc", c.vb, flat[1])):
        want, src = was.copy(), chain.numpy()
        for s in range(len(rows)):
            for t in range(c.row0[s], c.row0[s + 1]):
                if pos[t] >= c.room:
                    continue
                pg, off = c.table[s, pos[t] // page], pos[t] % page
                want[pg, :page * size].reshape(nkv, page, -1)[:, off] = src[:n * size].reshape(nkv, n, -1)[:, t]
                if kv == KV_I8:
                    want[pg, page * size:].reshape(nkv, page, 4)[:, off] = src[n * size:].reshape(nkv, n, 4)[:, t]
        caches.append((name, d[name].numpy(), want))
    got_q, want_q = d["q"].numpy(), up["q"].numpy()
    for x in (*d.values(), *up.values(), *flat):
        x.free()
    assert_bits_equal(got_q, want_q, "q")
    for name, got, want in caches:
        assert_bits_equal(got, want, name)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("rows,ctx,lens,nh,groups", [
    ([1, 2, 1, 2], [63, 62, 20, 62], [64, 66, 21, MOST], 8, ()),      # 4 to 8 query rows
    ([9, 1, 40], [55, 30, 24], [70, 31, 80], 8, ()),                  # many
    ([1, 1], [63, 63], [65, 90], 4, [(0, 64)]),                       # all that they see is shared: 4 query rows
    ([1, 2, 1], [63, 62, 63], [71, 70, MOST], 8, [(0, 64)]),          # and 16
    ([2, 1, 1], [62, 63, 40], [66, 65, 41], 8, [(0, 40), (2, 0)]),
])
def test_attention(dev, rows, ctx, lens, nh, groups, kv):
    c = shorten(Case(np.random.default_rng(len(rows) + kv), rows, ctx, nh, 2, 128, 16, kv, groups), lens)
    want, tol = c.reference()
    c.poison()
    c.len = np.asarray(lens)
    if groups and groups[0][1] == 64:
        c.shared[0] = MOST                 # no more than the table holds
    err = np.abs(attend(dev, c, fill=np.nan) - want).max(1)
    assert (err <= tol).all(), (err, tol)
