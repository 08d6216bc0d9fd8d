"""GPU: rows of a padded batch behind the last sequence. Their memory is there, like that of all n rows; whatever it
holds, the other rows' results have the same bits and nothing of theirs is written."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import A8
from tests.test_gpu_attn_batch import KV_F16, KV_F32, KV_I8, Case
from tests.test_gpu_q4k import assert_bits_equal


def step(dev, c, q, k, v, where, tables, norms):
    """(q, kc, vc, o, codes, d, fs) after the prep and the attention of a batch."""
    live, nb, span = int(c.row0[-1]), c.nh * c.hd // 32, len(tables[0])
    d = c.upload(dev)
    up = [dev.to_device(x) for x in (k, v, where, *tables, *norms)]
    a8 = [dev.to_device(x) for x in (np.full((nb, c.n, 32), 7, np.int8), np.full((nb, c.n), 7, np.float32), np.full((nb, c.n), 7, np.float32))]
    w = c.work(dev)
    dev.upload(d["q"], q)
    a = c.args(d, [x.ptr for x in a8], rot=2 * tables[0].shape[1], k_in=up[0].ptr, v_in=up[1].ptr, rope_pos=up[2].ptr, rope_cos=up[3].ptr,
               rope_sin=up[4].ptr, q_norm=up[5].ptr, k_norm=up[6].ptr, eps=1e-6, rope_rows=span, axes=where.shape[1])
    dev.attn_batch_prep(a)
    dev.attn_batch(a, w)
    dev.sync()
    out = [d["q"].numpy(), d["kc"].numpy(), d["vc"].numpy(), d["o"].numpy(), *[x.numpy() for x in a8]]
    for x in (*d.values(), *up, *a8, w):
        x.free()
    assert (out[3][live:] == 7).all() and all((x[:, live:] == 7).all() for x in out[4:])
    assert_bits_equal(out[0][live:], q[live:], "q of the padding")
    return [out[0][:live], out[1], out[2], out[3][:live]] + [x[:, :live] for x in out[4:]]


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [KV_F32, KV_F16, KV_I8])
@pytest.mark.parametrize("rows,ctx,pad", [([1, 2, 0], [40, 17, 5], 1), ([1, 9, 1], [40, 3, 200], 70), ([30, 1, 100], [0, 300, 20], 200)])
def test_what_the_padding_holds_does_not_matter(dev, rows, ctx, pad, kv):
    """Few rows and many, whose parts are joined by workgroups and by waves."""
    nh, nkv, hd, span, axes = 8, 2, 128, 50, 3
    rng = np.random.default_rng(sum(rows) + kv)
    c = Case(rng, rows, ctx, nh, nkv, hd, 16, kv, pad=pad)
    live = int(c.row0[-1])
    k, v = rng.standard_normal((2, c.n, nkv * hd)).astype(np.float32)
    where = rng.integers(0, span, (c.n, axes)).astype(np.int32)
    tables, norms = rng.uniform(-1, 1, (2, span, 32)).astype(np.float32), rng.uniform(0.5, 1.5, (2, hd)).astype(np.float32)
    want = step(dev, c, c.q, k, v, where, tables, norms)
    q = c.q.copy()
    for x in (q, k, v):
        x[live:] = rng.choice(np.array([np.nan, np.inf, -np.inf, 3e38], np.float32), x[live:].shape)
    where[live:] = rng.choice(np.array([-2 ** 31, 2 ** 31 - 1, -1], np.int32), where[live:].shape)
    for got, same in zip(step(dev, c, q, k, v, where, tables, norms), want):
        assert_bits_equal(got, same, "rows of sequences")
