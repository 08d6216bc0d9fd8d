"""GPU: nmx_sample against its definition in 64 bits (numpy sort, cumulative sums).

Bar: tokens equal, prob within 4e-7 relative. The token can only differ where the uniform number lies
within the weights' error (2^-41 of the mass) of a boundary between two tokens, about 1e-8 of the
draws below; prob is a quotient of weights right to 2^-41 rounded once to 32 bits (2^-24 = 6e-8),
the reference's quotient is not rounded."""
from __future__ import annotations

import numpy as np
import pytest

from nibblemac_amd.nmx import SAMPLE_PARAMS, NmxError

CHUNK = 8192  # logits of one workgroup: sizes on both sides of its multiples


def reference(l, T, top_k, top_p, min_p, u):
    """One row: (token, prob)."""
    l = np.where(np.isnan(l), -np.inf, np.minimum(l.astype(np.float64), np.float64(np.finfo(np.float32).max)))
    if not (l > -np.inf).any():
        return -1, 0.0
    T, top_p, min_p, u = (float(np.float32(x)) for x in (T, top_p, min_p, u))
    if not T > 0:
        return int(np.argmax(l)), 1.0
    order = np.lexsort((np.arange(len(l)), -l))
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp((l - l.max()) / T) if T < np.inf else (l > -np.inf).astype(float)
    if 0 < top_k < len(l):
        order = order[:top_k]
    if top_p < 1:
        reach = np.cumsum(w[order])
        order = order[:1 + min(np.searchsorted(reach, max(top_p, 0.0) * reach[-1]), len(order) - 1)]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    order = np.sort(order[w[order] > 0])
    reach = np.cumsum(w[order])
    u = u if u > 0 else 0.0
    i = min(np.searchsorted(reach, u * reach[-1], side="right"), len(order) - 1)
    return int(order[i]), w[order[i]] / reach[-1]


def records(n, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    r = np.zeros(n, SAMPLE_PARAMS)
    r["temperature"], r["top_k"], r["top_p"], r["min_p"] = T, top_k, top_p, min_p
    return r


def sample(dev, logits, par, u, stride=None, times=1):
    """The device's tokens and probs; the buffers hold 7s before."""
    n, vocab = logits.shape
    stride = stride or vocab
    wide = np.full((n, stride), 1e30, np.float32)
    wide[:, :vocab] = logits
    bufs = [dev.to_device(x) for x in (wide, par, u.astype(np.float32), np.full(n + 1, 7, np.int32),
                                       np.full(n + 1, 7, np.float32))]
    work = dev.alloc(dev.sample_work_bytes(n, vocab))
    for _ in range(times):
        dev.sample(bufs[0], stride, vocab, n, bufs[1], bufs[2], work, bufs[3], prob=bufs[4],
                   per_row=len(par) > 1 or n == 1)
    dev.sync()
    tok, prob = bufs[3].numpy(), bufs[4].numpy()
    assert tok[n] == 7 and prob[n] == 7
    for b in (*bufs, work):
        b.free()
    return tok[:n], prob[:n]


def check(dev, logits, par, u, stride=None):
    tok, prob = sample(dev, logits, par, u, stride, times=2)
    for r in range(len(logits)):
        p = par[r if len(par) > 1 else 0]
        want = reference(logits[r], p["temperature"], p["top_k"], p["top_p"], p["min_p"], u[r])
        assert tok[r] == want[0], (r, p, u[r], tok[r], want)
        assert abs(prob[r] - want[1]) <= 4e-7 * want[1], (r, p, prob[r], want)


def rows(rng, n, vocab, spread=2.0, peaks=20):
    l = (rng.standard_normal((n, vocab)) * spread).astype(np.float32)
    for r in range(n if peaks else 0):
        l[r, rng.integers(0, vocab, peaks)] += rng.uniform(3, 12, peaks).astype(np.float32)
    return l


FILTERS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.999), dict(min_p=0.05),
           dict(top_k=20, top_p=0.8), dict(top_k=3000, top_p=0.99, min_p=0.001), dict(T=0.0),
           dict(T=0.3, top_p=0.95), dict(T=1.7, top_k=4000)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, CHUNK - 1, CHUNK, CHUNK + 1, 3 * CHUNK + 17, 248320])
def test_filters(dev, vocab):
    print(f"[case] sample filters vocab={vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    par = np.concatenate([records(2, **f) for f in FILTERS])
    u = rng.random(len(par), np.float32)
    check(dev, rows(rng, len(par), vocab, peaks=min(20, vocab // 4)), par, u, stride=vocab + vocab % 5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "two_values", "quantized", "far_apart", "huge", "zeros_of_both_signs", "steps"])
def test_ties_and_ranges(dev, kind):
    """Ties at the borders of every filter, more members in a bin than the list holds, magnitudes at
    the ends of the type."""
    print(f"[case] sample {kind}", flush=True)
    rng = np.random.default_rng(len(kind))
    par = np.concatenate([records(3, **f) for f in FILTERS + [dict(top_k=9001, top_p=0.5), dict(T=1e-30), dict(T=np.inf),
                                                             dict(T=1e30, top_k=700), dict(T=1e-3, top_p=0.9)]])
    n, vocab = len(par), 2 * CHUNK + 300
    l = np.zeros((n, vocab), np.float32)
    if kind == "equal":
        l += 1.5
    elif kind == "two_values":
        l[:, ::3] = 0.25
    elif kind == "quantized":
        l = np.round(rng.standard_normal((n, vocab)) * 4).astype(np.float32) / 4
    elif kind == "far_apart":
        l = (rng.standard_normal((n, vocab)) * 40).astype(np.float32)
    elif kind == "huge":
        l = (rng.uniform(-1, 1, (n, vocab)) * 3e38).astype(np.float32)
        l[:, 5] = l[:, 9000] = 3.4e38
    elif kind == "zeros_of_both_signs":
        l = np.where(rng.random((n, vocab)) < 0.5, np.float32(-0.0), np.float32(0.0))
    else:       # one chunk 20 nats below the other, one 40
        l = rng.standard_normal((n, vocab)).astype(np.float32)
        l[:, :CHUNK] -= 20
        l[:, 2 * CHUNK:] -= 40
    check(dev, l, par, rng.random(n, np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("ties", [False, True])
def test_few_and_more_tokens(dev, ties):
    """Prefixes about the sizes at which a row is decided by one wave, by one workgroup's threads, and
    by its bins: by count, by mass and by border, over one chunk and over three."""
    print(f"[case] sample few tokens ties={ties}", flush=True)
    rng = np.random.default_rng(11 + ties)
    ks = [2, 33, 63, 64, 65, 127, 128, 129, 255, 256, 500, 511, 512, 513, 1000, 1023, 1024, 1025, 2000]
    for vocab in (2777, 2 * CHUNK + 300):
        par = np.concatenate([records(1, **f) for k in ks for f in (dict(top_k=k), dict(top_k=k, top_p=0.97),
                                                                   dict(top_k=k, min_p=0.003, T=1.5))] +
                             [records(1, top_p=p, T=t) for p in (0.3, 0.6, 0.8, 0.9, 0.95, 0.99) for t in (0.5, 1.0, 2.0)] +
                             [records(1, min_p=m, T=t) for m in (0.3, 0.03, 0.003) for t in (0.5, 1.0, 2.0)])
        l = (rng.standard_normal((len(par), vocab)) * 2.5).astype(np.float32)
        if ties:
            l = np.round(l * 8) / 8
        u = rng.random(len(par), np.float32)
        u[::7] = 0.0
        u[3::7] = 1.0 - 2.0 ** -24
        check(dev, l.astype(np.float32), par, u)


@pytest.mark.gpu
@pytest.mark.parametrize("n, vocab", [(4096, 33), (3, 1 << 20)])
def test_largest_sizes(dev, n, vocab):
    print(f"[case] sample {n} x {vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    par = np.concatenate([records(1, **FILTERS[r % len(FILTERS)]) for r in range(n)])
    check(dev, rows(rng, n, vocab, peaks=4), par, rng.random(n, np.float32), stride=vocab + 1)


@pytest.mark.gpu
def test_masked_values(dev):
    """-inf, NaN, +inf and the lowest finite value as masks; rows that nothing is left of."""
    print("[case] sample masks", flush=True)
    rng = np.random.default_rng(3)
    vocab = CHUNK + 100
    for f in (dict(), dict(top_k=5), dict(top_p=0.7), dict(min_p=0.1), dict(T=0.0)):
        l = rows(rng, 8, vocab)
        l[0, :CHUNK] = -np.inf
        l[1, 10:] = -np.inf
        l[2] = -np.inf
        l[3] = np.nan
        l[4, rng.random(vocab) < 0.5] = np.nan
        l[5, [7, CHUNK + 3]] = np.inf
        l[6] = np.finfo(np.float32).min
        l[7, 50:] = np.finfo(np.float32).min
        check(dev, l, records(8, **f), rng.random(8, np.float32))


@pytest.mark.gpu
def test_uniform_numbers(dev):
    """u at the ends of its range and outside it; one record for all rows."""
    print("[case] sample u", flush=True)
    rng = np.random.default_rng(4)
    u = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan, 2.0 ** -24, 0.5], np.float32)
    for f in (dict(), dict(top_p=0.9), dict(top_k=40, min_p=0.01)):
        check(dev, rows(rng, 8, 20000), records(1, **f), u)


@pytest.mark.gpu
def test_parameters_outside_their_range(dev):
    print("[case] sample odd parameters", flush=True)
    rng = np.random.default_rng(5)
    par = np.concatenate([records(1, **f) for f in (
        dict(T=-1.0), dict(T=np.nan), dict(top_k=-3), dict(top_k=1 << 30), dict(top_p=0.0), dict(top_p=-1.0),
        dict(top_p=np.nan), dict(top_p=7.0), dict(min_p=-1.0), dict(min_p=np.nan), dict(min_p=1.0), dict(min_p=3.0),
        dict(top_k=1 << 30, top_p=0.5), dict(min_p=1e-40), dict(top_p=1e-40))])
    check(dev, rows(rng, len(par), 9000), par, rng.random(len(par), np.float32))


@pytest.mark.gpu
def test_draws_follow_the_weights(dev):
    """4096 draws of one row: counts within 6 sigma of the weights' shares."""
    print("[case] sample counts", flush=True)
    rng = np.random.default_rng(6)
    l = np.tile(rng.standard_normal(40).astype(np.float32), (4096, 1))
    u = ((np.arange(4096) + 0.5) / 4096).astype(np.float32)
    tok, _ = sample(dev, l, records(1, T=0.9), u)
    w = np.exp(l[0].astype(np.float64) / float(np.float32(0.9)))
    assert np.abs(np.bincount(tok, minlength=40) - 4096 * w / w.sum()).max() <= 1.0  # u is a grid


@pytest.mark.gpu
def test_captured_call_reads_its_inputs_anew(dev):
    """One captured call, replayed with other logits, parameters and numbers."""
    print("[case] sample graph", flush=True)
    rng = np.random.default_rng(7)
    n, vocab = 5, 20000
    bufs = [dev.empty((n, vocab), np.float32), dev.alloc(16 * n), dev.empty(n, np.float32)]
    tok, prob = dev.empty(n, np.int32), dev.empty(n, np.float32)
    work = dev.alloc(dev.sample_work_bytes(n, vocab))
    dev.graph_begin()
    dev.sample(bufs[0], vocab, vocab, n, bufs[1], bufs[2], work, tok, prob=prob)
    g = dev.graph_end()
    for f in (dict(), dict(top_p=0.8), dict(T=0.0), dict(top_k=30, T=0.6), dict()):
        l, u, par = rows(rng, n, vocab), rng.random(n, np.float32), records(n, **f)
        for b, x in zip(bufs, (l, par, u)):
            dev.upload(b, x)
        dev.graph_launch(g)
        dev.sync()
        want_t, want_p = sample(dev, l, par, u)
        assert np.array_equal(tok.numpy(), want_t) and np.array_equal(prob.numpy(), want_p)
        check(dev, l, par, u)
    dev.graph_destroy(g)



def test_work_bytes_of_refused_shapes():
    from nibblemac_amd.nmx import load_library

    f = load_library().nmx_sample_work_bytes
    assert f(0, 100) == f(1, 0) == f(4097, 100) == f(1, (1 << 20) + 1) == f(-1, -1) == 0
    assert 0 < f(1, 1) == f(1, CHUNK) and f(1, CHUNK + 1) == 2 * f(1, 1) and f(4096, 1 << 20) == 4096 * 128 * f(1, 1)


@pytest.mark.gpu
def test_refusals(dev):
    print("[case] sample refusals", flush=True)
    n, vocab = 2, 100
    l, par, u = dev.zeros((n, vocab), np.float32), dev.zeros(4 * n, np.float32), dev.zeros(n, np.float32)
    tok, prob, work = dev.zeros(n, np.int32), dev.zeros(n, np.float32), dev.zeros(dev.sample_work_bytes(n, vocab), np.uint8)
    good = dict(logits=l, stride=vocab, vocab=vocab, n=n, params=par, u=u, work=work, tok=tok, prob=prob)
    for bad in (dict(n=0), dict(n=4097), dict(vocab=0), dict(vocab=(1 << 20) + 1, stride=1 << 21), dict(stride=99),
                dict(logits=None), dict(params=None), dict(u=None), dict(work=None), dict(tok=None),
                dict(work=work.ptr + 8), dict(tok=u), dict(tok=work), dict(prob=tok), dict(prob=l), dict(work=l)):
        with pytest.raises(NmxError, match="nmx_sample"):
            dev.sample(**{**good, **bad})
    dev.sync()
    assert not tok.numpy().any() and not work.numpy().any()


MIN_P_ROWS = [  # T, min_p, the maximum
    (1.0, 1.0, 0.0), (1.0, 1.0, 1.5), (np.inf, 1.0, 1.5), (np.inf, 0.5, -2.0), (1e17, 1.0, 10.0), (1e17, 3.0, 0.0), (1e30, 0.5, 3.0),
    (1.0, float(np.exp(-1)), 1.0), (1.0, 0.5, float(np.log(2))), (2.0, 0.3, 0.0), (0.7, 0.999, 0.0), (1.0, 1.0, 3.4e38),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["zeros", "zeros_of_both_signs", "next_to_zero", "tiny", "spread"])
def test_min_p_border_over_many_tokens(dev, kind):
    """More tokens than are decided among themselves, min-p alone and beside the other filters, where the
    border lies among logits next to 0 (floats are dense there), or the weights are alike over billions
    of floats (a high temperature, a min_p of 1 or more). No weight lies within 2^-40 of min_p of the
    border: a kernel's weight is right to 2^-43."""
    print(f"[case] sample min_p border {kind}", flush=True)
    rng = np.random.default_rng(len(kind))
    vocab = CHUNK + 3000
    par = np.concatenate([records(1, T=T, min_p=m, **f) for T, m, _ in MIN_P_ROWS for f in (dict(), dict(top_k=5000), dict(top_p=0.97))])
    n = len(par)
    l = np.zeros((n, vocab), np.float32)
    if kind == "zeros_of_both_signs":
        l = np.where(rng.random((n, vocab)) < 0.5, np.float32(-0.0), np.float32(0.0))
    elif kind == "next_to_zero":
        l = (10.0 ** rng.uniform(-12, -2, (n, vocab)) * rng.choice([-1, 1], (n, vocab))).astype(np.float32)
    elif kind == "tiny":    # down to the subnormals: all of one weight
        l = (10.0 ** rng.uniform(-44, -20, (n, vocab)) * rng.choice([-1, 1], (n, vocab))).astype(np.float32)
    elif kind == "spread":
        l = (rng.standard_normal((n, vocab)) * 0.3).astype(np.float32)
    if not kind.startswith("zeros"):
        l = np.minimum(l, np.repeat([m for _, _, m in MIN_P_ROWS], 3)[:, None]).astype(np.float32)
    l[np.arange(n), rng.integers(0, vocab, n)] = np.repeat([m for _, _, m in MIN_P_ROWS], 3)
    for r in range(n):
        x, m = l[r].astype(np.float64), float(par["min_p"][r])
        T = float(par["temperature"][r])
        w = np.exp((x - x.max()) / T) if T < np.inf else np.ones(vocab)
        near = np.abs(w / min(m, 1.0) - 1)
        assert not ((near < 2.0 ** -40) & (near > 0) & (m < 1)).any()
    check(dev, l, par, rng.random(n, np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("f", [dict(), dict(min_p=1e-12), dict(top_p=0.999999), dict(top_k=9000), dict(top_k=9000, top_p=0.999999)],
                         ids=lambda f: "_".join(f) or "none")
def test_from_one_on_the_last_token(dev, f):
    """u of 1 and more takes the last kept token, however little it weighs: the last ones of each row weigh
    less than the roundings of the row's sums."""
    print(f"[case] sample u = 1 {f}", flush=True)
    rng = np.random.default_rng(9)
    n, vocab = 64, 2 * CHUNK + 1000
    l = rng.standard_normal((n, vocab)).astype(np.float32)
    for r in range(n):
        if f:       # within reach of a filter, one token behind the others
            l[r, -1] = l[r].max() - (26 if "min_p" in f else 0.5)
        else:
            l[r, -700 if r % 2 else -2:] = l[r].max() - 45
    par = records(1, **f)
    u = np.where(np.arange(n) % 3, 1.0, 2.0).astype(np.float32)
    check(dev, l, par, u)


@pytest.mark.gpu
@pytest.mark.parametrize("offset,T", [(1e4, 0.002), (-1e4, 0.002), (1e6, 0.2), (3e4, 0.01), (1e30, 2e23)])
def test_logits_far_from_zero(dev, offset, T):
    """Logits about an offset, many temperatures away from 0: the weights are those of the differences to
    the maximum. Eight values, 700 tokens each; top-p ends 2^-38 to 2^-32.5 of the mass from a token's
    end, where weights right to 2^-40 of themselves decide alike and ones of 2^-31 do not."""
    print(f"[case] sample offset {offset} T={T}", flush=True)
    rng = np.random.default_rng(12)
    T = float(np.float32(T))
    values = np.sort((np.float32(offset) + np.spacing(np.float32(offset)) * rng.permutation(12)[:8]).astype(np.float32))[::-1]
    w = np.exp((values.astype(np.float64) - float(values[0])) / T)
    assert len(set(values)) == 8 and w[-1] > 1e-4
    ends = np.cumsum(np.repeat(w, 700)) / (700 * w.sum())
    p = ends.astype(np.float32)
    off = np.abs(p - ends)
    p = p[(off > 2.0 ** -38) & (off < 2.0 ** -32.5) & (p < 1)]
    assert len(p) >= 10
    l = np.full((len(p), CHUNK + 500), values[-1] - np.float32(400 * T), np.float32)
    l[:, 1000:6600] = np.repeat(values, 700)
    par = records(len(p))
    par["temperature"], par["top_p"] = T, p
    check(dev, l, par, np.ones(len(p), np.float32))
    check(dev, l, par, rng.random(len(p), np.float32))
