"""The operators of a step of many requests at once, as cases that can be timed and compared.

A program that serves a batch of sequences with this device layer keeps their KV rows in pages, reads a
prefix that many of them begin with once, and gives each request the low-rank adapter it asks for:

    pages   the tables of a step: each sequence goes on, is cut back, forks from another one or ends, takes
            pages for its new rows, and copies the one that it would write into beside others; with pack,
            the used pages move to the lowest numbers (nmx_pages_update)
    prep    query and key norms, rotary positions of several axes (time, height, width), K and V rows stored
            into their pages (nmx_attn_batch_prep)
    attn    gated causal attention of every sequence's rows over its pages, a shared prefix read once for
            its group (nmx_attn_batch)
    lora    y += scale B (A x) of each row's own adapter, beside the projections that share x (nmx_lora)
    lin     the Gated DeltaNet mixer over the rows of many sequences, each from the state of its own or of
            the sequence that it forks from (nmx_lin_mix_batch)

Sizes are those of the 0.8B shape (hidden 1024, FFN 3584, 8 query and 2 KV heads of 256 of which 64 rotate,
7 caches of K and V with the MTP layer's, 16 DeltaNet heads of 128 x 128, conv of 4) and, in the drawn cases,
of the tests' other head layouts. Where `own` is false, `run` computes them in elementary torch operations;
where it is true, through nibblemac_amd.nmx.Device.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

F16, BF16, F32, F64, I32 = torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.int32
KV_F32, KV_F16, KV_I8 = 0, 1, 2
HIDDEN, FFN = 1024, 3584
HEADS, DK, DV, CONV_K = 16, 128, 128, 4          # a DeltaNet layer
CHANNELS = HEADS * (2 * DK + DV)
EPS = 1e-6
QSCALE = float(np.float32(1 / math.sqrt(DK)))
W_TYPES = (F32, F16, BF16)


# ---- the cases ---------------------------------------------------------------------------
# `lens` seeds the lengths of a case (and which sequences fork or end), so that its work is known from it.
def listed():
    return [
        # a step of 64 chats: most go on by a token, a few fork from another one or end
        dict(name="pages_step", kind="pages", seqs=64, page=32, npages=640, lo=20, hi=300, add=1, fork=5, end=3,
             pack=0, caches=14, nkv=2, hd=256, kv=KV_F16, lens=1),
        # a quarter of the chats ended: the others' pages move together
        dict(name="pages_pack", kind="pages", seqs=64, page=16, npages=1200, lo=20, hi=400, add=4, fork=0, end=16,
             pack=1, caches=14, nkv=2, hd=256, kv=KV_F16, lens=2),
        # a token of each of 8 sequences, text and video positions
        dict(name="prep_step", kind="prep", seqs=8, most=1, ctx=900, nh=8, nkv=2, hd=256, rot=64, axes=3, page=64,
             kv=KV_F16, lens=3),
        # prompts with pictures among single tokens
        dict(name="prep_prompt", kind="prep", seqs=12, most=120, ctx=2000, nh=8, nkv=2, hd=256, rot=64, axes=3,
             page=64, kv=KV_F32, lens=4),
        # four chats, a token each: latency
        dict(name="attn_few", kind="attn", seqs=4, most=1, lo=300, hi=700, shared=0, nh=8, nkv=2, hd=256, page=16,
             kv=KV_F32, lens=5),
        # 48 chats of uneven lengths, a token each
        dict(name="attn_chat", kind="attn", seqs=48, most=1, lo=50, hi=6000, shared=0, nh=8, nkv=2, hd=256, page=64,
             kv=KV_F16, lens=6),
        # pieces of prompts among single tokens, int8 caches, a system prompt that all begin with
        dict(name="attn_mixed", kind="attn", seqs=20, most=90, lo=20, hi=3000, shared=700, nh=8, nkv=2, hd=256,
             page=32, kv=KV_I8, lens=7),
        # 64 questions about one long document
        dict(name="attn_prefix", kind="attn", seqs=64, most=1, lo=20, hi=1500, shared=30000, nh=8, nkv=2, hd=256,
             page=64, kv=KV_F16, lens=8),
        # the attention projections of 8 requests with 5 small adapters
        dict(name="lora_step", kind="lora", n=8, cols=HIDDEN, rows="4096 512 512", adapters=5, rank=16, ragged=0,
             w=1, lens=9),
        # gate and up projections of 64 requests, 40 adapters of ranks up to 64
        dict(name="lora_many", kind="lora", n=64, cols=HIDDEN, rows=f"{FFN} {FFN}", adapters=40, rank=64, ragged=1, w=2,
             lens=10),
        # a DeltaNet layer for four sequences, in place
        dict(name="lin_step", kind="lin", seqs=4, most=1, fork=0, lens=11),
        # for 64, some of which fork from others or start
        dict(name="lin_batch", kind="lin", seqs=64, most=1, fork=6, lens=12),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["pages", "prep", "attn", "attn", "attn", "lora", "lora", "lin"])
    lens, page = rng.randrange(1 << 30), rng.choice([16, 32, 64, 128])
    if kind == "pages":
        seqs, hi = _log(rng, 1, 64), _log(rng, 8, 300)
        npages = seqs * (2 + (hi + 8) // page) + rng.randint(0, 40)
        return dict(kind=kind, seqs=seqs, page=page, npages=npages, lo=rng.randint(0, 7), hi=hi,
                    add=rng.choice([1, 1, 2, 5]), fork=rng.randint(0, seqs // 4), end=rng.randint(0, seqs // 4),
                    pack=rng.choice([0, 1]), caches=rng.choice([2, 6, 14]), nkv=2, hd=rng.choice([64, 128]),
                    kv=rng.choice([KV_F32, KV_F16]), lens=lens)
    nh, nkv, hd = rng.choice([(8, 2, 256), (8, 2, 256), (8, 2, 256), (6, 2, 128), (4, 4, 64), (16, 2, 256),
                              (8, 1, 512), (4, 2, 192)])
    if kind == "prep":
        return dict(kind=kind, seqs=_log(rng, 1, 20), most=rng.choice([1, 1, _log(rng, 2, 25)]),
                    ctx=_log(rng, 1, 2000), nh=nh, nkv=nkv, hd=hd, rot=rng.choice([hd, hd // 2, 64]),
                    axes=rng.choice([1, 3, 3]), page=page, kv=rng.choice([KV_F32, KV_F16]), lens=lens)
    if kind == "attn":
        seqs, most = _log(rng, 1, 64), rng.choice([1, 1, 1, _log(rng, 2, 120)])
        hi = _log(rng, 1, min(8000, 400000 // (seqs * most)))
        return dict(kind=kind, seqs=seqs, most=most, lo=rng.randint(0, hi), hi=hi,
                    shared=rng.choice([0, 0, _log(rng, 16, min(20000, 500000 // (seqs * most)))]), nh=nh, nkv=nkv, hd=hd,
                    page=page, kv=rng.choice([KV_F32, KV_F16, KV_I8]), lens=lens)
    if kind == "lora":
        n, rank = rng.choice([_log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 65, 300)]), _log(rng, 1, 96)
        count = rng.randint(1, 3)
        return dict(kind=kind, n=n, cols=rng.choice([256, HIDDEN, HIDDEN, 2048, FFN]),
                    rows=" ".join(rng.choice(["16", "512", "1000", "2048", str(FFN)]) for _ in range(count)), adapters=_log(rng, 1, 30),
                    rank=rank, ragged=rng.choice([0, 1]), w=rng.choice([0, 1, 2]), lens=lens)
    seqs = _log(rng, 1, 64)
    return dict(kind=kind, seqs=seqs, most=rng.choice([1, 1, rng.randint(2, 6)]), fork=rng.randint(0, seqs // 2),
                lens=lens)


# ---- lengths and tables, known from the case ----------------------------------------------
def _rows_of(c):
    """Rows of each sequence: all `most` = 1, or single tokens with pieces of up to `most` among them."""
    r = np.random.default_rng(c["lens"])
    if c["most"] == 1:
        return np.ones(c["seqs"], np.int64)
    rows = np.where(r.random(c["seqs"]) < 0.7, 1, r.integers(1, c["most"] + 1, c["seqs"]))
    rows[r.integers(0, c["seqs"])] = c["most"]
    while rows.sum() > 512:
        rows[rows.argmax()] //= 2
    return rows


def _attn_lens(c):
    """Rows in the cache of each sequence: the shared prefix, its own and those of this step."""
    r = np.random.default_rng(c["lens"] + 1)
    own_rows = np.floor(np.exp(r.uniform(math.log(c["lo"] + 1), math.log(c["hi"] + 1), c["seqs"]))).astype(np.int64) - 1
    return c["shared"] + own_rows + _rows_of(c)


def _pages_plan(c):
    """Lengths, and what becomes of each sequence: (len, from, keep, add)."""
    r = np.random.default_rng(c["lens"])
    seqs = c["seqs"]
    ln = r.integers(c["lo"], c["hi"] + 1, seqs)
    src, add = np.arange(seqs), np.full(seqs, c["add"])
    order = r.permutation(seqs)
    ends, forks, stay = order[:c["end"]], order[c["end"]:c["end"] + c["fork"]], order[c["end"] + c["fork"]:]
    src[ends], add[ends] = -1, 0
    if len(stay):
        src[forks] = stay[r.integers(0, min(2, len(stay)), len(forks))]
    keep = np.where(src < 0, 0, ln[src.clip(0)])
    cut = r.random(seqs) < 0.15          # drafts that were not accepted
    keep = np.where(cut, np.maximum(keep - 2, 0), keep)
    return ln, src, keep, add


# ---- inputs ------------------------------------------------------------------------------
class _Inputs:
    """Seeded inputs of one case, made on the GPU; the same numbers for every caller."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))
        self.host = np.random.default_rng(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=F32) * std

    def uniform(self, lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(shape, generator=self.g, device="cuda", dtype=F32)

    def cache(self, kv, npages, nkv, page, hd):
        """Pages of rows of unit variance: [npages][nkv][page][hd], an int8 page with its scales behind."""
        rows = self.normal(npages, nkv, page, hd)
        if kv != KV_I8:
            return rows if kv == KV_F32 else rows.half()
        amax = rows.abs().amax(3)
        codes = torch.round(rows * (127.0 / amax)[..., None]).to(torch.int8)
        return torch.cat([codes.view(npages, -1), (amax / 127.0).view(npages, -1).view(torch.int8)], 1).contiguous()


def _dev(v):
    return torch.tensor(np.asarray(v), device="cuda", dtype=I32)


def _pages_inputs(c, x):
    seqs, page, npages = c["seqs"], c["page"], c["npages"]
    ln, src, keep, add = _pages_plan(c)
    wide = int(max(ln.max(), (keep + add).max()) // page + 2)
    perm, at = x.host.permutation(npages), 0
    table, refs = np.full((seqs, wide), -1), np.zeros(npages, np.int64)
    for s in range(seqs):
        k = -(-int(ln[s]) // page)
        table[s, :k] = perm[at:at + k]
        at += k
    refs[perm[:at]] = 1
    book = _dev(np.concatenate([table.ravel(), ln, refs]))
    a, b = seqs * wide, seqs * wide + seqs
    # a pass that packs finds nothing to move the next time: it starts from a copy of the tables
    return dict(book=book, start=book.clone(), table=book[:a].view(seqs, wide), len=book[a:b], refs=book[b:], src=_dev(src),
                keep=_dev(keep), add=_dev(add), out=_dev([-7] * 4),
                kv=[x.cache(c["kv"], npages, c["nkv"], page, c["hd"]) for _ in range(c["caches"])])


def _tables(c, x, lens, shared):
    """A table of random pages for every sequence, the whole pages of the first `shared` rows in common."""
    page, seqs, common = c["page"], c["seqs"], shared // c["page"]
    counts = -(-lens // page)
    npages = int(common + (counts - common).sum()) + 3
    perm, at = x.host.permutation(npages), common
    table = np.full((seqs, int(counts.max()) + 1), -1)
    for s in range(seqs):
        table[s, :common] = perm[:common]
        table[s, common:counts[s]] = perm[at:at + counts[s] - common]
        at += counts[s] - common
    return table, npages


def _row0(c):
    return np.concatenate([[0], np.cumsum(_rows_of(c))])


def _prep_inputs(c, x):
    nh, nkv, hd, h2 = c["nh"], c["nkv"], c["hd"], c["rot"] // 2
    row0, r = _row0(c), np.random.default_rng(c["lens"] + 1)
    lens, n = r.integers(0, c["ctx"] + 1, c["seqs"]) + np.diff(row0), int(row0[-1])
    table, npages = _tables(c, x, lens, 0)
    span = int(lens.max()) + 64
    angle = torch.outer(torch.arange(span, device="cuda", dtype=F64),
                        1e7 ** (-torch.arange(h2, device="cuda", dtype=F64) / h2))
    # the axes take turns over the frequencies, the slowest ones are time's
    axis = np.array([i % 3 if c["axes"] == 3 and i < h2 * 7 // 8 else 0 for i in range(h2)], np.uint8)
    return dict(row0=_dev(row0), len=_dev(lens), table=_dev(table), npages=npages, n=n, span=span, axis=axis,
                where=_dev(x.host.integers(0, span, (n, c["axes"]))), cos=torch.cos(angle).float(), sin=torch.sin(angle).float(),
                q=x.normal(n, nh, 2 * hd), k=x.normal(n, nkv, hd), v=x.normal(n, nkv, hd),
                qn=x.uniform(0.8, 1.2, hd), kn=x.uniform(0.8, 1.2, hd),
                kc=x.cache(c["kv"], npages, nkv, c["page"], hd), vc=x.cache(c["kv"], npages, nkv, c["page"], hd))


def _attn_inputs(c, x):
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    row0, lens = _row0(c), _attn_lens(c)
    n, shared = int(row0[-1]), c["shared"] // c["page"] * c["page"]
    table, npages = _tables(c, x, lens, shared)
    return dict(row0=_dev(row0), len=_dev(lens), table=_dev(table), npages=npages, n=n, lens=lens, host0=row0,
                group0=_dev([0, c["seqs"]]), shared=_dev([shared]), q=x.normal(n, nh, 2 * hd),
                kc=x.cache(c["kv"], npages, nkv, c["page"], hd), vc=x.cache(c["kv"], npages, nkv, c["page"], hd),
                o=torch.zeros(n, nh * hd, device="cuda", dtype=F32))


def _lora_rows(c):
    return [int(r) for r in c["rows"].split()]


def _lora_shape(c):
    """(the adapter of each row, the rank of each adapter): one row in ten without one."""
    r = np.random.default_rng(c["lens"])
    ad = np.where(r.random(c["n"]) < 0.1, -1, r.integers(0, c["adapters"], c["n"]))
    ranks = r.integers(max(1, c["rank"] // 4), c["rank"] + 1, c["adapters"]) if c["ragged"] else np.full(c["adapters"], c["rank"])
    return ad, ranks


def _lora_inputs(c, x):
    n, cols, R, m = c["n"], c["cols"], c["rank"], c["adapters"]
    ad, ranks = _lora_shape(c)
    wt = W_TYPES[c["w"]]
    return dict(x=x.normal(n, cols), ad=_dev(ad), ranks=_dev(ranks) if c["ragged"] else None,
                scale=x.uniform(0.5, 2.0, m), A=[x.normal(m, R, cols, std=cols ** -0.5).to(wt) for _ in _lora_rows(c)],
                B=[x.normal(m, r, R, std=0.05).to(wt) for r in _lora_rows(c)], y=[x.normal(n, r) for r in _lora_rows(c)])


def _state_at():
    """Position of element (head, column j, key i) of the recurrent state: columns in groups of 16,
    within a group the float4 slot of every lane contiguous (nmx_state_index, include/nmx.h)."""
    h, j, i = torch.meshgrid(*(torch.arange(d, device="cuda") for d in (HEADS, DV, DK)), indexing="ij")
    return (h * DV + j // 16 * 16) * DK + ((i % (DK // 4)) // 4 * 64 + 4 * (j % 16) + i // (DK // 4)) * 4 + i % 4


def _lin_from(c):
    """The state that each sequence starts from: its own, another one's, or (-1) none yet."""
    r = np.random.default_rng(c["lens"] + 1)
    src = np.arange(c["seqs"])
    for s in r.permutation(c["seqs"])[:c["fork"]]:
        src[s] = r.integers(-1, c["seqs"])
    return src


def _lin_inputs(c, x):
    seqs, row0 = c["seqs"], _row0(c)
    n = int(row0[-1])
    zeros = lambda *s: torch.zeros(s, device="cuda", dtype=F32)  # noqa: E731
    t = dict(row0=_dev(row0), n=n, host0=row0, raw=x.normal(n, CHANNELS), z=x.normal(n, HEADS * DV), b=x.normal(n, HEADS),
             a=x.normal(n, HEADS), conv=x.normal(seqs, CONV_K - 1, CHANNELS, std=0.5),
             conv_w=x.uniform(-0.5, 0.5, CHANNELS, CONV_K), A_log=x.uniform(math.log(0.2), math.log(0.4), HEADS),
             dt_bias=x.uniform(-4.5, -3.5, HEADS), norm=x.uniform(0.8, 1.2, DV),
             rec=x.normal(seqs, HEADS * DV * DK, std=0.05), at=_state_at(), y=zeros(n, HEADS * DV), src=None)
    t["conv_out"], t["rec_out"] = t["conv"], t["rec"]
    if c["fork"]:
        t.update(src=_dev(_lin_from(c)), conv_out=torch.zeros_like(t["conv"]), rec_out=torch.zeros_like(t["rec"]))
    return t


def prepare(case, seed):
    """The inputs on the GPU and the buffers that a program holds for its outputs."""
    made = dict(pages=_pages_inputs, prep=_prep_inputs, attn=_attn_inputs, lora=_lora_inputs, lin=_lin_inputs)
    return dict(case=case, t=made[case["kind"]](case, _Inputs(seed)), call=None)


# ---- the framework's calls ---------------------------------------------------------------
_device = None


def _ctx():
    """The program's one context (a device and its stream)."""
    global _device
    if _device is None:
        from nibblemac_amd.nmx import Device

        _device = Device(0)
    return _device


def _p(t):
    return None if t is None else t.data_ptr()


def _pages_of(c, t, npages):
    from nibblemac_amd.nmx import Pages

    return Pages(seqs=c["seqs"], npages=npages, page=c["page"], max_pages=t["table"].shape[1], table=_p(t["table"]),
                 len=_p(t["len"]), nkv=c["nkv"], hd=c["hd"], kv_dtype=c["kv"])


def _bytes(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device="cuda")


def _pages_call(c, t):
    from nibblemac_amd.nmx import pages_args

    dev = _ctx()
    args = pages_args(_pages_of(c, t, c["npages"]), _p(t["refs"]), _p(t["src"]), _p(t["keep"]), _p(t["add"]),
                      [_p(k) for k in t["kv"]], _p(t["out"]), pack=c["pack"])
    work = _bytes(dev.pages_work_bytes(c["npages"], c["seqs"], t["table"].shape[1]))

    book, start, size = _p(t["book"]), _p(t["start"]), 4 * t["book"].numel()

    def call():
        if c["pack"]:
            dev.copy(book, start, size)
        dev.pages_update(args, work.data_ptr())
        return _pages_out(t)

    return call


def _attn_args(c, t, **more):
    from nibblemac_amd.nmx import A8, AttnBatchArgs

    return AttnBatchArgs(pages=_pages_of(c, t, t["npages"]), n=t["n"], row0=_p(t["row0"]), nh=c["nh"], q=_p(t["q"]),
                         kc=_p(t["kc"]), vc=_p(t["vc"]), a8=A8(None, None, None), **more)


def _prep_call(c, t):
    dev, axis = _ctx(), t["axis"]
    args = _attn_args(c, t, rot=c["rot"], k_in=_p(t["k"]), v_in=_p(t["v"]), q_norm=_p(t["qn"]), k_norm=_p(t["kn"]),
                      eps=EPS, rope_cos=_p(t["cos"]), rope_sin=_p(t["sin"]), rope_rows=t["span"], axes=c["axes"],
                      axis=axis.ctypes.data, rope_pos=_p(t["where"]))

    def call():
        dev.attn_batch_prep(args)
        return {k: t[k] for k in ("q", "kc", "vc")}

    return call


def _attn_call(c, t):
    dev, groups = _ctx(), int(c["shared"] > 0)
    args = _attn_args(c, t, scale=np.float32(1 / math.sqrt(c["hd"])), groups=groups, group0=_p(t["group0"]),
                      shared=_p(t["shared"]), o=_p(t["o"]))
    work = _bytes(dev.attn_batch_work_bytes(t["n"], c["seqs"], groups, c["nh"], c["nkv"], c["hd"]))

    def call():
        dev.attn_batch(args, work.data_ptr())
        return dict(o=t["o"])

    return call


def _lora_call(c, t):
    from nibblemac_amd.nmx import lora_args

    dev, n, rows = _ctx(), c["n"], _lora_rows(c)
    args = lora_args(n, c["cols"], _p(t["x"]), c["cols"], c["adapters"], c["rank"], c["w"], _p(t["ad"]), _p(t["scale"]),
                     [(r, _p(a), _p(b), _p(y), r) for r, a, b, y in zip(rows, t["A"], t["B"], t["y"])],
                     ranks=_p(t["ranks"]))
    work = _bytes(dev.lora_work_bytes(n, len(rows), c["rank"]))

    def call():
        dev.lora(args, work.data_ptr())
        return dict(y=t["y"])

    return call


def _lin_call(c, t):
    from nibblemac_amd.nmx import A8, LinArgs, LinBatch, LinMixArgs, LinPreArgs

    dev, n, vd = _ctx(), t["n"], HEADS * DV
    pre = LinPreArgs(n=n, C=CHANNELS, conv_k=CONV_K, dk=DK, kd=HEADS * DK, raw=_p(t["raw"]), raw_stride=CHANNELS,
                     state=_p(t["conv"]), conv_w=_p(t["conv_w"]), qscale=QSCALE, l2eps=EPS, b_in=_p(t["b"]),
                     a_in=_p(t["a"]), g_stride=HEADS, heads=HEADS, A_log=_p(t["A_log"]), dt_bias=_p(t["dt_bias"]))
    rule = LinArgs(n=n, heads=HEADS, rep=1, dk=DK, dv=DV, S=_p(t["rec"]))
    mix = LinMixArgs(pre, rule, _p(t["z"]), vd, _p(t["norm"]), EPS, _p(t["y"]), vd, A8(None, None, None))
    batch = LinBatch(seqs=c["seqs"], most=int(np.diff(t["host0"]).max()), row0=_p(t["row0"]), src=_p(t["src"]),
                     state_out=_p(t["conv_out"]), S_out=_p(t["rec_out"]))

    def call():
        dev.lin_mix_batch(mix, batch)
        return dict(y=t["y"], conv=t["conv_out"], rec=t["rec_out"])

    return call


def run(state):
    c, t = state["case"], state["t"]
    if not own:
        return dict(pages=_pages_plain, prep=_prep_plain, attn=_attn_plain, lora=_lora_plain, lin=_lin_plain)[c["kind"]](c, t)
    if state["call"] is None:
        made = dict(pages=_pages_call, prep=_prep_call, attn=_attn_call, lora=_lora_call, lin=_lin_call)
        state["call"] = made[c["kind"]](c, t)
    return state["call"]()


# ---- the plain forms ---------------------------------------------------------------------
def _pages_out(t):
    """Tables and caches after the step: it computes nothing."""
    return {k: t[k] for k in ("table", "len", "refs", "out", "kv")}


def _pages_plain(c, t):
    """The new table of a sequence is the first pages of its source's, then fresh ones, lowest numbers first in
    the sequences' order (a page copied before it is written comes before those of its new rows)."""
    page, npages, seqs = c["page"], c["npages"], c["seqs"]
    if c["pack"]:
        t["book"].copy_(t["start"])
    table, ln, dev = t["table"], t["len"].long(), t["table"].device
    wide = table.shape[1]
    src, keep, add = t["src"].long(), t["keep"].long(), t["add"].long()
    seq, col = torch.arange(seqs, device=dev), torch.arange(wide, device=dev)
    keep = torch.where(src < 0, 0, torch.minimum(keep, ln[src.clamp(min=0)]))
    kept, all_ = (keep + page - 1) // page, (keep + add + page - 1) // page
    new = torch.where(col[None] < kept[:, None], table[src.clamp(min=0)], -1).long()
    bins = lambda pages: torch.zeros(npages + 1, device=dev, dtype=torch.long).scatter_add_(  # noqa: E731
        0, torch.where(pages < 0, npages, pages).reshape(-1), torch.ones_like(pages).reshape(-1))
    held = bins(new)
    last = torch.where((keep % page > 0) & (add > 0), new.gather(1, (kept - 1).clamp(min=0)[:, None])[:, 0], -1)
    same = (last[:, None] == last[None, :]) & (last >= 0)[None, :]
    first = ~(same & (seq[None, :] < seq[:, None])).any(1)
    others = held[last.clamp(min=0)]
    copy = (last >= 0) & (others > 1) & ~((others == same.sum(1)) & first)
    held[:npages].sub_(bins(torch.where(copy, last, -1))[:npages])
    need = all_ - kept + copy.long()
    free = torch.sort(torch.where(held[:npages] == 0, 0, 1), stable=True).indices      # free pages first, in order
    base = need.cumsum(0) - need
    taken = need.sum()
    fresh = base[:, None] + col[None] - (kept - copy.long())[:, None]
    grown = (col[None] >= (kept - copy.long())[:, None]) & (col[None] < all_[:, None])
    new = torch.where(grown, free[fresh.clamp(0, npages - 1)], new)
    dst = free[base.clamp(max=npages - 1)]
    for k in t["kv"]:
        k4 = k.view(npages, c["nkv"], page, c["hd"])
        row = torch.arange(page, device=dev)
        take = (copy[:, None] & (row[None] < (keep % page)[:, None]))[:, None, :, None]
        to = torch.where(copy, dst, free[npages - 1])       # the last one of them is nobody's page or stays as it is
        k4[to] = torch.where(take, k4[torch.where(copy, last, free[npages - 1])], k4[to])
    held = bins(new)[:npages]
    used = (held > 0).sum()
    if c["pack"]:
        at = torch.arange(npages, device=dev)
        moves = (held > 0) & (at >= used)
        empty = (held == 0) & (at < used)               # as many as pages that move
        order = lambda hit: torch.sort(torch.where(hit, 0, 1), stable=True).indices  # noqa: E731
        rank = lambda hit: (hit.long().cumsum(0) - 1).clamp(min=0)  # noqa: E731
        to = torch.where(moves, order(empty)[rank(moves)], at)
        back = torch.where(empty, order(moves)[rank(empty)], at)
        new = torch.where(new >= 0, to[new.clamp(min=0)], -1)
        for k in t["kv"]:
            k.copy_(k[back])
        held = bins(new)[:npages]
    t["table"].copy_(new)
    t["len"].copy_(keep + add)
    t["refs"].copy_(held)
    moved = moves.sum() if c["pack"] else torch.zeros_like(used)
    t["out"].copy_(torch.stack([torch.zeros_like(used), taken, used if c["pack"] else torch.zeros_like(used), moved]))
    return _pages_out(t)


def _seq_of(row0, n):
    """The sequence of each row."""
    return (torch.arange(n, device=row0.device)[:, None] >= row0[None, :].long()).sum(1) - 1


def _prep_plain(c, t):
    n, hd, h2, page, kv = t["n"], c["hd"], c["rot"] // 2, c["page"], c["kv"]
    q, k = t["q"][..., :hd], t["k"]
    axis = torch.as_tensor(t["axis"], device=q.device).long()
    at = t["where"].long()[:, axis]                                    # [n][h2]: the frequency's position
    cos, sin = (f.gather(0, at)[:, None] for f in (t["cos"], t["sin"]))

    def rows(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :h2], x[..., h2:2 * h2]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h2:]], -1)

    t["q"][..., :hd] = rows(q, t["qn"])
    s = _seq_of(t["row0"], n)
    slot = t["len"].long()[s] - t["row0"].long()[s + 1] + torch.arange(n, device=q.device)
    pg = t["table"].long()[s, slot // page]
    for cache, x in ((t["kc"], rows(k, t["kn"])), (t["vc"], t["v"])):
        cache[pg, :, slot % page] = x.to(cache.dtype)
    return {x: t[x] for x in ("q", "kc", "vc")}


def _rows32(c, t, name, s, length):
    """The cache rows of sequence s: [nkv][length][hd] in 32 bits."""
    page, nkv, hd = c["page"], c["nkv"], c["hd"]
    pg = t["table"][s, :-(-length // page)].long()
    x = t[name][pg]
    if c["kv"] == KV_I8:
        codes, scale = x[:, :nkv * page * hd].view(-1, nkv, page, hd), x[:, nkv * page * hd:].contiguous().view(F32).view(-1, nkv, page, 1)
        x = codes.float() * scale
    return x.float().transpose(0, 1).reshape(nkv, -1, hd)[:, :length].contiguous()


def _attn_plain(c, t):
    nh, nkv, hd, rep, outs = c["nh"], c["nkv"], c["hd"], c["nh"] // c["nkv"], []
    scale = float(np.float32(1 / math.sqrt(hd)))
    for s in range(c["seqs"]):
        r0, r1, length = int(t["host0"][s]), int(t["host0"][s + 1]), int(t["lens"][s])
        m = r1 - r0
        k, v = (_rows32(c, t, x, s, length) for x in ("kc", "vc"))
        q = t["q"][r0:r1, :, :hd].reshape(m, nkv, rep, hd).permute(1, 0, 2, 3).reshape(nkv, m * rep, hd)
        sc = (torch.bmm(q.contiguous(), k.transpose(1, 2).contiguous()) * scale).view(nkv, m, rep, length)
        hide = torch.arange(length, device=q.device)[None] > (length - m + torch.arange(m, device=q.device))[:, None]
        sc.masked_fill_(hide[None, :, None], -math.inf)
        p = torch.exp(sc - sc.amax(3, keepdim=True))
        o = torch.bmm(p.view(nkv, m * rep, length), v).view(nkv, m, rep, hd) / p.sum(3, keepdim=True)
        outs.append(o.permute(1, 0, 2, 3).reshape(m, nh, hd))
    return dict(o=(torch.cat(outs) / (1 + torch.exp(-t["q"][..., hd:]))).reshape(t["n"], nh * hd))


def _lora_plain(c, t):
    R, dev = c["rank"], t["x"].device
    ranks = t["ranks"] if t["ranks"] is not None else torch.full((c["adapters"],), R, device=dev)
    live = (torch.arange(R, device=dev)[None] < ranks[:, None]).float()
    for A, B, y in zip(t["A"], t["B"], t["y"]):
        for m in range(c["adapters"]):
            mine = (t["ad"] == m).float()[:, None] * t["scale"][m]
            y += mine * (((t["x"] @ A[m].float().T) * live[m]) @ B[m].float().T)
    return dict(y=t["y"])


def _lin_plain(c, t):
    """The recurrence row by row, all sequences that have such a row together."""
    seqs, n, dev = c["seqs"], t["n"], t["raw"].device
    row0, rows = t["row0"].long(), torch.as_tensor(np.diff(t["host0"]), device=dev)
    src = torch.arange(seqs, device=dev) if t["src"] is None else t["src"].long()
    old = (src >= 0).float()
    win = t["conv"][src.clamp(min=0)] * old[:, None, None]
    R = t["rec"][src.clamp(min=0)] * old[:, None]
    R = R[:, t["at"].reshape(-1)].view(seqs, HEADS, DV, DK)
    out = torch.zeros(n + 1, HEADS * DV, device=dev)
    for i in range(int(np.diff(t["host0"]).max())):
        on = rows > i
        at = torch.where(on, row0[:-1] + i, 0)
        seen = torch.cat([win, t["raw"][at][:, None]], 1)
        acc = (seen * t["conv_w"].T[None]).sum(1)
        conv = acc / (1 + torch.exp(-acc))
        q, k = (conv[:, j * HEADS * DK:(j + 1) * HEADS * DK].view(seqs, HEADS, DK) for j in (0, 1))
        v = conv[:, 2 * HEADS * DK:].view(seqs, HEADS, DV)
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
        beta = 1 / (1 + torch.exp(-t["b"][at]))
        sp = t["a"][at] + t["dt_bias"]
        sp = torch.where(sp > 20, sp, torch.log1p(torch.exp(sp)))
        S = R * torch.exp(-torch.exp(t["A_log"]) * sp)[:, :, None, None]
        delta = (v - (S * k[:, :, None]).sum(-1)) * beta[..., None]
        S = S + delta[..., None] * k[:, :, None]
        o = (S * (q * QSCALE)[:, :, None]).sum(-1)
        y = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * t["norm"]
        z = t["z"][at].view(seqs, HEADS, DV)
        y = (y * (z / (1 + torch.exp(-z)))).view(seqs, -1)
        out[torch.where(on, at, n)] = y          # row n: what no sequence has
        R = torch.where(on[:, None, None, None], S, R)
        win = torch.where(on[:, None, None], seen[:, 1:], win)
    rec = torch.empty_like(t["rec_out"])
    rec[:, t["at"].reshape(-1)] = R.view(seqs, -1)
    t["rec_out"].copy_(rec)
    t["conv_out"].copy_(win)
    t["y"].copy_(out[:n])
    return dict(y=t["y"], conv=t["conv_out"], rec=t["rec_out"])


# ---- what a pass cannot do without -------------------------------------------------------
def _kv_row(kv, hd):
    return hd + 4 if kv == KV_I8 else hd * (2 if kv == KV_F16 else 4)


def work(case):
    c = case
    if c["kind"] == "pages":
        ln, src, keep, add = _pages_plan(c)
        row = c["nkv"] * _kv_row(c["kv"], c["hd"]) * c["caches"]
        t = _pages_host(c, *_pages_start(c))
        return dict(bytes=2 * row * (sum(x[2] for x in t["copies"]) + c["page"] * len(t["moves"])) + 20 * c["seqs"] + 4 * c["npages"], flops=0)
    if c["kind"] == "prep":
        n = int(_row0(c)[-1])
        hd, nh, nkv = c["hd"], c["nh"], c["nkv"]
        return dict(bytes=4 * n * hd * (2 * nh + 2 * nkv) + 2 * n * nkv * _kv_row(c["kv"], hd) + 8 * n * c["rot"] // 2,
                    flops=n * (nh + nkv) * (4 * hd + 3 * c["rot"]))
    if c["kind"] == "attn":
        rows, lens = _rows_of(c), _attn_lens(c)
        shared = c["shared"] // c["page"] * c["page"]
        held = shared + int((lens - shared).sum())
        seen = int((rows * (lens - rows) + rows * (rows + 1) // 2).sum())
        return dict(bytes=2 * c["nkv"] * held * _kv_row(c["kv"], c["hd"]) + 12 * int(rows.sum()) * c["nh"] * c["hd"],
                    flops=4 * c["nh"] * c["hd"] * seen)
    if c["kind"] == "lora":
        ad, ranks = _lora_shape(c)
        size, on = (4, 2, 2)[c["w"]], ad[ad >= 0]
        rows = _lora_rows(c)
        both = len(rows) * c["cols"] + sum(rows)
        return dict(bytes=size * both * int(ranks[np.unique(on)].sum()) + 4 * c["n"] * c["cols"] + 8 * len(on) * sum(rows),
                    flops=2 * both * int(ranks[on].sum()))
    n, seqs = int(_row0(c)[-1]), c["seqs"]
    fresh = int((_lin_from(c) < 0).sum()) if c["fork"] else 0
    state = HEADS * DK * DV * 4 + 3 * CHANNELS * 4
    return dict(bytes=state * (2 * seqs - fresh) + n * (CHANNELS + 2 * HEADS * DV + 2 * HEADS) * 4 + CHANNELS * CONV_K * 4,
                flops=7 * n * HEADS * DK * DV + 2 * CONV_K * n * CHANNELS)


# ---- the results in 64 bits --------------------------------------------------------------
def exact(case, seed):
    t = prepare(case, seed)["t"]
    return dict(pages=_pages_64, prep=_prep_64, attn=_attn_64, lora=_lora_64, lin=_lin_64)[case["kind"]](case, t)


def _pages_start(c):
    """A start with pages in order (what is copied does not depend on their numbers but for pack)."""
    ln, src, keep, add = _pages_plan(c)
    table, at = [], 0
    perm = np.random.default_rng(1).permutation(c["npages"]).tolist()
    for s in range(c["seqs"]):
        k = -(-int(ln[s]) // c["page"])
        table.append(perm[at:at + k])
        at += k
    return table, ln.tolist(), src.tolist(), keep.tolist(), add.tolist()


def _pages_host(c, table, ln, src, keep, add):
    """The step in Python lists, one sequence after the other."""
    page, seqs = c["page"], c["seqs"]
    keep = [0 if src[s] < 0 else min(keep[s], ln[src[s]]) for s in range(seqs)]
    new = [[] if src[s] < 0 else list(table[src[s]][:-(-keep[s] // page)]) for s in range(seqs)]
    holders = {}
    for s in range(seqs):
        for i, p in enumerate(new[s]):
            writes = add[s] > 0 and keep[s] % page > 0 and i == len(new[s]) - 1
            holders.setdefault(p, []).append((s, writes))
    copies, want = [], []
    for s in range(seqs):
        p = new[s][-1] if new[s] else None
        who = holders.get(p, [])
        if (s, True) in who and len(who) > 1 and not (all(w for _, w in who) and who[0][0] == s):
            copies.append([p, None, keep[s] % page, s])
            new[s].pop()
        want.append(-(-(keep[s] + add[s]) // page) - len(new[s]))
    used = {p for x in new for p in x}
    free = iter(sorted(set(range(c["npages"])) - used))
    for s in range(seqs):
        new[s] += [next(free) for _ in range(want[s])]
    for x in copies:
        x[1] = new[x[3]][-(-keep[x[3]] // page) - 1]
    used = sorted({p for x in new for p in x})
    moves = []
    if c["pack"]:
        holes = sorted(set(range(len(used))) - set(used))
        moves = list(zip([p for p in used if p >= len(used)], holes))
        to = dict(moves)
        new = [[to.get(p, p) for p in x] for x in new]
    return dict(table=new, len=[k + a for k, a in zip(keep, add)], copies=[x[:3] for x in copies], moves=moves,
                out=[0, sum(want), len(used) if c["pack"] else 0, len(moves)])


def _pages_64(c, t):
    table, ln = [[p for p in x if p >= 0] for x in t["table"].tolist()], t["len"].tolist()
    h = _pages_host(c, table, ln, t["src"].tolist(), t["keep"].tolist(), t["add"].tolist())
    wide, kv = t["table"].shape[1], [k.double() for k in t["kv"]]
    for k in kv:
        for a, b, rows in h["copies"]:
            k[b, :, :rows] = k[a, :, :rows]
        for a, b in h["moves"]:
            k[b] = k[a]
    refs = [0] * c["npages"]
    for x in h["table"]:
        for p in x:
            refs[p] += 1
    ints = lambda v: torch.tensor(v, dtype=I32)  # noqa: E731
    return dict(table=ints([x + [-1] * (wide - len(x)) for x in h["table"]]), len=ints(h["len"]), refs=ints(refs),
                out=ints(h["out"]), kv=kv)


def _prep_64(c, t):
    n, hd, h2, page = t["n"], c["hd"], c["rot"] // 2, c["page"]
    q, kc, vc = t["q"].double(), t["kc"].double(), t["vc"].double()
    row0, lens, table, where = (t[k].tolist() for k in ("row0", "len", "table", "where"))
    turn = torch.complex(t["cos"].double(), t["sin"].double())
    for s in range(c["seqs"]):
        for r in range(row0[s], row0[s + 1]):
            w = torch.stack([turn[where[r][a], i] for i, a in enumerate(t["axis"])]) if h2 else None
            slot = lens[s] - row0[s + 1] + r
            for x, norm, put in ((t["q"][r, :, :hd], t["qn"], q[r]), (t["k"][r], t["kn"], kc[table[s][slot // page], :, slot % page])):
                x = x.double()
                x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * norm.double()
                if h2:
                    z = torch.complex(x[:, :h2].contiguous(), x[:, h2:2 * h2].contiguous()) * w
                    x = torch.cat([z.real, z.imag, x[:, 2 * h2:]], 1)
                put[:, :hd] = x
            vc[table[s][slot // page], :, slot % page] = t["v"][r].double()
    return dict(q=q, kc=kc, vc=vc)


def _attn_64(c, t):
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    rep, out = nh // nkv, torch.empty(t["n"], nh, hd, dtype=F64, device="cuda")
    size = nkv * page * hd
    for s in range(c["seqs"]):
        r0, r1, length = int(t["host0"][s]), int(t["host0"][s + 1]), int(t["lens"][s])
        pg = t["table"][s, :-(-length // page)].long()
        last = torch.arange(length - (r1 - r0), length, device="cuda")
        for g in range(nkv):
            k, v = (t[x].index_select(0, pg) for x in ("kc", "vc"))
            if c["kv"] == KV_I8:
                k, v = (x[:, :size].view(-1, nkv, page, hd)[:, g].double()
                        * x[:, size:].contiguous().view(F32).view(-1, nkv, page)[:, g, :, None].double() for x in (k, v))
            else:
                k, v = k[:, g].double(), v[:, g].double()
            k, v = k.reshape(-1, hd)[:length], v.reshape(-1, hd)[:length]
            for h in range(g * rep, g * rep + rep):
                a = (t["q"][r0:r1, h, :hd].double() @ k.T) * float(np.float32(1 / math.sqrt(hd)))
                a[torch.arange(length, device="cuda")[None] > last[:, None]] = -math.inf
                out[r0:r1, h] = torch.softmax(a, 1) @ v
    return dict(o=(out * torch.sigmoid(t["q"][..., hd:].double())).reshape(t["n"], nh * hd))


def _lora_64(c, t):
    ad, scale, ys = t["ad"].tolist(), t["scale"].double(), []
    ranks = [c["rank"]] * c["adapters"] if t["ranks"] is None else t["ranks"].tolist()
    for A, B, y in zip(t["A"], t["B"], t["y"]):
        y = y.double()
        for m in sorted({a for a in ad if a >= 0}):
            at = torch.tensor([r for r, a in enumerate(ad) if a == m], device="cuda")
            low = t["x"][at].double() @ A[m, :ranks[m]].double().T
            y[at] += scale[m] * (low @ B[m, :, :ranks[m]].double().T)
        ys.append(y)
    return dict(y=ys)


def _lin_64(c, t):
    """Sequence by sequence, row by row, with the state's update as one matrix: S (I - beta k k^T) d + beta v k^T."""
    row0, src = t["host0"].tolist(), list(range(c["seqs"])) if t["src"] is None else t["src"].tolist()
    d = {k: t[k].double() for k in ("raw", "z", "b", "a", "conv", "conv_w", "A_log", "dt_bias", "norm")}
    y, conv = torch.zeros(t["n"], HEADS * DV, dtype=F64, device="cuda"), torch.zeros_like(d["conv"])
    rec, eye = torch.zeros(t["rec"].shape, dtype=F64, device="cuda"), torch.eye(DK, dtype=F64, device="cuda")
    zero = torch.zeros(HEADS, DV, DK, dtype=F64, device="cuda")
    for s in range(c["seqs"]):
        S = t["rec"][src[s]].double()[t["at"]] if src[s] >= 0 else zero
        past = d["conv"][src[s]] if src[s] >= 0 else torch.zeros_like(d["conv"][0])
        seen = torch.cat([past, d["raw"][row0[s]:row0[s + 1]]])
        for i, r in enumerate(range(row0[s], row0[s + 1])):
            x = torch.nn.functional.silu((seen[i:i + CONV_K].T * d["conv_w"]).sum(1))
            q, k, v = x.split([HEADS * DK, HEADS * DK, HEADS * DV])
            q, k, v = q.view(HEADS, DK), k.view(HEADS, DK), v.view(HEADS, DV, 1)
            q, k = (e * torch.rsqrt(e.square().sum(1, keepdim=True) + EPS) for e in (q, k))
            beta = torch.sigmoid(d["b"][r])[:, None, None]
            decay = torch.exp(-torch.exp(d["A_log"]) * torch.nn.functional.softplus(d["a"][r] + d["dt_bias"], threshold=50.0))
            kk = k[:, :, None] * k[:, None, :]
            S = decay[:, None, None] * (S @ (eye - beta * kk)) + beta * v * k[:, None, :]
            o = (S @ q[:, :, None])[..., 0] * QSCALE
            o = o * torch.rsqrt(o.square().mean(1, keepdim=True) + EPS) * d["norm"]
            z = d["z"][r].view(HEADS, DV)
            y[r] = (o * z * torch.sigmoid(z)).reshape(-1)
        rec[s, t["at"].reshape(-1)] = S.reshape(-1)
        conv[s] = seen[-(CONV_K - 1):]
    return dict(y=y, conv=conv, rec=rec)
