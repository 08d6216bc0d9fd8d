"""The operators of a tree verify pass, as cases that can be timed and compared.

A speculative round that drafts a tree of tokens (a node's children are the candidates after it) and
verifies it in one pass needs, beside the products and norms of a chain's verify pass:

    attn    gated attention of the tree's nodes over the KV cache: a node sees the context and its
            own ancestors (nmx_attn_tree)
    lin     the Gated DeltaNet mixer with the conv window and the recurrent state of each node taken
            along its ancestors, every node's update logged (nmx_lin_mix_tree)
    sample  tokens drawn from rows of logits with temperature, top-k, top-p and min-p, from given
            uniform numbers (nmx_sample)
    commit  the walk from the root along the drafts that were chosen, and the move of what the walk
            accepted: KV rows, conv states, logged updates (nmx_tree_commit)

Sizes are those of the 0.8B shape (8 query and 2 KV heads of 256, 16 DeltaNet heads of 128 x 128,
conv of 4 over 6144 channels, 18 DeltaNet layers, vocabulary 248320, draft vocabulary 32768) and, in
the drawn cases, of the tests' other head layouts. Where `own` is false, `run` computes them in
elementary torch operations; where it is true, through nibblemac_amd.nmx.Device.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
KV_F32, KV_F16, KV_I8 = 0, 1, 2
VOCAB, DRAFT_VOCAB = 248320, 32768
HEADS, DK, DV, CONV_K = 16, 128, 128, 4          # a DeltaNet layer
CHANNELS = HEADS * (2 * DK + DV)
LOG_ROW = DK + DV + 1                            # k | delta | decay of one head
LIN_LAYERS, KV_LAYERS = 18, 7                    # the MTP layer's cache among the latter
EPS = 1e-6
QSCALE = float(np.float32(1 / math.sqrt(DK)))


# ---- the cases ---------------------------------------------------------------------------
def listed():
    return [
        # a plain sampled step, the usual settings of a chat model
        dict(name="sample_step", kind="sample", n=1, vocab=VOCAB, stride=VOCAB, temperature=0.7,
             top_k=20, top_p=0.8, min_p=0.0, spread=2.0, peaks=40),
        # one draft drawn over the draft vocabulary, min-p alone
        dict(name="sample_draft", kind="sample", n=1, vocab=DRAFT_VOCAB, stride=DRAFT_VOCAB,
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.05, spread=2.0, peaks=20),
        # the rows of a verify pass of 4 drafts at the temperature alone
        dict(name="sample_verify", kind="sample", n=5, vocab=VOCAB, stride=VOCAB, temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0, spread=2.0, peaks=40),
        # every node of a large tree, nucleus sampling from rows without strong peaks
        dict(name="sample_tree", kind="sample", n=64, vocab=VOCAB, stride=VOCAB, temperature=0.8,
             top_k=0, top_p=0.95, min_p=0.0, spread=2.5, peaks=5),
        # a single token (a tree of one node) in a long document's context, binary16 cache
        dict(name="attn_step", kind="attn", n=1, nh=8, nkv=2, hd=256, pos=20000, max_ctx=32768,
             kv=KV_F16),
        # a small tree in a chat's context
        dict(name="attn_chat", kind="attn", n=9, nh=8, nkv=2, hd=256, pos=600, max_ctx=1024,
             kv=KV_F32),
        # a ragged tree in an int8 cache
        dict(name="attn_ragged", kind="attn", n=37, nh=8, nkv=2, hd=256, pos=4001, max_ctx=8192,
             kv=KV_I8),
        # the largest tree over a book, binary16 cache
        dict(name="attn_book", kind="attn", n=64, nh=8, nkv=2, hd=256, pos=100000, max_ctx=131072,
             kv=KV_F16),
        # a DeltaNet layer over a small tree, two accepted tokens of the last round replayed first
        dict(name="lin_small", kind="lin", n=9, keep=2),
        # the largest tree
        dict(name="lin_tree", kind="lin", n=64, keep=5),
        # a small tree whose first branch was accepted, chat context
        dict(name="commit_small", kind="commit", n=9, accept=3, pos=600, max_ctx=1024, kv=KV_F32),
        # the largest tree, a deep branch accepted
        dict(name="commit_tree", kind="commit", n=64, accept=9, pos=4001, max_ctx=8192, kv=KV_F16),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "sample", "attn", "attn", "attn", "lin", "commit"])
    kv = rng.choice([KV_F32, KV_F16, KV_I8])
    if kind == "sample":
        n, vocab = _log(rng, 1, 64), _log(rng, 100, VOCAB)
        return dict(kind=kind, n=n, vocab=vocab, stride=vocab + rng.choice([0, 0, 1, 32]),
                    temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5]),
                    top_k=rng.choice([0, 0, 1, 20, 50, _log(rng, 2, vocab)]),
                    top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.999]),
                    min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), spread=rng.choice([0.5, 2.0, 2.5, 4.0]),
                    peaks=rng.choice([0, 5, 40]))
    if kind == "attn":
        n = _log(rng, 1, 64)
        nh, nkv, hd = rng.choice([(8, 2, 256), (8, 2, 256), (8, 2, 256), (6, 2, 128), (4, 4, 64),
                                  (16, 2, 256), (8, 1, 512), (4, 2, 192)])
        pos = _log(rng, 1, min(100000 if kv else 50000, 6400000 * 8 * 256 // (n * nh * hd)))
        return dict(kind=kind, n=n, nh=nh, nkv=nkv, hd=hd, pos=pos - 1,
                    max_ctx=pos - 1 + n + _log(rng, 1, 30000), kv=kv)
    if kind == "lin":
        return dict(kind=kind, n=_log(rng, 1, 64), keep=rng.randint(0, 8))
    n = _log(rng, 1, 64)
    return dict(kind=kind, n=n, accept=rng.randint(0, min(n - 1, 8)), pos=_log(rng, 1, 4000),
                max_ctx=rng.choice([4096, 5000]), kv=kv)


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

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=I32)

    def tree(self, n, spine=0):
        """Parents of n nodes in an order that puts parents first: node 0 is the root, a node's
        parent one of the 12 nodes before it; a branch of `spine` drafts at nodes of its own."""
        parent = np.full(n, -1, np.int64)
        for t in range(1, n):
            parent[t] = self.host.integers(max(0, t - 12), t)
        if spine:
            path = np.concatenate([[0], 1 + np.sort(self.host.choice(n - 1, spine, replace=False))])
            parent[path[1:]] = path[:-1]
            return torch.tensor(parent, device="cuda", dtype=I32), path
        return torch.tensor(parent, device="cuda", dtype=I32), None

    def cache(self, kv, nkv, ctx, hd):
        """KV rows of unit variance in the cache's format (int8 rows with their scales behind)."""
        rows = self.normal(nkv, ctx, hd)
        if kv == KV_F32:
            return rows
        if kv == KV_F16:
            return rows.half()
        amax = rows.abs().amax(2)
        codes = torch.round(rows * (127.0 / amax)[..., None]).to(torch.int8)
        return torch.cat([codes.reshape(-1), (amax / 127.0).reshape(-1).view(torch.int8)])


def _state_at():
    """Position of element (head, column j, key i) of the recurrent state: columns in groups of 16,
    within a group the float4 slot of every lane contiguous (nmx_state_index, include/nmx.h)."""
    h, j, i = torch.meshgrid(*(torch.arange(d, device="cuda") for d in (HEADS, DV, DK)), indexing="ij")
    return (h * DV + j // 16 * 16) * DK + ((i % (DK // 4)) // 4 * 64 + 4 * (j % 16) + i // (DK // 4)) * 4 + i % 4


def _sample_inputs(c, x):
    n, vocab, stride = c["n"], c["vocab"], c["stride"]
    logits = x.normal(n, stride, std=c["spread"])
    if c["peaks"]:      # the few tokens that a trained model prefers
        at = x.ints(0, vocab, n, c["peaks"]).long()
        logits.scatter_add_(1, at, x.uniform(3.0, 12.0, n, c["peaks"]))
    par = torch.tensor([[c["temperature"], c["top_p"], c["min_p"], 0.0]], device="cuda", dtype=F32).repeat(n, 1)
    par.view(I32)[:, 3] = c["top_k"]    # records of three floats and a whole number
    return dict(logits=logits, par=par, u=torch.rand(n, generator=x.g, device="cuda", dtype=F32),
                tok=torch.zeros(n, device="cuda", dtype=I32), prob=torch.zeros(n, device="cuda", dtype=F32))


def _attn_inputs(c, x):
    n, nh, nkv, hd, ctx = c["n"], c["nh"], c["nkv"], c["hd"], c["max_ctx"]
    parent, _ = x.tree(n)
    return dict(q=x.normal(n, nh, 2 * hd), kc=x.cache(c["kv"], nkv, ctx, hd), vc=x.cache(c["kv"], nkv, ctx, hd),
                parent=parent, pos=torch.tensor([c["pos"]], device="cuda", dtype=I32),
                o=torch.zeros(n, nh * hd, device="cuda", dtype=F32))


def _lin_inputs(c, x):
    n, keep = c["n"], c["keep"]
    parent, _ = x.tree(n)
    pend = x.normal(max(keep, 1), HEADS, LOG_ROW, std=0.1)
    pend[:, :, DK + DV] = x.uniform(0.9, 0.99, max(keep, 1), HEADS)
    zeros = lambda *s: torch.zeros(s, device="cuda", dtype=F32)  # noqa: E731
    return dict(parent=parent, raw=x.normal(n, CHANNELS), z=x.normal(n, HEADS * DV), b=x.normal(n, HEADS),
                a=x.normal(n, HEADS), conv=x.normal(CONV_K - 1, CHANNELS, std=0.5),
                conv_w=x.uniform(-0.5, 0.5, CHANNELS, CONV_K),
                A_log=x.uniform(math.log(0.2), math.log(0.4), HEADS), dt_bias=x.uniform(-4.5, -3.5, HEADS),
                norm=x.uniform(0.8, 1.2, DV), rec=x.normal(HEADS * DV * DK, std=0.05), pend=pend, at=_state_at(),
                cv=zeros(n, CHANNELS), beta=zeros(n, HEADS), decay=zeros(n, HEADS), o=zeros(n, HEADS * DV),
                y=zeros(n, HEADS * DV), log=zeros(n, HEADS, LOG_ROW), xin=zeros(n, CHANNELS))


def _commit_inputs(c, x):
    n, accept = c["n"], c["accept"]
    parent, path = x.tree(n, accept)
    path = path if path is not None else np.zeros(1, np.int64)
    tok = x.host.permutation(VOCAB)[:2 * n]
    choice = tok[n:].copy()             # tokens that no node has
    tok = tok[:n]
    choice[path[:-1]] = tok[path[1:]]   # but along the accepted branch
    if accept:                          # a later child of the root with the accepted child's token
        par = parent.cpu().numpy()
        twin = [t for t in range(path[1] + 1, n) if par[t] == 0]
        if twin:
            tok[twin[0]] = tok[path[1]]
    dev = lambda v: torch.tensor(v, device="cuda", dtype=I32)  # noqa: E731
    return dict(parent=parent, tok=dev(tok), choice=dev(choice), pos=dev([c["pos"]]), out=dev([-7] * (2 + n)),
                state=x.normal(LIN_LAYERS, CONV_K - 1, CHANNELS), xin=x.normal(LIN_LAYERS, n, CHANNELS),
                log=x.normal(LIN_LAYERS, n, HEADS * LOG_ROW), pend=x.normal(LIN_LAYERS, n, HEADS * LOG_ROW),
                kv=[x.cache(c["kv"], 2, c["max_ctx"], 256) for _ in range(2 * KV_LAYERS)])


def prepare(case, seed):
    """The inputs on the GPU and the buffers that a program holds for its outputs."""
    made = dict(sample=_sample_inputs, attn=_attn_inputs, lin=_lin_inputs, commit=_commit_inputs)
    return dict(case=case, t=made[case["kind"]](case, _Inputs(seed)), call=None)


# ---- the framework's calls ---------------------------------------------------------------
_device = None


def _dev():
    """The program's one context (a device and its stream)."""
    global _device
    if _device is None:
        from nibblemac_amd.nmx import Device

        _device = Device(0)
    return _device


def _p(t):
    return None if t is None else t.data_ptr()


def _sample_call(c, t):
    dev, n = _dev(), c["n"]
    work = torch.empty(dev.sample_work_bytes(n, c["vocab"]), dtype=torch.uint8, device="cuda")
    args = [_p(t[k]) for k in ("logits", "par", "u", "tok", "prob")]

    def call():
        logits, par, u, tok, prob = args
        dev.sample(logits, c["stride"], c["vocab"], n, par, u, work.data_ptr(), tok, prob=prob)
        return dict(tok=t["tok"], prob=t["prob"])

    return call


def _attn_call(c, t):
    from nibblemac_amd.nmx import A8, AttnArgs

    dev = _dev()
    work = torch.empty(dev.attn_tree_work_bytes(c["n"], c["nh"], c["nkv"], c["hd"]), dtype=torch.uint8,
                       device="cuda")
    a = AttnArgs(n=c["n"], nh=c["nh"], nkv=c["nkv"], hd=c["hd"], max_ctx=c["max_ctx"], q=_p(t["q"]),
                 scale=np.float32(1 / math.sqrt(c["hd"])), kc=_p(t["kc"]), vc=_p(t["vc"]), pos=_p(t["pos"]),
                 pos_off=0, o=_p(t["o"]), a8=A8(None, None, None), kv_dtype=c["kv"])
    parent = _p(t["parent"])

    def call():
        dev.attn_tree(a, parent, work.data_ptr())
        return dict(o=t["o"])

    return call


def _lin_call(c, t):
    from nibblemac_amd.nmx import A8, LinArgs, LinMixArgs, LinPreArgs

    dev, n, vd = _dev(), c["n"], HEADS * DV
    pre = LinPreArgs(n, CHANNELS, CONV_K, DK, HEADS * DK, _p(t["raw"]), CHANNELS, _p(t["cv"]), _p(t["conv"]),
                     _p(t["conv_w"]), _p(t["xin"]), QSCALE, EPS, _p(t["b"]), _p(t["a"]), HEADS, HEADS,
                     _p(t["A_log"]), None, _p(t["dt_bias"]), _p(t["beta"]), _p(t["decay"]))
    rule = LinArgs(n, HEADS, 1, DK, DV, CHANNELS, vd, _p(t["cv"]), _p(t["decay"]), _p(t["beta"]), _p(t["rec"]),
                   _p(t["o"]), _p(t["log"]), _p(t["pend"]), c["keep"], 1, None)
    args = LinMixArgs(pre, rule, _p(t["z"]), vd, _p(t["norm"]), EPS, _p(t["y"]), vd, A8(None, None, None))
    parent = _p(t["parent"])

    def call():
        dev.lin_mix_tree(args, parent)
        return {k: t[k] for k in ("y", "log", "rec", "xin")}

    return call


def _commit_call(c, t):
    from nibblemac_amd.nmx import tree_commit_args

    dev, n = _dev(), c["n"]
    args = tree_commit_args(n, _p(t["parent"]), _p(t["tok"]), _p(t["choice"]), _p(t["out"]),
                            lin=dict(layers=LIN_LAYERS, C=CHANNELS, conv_k=CONV_K, state=_p(t["state"]),
                                     xin=_p(t["xin"]), log=_p(t["log"]), pend=_p(t["pend"]), cap=n,
                                     row=HEADS * LOG_ROW),
                            kv=dict(caches=[_p(k) for k in t["kv"]], nkv=2, max_ctx=c["max_ctx"], hd=256,
                                    kv_dtype=c["kv"], pos=_p(t["pos"])))

    def call():
        dev.tree_commit(args)
        return _commit_out(t)

    return call


def run(state):
    c, t = state["case"], state["t"]
    if not own:
        return dict(sample=_sample_plain, attn=_attn_plain, lin=_lin_plain, commit=_commit_plain)[c["kind"]](c, t)
    if state["call"] is None:
        state["call"] = dict(sample=_sample_call, attn=_attn_call, lin=_lin_call, commit=_commit_call)[c["kind"]](c, t)
    return state["call"]()


# ---- the plain forms ---------------------------------------------------------------------
def _sample_plain(c, t):
    """Weights exp((l - max) / T) in 64 bits. In descending order (ties: lowest index first) the
    first top_k, of these the shortest run whose mass reaches top_p, of these the weights of at least
    min_p times the largest; the token where the running mass in index order passes u times the
    whole. T = 0: the first maximum."""
    n, vocab = c["n"], c["vocab"]
    l = t["logits"][:, :vocab]
    T, top_p, min_p = (t["par"][:, i:i + 1].double() for i in range(3))
    top_k = t["par"].view(I32)[:, 3:4].long()
    best = l.max(1, keepdim=True).values
    first = (l == best).to(I32).argmax(1).to(I32)
    w = torch.exp((l.double() - best.double()) / torch.where(T > 0, T, 1.0))
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    ws, rank = w.gather(1, order), torch.arange(vocab, device=l.device)
    ws = torch.where((top_k > 0) & (rank >= top_k), 0.0, ws)
    mass = ws.cumsum(1)
    ws = torch.where((top_p < 1) & (rank > 0) & (mass - ws >= top_p * mass[:, -1:]), 0.0, ws)
    ws = torch.where(ws >= min_p, ws, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    run_ = kept.cumsum(1)
    hit = (run_ > t["u"].double()[:, None] * run_[:, -1:]) & (kept > 0)
    tok = hit.to(I32).argmax(1)
    prob = kept.gather(1, tok[:, None])[:, 0] / run_[:, -1]
    greedy = (T <= 0)[:, 0]
    return dict(tok=torch.where(greedy, first, tok.to(I32)), prob=torch.where(greedy, 1.0, prob).float())


def _ancestors(parent):
    """[n][n] truth: column s is row t itself or one of its ancestors."""
    n = parent.numel()
    step = torch.eye(n, device=parent.device, dtype=F64)
    step = step + (parent[:, None] == torch.arange(n, device=parent.device)[None, :]).double()
    return torch.linalg.matrix_power(step.clamp(max=1.0), n) > 0


def _rows32(cache, kv, nkv, ctx, hd, upto):
    """The first `upto` rows of every KV head, in 32 bits."""
    if kv != KV_I8:
        return cache[:, :upto].float()
    codes = cache[:nkv * ctx * hd].view(nkv, ctx, hd)[:, :upto].float()
    return codes * cache[nkv * ctx * hd:].view(F32).view(nkv, ctx)[:, :upto, None]


def _attn_plain(c, t):
    n, nh, nkv, hd, ctx, pos = c["n"], c["nh"], c["nkv"], c["hd"], c["max_ctx"], c["pos"]
    rep, length = nh // nkv, pos + n
    k, v = (_rows32(t[x], c["kv"], nkv, ctx, hd, length) for x in ("kc", "vc"))
    q = t["q"][..., :hd].reshape(n, nkv, rep, hd).permute(1, 0, 2, 3).reshape(nkv, n * rep, hd)
    s = (torch.bmm(q.contiguous(), k.transpose(1, 2).contiguous()) * float(np.float32(1 / math.sqrt(hd)))).view(nkv, n, rep, length)
    s[..., pos:].masked_fill_(~_ancestors(t["parent"])[None, :, None, :], -math.inf)
    p = torch.exp(s - s.amax(3, keepdim=True))
    o = torch.bmm(p.view(nkv, n * rep, length), v.contiguous()).view(nkv, n, rep, hd) / p.sum(3, keepdim=True)
    o = o.permute(1, 0, 2, 3).reshape(n, nh, hd)
    return dict(o=(o / (1 + torch.exp(-t["q"][..., hd:]))).reshape(n, nh * hd))


def _lin_plain(c, t):
    """The recurrence node by node, each from its parent's state."""
    n, dev = c["n"], t["raw"].device
    parent = t["parent"].long()
    # the conv window: the node, its ancestors, then the state's rows (the newest last)
    rows = torch.cat([t["conv"], t["raw"]])                      # node t is row t + K - 1
    above = torch.cat([torch.arange(-1, CONV_K - 2, device=dev).clamp(min=0),
                       torch.where(parent < 0, CONV_K - 2, parent + CONV_K - 1)])
    up = torch.arange(n, device=dev) + CONV_K - 1
    win = [up, above[up], above[above[up]], above[above[above[up]]]]
    acc = sum(t["conv_w"][:, CONV_K - 1 - j] * rows[at] for j, at in enumerate(win))
    conv = acc / (1 + torch.exp(-acc))
    q, k = (conv[:, i * HEADS * DK:(i + 1) * HEADS * DK].view(n, HEADS, DK) for i in (0, 1))
    v = conv[:, 2 * HEADS * DK:].view(n, HEADS, DV)
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
    q = q * QSCALE
    beta = 1 / (1 + torch.exp(-t["b"]))
    sp = t["a"] + t["dt_bias"]
    sp = torch.where(sp > 20, sp, torch.log1p(torch.exp(sp)))
    decay = torch.exp(-torch.exp(t["A_log"]) * sp)
    R = t["rec"][t["at"]]                                        # [heads][dv][dk]
    for r in t["pend"][:c["keep"]]:
        R = R * r[:, DK + DV, None, None] + r[:, DK:DK + DV, None] * r[:, None, :DK]
    if c["keep"]:
        t["rec"][t["at"].reshape(-1)] = R.reshape(-1)
    states = torch.empty(n + 1, *R.shape, device=dev)            # row 0: before the tree
    states[0] = R
    for i in range(n):
        S = states.index_select(0, parent[i:i + 1] + 1)[0] * decay[i, :, None, None]
        delta = (v[i] - (S * k[i, :, None, :]).sum(-1)) * beta[i, :, None]
        states[i + 1] = S + delta[:, :, None] * k[i, :, None, :]
        t["o"][i] = (states[i + 1] * q[i, :, None, :]).sum(-1).view(-1)
        t["log"][i] = torch.cat([k[i], delta, decay[i, :, None]], 1)
    o = t["o"].view(n, HEADS, DV)
    y = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * t["norm"]
    z = t["z"]
    return dict(y=y.reshape(n, -1) * (z / (1 + torch.exp(-z))), log=t["log"], rec=t["rec"], xin=t["raw"].clone())


def _commit_out(t):
    """The state after a commit: it computes nothing, so int8 caches are whole numbers to it."""
    return {k: t[k] for k in ("out", "state", "pend", "kv")}


def _commit_plain(c, t):
    n, pos, ctx, dev = c["n"], c["pos"], c["max_ctx"], t["tok"].device
    parent, at = t["parent"].long(), torch.arange(n, device=t["tok"].device)
    hit = (t["tok"] == t["choice"][parent.clamp(min=0)]) & (parent >= 0)
    twin = (parent[:, None] == parent[None, :]) & hit[None, :] & (at[None, :] < at[:, None])
    hit = (hit & ~twin.any(1)) | (at == 0)                       # the first child that matches
    on = ~(_ancestors(t["parent"]) & ~hit[None, :]).any(1)       # every ancestor matches
    src = torch.sort(torch.where(on, at, at + n)).values         # the path first
    e = on.sum()
    src = torch.where(at < e, src, at)
    last = t["choice"][src[e - 1]]
    t["out"].copy_(torch.cat([(e - 1)[None].to(I32), last[None], torch.where(at < e, src, -1).to(I32)]))
    t["pend"].copy_(torch.where((at < e)[None, :, None], t["log"][:, src], t["pend"]))
    rows = torch.cat([t["state"], t["xin"][:, src]], 1)
    t["state"].copy_(rows[:, e + torch.arange(CONV_K - 1, device=dev)])
    for k in t["kv"]:
        r = k if c["kv"] != KV_I8 else k[:2 * ctx * 256].view(2, ctx, 256)
        r[:, pos:pos + n] = r[:, pos + src]
        if c["kv"] == KV_I8:
            s = k[2 * ctx * 256:].view(F32).view(2, ctx)
            s[:, pos:pos + n] = s[:, pos + src]
    return _commit_out(t)


# ---- what a pass cannot do without -------------------------------------------------------
def _kv_row(kv, hd):
    return hd + 4 if kv == KV_I8 else hd * (2 if kv == KV_F16 else 4)


def work(case):
    c, n = case, case["n"]
    if c["kind"] == "sample":      # a weight's exponential: about ten products and sums
        return dict(bytes=n * (4 * c["vocab"] + 28), flops=n * c["vocab"] * (10 if c["temperature"] > 0 else 1))
    if c["kind"] == "attn":
        length, hd = c["pos"] + n, c["hd"]
        return dict(bytes=2 * c["nkv"] * length * _kv_row(c["kv"], hd) + 12 * n * c["nh"] * hd,
                    flops=4 * n * c["nh"] * hd * (c["pos"] + 1))
    if c["kind"] == "lin":
        by = HEADS * DK * DV * 4 * (2 if c["keep"] else 1) + (n + c["keep"]) * HEADS * LOG_ROW * 4
        by += n * CHANNELS * 4 * 2 + n * HEADS * (2 * DV + 2) * 4 + CHANNELS * (CONV_K * 2 - 1) * 4
        return dict(bytes=by, flops=HEADS * DK * DV * (4 * n + 3 * c["keep"]) + 2 * CONV_K * n * CHANNELS)
    e = c["accept"] + 1
    by = 2 * LIN_LAYERS * 4 * (e * HEADS * LOG_ROW + (CONV_K - 1) * CHANNELS)
    return dict(bytes=by + 2 * 2 * KV_LAYERS * 2 * c["accept"] * _kv_row(c["kv"], 256), flops=0)


# ---- the results in 64 bits --------------------------------------------------------------
def exact(case, seed):
    t = prepare(case, seed)["t"]
    return dict(sample=_sample_64, attn=_attn_64, lin=_lin_64, commit=_commit_64)[case["kind"]](case, t)


def _sample_64(c, t):
    n, vocab = c["n"], c["vocab"]
    logits, u = t["logits"][:, :vocab].cpu().numpy().astype(np.float64), t["u"].cpu().numpy().astype(np.float64)
    T, top_p, min_p = (float(np.float32(c[k])) for k in ("temperature", "top_p", "min_p"))
    tok, prob = np.zeros(n, np.int64), np.ones(n)
    for r in range(n):
        l = logits[r]
        if T <= 0:
            tok[r] = np.argmax(l)
            continue
        order = np.lexsort((np.arange(vocab), -l))
        if c["top_k"] > 0:
            order = order[:c["top_k"]]
        p = np.exp((l[order] - l[order[0]]) / T)
        if top_p < 1:
            reach = np.cumsum(p)
            order = order[:1 + np.searchsorted(reach, top_p * reach[-1])]
            p = p[:len(order)]
        order = np.sort(order[p >= min_p])
        p = np.exp((l[order] - l.max()) / T)
        reach = np.cumsum(p)
        i = np.searchsorted(reach, u[r] * reach[-1], side="right")
        tok[r], prob[r] = order[i], p[i] / reach[-1]
    return dict(tok=torch.tensor(tok, dtype=I32), prob=torch.tensor(prob))


def _attn_64(c, t):
    n, nh, nkv, hd, ctx, pos = c["n"], c["nh"], c["nkv"], c["hd"], c["max_ctx"], c["pos"]
    par, seen = t["parent"].tolist(), torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = par[j]
    hide = ~torch.cat([torch.ones(n, pos, dtype=torch.bool), seen], 1).cuda()
    out = torch.empty(n, nh, hd, dtype=F64, device="cuda")
    for h in range(nh):
        g = h // (nh // nkv)
        if c["kv"] == KV_I8:
            at = slice(g * ctx * hd, (g * ctx + pos + n) * hd)
            k, v = (t[x][at].double().view(-1, hd) * t[x][nkv * ctx * hd:].view(F32)[g * ctx:g * ctx + pos + n, None].double()
                    for x in ("kc", "vc"))
        else:
            k, v = (t[x][g, :pos + n].double() for x in ("kc", "vc"))
        s = (t["q"][:, h, :hd].double() @ k.T) * float(np.float32(1 / math.sqrt(hd)))
        out[:, h] = torch.softmax(s.masked_fill(hide, -math.inf), 1) @ v
    return dict(o=(out * torch.sigmoid(t["q"][..., hd:].double())).reshape(n, nh * hd))


def _lin_64(c, t):
    """In closed form: with G the product of the decays along a node's ancestors, a node's delta
    solves a triangular system over its ancestors and its output is a sum over them."""
    n = c["n"]
    par, K1 = t["parent"].tolist(), CONV_K - 1
    d = {k: v.double() for k, v in t.items() if torch.is_tensor(v) and v.dtype == F32}
    rows, conv = torch.cat([d["conv"], d["raw"]]), torch.empty_like(d["raw"])
    for i in range(n):
        chain, j = [], i
        while j >= 0:
            chain.append(j + K1)
            j = par[j]
        chain = (chain + list(range(K1 - 1, -1, -1)))[:CONV_K][::-1]
        conv[i] = (rows[chain] * d["conv_w"].T).sum(0)
    conv = conv * torch.sigmoid(conv)
    q, k, v = (conv[:, i * HEADS * DK:(i + 1) * HEADS * DK].view(n, HEADS, DK).transpose(0, 1) for i in range(3))
    q, k = (torch.nn.functional.normalize(x, dim=2, eps=0) * torch.sqrt(1 - EPS / ((x * x).sum(2, keepdim=True) + EPS))
            for x in (q, k))
    beta = torch.sigmoid(d["b"]).T
    logdec = (-torch.exp(d["A_log"]) * torch.nn.functional.softplus(d["a"] + d["dt_bias"], threshold=50.0)).T
    seen, path = torch.zeros(n, n, dtype=F64, device="cuda"), torch.zeros(n, dtype=F64, device="cuda")
    for i in range(n):
        if par[i] >= 0:
            seen[i] = seen[par[i]]
        seen[i, i] = 1
    cum = logdec @ seen.T                                        # the decays from the state to a node
    R = d["rec"][t["at"]]
    for r in d["pend"][:c["keep"]]:
        R = torch.addcmul(R * r[:, None, DK + DV:], r[:, DK:DK + DV, None], r[:, None, :DK])
    gap = torch.exp((cum[:, :, None] - cum[:, None, :]).clamp(max=0)) * seen
    A = beta[:, :, None] * gap * (k @ k.transpose(1, 2)) * (1 - torch.eye(n, device="cuda", dtype=F64))
    rhs = beta[:, :, None] * (v - torch.exp(cum)[:, :, None] * (k @ R.transpose(1, 2)))
    delta = torch.linalg.solve_triangular(A + torch.eye(n, device="cuda", dtype=F64), rhs, upper=False)
    o = torch.exp(cum)[:, :, None] * (q @ R.transpose(1, 2)) + (gap * (q @ k.transpose(1, 2))) @ delta
    o = (o * QSCALE).transpose(0, 1)
    y = o * torch.rsqrt((o * o).mean(2, keepdim=True) + EPS) * d["norm"]
    z = d["z"].view(n, HEADS, DV)
    rec = torch.empty_like(d["rec"])
    rec[t["at"].reshape(-1)] = R.reshape(-1)
    log = torch.cat([k, delta, torch.exp(logdec)[:, :, None]], 2).transpose(0, 1)
    return dict(y=(y * z * torch.sigmoid(z)).reshape(n, -1), log=log, rec=rec, xin=d["raw"])


def _commit_64(c, t):
    n, pos = c["n"], c["pos"]
    par, tok, choice = (t[k].tolist() for k in ("parent", "tok", "choice"))
    path = [0]
    while True:
        nxt = [i for i in range(n) if par[i] == path[-1] and tok[i] == choice[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    e, pend = len(path), t["pend"].double()
    pend[:, :e] = t["log"][:, path].double()
    state = torch.cat([t["state"], t["xin"][:, path]], 1)[:, -(CONV_K - 1):].double()
    kv = [None if c["kv"] == KV_I8 else k.double() for k in t["kv"]]
    for r in kv:
        if r is not None:
            r[:, pos:pos + e] = r[:, [pos + i for i in path]]
    out = [e - 1, choice[path[-1]]] + path + [-1] * (n - e)
    return dict(out=torch.tensor(out, dtype=I32), state=state, pend=pend, kv=kv)
