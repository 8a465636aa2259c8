"""Measured cases of the operators around drafted tokens and the int8 cache.

Kinds:
  rope    per-head norms of q and k, and the rotation, of fused qkv rows at the
          positions of a draft tree or of consecutive tokens
  cache   K/V rows quantised into an int8 cache as they are written, the
          accepted path's rows kept, and those rows read back
  attend  attention of a draft tree (or of consecutive tokens) over an f32 or an
          int8 cache
  draft   a drafted chain against the target's probabilities, by rejection
  tree    a drafted tree against the target's probabilities, by sampled tokens

Sequence s of a batch has context length _lens(case)[s]; draft node i of it
lies at cache row len + i; its parent is parents[s][i] (-1: the context).
"""
import math
import random

import numpy as np
import torch
import torch.utils.dlpack

own = False  # run() computes plain forms; true: it calls the framework's operators

# (query heads, KV heads, head size) of this repository's configurations: the
# smallest model, the 7B and the 8B shape; GPT-2 small's and Whisper large's
# heads; then head sizes off the powers of two
TINY = dict(nq=6, nkv=6, hd=48)
L7B = dict(nq=32, nkv=32, hd=128)
L8B = dict(nq=32, nkv=8, hd=128)
OTHER = [dict(nq=12, nkv=12, hd=64), dict(nq=20, nkv=20, hd=64), dict(nq=10, nkv=2, hd=80), dict(nq=9, nkv=3, hd=100)]
EPS = 1e-6


def listed():
    return [
        # one decode token of the 8B shape: nothing but latency
        dict(name="rope_token_8b", kind="rope", **L8B, seqs=1, rows=1, start=511, tree=False, norm=True),
        # a long prompt's q, k and v of the 7B shape
        dict(name="rope_prompt_7b", kind="rope", **L7B, seqs=1, rows=2047, start=0, tree=False, norm=False),
        # eight sequences' draft trees written, the accepted paths kept
        dict(name="cache_tree_8b", kind="cache", **L8B, seqs=8, rows=26, start=1000, keep=5),
        # a prompt written and read back whole
        dict(name="cache_prompt_7b", kind="cache", **L7B, seqs=1, rows=2047, start=0, keep=0),
        # one token of the smallest model over a short f32 cache: latency
        dict(name="attend_token_tiny", kind="attend", **TINY, seqs=1, rows=1, len=77, tree=False, cache="f32"),
        # four sequences' draft trees over the f32 cache
        dict(name="attend_tree_8b", kind="attend", **L8B, seqs=4, rows=26, len=2047, tree=True, cache="f32"),
        # one token over a long int8 context
        dict(name="attend_long_8b_int8", kind="attend", **L8B, seqs=1, rows=1, len=65001, tree=False, cache="int8"),
        # wide trees of eight sequences over int8 caches
        dict(name="attend_tree_8b_int8", kind="attend", **L8B, seqs=8, rows=64, len=4000, tree=True, cache="int8"),
        # the next chunk of a prompt over an int8 cache
        dict(name="attend_chunk_7b_int8", kind="attend", **L7B, seqs=1, rows=512, len=1500, tree=False, cache="int8"),
        # a short drafted chain of one request
        dict(name="draft_7b", kind="draft", vocab=32000, seqs=1, rows=4),
        # sixteen requests' chains, the largest vocabulary
        dict(name="draft_8b", kind="draft", vocab=128256, seqs=16, rows=8),
        # four requests' drafted trees
        dict(name="tree_8b", kind="tree", vocab=128256, seqs=4, rows=31),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "cache", "attend", "attend", "attend", "draft", "tree"])
    dims = dict(rng.choice([TINY, L7B, L8B, L8B] + OTHER))
    seqs = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    heads = dims["nq"] + 2 * dims["nkv"]
    if kind == "rope":
        tree = rng.random() < 0.5
        rows = _log(rng, 1, 64 if tree else max(2, min(4096, 2047 * 96 * 128 // (heads * dims["hd"] * seqs))))
        return dict(kind=kind, **dims, seqs=seqs, rows=rows, start=_log(rng, 1, 100000), tree=tree, norm=rng.random() < 0.6)
    if kind == "cache":
        keep = rng.randint(1, 8) if rng.random() < 0.6 else 0
        rows = _log(rng, max(1, 2 * keep), 64) if keep else _log(rng, 1, max(2, min(4096, 2047 * 32 * 128 // (dims["nkv"] * dims["hd"] * seqs))))
        return dict(kind=kind, **dims, seqs=seqs, rows=rows, start=_log(rng, 1, 2000) - 1, keep=keep)
    if kind == "attend":
        cache = rng.choice(["f32", "int8", "int8"])
        shape = rng.choice(["token", "tree", "tree", "chunk"])
        rows = 1 if shape == "token" else _log(rng, 2, 64) if shape == "tree" else _log(rng, 2, 768)
        # products at most the widest listed trees', cache at most the longest's
        most = min(64 * 4000 * 32 * 128 * 8 // (rows * dims["nq"] * dims["hd"] * seqs), 8 * 4000 * 8 * 128 // (dims["nkv"] * dims["hd"] * seqs), 65001)
        return dict(kind=kind, **dims, seqs=seqs, rows=rows, len=_log(rng, 1, max(2, most - rows)) - 1, tree=shape == "tree", cache=cache)
    vocab = rng.choice([32000, 50257, 128256, _log(rng, 1000, 128256)])
    rows = _log(rng, 1, 16) if kind == "draft" else _log(rng, 2, 64)
    return dict(kind=kind, vocab=vocab, seqs=max(1, min(seqs, 16 * 9 * 128256 // ((rows + 1) * vocab))), rows=rows)


def _lens(c):
    """Context lengths of the batch's sequences: ragged, the first the longest."""
    n = c["len"] if c["kind"] == "attend" else c["start"]
    return [n - s * n // (2 * c["seqs"]) for s in range(c["seqs"])]


def _chain(c):
    return np.tile(np.arange(-1, c["rows"] - 1, dtype=np.int64), (c["seqs"], 1))


def _tree(c, seed):
    """parents [seqs, rows]: a few children a node, paths of some length."""
    r = random.Random(int(seed) * 131 + 7)
    return np.array([[-1 if i == 0 else r.randint(max(-1, i - 7), i - 1) for i in range(c["rows"])] for _ in range(c["seqs"])],
                    dtype=np.int64)


# ------------------------------------------------------------------- inputs
class _Draw:
    """Seeded tensors on the GPU, the same for prepare and exact."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std).add_(mean)

    def heads(self, *shape):
        # key and query rows: a few channels carry larger values
        x = self.normal(*shape)
        x[..., torch.randint(0, shape[-1], (2,), generator=self.g, device="cuda")] *= 5.0
        return x


def _inputs(c, seed):
    d = _Draw(seed)
    if c["kind"] == "rope":
        hd = c["hd"]
        t = dict(qkv=d.heads(c["seqs"] * c["rows"], c["nq"] + 2 * c["nkv"], hd),
                 freqs=(500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)).float())
        if c["norm"]:
            t["qw"], t["kw"] = d.normal(hd, std=0.1, mean=1.0), d.normal(hd, std=0.1, mean=1.0)
        t["parents"] = _tree(c, seed) if c["tree"] else None
        return t
    if c["kind"] == "cache":
        t = dict(k=d.heads(c["seqs"], c["rows"], c["nkv"], c["hd"]), v=d.normal(c["seqs"], c["rows"], c["nkv"], c["hd"]))
        r = random.Random(int(seed) * 17 + 3)  # the accepted nodes, in order
        t["paths"] = np.array([sorted(r.sample(range(c["rows"]), c["keep"])) for _ in range(c["seqs"])], dtype=np.int64) if c["keep"] else None
        return t
    if c["kind"] == "attend":
        n = c["len"] + c["rows"]
        t = dict(q=d.heads(c["seqs"], c["rows"], c["nq"], c["hd"]), k=d.heads(c["seqs"], n, c["nkv"], c["hd"]),
                 v=d.normal(c["seqs"], n, c["nkv"], c["hd"]))
        t["parents"] = _tree(c, seed) if c["tree"] else None
        return t
    # a model's next-token distributions: most of the mass on a few tokens of
    # each row, drafted by a smaller model that sees them with some noise
    n, m, V = c["seqs"], c["rows"], c["vocab"]
    lg = d.normal(n, m + 1, V, std=1.5)
    lg.scatter_add_(2, torch.randint(0, V, (n, m + 1, 6), generator=d.g, device="cuda"), d.normal(n, m + 1, 6, mean=12.0))
    near = lg + d.normal(n, m + 1, V, std=0.5)
    t = dict(p=torch.softmax(lg, -1), u=torch.rand(n, m + 1, generator=d.g, device="cuda", dtype=torch.float64))
    if c["kind"] == "draft":
        t["q"] = torch.softmax(near[:, :m], -1).contiguous()
        t["tokens"] = torch.multinomial(t["q"].reshape(n * m, V), 1, generator=d.g).reshape(n, m)
        return t
    t["parents"] = _tree(c, seed)
    rank = np.array([[int((row[:i] == row[i]).sum()) for i in range(m)] for row in t["parents"]])  # among its siblings
    top = near.topk(min(V, int(rank.max()) + 1), -1).indices
    s = torch.arange(n, device="cuda")[:, None]
    t["tokens"] = top[s, torch.from_numpy(t["parents"] + 1).cuda(), torch.from_numpy(rank).cuda()]
    return t


def _quantised(x):
    """(int8 values, scale) of rows [..., hd], one scale a row: ties away from zero."""
    s = (x.abs().amax(-1, keepdim=True).double() / 127.0).float()
    r = x.double() / s.double()
    return (torch.sign(r) * torch.floor(r.abs() + 0.5)).clamp_(-127, 127).to(torch.int8), s


def prepare(case, seed):
    """A program's tensors; an int8 cache holds its context rows, quantised."""
    c, t = case, _inputs(case, seed)
    s = dict(c=c, start=_lens(c) if "vocab" not in c else None, **t)
    if c["kind"] in ("draft", "tree"):
        # token ids, random numbers and parents are host values in a program,
        # the plain form's indices device ones
        s["host"] = {n: t[n].cpu().numpy() for n in ("tokens", "u")}
    for n in ("parents", "paths"):
        if t.get(n) is not None:
            s[n + "_dev"] = torch.from_numpy(t[n]).cuda()
    if "start" in s and s["start"] is not None:
        s["start_dev"] = torch.tensor(s["start"], device="cuda")
    if c["kind"] == "cache":
        s["max"] = c["start"] + c["rows"] + 16
        s["store"] = [torch.zeros(c["seqs"], s["max"], c["nkv"], w, device="cuda", dtype=d)
                      for w, d in ((c["hd"], torch.int8), (1, torch.float32)) * 2]
    if c["kind"] == "attend" and c["cache"] == "int8":
        (s["kq"], s["ks"]), (s["vq"], s["vs"]) = _quantised(t["k"]), _quantised(t["v"])
    if own:  # the same values in the framework's storages and caches
        s.update(_handles(s, c))
    if c["kind"] == "attend" and c["cache"] == "int8":
        del s["k"], s["v"]
    return s


def _handles(s, c):
    import esolearn_amd as E

    B = E.HipBackend
    E.init(0)

    def hold(t):
        x = B.zeros(t.numel())
        B.synchronize()
        torch.from_dlpack(x).copy_(t.reshape(-1))
        torch.cuda.synchronize()
        return x

    h = {"B": B}
    for n in ("qkv", "freqs", "qw", "kw", "q", "p"):
        if n in s:
            h["h_" + n] = hold(s[n])
    if c["kind"] == "cache":
        h["h_k"], h["h_v"] = hold(s["k"]), hold(s["v"])
        h["caches"] = [B.kv8_new(s["max"], c["nkv"], c["hd"]) for _ in range(c["seqs"])]
    if c["kind"] == "attend" and c["cache"] == "f32":
        h["kc"], h["vc"] = [hold(x) for x in s["k"]], [hold(x) for x in s["v"]]
    if c["kind"] == "attend" and c["cache"] == "int8":
        n = c["len"] + c["rows"]
        h["caches"] = [B.kv8_new(n, c["nkv"], c["hd"]) for _ in range(c["seqs"])]
        for i, cache in enumerate(h["caches"]):
            B.kv8_write([cache], hold(s["k"][i]), hold(s["v"][i]), [0], n)
    return h


# --------------------------------------------------------------------- runs
def run(s):
    return (_OWN if own else _PLAIN)[s["c"]["kind"]](s, s["c"])


def _view(x, *shape):
    # the storage itself: whoever reads the outputs waits for the device first
    return torch.utils.dlpack.from_dlpack(x.__dlpack__(stream=-1)).view(*shape)


def _own_rope(s, c):
    q, k, v = s["B"].qk_norm_rope(s["h_qkv"], s["start"], c["rows"], c["nq"], c["nkv"], c["hd"], s["h_freqs"],
                                  q_weight=s.get("h_qw"), k_weight=s.get("h_kw"), eps=EPS, q_scale=1.0 / math.sqrt(c["hd"]),
                                  parents=s["parents"])
    n = c["seqs"] * c["rows"]
    return {"q": _view(q, n, c["nq"], c["hd"]), "k": _view(k, n, c["nkv"], c["hd"]), "v": _view(v, n, c["nkv"], c["hd"])}


def _own_cache(s, c):
    B, n = s["B"], c["keep"] or c["rows"]
    B.kv8_write(s["caches"], s["h_k"], s["h_v"], s["start"], c["rows"])
    if c["keep"]:
        B.kv8_keep(s["caches"], s["start"], s["paths"])
    k, v = B.kv8_read(s["caches"], s["start"], n)
    return {"k": _view(k, c["seqs"], n, c["nkv"], c["hd"]), "v": _view(v, c["seqs"], n, c["nkv"], c["hd"])}


def _own_attend(s, c):
    scale = 1.0 / math.sqrt(c["hd"])
    if c["cache"] == "int8":
        o = s["B"].kv8_tree_attention(s["h_q"], s["caches"], s["start"], c["rows"], c["nq"], scale, parents=s["parents"])
    else:
        o = s["B"].tree_attention(s["h_q"], s["kc"], s["vc"], s["start"], c["rows"], c["nq"], c["nkv"], c["hd"], scale,
                                  parents=s["parents"])
    return _view(o, c["seqs"], c["rows"], c["nq"], c["hd"])


def _own_draft(s, c):
    n, token = s["B"].verify_draft(s["h_p"], s["h_q"], s["host"]["tokens"], s["host"]["u"], c["vocab"])
    return {"accepted": n, "token": token}


def _own_tree(s, c):
    paths, n, token = s["B"].verify_tree(s["h_p"], s["host"]["tokens"], s["parents"], s["host"]["u"], c["vocab"])
    return {"paths": paths, "accepted": n, "token": token}


def _ancestors(s, c):
    """[seqs or 1, rows, rows]: node i's ancestors and itself."""
    m = c["rows"]
    if s["parents"] is None:
        return torch.ones(1, m, m, device="cuda", dtype=torch.bool).tril()
    # (1 + P)^n holds binomials of the distances along the paths: exact at 64
    up = torch.nn.functional.one_hot(s["parents_dev"] + 1, m + 1)[..., 1:].double() + torch.eye(m, device="cuda", dtype=torch.float64)
    return torch.linalg.matrix_power(up, 64) > 0


def _plain_rope(s, c):
    n, m, hd, nq, nkv = c["seqs"], c["rows"], c["hd"], c["nq"], c["nkv"]
    if s["parents"] is None:
        depth = torch.arange(m, device="cuda")[None]
    else:
        depth = _ancestors(s, c).sum(-1) - 1
    pos = (s["start_dev"][:, None] + depth).reshape(n * m, 1, 1)
    ang = pos.double() * s["freqs"].double()
    co, si = ang.cos().float(), ang.sin().float()
    q, k, v = s["qkv"].split([nq, nkv, nkv], 1)
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["qw"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["kw"]

    def turn(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * co - b * si, a * si + b * co), -1).reshape(x.shape)

    return {"q": turn(q) * (1.0 / math.sqrt(hd)), "k": turn(k), "v": v.contiguous()}


def _plain_cache(s, c):
    n, m, keep = c["seqs"], c["rows"], c["keep"]
    (kq, ks), (vq, vs) = _quantised(s["k"]), _quantised(s["v"])
    at = torch.arange(n, device="cuda")[:, None]
    rows = s["start_dev"][:, None] + torch.arange(m, device="cuda")
    KQ, KS, VQ, VS = s["store"]
    KQ[at, rows], KS[at, rows], VQ[at, rows], VS[at, rows] = kq, ks, vq, vs
    if keep:
        src, rows = s["start_dev"][:, None] + s["paths_dev"], rows[:, :keep]
        KQ[at, rows], KS[at, rows], VQ[at, rows], VS[at, rows] = KQ[at, src], KS[at, src], VQ[at, src], VS[at, src]
    return {"k": KQ[at, rows].float() * KS[at, rows], "v": VQ[at, rows].float() * VS[at, rows]}


def _plain_attend(s, c):
    n, m, hd, nq, nkv = c["seqs"], c["rows"], c["hd"], c["nq"], c["nkv"]
    k, v = (s["kq"].float() * s["ks"], s["vq"].float() * s["vs"]) if c["cache"] == "int8" else (s["k"], s["v"])
    keys = torch.arange(k.shape[1], device="cuda")
    draft = keys - s["start_dev"][:, None]  # the draft node of a cache row
    sees = (draft < 0)[:, None, :] | (((draft >= 0) & (draft < m))[:, None, :] & torch.gather(
        _ancestors(s, c).expand(n, m, m), 2, draft.clamp(0, m - 1)[:, None, :].expand(n, m, -1)))
    q = s["q"].reshape(n, m, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(hd))
    sc = sc.reshape(n, nkv, nq // nkv, m, -1).masked_fill(~sees[:, None, None], -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).reshape(n, nkv, -1, sc.shape[-1])
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())
    return o.reshape(n, nkv, nq // nkv, m, hd).permute(0, 3, 1, 2, 4).reshape(n, m, nq, hd)


def _pick(w, u):
    """The lowest index whose running sum of w [.., V] passes u times the whole."""
    cum = w.double().cumsum(-1)
    return torch.searchsorted(cum, (u * cum[..., -1])[..., None], right=True)[..., 0].clamp_(max=w.shape[-1] - 1)


def _plain_draft(s, c):
    m, at = c["rows"], torch.arange(c["seqs"], device="cuda")
    x = s["tokens"][..., None]
    p, q = s["p"][:, :m].gather(2, x)[..., 0].double(), s["q"].gather(2, x)[..., 0].double()
    n = (s["u"][:, :m] * q < p).long().cumprod(-1).sum(-1)
    row, less = s["p"][at, n].double(), s["q"][at, n.clamp(max=m - 1)].double()
    w = torch.where((n < m)[:, None], (row - less).clamp_(min=0.0), row)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, row)
    return {"accepted": n, "token": _pick(w, s["u"][:, m])}


def _plain_tree(s, c):
    m = c["rows"]
    t = _pick(s["p"], s["u"])
    match = t.gather(1, s["parents_dev"] + 1) == s["tokens"]
    # a node is accepted where it and all its ancestors match
    ok = (match[:, None, :] | ~_ancestors(s, c)).all(-1)
    n = ok.sum(-1)
    node = torch.arange(m, device="cuda")
    order = torch.where(ok, node, m).sort(-1).values
    last = torch.where(ok, node + 1, 0).amax(-1)
    return {"paths": torch.where(order < m, order, -1), "accepted": n, "token": t.gather(1, last[:, None])[:, 0]}


_OWN = {"rope": _own_rope, "cache": _own_cache, "attend": _own_attend, "draft": _own_draft, "tree": _own_tree}
_PLAIN = {"rope": _plain_rope, "cache": _plain_cache, "attend": _plain_attend, "draft": _plain_draft, "tree": _plain_tree}


# -------------------------------------------------------------------- exact
def _paths(parents):
    """For each node its path from the context down to itself."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _step_values(x):
    """The values that int8 rows [..., hd] stand for, in float64."""
    x = x.double()
    s = (x.abs().max(-1, keepdim=True).values / 127).float().double()
    return torch.where(x < 0, -1.0, 1.0) * torch.floor(x.abs() / s + 0.5).clamp(max=127) * s


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    n, m = c["seqs"], c["rows"]
    if c["kind"] == "rope":
        nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
        parents = t["parents"] if t["parents"] is not None else _chain(c)
        depth = [[len(p) - 1 for p in _paths(r)] for r in parents] if c["tree"] else [list(range(m))] * n
        pos = torch.tensor([[a + d for d in r] for a, r in zip(_lens(c), depth)], device="cuda").reshape(-1).double()
        z = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), pos[:, None, None] * t["freqs"].double())
        x = t["qkv"].double()

        def head(x, w):
            if w is not None:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2).contiguous()) * z).reshape(x.shape)

        return {"q": head(x[:, :nq], t.get("qw")) / math.sqrt(hd), "k": head(x[:, nq:nq + nkv], t.get("kw")), "v": x[:, nq + nkv:]}
    if c["kind"] == "cache":
        if c["keep"]:
            at = torch.from_numpy(t["paths"]).cuda()
            t = {x: torch.stack([t[x][i, at[i]] for i in range(n)]) for x in ("k", "v")}
        return {"k": _step_values(t["k"]), "v": _step_values(t["v"])}
    if c["kind"] == "attend":
        nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
        k, v = (_step_values(t["k"]), _step_values(t["v"])) if c["cache"] == "int8" else (t["k"], t["v"])
        out = torch.empty(n, m, nq, hd, device="cuda", dtype=torch.float64)
        for i, ln in enumerate(_lens(c)):
            sees = torch.zeros(m, ln + m, device="cuda", dtype=torch.bool)
            sees[:, :ln] = True
            if c["tree"]:
                for j, path in enumerate(_paths(t["parents"][i])):
                    sees[j, [ln + a for a in path]] = True
            else:
                sees[:, ln:] = torch.ones(m, m, device="cuda", dtype=torch.bool).tril()
            for h in range(nq):
                g = h // (nq // nkv)
                kk, vv = k[i, :ln + m, g].double(), v[i, :ln + m, g].double().contiguous()
                sc = t["q"][i, :, h].double() @ kk.t().contiguous() / math.sqrt(hd)
                out[i, :, h] = torch.softmax(sc.masked_fill_(~sees, -math.inf), -1) @ vv
        return out
    # counts and tokens are whole numbers: compared with the plain form's
    return None


# --------------------------------------------------------------------- work
def work(case):
    c = case
    n, m = c["seqs"], c["rows"]
    if c["kind"] == "draft":
        # one row of p and of q a sequence, whichever the draft ends at
        return {"bytes": 8.0 * n * (c["vocab"] + m), "flops": 3.0 * n * c["vocab"]}
    if c["kind"] == "tree":
        # the rows that a walk of a few nodes visits
        return {"bytes": 4.0 * n * c["vocab"] * min(m + 1, 4), "flops": 1.0 * n * c["vocab"] * min(m + 1, 4)}
    kv = c["nkv"] * c["hd"]
    if c["kind"] == "rope":
        e = n * m * (c["nq"] + 2 * c["nkv"]) * c["hd"]
        return {"bytes": 8.0 * e, "flops": 7.0 * e}
    if c["kind"] == "cache":
        back = c["keep"] or m
        return {"bytes": 2.0 * n * (m * (5.0 * kv + 4 * c["nkv"]) + back * (5.0 * kv + 4 * c["nkv"])), "flops": 2.0 * n * kv * (3 * m + back)}
    rows = sum(_lens(c)) + n * m
    # of the drafted rows a chain's node sees half, a tree's a few
    pairs = m * sum(_lens(c)) + n * m * ((m + 1) / 2 if not c["tree"] else min(m, 6))
    row = 2.0 * (kv + 4 * c["nkv"]) if c["cache"] == "int8" else 8.0 * kv
    return {"bytes": rows * row + 8.0 * n * m * c["nq"] * c["hd"], "flops": 4.0 * pairs * c["nq"] * c["hd"]}
