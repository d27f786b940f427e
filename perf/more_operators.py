"""Operators of bounded and quantised key caches: their cases, plain forms and exact results.

  window   masked_attention over mask_spans with a sliding window and a few first tokens
           of each document that stay visible (sinks); with "grad" also dq, dk and dv
  step     paged_step, new tokens over a paged K/V cache, each with one or more of
             window, sinks   the same rule for serving: pages between the two are gone
             tree            the new tokens are drafts in a tree: each attends what is
                             cached and its own ancestors; paged_keep then keeps one path
             held            pages of 8 bits ("int8", "e4m3") with a scale for each token
                             and head: the new rows are quantised as they are written and
                             read back by paged_read

``run`` computes them in elementary torch operations in 32 bits (64 next to a rounding's
border), or, where ``own`` is true, by the calls a user of ssa_amd makes.  q, k and v are
N(0, 1), as heads after a normalisation of q and k are; gradients coming in are N(0, 1) too.
"""

import math
import random

import torch

own = False
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
MOST = {"int8": 127.0, "e4m3": 448.0}   # the largest value that 8 bits hold
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _window(name, dtype, B, n, h_q, h_kv, d, window, sinks, docs=1, grad=False):
    """docs: documents in a sequence, of unlike lengths (1: the sequence is one)."""
    c = {"op": "window", "dtype": dtype, "B": B, "n": n, "h_q": h_q, "h_kv": h_kv, "d": d, "window": window,
         "sinks": sinks, "docs": docs, "grad": grad}
    return {"name": name, **c} if name else c


def _step(name, dtype, h_q, h_kv, d, page, one, chunks, new, ctx, window=0, sinks=0, tree=False, held=""):
    """`one` sequences with a single new token and `chunks` with up to `new` of them, each
    over up to `ctx` cached tokens; the longest of each kind has just as many."""
    c = {"op": "step", "dtype": dtype, "h_q": h_q, "h_kv": h_kv, "d": d, "page": page, "one": one,
         "chunks": chunks, "new": new, "ctx": ctx, "window": window, "sinks": sinks, "tree": tree, "held": held}
    return {"name": name, **c} if name else c


def listed():
    return [
        # The smallest windowed call: the layer's default heads over one short prompt of a
        # ragged length. Latency.
        _window("window-203", "fp32", 1, 203, 8, 2, 64, 50, 4),
        # The README's heads trained with a window, fp32.
        _window("window-grad-readme", "fp32", 2, 1024, 8, 2, 64, 256, 4, grad=True),
        # Packed fine-tuning of a windowed layer: six documents in 8192 tokens.
        _window("window-grad-packed", "bf16", 1, 8192, 32, 8, 128, 1024, 16, docs=6, grad=True),
        # A training step's windowed layer over one long odd sequence.
        _window("window-grad-long", "bf16", 1, 16001, 16, 4, 128, 1000, 4, grad=True),
        # One token each of 24 long conversations whose caches keep sinks and a window.
        _step("ring-24-tokens", "bf16", 32, 8, 128, 64, 24, 0, 0, 32767, window=4096, sinks=4),
        # A chunk of a long prompt behind what its window leaves of it.
        _step("ring-chunk-2k", "bf16", 32, 8, 128, 64, 0, 1, 2048, 30720, window=4096, sinks=4),
        # The smallest tree: seven drafted tokens of one short sequence, fp32. Latency.
        _step("tree-7", "fp32", 8, 2, 64, 16, 0, 1, 7, 203, tree=True),
        # Verifying up to 32 drafted tokens for each of 16 sequences.
        _step("tree-16x32", "bf16", 32, 8, 128, 64, 0, 16, 32, 8191, tree=True),
        # One token of one short sequence over an int8 cache, fp32 queries. Latency.
        _step("int8-token", "fp32", 8, 2, 64, 16, 1, 0, 0, 203, held="int8"),
        # A serving batch's step over an int8 cache: 32 sequences of unlike lengths.
        _step("int8-32-tokens", "bf16", 32, 8, 128, 64, 32, 0, 0, 8191, held="int8"),
        # One token against the longest cache, of e4m3: the work split over the keys.
        _step("e4m3-token-128k", "bf16", 16, 2, 128, 16, 1, 0, 0, 131071, held="e4m3"),
        # A chunk of a long prompt behind an int8 cache. The largest.
        _step("int8-chunk-2k", "bf16", 32, 8, 128, 64, 0, 1, 2048, 30720, held="int8"),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; every second one odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n | 1 if rng.random() < 0.5 else n


HEADS = ((32, 8, 128), (16, 2, 128), (28, 4, 128), (16, 4, 64), (12, 4, 128), (8, 2, 64), (8, 8, 80), (6, 2, 96))


def draw(rng):
    op = rng.choice(("window", "window", "step", "step", "step"))
    h_q, h_kv, d = rng.choice(HEADS)
    dtype = "fp32" if rng.random() < 0.25 else "bf16"
    sinks = rng.choice((0, 1, 4, 4, 16, _spread(rng, 1, 200)))
    if op == "window":
        n = _spread(rng, 64, 2048 if dtype == "fp32" else 12000)
        B = rng.choice([b for b in (1, 2, 4) if b * n <= 12000])
        docs = rng.choice((1, 1, rng.randint(2, 12)))
        return _window("", dtype, B, n, h_q, h_kv, d, _spread(rng, 16, 4096), max(sinks, 1), docs, rng.random() < 0.6)
    page = rng.choice((16, 32, 64, 128))
    kind = rng.choice(("ring", "tree", "held", "held", "both"))
    held = rng.choice(("int8", "e4m3")) if kind in ("held", "both") else ""
    window = _spread(rng, 16, 8192) if kind in ("ring", "both") else 0
    tree = kind == "tree" or (kind == "both" and rng.random() < 0.5)
    if not window:
        sinks = 0
    if tree:
        ctx = _spread(rng, 16, 16384)
        return _step("", dtype, h_q, h_kv, d, page, 0, min(_spread(rng, 1, 32), max(1, 131072 // ctx)),
                     _spread(rng, 2, 63), ctx, window, sinks, True, held)
    shape = rng.choice(("tokens", "tokens", "chunk", "mixed"))
    if shape == "tokens":
        ctx = _spread(rng, 16, 65536)
        one = min(_spread(rng, 1, 64), max(1, 262144 // ctx))
        return _step("", dtype, h_q, h_kv, d, page, one, 0, 0, ctx, window, sinks, held=held)
    if shape == "chunk":
        return _step("", dtype, h_q, h_kv, d, page, 0, 1, _spread(rng, 2, 1024), _spread(rng, 16, 16384), window, sinks,
                     held=held)
    return _step("", dtype, h_q, h_kv, d, page, rng.randint(1, 12), rng.randint(1, 3), _spread(rng, 2, 400),
                 _spread(rng, 16, 8192), window, sinks, held=held)


# ---- sizes that follow from a case, the same for every seed -------------------


def _doc_lengths(c):
    """Lengths of a sequence's documents: unlike each other, their sum n less a padded end of up to 3%
    where there are several."""
    n, docs = c["n"], min(c["docs"], c["n"])
    if docs == 1:
        return [n]
    r = random.Random(n * 131 + docs)
    w = [math.exp(r.gauss(0.0, 0.7)) for _ in range(docs)]
    total = n - n // 32
    lens = [max(1, int(total * x / sum(w))) for x in w]
    lens[0] += max(0, total - sum(lens))
    return lens


def _sequences(c):
    """(new tokens, cached tokens) of a step's sequences."""
    r = random.Random(c["ctx"] * 131 + c["one"] * 17 + c["chunks"])
    some = lambda most: max(1, int(most * (1.0 - 0.75 * r.random())))  # noqa: E731
    ones = [(1, c["ctx"] if i == 0 else some(c["ctx"])) for i in range(c["one"])]
    return ones + [(c["new"], c["ctx"]) if i == 0 else (some(c["new"]), some(c["ctx"])) for i in range(c["chunks"])]


def _drafts(m, r):
    """Parents of m drafted tokens (-1: the cached tokens), every one behind its parent, and the path
    that is kept: a token's ancestors and itself."""
    parents = [max(-1, i - 1 - int(r.expovariate(0.7))) for i in range(m)]
    path, at = [], r.randrange(m)
    while at >= 0:
        path.append(at)
        at = parents[at]
    return parents, path[::-1]


def _seen_keys(c, pos):
    """How many of the keys 0 .. pos a token at pos sees."""
    if not c["window"]:
        return pos + 1
    first = max(0, pos + 1 - c["window"])
    return pos + 1 - first + min(c["sinks"], first)


def _live(c, L, x):
    """Whether page x of a sequence with L cached keys holds a key that a later token sees."""
    P = c["page"]
    return not c["window"] or x * P < c["sinks"] or (x + 1) * P > L + 1 - c["window"]


def work(c):
    e = 4 if c["dtype"] == "fp32" else 2
    d, h_q, h_kv = c["d"], c["h_q"], c["h_kv"]
    if c["op"] == "window":
        pairs = c["B"] * sum(sum(_seen_keys(c, i) for i in range(x)) for x in _doc_lengths(c))
        q, kv = c["B"] * c["n"] * h_q * d * e, 2 * c["B"] * c["n"] * h_kv * d * e
        # forward: q, k, v, out; backward: q, k, v, out, dout read and the gradients written
        return {"bytes": 2 * q + kv + ((3 * q + kv) + (q + kv) if c["grad"] else 0),
                "flops": (14 if c["grad"] else 4) * d * h_q * pairs}
    held = d + 4 if c["held"] else d * e    # bytes of a cached row of one head
    pairs = rows = moved = new = 0
    r = random.Random(c["ctx"] + c["new"])
    for m, L in _sequences(c):
        new += m
        first = max(0, L + 1 - c["window"]) if c["window"] else 0
        rows += L - first + min(c["sinks"], first)
        if c["tree"]:
            parents, path = _drafts(m, r)
            depth = []
            for x in parents:
                depth.append(depth[x] + 1 if x >= 0 else 0)
            pairs += sum(_seen_keys(c, L + x) for x in depth)
            moved += sum(x != i for i, x in enumerate(path))
        else:
            pairs += sum(_seen_keys(c, L + t) for t in range(m))
    size = 2 * new * h_q * d * e + 2 * rows * h_kv * held + 2 * new * h_kv * (d * e + held) + 4 * moved * h_kv * held
    if c["held"]:
        size += 2 * new * h_kv * (held + d * e)  # read back
    return {"bytes": size, "flops": 4 * d * h_q * pairs}


# ---- inputs -------------------------------------------------------------------


def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + part)


def _randn(c, seed, part, *shape):
    return torch.randn(*shape, generator=_gen(seed, part), device=DEV).to(DTYPES[c["dtype"]])


def _prepare_window(c, seed):
    B, n = c["B"], c["n"]
    s = {"q": _randn(c, seed, 1, B, n, c["h_q"], c["d"]), "k": _randn(c, seed, 2, B, n, c["h_kv"], c["d"]),
         "v": _randn(c, seed, 3, B, n, c["h_kv"], c["d"]), "starts": None}
    if c["docs"] > 1:  # the same documents in another order for every seed and sequence
        starts = []
        for b in range(B):
            lens = _doc_lengths(c)
            random.Random(1009 * seed + b).shuffle(lens)
            starts.append([sum(lens[:i]) for i in range(len(lens) + 1)])
        s["starts"] = torch.tensor(starts, device=DEV, dtype=torch.int32)
    if c["grad"]:
        s["dout"] = _randn(c, seed, 4, B, n, c["h_q"], c["d"])
        for name in "qkv":
            s[name].requires_grad_(True)
    return s


def _pool(c, pages, g):
    """A pool of cached rows: values of the case's type, or 8-bit codes and their scales."""
    shape = (pages, c["page"], c["h_kv"], c["d"])
    if not c["held"]:
        return torch.randn(*shape, generator=g, device=DEV, dtype=DTYPES[c["dtype"]]), None
    x = torch.randn(*shape, generator=g, device=DEV)
    scale = x.abs().amax(-1) / MOST[c["held"]]
    x = x.div_(scale[..., None])
    # scales of a page lie by heads: a head's tokens are neighbours
    scale = scale.transpose(1, 2).contiguous().transpose(1, 2)
    return (x.round_() if c["held"] == "int8" else x).to(CODES[c["held"]]), scale


def _prepare_step(c, seed):
    seqs, P = _sequences(c), c["page"]
    new, total = [m for m, _ in seqs], [m + L for m, L in seqs]
    counts = [(t + P - 1) // P for t in total]
    live = [[x for x in range(n) if _live(c, L, x)] for n, (_, L) in zip(counts, seqs)]
    pages = sum(len(x) for x in live) + 3
    perm = torch.randperm(pages, generator=_gen(seed, 5), device=DEV).to(torch.int32)
    table = torch.zeros(len(seqs), max(counts), device=DEV, dtype=torch.int32)
    at = 0
    for b, x in enumerate(live):  # each sequence's pages, scattered over the pool; those that are gone: 0
        table[b, torch.tensor(x, device=DEV)] = perm[at:at + len(x)]
        at += len(x)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    T = starts[-1]
    g = _gen(seed, 6)
    s = {"table": table, "starts": torch.tensor(starts, device=DEV, dtype=torch.int32),
         "cached": torch.tensor([L for _, L in seqs], device=DEV, dtype=torch.int32),
         "q": _randn(c, seed, 1, T, c["h_q"], c["d"]), "k": _randn(c, seed, 2, T, c["h_kv"], c["d"]),
         "v": _randn(c, seed, 3, T, c["h_kv"], c["d"]), "max_new": max(new), "max_len": max(total),
         "parents": None, "kept": None}
    s["k_pages"], s["k_scales"] = _pool(c, pages, g)
    s["v_pages"], s["v_scales"] = _pool(c, pages, g)
    if c["tree"]:
        r = random.Random(7919 * seed + T)
        drafts = [_drafts(m, r) for m in new]
        s["parents"] = torch.tensor([x for parents, _ in drafts for x in parents], device=DEV, dtype=torch.int32)
        most = max(len(path) for _, path in drafts)
        s["kept"] = torch.tensor([path + [-1] * (most - len(path)) for _, path in drafts], device=DEV, dtype=torch.int32)
    return s


def prepare(case, seed):
    s = (_prepare_window if case["op"] == "window" else _prepare_step)(case, seed)
    return {"case": case, **s}


# ---- the framework's calls ----------------------------------------------------


def _own(s):
    import ssa_amd

    c = s["case"]
    if c["op"] == "window":
        spans = ssa_amd.mask_spans(c["n"], c["B"], doc_starts=s["starts"], window=c["window"], sinks=c["sinks"],
                                   device=s["q"].device)
        out = ssa_amd.masked_attention(s["q"], s["k"], s["v"], spans)
        if not c["grad"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    pools = (s["k_pages"], s["v_pages"])
    scales = {"k_scales": s["k_scales"], "v_scales": s["v_scales"]} if c["held"] else {}
    rule = {"window": c["window"], "sinks": c["sinks"]} if c["window"] else {}
    out = ssa_amd.paged_step(s["q"], s["k"], s["v"], *pools, s["table"], s["starts"], s["cached"], parents=s["parents"],
                             max_new=s["max_new"], max_len=s["max_len"], **rule, **scales)
    if c["tree"]:
        ssa_amd.paged_keep(*pools, s["table"], s["cached"], s["kept"], **scales)
    if c["held"]:  # the new rows as the cache holds them
        k, v = ssa_amd.paged_read(*pools, s["table"], s["starts"], s["cached"], len(s["q"]), dtype=s["q"].dtype, **scales)
        return {"out": out, "k": k, "v": v, **scales}
    return {"out": out, "k_pages": pools[0], "v_pages": pools[1]}


# ---- the plain forms ----------------------------------------------------------


def _scores(c, q, k):
    """Scores [B, h_kv, g, m, n] of q [B, h_kv, g, m, d] and k [B, h_kv, n, d]."""
    return torch.matmul(q, k.transpose(2, 3).contiguous()[:, :, None]).div_(math.sqrt(c["d"]))


def _softmax(s, seen):
    """Softmax over the seen keys; rows that see none are zeros."""
    s = s.masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _plain_window(c, s):
    B, n, h_q, d = s["q"].shape
    h_kv = c["h_kv"]
    g = h_q // h_kv
    row = torch.arange(n, device=DEV, dtype=torch.int32).expand(B, n).contiguous()
    opened = torch.zeros(B, n, device=DEV, dtype=torch.int32)     # where the row's document starts
    inside = opened == 0
    if s["starts"] is not None:
        doc = torch.searchsorted(s["starts"], row, right=True) - 1
        inside = doc < s["starts"].shape[1] - 1
        opened = s["starts"].gather(1, doc)
    i, j = row[:, :, None], row[:, None, :]
    near = j > i - c["window"]
    first = j < opened[:, :, None] + c["sinks"]
    seen = (j <= i) & (j >= opened[:, :, None]) & (near | first) & inside[:, :, None]

    heads = lambda x: x.detach().float().view(B, n, h_kv, -1, d).permute(0, 2, 3, 1, 4).contiguous()  # noqa: E731
    back = lambda x, t: x.permute(0, 3, 1, 2, 4).reshape(t.shape).to(t.dtype)  # noqa: E731
    q, k, v = heads(s["q"]), heads(s["k"])[:, :, 0], heads(s["v"])[:, :, 0]
    p = _softmax(_scores(c, q, k), seen[:, None, None])
    o = torch.matmul(p, v[:, :, None])
    if not c["grad"]:
        return {"out": back(o, s["q"])}
    do = heads(s["dout"])
    flat = lambda x: x.reshape(B, h_kv, g * n, -1)  # noqa: E731
    dv = torch.matmul(flat(p).transpose(2, 3), flat(do))
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()[:, :, None]).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    ds.div_(math.sqrt(d))
    dq = torch.matmul(ds, k[:, :, None])
    dk = torch.matmul(flat(ds).transpose(2, 3), flat(q))
    return {"out": back(o, s["q"]), "dq": back(dq, s["q"]), "dk": back(dk[:, :, None], s["k"]),
            "dv": back(dv[:, :, None], s["v"])}


def _quantise(c, x):
    """Codes and scales of rows x [..., d]; the quotients in 64 bits."""
    scale = (x.float().abs().amax(-1).double() / MOST[c["held"]]).float()
    y = x.double() / torch.where(scale > 0, scale, 1.0).double()[..., None]
    if c["held"] == "int8":
        return y.round().to(torch.int8), scale
    ulp = torch.pow(2.0, torch.frexp(y)[1].clamp(min=-5).double() - 4.0)  # of e4m3: 3 bits behind the first
    return (y / ulp).round().mul_(ulp).float().to(torch.float8_e4m3fn), scale


def _values(codes, scale):
    return codes.float() if scale is None else codes.float() * scale[..., None]


def _plain_step(c, s):
    h_q, h_kv, d, P = c["h_q"], c["h_kv"], c["d"], c["page"]
    T, B = s["q"].shape[0], s["table"].shape[0]
    starts, cached, table = s["starts"].long(), s["cached"].long(), s["table"].long()
    token = torch.arange(T, device=DEV)
    seq = torch.searchsorted(starts, token, right=True) - 1
    at = token - starts[seq]
    slot = cached[seq] + at
    page, row = table[seq, slot // P], slot % P
    for x in "kv":
        if c["held"]:
            s[x + "_pages"].view(torch.int8)[page, row], s[x + "_scales"][page, row] = (
                t if t.dtype == torch.float32 else t.view(torch.int8) for t in _quantise(c, s[x]))
        else:
            s[x + "_pages"][page, row] = s[x]
    wide, M = table.shape[1] * P, s["max_new"]
    spots = table[:, :, None] * P + torch.arange(P, device=DEV)

    def keys(x):
        pages, scale = s[x + "_pages"], s[x + "_scales"]
        flat = pages.view(torch.int8).flatten(0, 1)[spots.flatten()].view(pages.dtype) if c["held"] else pages.flatten(0, 1)[spots.flatten()]
        rows = _values(flat, None if scale is None else scale.reshape(-1, h_kv)[spots.flatten()]).view(B, wide, h_kv, d)
        rows[seq, slot] = s[x].float()  # a call's own tokens are attended as they are given
        return rows.transpose(1, 2).contiguous()

    q = torch.zeros(B, M, h_q, d, device=DEV)
    q[seq, at] = s["q"].float()
    q = q.view(B, M, h_kv, -1, d).permute(0, 2, 3, 1, 4).contiguous()

    # every key's position and, of new ones, which rows they are ancestors of
    kpos = torch.arange(wide, device=DEV).expand(B, wide).clone()
    qpos = cached[:, None] + torch.arange(M, device=DEV)
    family = torch.ones(M, M, dtype=torch.bool, device=DEV).tril().expand(B, M, M).clone()
    if c["tree"]:
        parent = torch.full((B, M), -1, device=DEV)
        parent[seq, at] = s["parents"].long()
        family = torch.eye(M, dtype=torch.bool, device=DEV).expand(B, M, M).clone()
        up = parent
        for _ in range(M):
            b, i = (up >= 0).nonzero(as_tuple=True)
            family[b, i, up[b, i]] = True
            up = torch.where(up >= 0, parent.gather(1, up.clamp(min=0)), up)
        qpos = cached[:, None] + family.sum(-1) - 1
        kpos[seq, slot] = qpos[seq, at]
    seen = (torch.arange(wide, device=DEV) < cached[:, None])[:, None].expand(B, M, wide).clone()
    seen[seq, :, slot] = family[seq, :, at]
    if c["window"]:
        seen &= (kpos[:, None] > qpos[:, :, None] - c["window"]) | (kpos[:, None] < c["sinks"])
    p = _softmax(_scores(c, q, keys("k")), seen[:, None, None])
    o = torch.matmul(p, keys("v")[:, :, None]).permute(0, 3, 1, 2, 4).reshape(B, M, h_q, d)
    out = o[seq, at].to(s["q"].dtype)
    if c["tree"]:
        b, t = (s["kept"] >= 0).nonzero(as_tuple=True)
        src, dst = cached[b] + s["kept"].long()[b, t], cached[b] + t
        for x in "kv":
            pages = s[x + "_pages"].view(torch.int8) if c["held"] else s[x + "_pages"]
            pages[table[b, dst // P], dst % P] = pages[table[b, src // P], src % P]
            if c["held"]:
                scale = s[x + "_scales"]
                scale[table[b, dst // P], dst % P] = scale[table[b, src // P], src % P]
    if not c["held"]:
        return {"out": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    res = {"out": out, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    for x in "kv":
        codes = s[x + "_pages"].view(torch.int8)[page, row].view(CODES[c["held"]])
        res[x] = _values(codes, s[x + "_scales"][page, row]).to(s["q"].dtype)
    return res


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    return (_plain_window if c["op"] == "window" else _plain_step)(c, state)


# ---- from the definitions, in 64 bits -----------------------------------------


def _attend64(c, q, k, v, see, dout=None):
    """One head's rows q [m, d] over the keys that each sees: out and, with dout, dq and its parts of dk and dv."""
    s = torch.where(see, q @ k.T / math.sqrt(c["d"]), -math.inf)
    w = torch.where(see, torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)), 0.0)
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    o = w @ v
    if dout is None:
        return o
    dw = dout @ v.T
    ds = w * (dw - (w * dw).sum(-1, keepdim=True)) / math.sqrt(c["d"])
    return o, ds @ k, ds.T @ q, w.T @ dout


def _exact_window(c, s):
    B, n, g = c["B"], c["n"], c["h_q"] // c["h_kv"]
    q, k, v = (s[x].detach().double() for x in "qkv")
    res = {"out": torch.zeros_like(q)}
    if c["grad"]:
        res |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    for b in range(B):
        bounds = [0, n] if s["starts"] is None else s["starts"][b].tolist()
        for a, e in zip(bounds, bounds[1:]):  # a document by itself
            i = torch.arange(e - a, device=DEV)
            back = i[:, None] - i[None]
            see = (back >= 0) & ((back < c["window"]) | (i[None] < c["sinks"]))
            for h in range(c["h_q"]):
                kv = h // g
                args = (c, q[b, a:e, h], k[b, a:e, kv], v[b, a:e, kv], see)
                if c["grad"]:
                    o, dq, dk, dv = _attend64(*args, dout=s["dout"][b, a:e, h].double())
                    res["dq"][b, a:e, h] = dq
                    res["dk"][b, a:e, kv] += dk
                    res["dv"][b, a:e, kv] += dv
                else:
                    o = _attend64(*args)
                res["out"][b, a:e, h] = o
    return res


def _exact_held(c, x):
    """Scales [m, h_kv] of rows x [m, h_kv, d] (floats), and what they and 8 bits stand for, in 64 bits."""
    scale = (x.abs().amax(-1, keepdim=True) / MOST[c["held"]]).float().double()
    y = x / scale.clamp(min=1e-300)
    if c["held"] == "int8":
        return scale[..., 0], torch.round(y) * scale
    # e4m3: multiples of 2^-9 up to 2^-6, from there on eight a factor of two
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return scale[..., 0], torch.round(y / step) * step * scale


def _exact_step(c, s):
    P, g, h_kv, d = c["page"], c["h_q"] // c["h_kv"], c["h_kv"], c["d"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    new = {x: torch.zeros_like(s[x], dtype=torch.float64) for x in "kv"}
    pools = {x: s[x + ("_scales" if c["held"] else "_pages")].double() for x in "kv"}
    at = 0
    for b, (m, L) in enumerate(_sequences(c)):
        where = torch.arange(L + m, device=DEV)
        page, row = s["table"][b].long()[where // P], where % P
        rows = {}
        for x in "kv":
            mine = s[x][at:at + m].double()
            if c["held"]:
                codes = s[x + "_pages"].view(torch.int8)[page[:L], row[:L]].view(CODES[c["held"]])
                old = codes.float().double() * s[x + "_scales"][page[:L], row[:L]].double()[..., None]
                pools[x][page[L:], row[L:]], new[x][at:at + m] = _exact_held(c, mine)
            else:
                old = s[x + "_pages"][page[:L], row[:L]].double()
                pools[x][page[L:], row[L:]] = mine
            rows[x] = torch.cat((old, mine))
        kpos, qpos = where.clone(), L + torch.arange(m, device=DEV)
        see = where[None] <= qpos[:, None]
        if c["tree"]:
            parents = s["parents"][at:at + m].tolist()
            see[:, L:] = False
            for i in range(m):
                x, depth = i, -1
                while x >= 0:
                    see[i, L + x] = True
                    x, depth = parents[x], depth + 1
                qpos[i] = kpos[L + i] = L + depth
        if c["window"]:
            see &= (qpos[:, None] - kpos[None] < c["window"]) | (kpos[None] < c["sinks"])
        for h in range(c["h_q"]):
            out[at:at + m, h] = _attend64(c, s["q"][at:at + m, h].double(), rows["k"][:, h // g], rows["v"][:, h // g], see)
        if c["tree"]:
            for t, x in enumerate(y for y in s["kept"][b].tolist() if y >= 0):
                for y in "kv":
                    pools[y][page[L + t], row[L + t]] = pools[y][page[L + x], row[L + x]]  # (no token comes before its slot)
                    new[y][at + t] = new[y][at + x]
        at += m
    if c["held"]:
        return {"out": out, "k": new["k"], "v": new["v"], "k_scales": pools["k"], "v_scales": pools["v"]}
    return {"out": out, "k_pages": pools["k"], "v_pages": pools["v"]}


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_window if case["op"] == "window" else _exact_step)(case, s)
