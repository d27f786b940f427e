"""Operators beside the selective attention: their cases, plain forms and exact results.

  masked   masked_attention: softmax attention whose rows see one key interval each
           (causal, documents, prefixes), with capped scores and a distance bias;
           with "grad" also dq, dk and dv
  paged    paged_step: new tokens of several sequences appended to a paged K/V cache
           and attended over it, chunks and single tokens in one ragged batch
  axes     rope_axes: rotary positions with several axes (time, height, width) on q
           and k; with "grad" the rotation's gradients

``run`` computes them in elementary torch operations in 32 bits, or, where ``own``
is true, by the calls a user of ssa_amd makes.  q, k and v are N(0, 1), as heads
after a normalisation of q and k are; gradients coming in are N(0, 1) too.
"""

import math
import random

import torch

own = False
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _masked(name, dtype, B, n, h_q, h_kv, d, mask, cap=0.0, slopes=False, grad=False, docs=1):
    """mask: "causal", "full", "docs" or "prefix" (every document opens with a part that
    sees itself whole); docs: documents in a sequence, of unlike lengths."""
    c = {"op": "masked", "dtype": dtype, "B": B, "n": n, "h_q": h_q, "h_kv": h_kv, "d": d, "mask": mask,
         "docs": docs, "cap": cap, "slopes": slopes, "grad": grad}
    return {"name": name, **c} if name else c


def _paged(name, dtype, h_q, h_kv, d, page, one, chunks, new, ctx, cap=0.0, slopes=False):
    """`one` sequences with a single new token and `chunks` with up to `new` of them, each
    over up to `ctx` cached tokens; the longest of each kind has just as many."""
    c = {"op": "paged", "dtype": dtype, "h_q": h_q, "h_kv": h_kv, "d": d, "page": page, "one": one,
         "chunks": chunks, "new": new, "ctx": ctx, "cap": cap, "slopes": slopes}
    return {"name": name, **c} if name else c


def _axes(name, dtype, B, n, h_q, h_kv, d, rot, axes, grad=False):
    c = {"op": "axes", "dtype": dtype, "B": B, "n": n, "h_q": h_q, "h_kv": h_kv, "d": d, "rot": rot, "axes": axes,
         "grad": grad}
    return {"name": name, **c} if name else c


def listed():
    return [
        # The smallest dense call: the layer's default heads over one short prompt of a ragged
        # length, scores with a distance bias. Latency.
        _masked("masked-203", "fp32", 1, 203, 8, 2, 64, "causal", slopes=True),
        # The README's heads trained with a prefix that sees itself whole, fp32.
        _masked("masked-grad-readme", "fp32", 2, 1024, 8, 2, 64, "prefix", grad=True),
        # A training step's attention on short odd sequences with capped scores, d = 64.
        _masked("masked-grad-capped", "bf16", 2, 4001, 16, 4, 64, "causal", cap=30.0, grad=True),
        # Packed fine-tuning: twelve documents of image prefix and text in 8192 tokens.
        _masked("masked-grad-packed", "bf16", 1, 8192, 32, 8, 128, "prefix", docs=12, grad=True),
        # The largest dense call: one long causal prompt through an attention layer.
        _masked("masked-16k", "bf16", 1, 16384, 32, 8, 128, "causal"),
        # The smallest serving call: one token of one short sequence, fp32. Latency.
        _paged("paged-token", "fp32", 8, 2, 64, 16, 1, 0, 0, 203),
        # A serving batch's step: 32 sequences of unlike lengths, one token each.
        _paged("paged-32-tokens", "bf16", 32, 8, 128, 64, 32, 0, 0, 8191),
        # One token against the longest cache: few heads, the work split over the keys.
        _paged("paged-token-128k", "bf16", 16, 2, 128, 16, 1, 0, 0, 131071),
        # A chunk of a long prompt against what is cached of it.
        _paged("paged-chunk-2k", "bf16", 32, 8, 128, 64, 0, 1, 2048, 30720),
        # Chunks of two prompts among the single tokens of seven sequences, capped scores.
        _paged("paged-mixed", "bf16", 28, 4, 128, 32, 7, 2, 500, 6001, cap=50.0),
        # Image positions of a small layer trained in fp32: forward and backward, half the features.
        _axes("axes-grad", "fp32", 2, 1001, 16, 4, 64, 32, 2, grad=True),
        # A long video prompt's q and k: time, height and width.
        _axes("axes-32k", "bf16", 1, 32768, 32, 8, 128, 128, 3),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; every second one odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n | 1 if rng.random() < 0.5 else n


HEADS = ((32, 8, 128), (16, 2, 128), (28, 4, 128), (16, 4, 64), (12, 4, 128), (8, 2, 64), (8, 8, 80), (6, 2, 96))


def draw(rng):
    op = rng.choice(("masked", "masked", "masked", "paged", "paged", "axes"))
    h_q, h_kv, d = rng.choice(HEADS)
    dtype = "fp32" if rng.random() < 0.25 else "bf16"
    cap = rng.choice((0.0, 0.0, 20.0, 30.0, 50.0))
    slopes = rng.random() < 0.3
    if op == "axes":
        B = rng.choice((1, 1, 2, 4))
        rot = rng.choice((d, d, d // 2))
        return _axes("", dtype, B, _spread(rng, 1, 32768 // B), h_q, h_kv, d, rot, rng.choice((2, 3, 3)),
                     grad=rng.random() < 0.5)
    if op == "masked":
        grad = rng.random() < 0.5
        mask = rng.choice(("causal", "full", "docs", "prefix"))
        n = _spread(rng, 64, 2048 if dtype == "fp32" else 4096 if mask == "full" else 8192)
        B = rng.choice([b for b in (1, 2, 4) if b * n <= 8192] or [1])
        docs = rng.randint(1, 16) if mask in ("docs", "prefix") else 1
        return _masked("", dtype, B, n, h_q, h_kv, d, mask, cap, slopes, grad, docs)
    page = rng.choice((16, 32, 64, 128))
    kind = rng.choice(("tokens", "tokens", "chunk", "mixed"))
    if kind == "tokens":
        ctx = _spread(rng, 16, 65536)
        one = min(_spread(rng, 1, 64), max(1, 262144 // ctx))
        return _paged("", dtype, h_q, h_kv, d, page, one, 0, 0, ctx, cap, slopes)
    if kind == "chunk":
        return _paged("", dtype, h_q, h_kv, d, page, 0, 1, _spread(rng, 2, 1024), _spread(rng, 16, 16384), cap, slopes)
    return _paged("", dtype, h_q, h_kv, d, page, rng.randint(1, 12), rng.randint(1, 3), _spread(rng, 2, 400),
                  _spread(rng, 16, 8192), cap, slopes)


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


def _prefix_of(c, length):
    return length // 3 if c["mask"] == "prefix" else 0


def _sequences(c):
    """(new tokens, cached tokens) of a paged case's sequences."""
    r = random.Random(c["ctx"] * 131 + c["one"] * 17 + c["chunks"])
    some = lambda most: max(1, int(most * (1.0 - 0.75 * r.random())))  # noqa: E731
    ones = [(1, c["ctx"] if i == 0 else some(c["ctx"])) for i in range(c["one"])]
    return ones + [(c["new"], c["ctx"]) if i == 0 else (some(c["new"]), some(c["ctx"])) for i in range(c["chunks"])]


def _pairs(c):
    """Visible (row, key) pairs of one head."""
    if c["op"] == "paged":
        return sum(m * L + m * (m + 1) // 2 for m, L in _sequences(c))
    if c["mask"] == "full":
        return c["B"] * c["n"] ** 2
    return c["B"] * sum(x * (x + 1) // 2 + _prefix_of(c, x) * (_prefix_of(c, x) - 1) // 2 for x in _doc_lengths(c))


def work(c):
    e = 4 if c["dtype"] == "fp32" else 2
    d, h_q, h_kv = c["d"], c["h_q"], c["h_kv"]
    if c["op"] == "axes":
        rows = c["B"] * c["n"]
        once = 2 * rows * (h_q + h_kv) * d * e + c["axes"] * rows * 8
        flops = 3 * rows * (h_q + h_kv) * c["rot"]
        return {"bytes": once * (2 if c["grad"] else 1), "flops": flops * (2 if c["grad"] else 1)}
    pairs = _pairs(c)
    if c["op"] == "masked":
        q, kv = c["B"] * c["n"] * h_q * d * e, 2 * c["B"] * c["n"] * h_kv * d * e
        # forward: q, k, v, out; backward: q, k, v, out, dout read and the gradients written
        return {"bytes": 2 * q + kv + ((3 * q + kv) + (q + kv) if c["grad"] else 0),
                "flops": (14 if c["grad"] else 4) * d * h_q * pairs}
    new, cached = (sum(x[i] for x in _sequences(c)) for i in (0, 1))
    return {"bytes": 2 * new * h_q * d * e + 2 * cached * h_kv * d * e + 4 * new * h_kv * d * e, "flops": 4 * d * h_q * pairs}


# ---- inputs -------------------------------------------------------------------


def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + part)


def _randn(c, seed, part, *shape):
    return torch.randn(*shape, generator=_gen(seed, part), device=DEV).to(DTYPES[c["dtype"]])


def _slopes(c):
    """The distance bias' geometric slopes, one a query head."""
    if not c["slopes"]:
        return None
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / c["h_q"]) for i in range(c["h_q"])], device=DEV)


def _prepare_masked(c, seed):
    B, n = c["B"], c["n"]
    s = {"q": _randn(c, seed, 1, B, n, c["h_q"], c["d"]), "k": _randn(c, seed, 2, B, n, c["h_kv"], c["d"]),
         "v": _randn(c, seed, 3, B, n, c["h_kv"], c["d"]), "slopes": _slopes(c), "starts": None, "prefix": None}
    if c["mask"] in ("docs", "prefix"):  # the same documents in another order for every seed and sequence
        starts, prefix = [], []
        for b in range(B):
            lens = _doc_lengths(c)
            random.Random(1009 * seed + b).shuffle(lens)
            starts.append([sum(lens[:i]) for i in range(len(lens) + 1)])
            prefix.append([_prefix_of(c, x) for x in lens])
        s["starts"] = torch.tensor(starts, device=DEV, dtype=torch.int32)
        s["prefix"] = torch.tensor(prefix, device=DEV, dtype=torch.int32)
    if c["grad"]:
        s["dout"] = _randn(c, seed, 4, B, n, c["h_q"], c["d"])
        for name in "qkv":
            s[name].requires_grad_(True)
    return s


def _prepare_paged(c, seed):
    seqs, P, dt = _sequences(c), c["page"], DTYPES[c["dtype"]]
    new, total = [m for m, _ in seqs], [m + L for m, L in seqs]
    counts = [(t + P - 1) // P for t in total]
    pages = sum(counts) + 3
    perm = torch.randperm(pages, generator=_gen(seed, 5), device=DEV).to(torch.int32)
    table = torch.zeros(len(seqs), max(counts), device=DEV, dtype=torch.int32)
    at = 0
    for b, x in enumerate(counts):  # each sequence's pages, scattered over the pool
        table[b, :x] = perm[at:at + x]
        at += x
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    T = starts[-1]
    g = _gen(seed, 6)
    return {"k_pages": torch.randn(pages, P, c["h_kv"], c["d"], generator=g, device=DEV, dtype=dt),
            "v_pages": torch.randn(pages, P, c["h_kv"], c["d"], generator=g, device=DEV, dtype=dt),
            "table": table, "starts": torch.tensor(starts, device=DEV, dtype=torch.int32),
            "cached": torch.tensor([L for _, L in seqs], device=DEV, dtype=torch.int32),
            "q": _randn(c, seed, 1, T, c["h_q"], c["d"]), "k": _randn(c, seed, 2, T, c["h_kv"], c["d"]),
            "v": _randn(c, seed, 3, T, c["h_kv"], c["d"]), "slopes": _slopes(c), "max_new": max(new), "max_len": max(total)}


def _sections(c):
    """Pairs of features on each axis: the first axis a quarter of them (half with two axes), the others the rest."""
    half, a = c["rot"] // 2, c["axes"]
    first = half // 4 if a == 3 else half // 2
    second = (half - first) // 2 if a == 3 else half - first
    return [first, second, half - first - second][:a]


def _prepare_axes(c, seed):
    B, n, a = c["B"], c["n"], c["axes"]
    i = torch.arange(n, device=DEV).expand(B, n)
    text = min(n, 16) + seed % 5  # a few words, then frames (or one image) of a grid 20 wide
    j = (i - text).clamp(min=0)
    grid = [j // 240, j // 20 % 12, j % 20] if a == 3 else [j // 20, j % 20]
    pos = torch.stack([torch.where(i < text, i, text + x) for x in grid])
    pos = pos + (torch.arange(B, device=DEV) * 1000 + 7000 * (seed % 7))[None, :, None]
    s = {"q": _randn(c, seed, 1, B, n, c["h_q"], c["d"]), "k": _randn(c, seed, 2, B, n, c["h_kv"], c["d"]), "pos": pos,
         "sections": _sections(c),
         "freqs": 1e6 ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"])}
    if c["grad"]:
        s["dq"], s["dk"] = _randn(c, seed, 3, B, n, c["h_q"], c["d"]), _randn(c, seed, 4, B, n, c["h_kv"], c["d"])
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    return s


def prepare(case, seed):
    s = {"masked": _prepare_masked, "paged": _prepare_paged, "axes": _prepare_axes}[case["op"]](case, seed)
    return {"case": case, **s}


# ---- the framework's calls ----------------------------------------------------


def _own(s):
    import ssa_amd

    c = s["case"]
    cap = c["cap"] or None if "cap" in c else None
    if c["op"] == "masked":
        spans = None
        if c["mask"] != "causal":
            spans = ssa_amd.mask_spans(c["n"], c["B"], causal=c["mask"] != "full", doc_starts=s["starts"],
                                       prefix_lens=s["prefix"], device=s["q"].device)
        out = ssa_amd.masked_attention(s["q"], s["k"], s["v"], spans, softcap=cap, slopes=s["slopes"])
        if not c["grad"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "paged":
        out = ssa_amd.paged_step(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["cached"],
                                 softcap=cap, slopes=s["slopes"], max_new=s["max_new"], max_len=s["max_len"])
        return {"out": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    q, k = ssa_amd.rope_axes(s["q"], s["k"], s["pos"], s["freqs"], s["sections"])
    if not c["grad"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


# ---- the plain forms ----------------------------------------------------------


def _scores(c, q, k, slopes, qpos, kpos):
    """Scores [B, h_kv, g, m, n] of q [B, h_kv, g, m, d] and k [B, h_kv, n, d] and, with a cap, the tanh
    they went through; qpos [B, m] and kpos [n]."""
    s = torch.matmul(q, k.transpose(2, 3).contiguous()[:, :, None]).div_(math.sqrt(c["d"]))
    t = None
    if c["cap"]:
        t = s.div_(c["cap"]).tanh_()
        s = t * c["cap"]
    if slopes is not None:
        far = (qpos[:, None, None, :, None] - kpos).abs().to(s.dtype)
        s = s - slopes.view(1, q.shape[1], q.shape[2], 1, 1) * far
    return s, t


def _softmax(s, seen):
    """Softmax over the seen keys; rows that see none are zeros."""
    s = s.masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _seen(c, s, n):
    """[B, n, n]: which keys each row sees."""
    i, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)[None, :]
    if c["mask"] in ("causal", "full"):
        return ((j <= i) if c["mask"] == "causal" else (j == j) | (i == i)).expand(c["B"], n, n)
    row = torch.arange(n, device=DEV, dtype=torch.int32).expand(c["B"], n).contiguous()
    doc = torch.searchsorted(s["starts"], row, right=True) - 1
    inside = doc < s["prefix"].shape[1]
    at = doc.clamp(max=s["prefix"].shape[1] - 1)
    opened = s["starts"].gather(1, at) + s["prefix"].gather(1, at)
    same = (doc[:, :, None] == doc[:, None, :]) & inside[:, :, None]
    return same & ((j <= i) | (j < opened[:, :, None]))


def _plain_masked(c, s):
    B, n, h_q, d = s["q"].shape
    h_kv = c["h_kv"]
    g = h_q // h_kv
    heads = lambda x: x.detach().float().view(B, n, h_kv, -1, d).permute(0, 2, 3, 1, 4).contiguous()  # noqa: E731
    back = lambda x, t: x.permute(0, 3, 1, 2, 4).reshape(t.shape).to(t.dtype)  # noqa: E731
    q, k, v = heads(s["q"]), heads(s["k"])[:, :, 0], heads(s["v"])[:, :, 0]
    at = torch.arange(n, device=DEV)
    score, t = _scores(c, q, k, s["slopes"], at.expand(B, n), at)
    p = _softmax(score, _seen(c, s, n)[:, None, None])
    o = torch.matmul(p, v[:, :, None])
    if not c["grad"]:
        return {"out": back(o, s["q"])}
    do = heads(s["dout"])
    flat = lambda x: x.reshape(B, h_kv, g * n, -1)  # noqa: E731
    dv = torch.matmul(flat(p).transpose(2, 3), flat(do))
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()[:, :, None]).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if t is not None:
        ds.mul_(1.0 - t * t)
    ds.div_(math.sqrt(d))
    dq = torch.matmul(ds, k[:, :, None])
    dk = torch.matmul(flat(ds).transpose(2, 3), flat(q))
    return {"out": back(o, s["q"]), "dq": back(dq, s["q"]), "dk": back(dk[:, :, None], s["k"]),
            "dv": back(dv[:, :, None], s["v"])}


def _plain_paged(c, s):
    h_q, h_kv, d, P = c["h_q"], c["h_kv"], c["d"], c["page"]
    T, B = s["q"].shape[0], s["table"].shape[0]
    starts, cached, table = s["starts"].long(), s["cached"].long(), s["table"].long()
    token = torch.arange(T, device=DEV)
    seq = torch.searchsorted(starts, token, right=True) - 1
    step = token - starts[seq]
    pos = cached[seq] + step
    page, row = table[seq, pos // P], pos % P
    s["k_pages"][page, row] = s["k"]
    s["v_pages"][page, row] = s["v"]
    wide = table.shape[1] * P
    keys = s["k_pages"][table].float().view(B, wide, h_kv, d).transpose(1, 2).contiguous()
    vals = s["v_pages"][table].float().view(B, wide, h_kv, d).transpose(1, 2).contiguous()
    q = torch.zeros(B, s["max_new"], h_q, d, device=DEV)
    q[seq, step] = s["q"].float()
    q = q.view(B, s["max_new"], h_kv, -1, d).permute(0, 2, 3, 1, 4).contiguous()
    qpos = cached[:, None] + torch.arange(s["max_new"], device=DEV)
    kpos = torch.arange(wide, device=DEV)
    score, _ = _scores(c, q, keys, s["slopes"], qpos, kpos)
    p = _softmax(score, (kpos <= qpos[:, :, None])[:, None, None])
    o = torch.matmul(p, vals[:, :, None]).permute(0, 3, 1, 2, 4).reshape(B, s["max_new"], h_q, d)
    return {"out": o[seq, step].to(s["q"].dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _turn(x, cos, sin, rot):
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1)


def _plain_axes(c, s):
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=DEV), torch.tensor(s["sections"], device=DEV),
                                   output_size=c["rot"] // 2)
    ang = s["pos"].double()[axis].permute(1, 2, 0) * s["freqs"]
    cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]
    out = {x: _turn(s[x].detach().float(), cos, sin, c["rot"]).to(s[x].dtype) for x in ("q", "k")}
    if c["grad"]:
        out |= {x: _turn(s[x].float(), cos, -sin, c["rot"]).to(s[x].dtype) for x in ("dq", "dk")}
    return out


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    return {"masked": _plain_masked, "paged": _plain_paged, "axes": _plain_axes}[c["op"]](c, state)


# ---- from the definitions, in 64 bits -----------------------------------------


def _attend64(c, q, k, v, lo, hi, qpos, slope, dout=None):
    """One head's rows q [m, d] over the keys [lo, hi) of each: out and, with dout, dq and its parts of dk and dv."""
    n = k.shape[0]
    j = torch.arange(n, device=DEV)
    see = (j[None] >= lo[:, None]) & (j[None] < hi[:, None])
    raw = q @ k.T / math.sqrt(c["d"])
    s = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
    if slope is not None:
        s = s - slope * (qpos[:, None] - j[None]).abs()
    s = torch.where(see, s, -math.inf)
    w = torch.where(see, torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)), 0.0)
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    o = w @ v
    if dout is None:
        return o
    dw = dout @ v.T
    ds = w * (dw - (w * dw).sum(-1, keepdim=True))
    if c["cap"]:
        ds = ds / torch.cosh(raw / c["cap"]) ** 2
    ds = ds / math.sqrt(c["d"])
    return o, ds @ k, ds.T @ q, w.T @ dout


def _exact_masked(c, s):
    B, n, g = c["B"], c["n"], c["h_q"] // c["h_kv"]
    q, k, v = (s[x].detach().double() for x in "qkv")
    res = {"out": torch.zeros_like(q)}
    if c["grad"]:
        res |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    i = torch.arange(n, device=DEV)
    for b in range(B):
        lo, hi = torch.zeros_like(i), (i + 1 if c["mask"] == "causal" else torch.full_like(i, n))
        if s["starts"] is not None:
            hi = torch.zeros_like(i)
            starts, prefix = s["starts"][b].tolist(), s["prefix"][b].tolist()
            for x in range(len(prefix)):
                a, e = starts[x], starts[x + 1]
                lo[a:e] = a
                hi[a:e] = (i[a:e] + 1).clamp(min=a + prefix[x])
        for h in range(c["h_q"]):
            kv = h // g
            slope = None if s["slopes"] is None else float(s["slopes"][h])
            args = (c, q[b, :, h], k[b, :, kv], v[b, :, kv], lo, hi, i, slope)
            if c["grad"]:
                o, dq, dk, dv = _attend64(*args, dout=s["dout"][b, :, h].double())
                res["dq"][b, :, h] = dq
                res["dk"][b, :, kv] += dk
                res["dv"][b, :, kv] += dv
            else:
                o = _attend64(*args)
            res["out"][b, :, h] = o
    return res


def _exact_paged(c, s):
    P, g = c["page"], c["h_q"] // c["h_kv"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    kp, vp = s["k_pages"].clone(), s["v_pages"].clone()
    at = 0
    for b, (m, L) in enumerate(_sequences(c)):
        where = torch.arange(L + m, device=DEV)
        page, row = s["table"][b].long()[where // P], where % P
        kp[page[L:], row[L:]] = s["k"][at:at + m]
        vp[page[L:], row[L:]] = s["v"][at:at + m]
        k, v = kp[page, row].double(), vp[page, row].double()
        qpos = L + torch.arange(m, device=DEV)
        for h in range(c["h_q"]):
            slope = None if s["slopes"] is None else float(s["slopes"][h])
            out[at:at + m, h] = _attend64(c, s["q"][at:at + m, h].double(), k[:, h // g], v[:, h // g],
                                          torch.zeros_like(qpos), qpos + 1, qpos, slope)
        at += m
    return {"out": out, "k_pages": kp.double(), "v_pages": vp.double()}


def _exact_axes(c, s):
    half, sections = c["rot"] // 2, s["sections"]
    axis = [a for a, x in enumerate(sections) for _ in range(x)]
    res = {x: s[x].detach().double() for x in ("q", "k") + (("dq", "dk") if c["grad"] else ())}
    for x, t in res.items():
        r = t.clone()
        for m in range(half):
            ang = (s["pos"][axis[m]].double() * float(s["freqs"][m]))[:, :, None]
            z = torch.complex(t[..., m], t[..., half + m]) * torch.polar(torch.ones_like(ang), -ang if x[0] == "d" else ang)
            r[..., m], r[..., half + m] = z.real, z.imag
        res[x] = r
    return res


def exact(case, seed):
    s = prepare(case, seed)
    return {"masked": _exact_masked, "paged": _exact_paged, "axes": _exact_axes}[case["op"]](case, s)
