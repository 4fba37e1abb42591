"""Operators of a language model's step beside those of ``operators.py``: new tokens
into a paged cache with their norms and rotations, attention of sequences that share
a prefix, tokens drawn from logits, and norms with the residual's addition.

``run`` computes them in elementary torch operations, in 32 bits (64 for the draws, whose
results turn on a border), where ``own`` is false, and through the package's entry points
where it is true; ``exact`` computes them from their definition in 64 bits.  The head
layout 16 / 8 / 128, the hidden width 1024 and the vocabularies are those of the Qwen3
shape that this repository is built for; the others are generic.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # The next token of eight answers into one layer: each decoding step makes this call
        # once a layer, and latency counts.
        {"name": "append_8x1", "kind": "append", "seqs": 8, "rows": 1, "before": 1000, "ragged": True, "heads": 16,
         "kv": 8, "dim": 128, "turned": 128, "interleaved": False, "norms": True, "page": 16, "type": "bf16"},
        # Three prompts of different lengths of a model that turns half of each head, pair by
        # pair, and has no norms there.
        {"name": "append_3x500", "kind": "append", "seqs": 3, "rows": 500, "before": 77, "ragged": True, "heads": 32,
         "kv": 4, "dim": 64, "turned": 32, "interleaved": True, "norms": False, "page": 64, "type": "f16"},
        # A chunk of four prompts of retrieved passages.
        {"name": "append_4x2048", "kind": "append", "seqs": 4, "rows": 2048, "before": 100, "ragged": False,
         "heads": 16, "kv": 8, "dim": 128, "turned": 128, "interleaved": False, "norms": True, "page": 16,
         "type": "bf16"},
        # A token of eight answers to one question over a few passages.
        {"name": "shared_8_of_2000", "kind": "shared", "groups": "8", "prefix": 2000, "own": 64, "heads": 16, "kv": 8,
         "dim": 128, "page": 16, "type": "bf16", "lse": False},
        # Questions over five long documents at once, some with one reader and some with many.
        {"name": "shared_5_groups", "kind": "shared", "groups": "1 12 3 7 2", "prefix": 30000, "own": 700,
         "heads": 32, "kv": 4, "dim": 64, "page": 64, "type": "f16", "lse": True},
        # Sixty-four samples of one long prompt, which go apart after it.
        {"name": "shared_64_of_8192", "kind": "shared", "groups": "64", "prefix": 8192, "own": 512, "heads": 16,
         "kv": 8, "dim": 128, "page": 16, "type": "bf16", "lse": True},
        # The next token of one answer: the smallest draw, at a small vocabulary.
        {"name": "sample_1x32768", "kind": "sample", "rows": 1, "vocab": 32768, "type": "bf16", "spread": 2.5,
         "filters": "all"},
        # Eight answers, each request with its own temperature and filters.
        {"name": "sample_8x155648", "kind": "sample", "rows": 8, "vocab": 155648, "type": "bf16", "spread": 2.5,
         "filters": "mixed"},
        # Sixty-four rows in 32 bits that are nearly flat, cut by their sum alone: almost every
        # token of the vocabulary stays a candidate.
        {"name": "sample_64x155648", "kind": "sample", "rows": 64, "vocab": 155648, "type": "f32", "spread": 1.0,
         "filters": "top_p"},
        # The norm between two products of a decoding step.
        {"name": "norm_8x1024", "kind": "norm", "rows": 8, "n": 1024, "add": True, "type": "bf16"},
        # Rows of an odd width, without an addition, at a prompt's start.
        {"name": "norm_1003x4099", "kind": "norm", "rows": 1003, "n": 4099, "add": False, "type": "f16"},
        # The same between two products of a long prompt.
        {"name": "norm_8192x1024", "kind": "norm", "rows": 8192, "n": 1024, "add": True, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], uniform over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


HEADS = [(16, 8, 128), (16, 8, 128), (32, 4, 64), (8, 8, 64), (32, 8, 128), (12, 1, 96), (28, 4, 128), (8, 2, 256)]


def draw(rng):
    kind = rng.choice(["append", "append", "shared", "shared", "shared", "sample", "sample", "norm"])
    heads, kv, dim = rng.choice(HEADS)
    at = {"page": rng.choice([16, 16, 32, 64, 128]), "heads": heads, "kv": kv, "dim": dim, "type": rng.choice(["bf16", "f16"])}
    if kind == "append":
        most = min(8192, (1 << 25) // ((heads + 2 * kv) * dim))
        rows = _log_int(rng, 1, min(2048, most))
        return {"kind": kind, "seqs": _log_int(rng, 1, max(1, min(64, most // rows))), "rows": rows,
                "before": rng.randint(0, 2000), "ragged": rng.random() < 0.5,
                "turned": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.4,
                "norms": rng.random() < 0.5, **at}
    if kind == "shared":
        groups = [_log_int(rng, 1, 32) for _ in range(rng.choice([1, 1, 2, rng.randint(1, 6)]))]
        # (no more bytes than the largest listed one reads, and its products)
        groups = groups[: max(1, 64 // max(groups))]
        most = min(32768, (8 << 20) // (kv * dim * len(groups)), 64 * 8192 * 2048 // (sum(groups) * heads * dim))
        return {"kind": kind, "groups": " ".join(map(str, groups)), "prefix": _log_int(rng, 1, most),
                "own": _log_int(rng, 1, max(1, min(1000, (16 << 20) // (kv * dim * sum(groups))))),
                "lse": rng.random() < 0.5, **at}
    if kind == "sample":
        vocab = _log_int(rng, 2, 160000)
        return {"kind": kind, "rows": _log_int(rng, 1, 64), "vocab": vocab, "type": rng.choice(["bf16", "f16", "f32"]),
                "spread": rng.choice([0.5, 1.0, 2.5, 6.0]), "filters": rng.choice(["none", "top_k", "top_p", "all", "mixed"])}
    n = _log_int(rng, 64, 16384)
    return {"kind": kind, "rows": _log_int(rng, 1, max(1, min(8192, (8 << 20) // n))), "n": n, "add": rng.random() < 0.7,
            "type": at["type"]}


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, torch.Generator(device=DEV).manual_seed(seed))


def run(state):
    return state["run"](state)


def work(case):
    return globals()["_work_" + case["kind"]](case)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed))


def _praghip():
    path = os.path.join(os.getcwd(), "privacy-rag_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import praghip
    return praghip


def _normal(g, *shape, type, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(type)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(g, need, c):
    """Pages at random places for sequences of need[s] pages each, and their tables."""
    count = sum(need)
    tables = torch.full((len(need), max(need) + 1), -1, dtype=torch.int32)
    order = torch.randperm(count + 3, generator=g, device=DEV)[:count].cpu().to(torch.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at: at + n]
        at += n
    shape = (count + 3, c["kv"], c["page"], c["dim"])
    return (_normal(g, *shape, type=TYPES[c["type"]]), _normal(g, *shape, type=TYPES[c["type"]]), tables)


# ------------------------------------------- new tokens into the cache (append)
def _stretches(c):
    """Each sequence's tokens before the call and in it: a function of the case."""
    rng = random.Random(c["seqs"] * 1000003 + c["before"])
    return [(c["before"] if not c["ragged"] or not i else rng.randint(0, c["before"]),
             c["rows"] if not c["ragged"] or not i else rng.randint(1, c["rows"])) for i in range(c["seqs"])]


def _prepare_append(c, g):
    pairs = _stretches(c)
    k_pages, v_pages, tables = _pages(g, [-(-(n + m) // c["page"]) for n, m in pairs], c)
    total, starts = sum(m for _, m in pairs), [sum(m for _, m in pairs[:i]) for i in range(len(pairs) + 1)]
    # the joint projection's rows, of which queries, keys and values are columns
    joint = _normal(g, total, c["heads"] + 2 * c["kv"], c["dim"], type=TYPES[c["type"]])
    q, k, v = joint.split((c["heads"], c["kv"], c["kv"]), 1)
    half = c["turned"] // 2
    places = torch.arange(tables.shape[1] * c["page"], dtype=torch.float64, device=DEV)
    angle = places[:, None] * 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    norms = [1 + _normal(g, c["dim"], type=torch.float32, scale=0.2).to(TYPES[c["type"]]) if c["norms"] else None for _ in "qk"]
    return {"run": _run_append, "q": q, "k": k, "v": v, "k_pages": k_pages, "v_pages": v_pages, "tables": tables.to(DEV),
            "lengths": _ints([n + m for n, m in pairs]), "starts": _ints(starts), "cos": angle.cos().float(),
            "sin": angle.sin().float(), "q_norm": norms[0], "k_norm": norms[1], "interleaved": c["interleaved"],
            "pairs": pairs}


def _run_append(s):
    if own:
        q = _praghip().page_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"],
                                   s["starts"], s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                   interleaved=s["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    starts, lengths, size = s["starts"].long(), s["lengths"].long(), s["k_pages"].shape[2]
    total = s["q"].shape[0]
    of = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), starts[1:] - starts[:-1], output_size=total)
    at = lengths[of] - starts[1:][of] + torch.arange(total, device=DEV)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    half = cos.shape[-1]

    def turned(x, norm):
        x = x.float()
        if norm is not None:
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * norm.float()
        if s["interleaved"]:
            a, b = x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]
            both = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half: 2 * half]
            both = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((both, x[..., 2 * half:]), -1).to(s["q"].dtype)

    entry = s["tables"].long()[of, at // size]
    s["k_pages"][entry, :, at % size] = turned(s["k"], s["k_norm"])
    s["v_pages"][entry, :, at % size] = s["v"]
    return turned(s["q"], s["q_norm"]), s["k_pages"], s["v_pages"]


def _exact_append(s):
    size = s["k_pages"].shape[2]
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    cos, sin = s["cos"].double(), s["sin"].double()
    half = cos.shape[1]
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + half)
    row = 0
    for n, (before, rows) in enumerate(s["pairs"]):
        place = torch.arange(before, before + rows, device=DEV)
        entry = s["tables"][n].long()[place // size]
        for x, weight, heads in ((s["q"], s["q_norm"], 0), (s["k"], s["k_norm"], 1)):
            y = x[row: row + rows].double()
            if weight is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * weight.double()
            a, b = y[..., first].clone(), y[..., second].clone()
            y[..., first] = a * cos[place][:, None] - b * sin[place][:, None]
            y[..., second] = a * sin[place][:, None] + b * cos[place][:, None]
            if heads:
                pools[0][entry, :, place % size] = y
            else:
                out[row: row + rows] = y
        pools[1][entry, :, place % size] = s["v"][row: row + rows].double()
        row += rows
    return (out, *pools)


def _work_append(c):
    tokens = sum(m for _, m in _stretches(c))
    values = tokens * (c["heads"] + c["kv"])
    return {"bytes": 4 * (values + tokens * c["kv"]) * c["dim"] + 4 * tokens * c["turned"],
            "flops": values * (3 * c["turned"] + (4 * c["dim"] if c["norms"] else 0))}


# --------------------------------------- sequences that share a prefix (shared)
def _members(c):
    """(shared tokens, the members' lengths) of each group: a function of the case."""
    groups = [int(n) for n in c["groups"].split()]
    rng = random.Random(sum(groups) * 1000003 + c["prefix"])
    out = []
    for i, n in enumerate(groups):
        shared = c["prefix"] if not i else rng.randint(1, c["prefix"])
        out.append((shared, [shared + (c["own"] if not j else rng.randint(0, c["own"])) for j in range(n)]))
    return out


def _prepare_shared(c, g):
    # as forks leave it: the prefix's full pages are everybody's, what follows is each one's
    # own (a page that the prefix ends in is a copy for each)
    groups, page = _members(c), c["page"]
    need, of = [], []
    for shared, lengths in groups:
        whole, first = shared // page, len(need)
        need.append(whole)
        for n in lengths:
            of.append((first, len(need)))
            need.append(-(-n // page) - whole)
    k, v, named = _pages(g, need, c)
    lengths = [n for _, group in groups for n in group]
    tables = torch.full((len(lengths), max(-(-n // page) for n in lengths) + 2), -1, dtype=torch.int32)
    for s, (a, b) in enumerate(of):
        tables[s, : need[a]] = named[a, : need[a]]
        tables[s, need[a]: need[a] + need[b]] = named[b, : need[b]]
    starts, first = [0], 0
    for shared, group in groups:
        last, rest = shared // page, shared % page
        if rest and len(group) > 1:
            entry = tables[first: first + len(group), last].long().to(DEV)
            for x in (k, v):
                x[entry[1:], :, :rest] = x[entry[:1], :, :rest]
        first += len(group)
        starts.append(first)
    q = _normal(g, len(lengths), c["heads"], c["dim"], type=TYPES[c["type"]])
    return {"run": _run_shared, "q": q, "k": k, "v": v, "tables": tables.to(DEV), "lengths": _ints(lengths),
            "groups": _ints(starts), "shared": _ints([n for n, _ in groups]), "longest": max(lengths), "lse": c["lse"],
            "members": groups}


def _run_shared(s):
    if own:
        return _praghip().paged_shared(s["q"], s["k"], s["v"], s["tables"], s["lengths"], s["groups"], s["shared"],
                                       max_length=s["longest"], lse=s["lse"])
    q, size = s["q"], s["k"].shape[2]
    seqs, heads, dim = q.shape
    kv = s["k"].shape[1]
    out = torch.empty((seqs, heads, dim), dtype=torch.float32, device=DEV)
    lse = torch.empty((seqs, heads), dtype=torch.float32, device=DEV)
    first = 0
    for shared, lengths in s["members"]:
        n, longest = len(lengths), max(lengths) - shared
        rows = slice(first, first + n)
        group = q[rows].float().view(n, kv, heads // kv, dim)
        # the prefix once for all, what follows for each
        at = torch.arange(shared, device=DEV)
        entry = s["tables"][first].long()[at // size]
        k, v = (s[x][entry, :, at % size].float().transpose(0, 1) for x in "kv")
        one = torch.matmul(group.transpose(0, 1).reshape(kv, -1, dim), k.transpose(1, 2)).view(kv, n, -1, shared).transpose(0, 1)
        at = shared + torch.arange(longest, device=DEV)[None].expand(n, -1)
        seen = at < s["lengths"][rows, None]
        entry = torch.gather(s["tables"][rows].long(), 1, torch.where(seen, at, 0) // size).clamp(min=0)
        k2, v2 = (s[x][entry, :, at % size].float().masked_fill(~seen[..., None, None], 0).transpose(1, 2) for x in "kv")
        two = torch.matmul(group, k2.transpose(2, 3)).masked_fill(~seen[:, None, None], -math.inf)
        scores = torch.cat((one, two), -1) / math.sqrt(dim)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - top)
        total = p.sum(-1, keepdim=True)
        p = p / total
        o = torch.matmul(p[..., :shared].transpose(0, 1).reshape(kv, -1, shared), v).view(kv, n, -1, dim).transpose(0, 1)
        out[rows] = (o + torch.matmul(p[..., shared:], v2)).reshape(n, heads, dim)
        lse[rows] = (top + torch.log(total)).reshape(n, heads)
        first += n
    out = out.to(q.dtype)
    return (out, lse) if s["lse"] else out


def _exact_shared(s):
    """Each sequence by itself, over its own table."""
    q, page = s["q"].double(), s["k"].shape[2]
    seqs, heads, dim = q.shape
    kv = s["k"].shape[1]
    out, lse = torch.zeros_like(q), torch.zeros((seqs, heads), dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n, device=DEV)
        entry = s["tables"][i].long()[at // page]
        k, v = (s[x][entry, :, at % page].double() for x in "kv")
        for h in range(heads):
            score = (k[:, h * kv // heads] @ q[i, h]) * dim ** -0.5
            lse[i, h] = torch.logsumexp(score, 0)
            out[i, h] = torch.exp(score - lse[i, h]) @ v[:, h * kv // heads]
    return (out, lse) if s["lse"] else out


def _work_shared(c):
    groups = _members(c)
    keys = sum(shared + sum(n - shared for n in group) for shared, group in groups)
    seqs, pairs = sum(len(group) for _, group in groups), sum(sum(group) for _, group in groups)
    return {"bytes": 4 * keys * c["kv"] * c["dim"] + 4 * seqs * c["heads"] * c["dim"], "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------ tokens from logits (sample)
def _prepare_sample(c, g):
    # a wide spread of unlikely tokens and a few that stand out, as a model's logits have them
    rows, vocab = c["rows"], c["vocab"]
    logits = torch.randn((rows, vocab), generator=g, device=DEV) * c["spread"]
    at = torch.randint(0, vocab, (rows, min(vocab, 12)), generator=g, device=DEV)
    logits.scatter_add_(1, at, torch.rand(at.shape, generator=g, device=DEV) * 5 * c["spread"])
    made = {"temperature": torch.rand(rows, generator=g, device=DEV) + 0.4,
            "top_k": torch.randint(1, 200, (rows,), generator=g, device=DEV, dtype=torch.int32),
            "top_p": torch.rand(rows, generator=g, device=DEV) * 0.6 + 0.4,
            "min_p": torch.rand(rows, generator=g, device=DEV) * 0.05}
    if c["filters"] == "mixed":  # greedy rows, and rows without one filter or the other
        turn = torch.arange(rows, device=DEV) % 5
        made["temperature"][turn == 4] = 0
        made["top_k"][turn % 2 == 0] = 0
        made["top_p"][turn == 1] = 1
        made["min_p"][turn == 2] = 0
    elif c["filters"] != "all":
        made = {x: made[x] for x in ("temperature", c["filters"]) if x in made}
    return {"run": _run_sample, "logits": logits.to(TYPES[c["type"]]),
            "uniform": torch.rand(rows, generator=g, device=DEV), "filters": made}


def _run_sample(s):
    if own:
        return _praghip().sample_tokens(s["logits"], s["uniform"], **s["filters"])
    x, f = s["logits"].double(), s["filters"]
    vocab = x.shape[1]
    top = x.amax(1, keepdim=True)
    t = f["temperature"].double()[:, None]
    index = torch.arange(vocab, device=DEV)[None]
    weight = torch.exp((x - top) / torch.where(t == 0, 1.0, t))
    if "top_k" in f or "top_p" in f:
        order = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices
        sorted_weight = torch.gather(weight, 1, order)
        if "top_k" in f:
            k = f["top_k"].long()[:, None]
            sorted_weight = torch.where((index < k) | (k == 0), sorted_weight, 0.0)
        if "top_p" in f:
            sums = torch.cumsum(sorted_weight, 1)
            p = f["top_p"].double()[:, None]
            # what stands before a token has to fall short of the share
            keep = (sums - sorted_weight < p * sums[:, -1:]) | (p >= 1)
            sorted_weight = torch.where(keep, sorted_weight, 0.0)
        weight = torch.zeros_like(weight).scatter_(1, order, sorted_weight)
    if "min_p" in f:
        weight = torch.where(weight >= f["min_p"].double()[:, None], weight, 0.0)
    sums = torch.cumsum(weight, 1)
    token = (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(1)
    token = torch.minimum(token, torch.where(weight > 0, index, -1).amax(1))
    return torch.where(t[:, 0] == 0, torch.where(x == top, index, vocab).amin(1), token)


def _exact_sample(s):
    out = []
    f = {name: value.tolist() for name, value in s["filters"].items()}
    for row, u in enumerate(s["uniform"].tolist()):
        x = s["logits"][row].double()
        n, t = x.numel(), f["temperature"][row]
        by = torch.argsort(-x, stable=True)  # the likeliest first, the lower index of two alike
        if not t:
            out.append(int(by[0]))
            continue
        weight = torch.softmax(x[by] / t, 0)
        count = f["top_k"][row] if f.get("top_k") and f["top_k"][row] else n
        weight, by = weight[:count], by[:count]
        if f.get("top_p") and f["top_p"][row] < 1:
            reached = torch.cumsum(weight, 0) >= f["top_p"][row] * weight.sum()
            count = int(torch.nonzero(reached)[0]) + 1 if bool(reached.any()) else len(by)
            weight, by = weight[:count], by[:count]
        if f.get("min_p"):
            here = weight >= f["min_p"][row] * weight[0]
            weight, by = weight[here], by[here]
        at, back = torch.sort(by)
        sums = torch.cumsum(weight[back], 0)
        i = int(torch.searchsorted(sums, u * float(sums[-1]), right=True))
        out.append(int(at[min(i, len(at) - 1)]))
    return torch.tensor(out, device=DEV)


def _work_sample(c):
    values = c["rows"] * c["vocab"]
    return {"bytes": values * BYTES[c["type"]] + 28 * c["rows"], "flops": 4 * values}


# ------------------------------------- norms with the residual's addition (norm)
def _prepare_norm(c, g):
    type = TYPES[c["type"]]
    x = _normal(g, c["rows"], c["n"], type=type)
    return {"run": _run_norm, "x": x, "residual": _normal(g, c["rows"], c["n"], type=type, scale=3.0) if c["add"] else None,
            "weight": (1 + 0.2 * torch.randn(c["n"], generator=g, device=DEV)).to(type)}


def _run_norm(s):
    if own:
        return _praghip().add_norm(s["x"], s["weight"], s["residual"])
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = (x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * s["weight"].float()).to(s["x"].dtype)
    return y if s["residual"] is None else (y, x.to(s["x"].dtype))


def _exact_norm(s):
    total = s["x"].double()
    if s["residual"] is not None:
        total = total + s["residual"].double()
    size = torch.sqrt((total ** 2).sum(1, keepdim=True) / total.shape[1] + 1e-6)
    y = total / size * s["weight"].double()
    return y if s["residual"] is None else (y, total)


def _work_norm(c):
    values = c["rows"] * c["n"]
    return {"bytes": 2 * values * (4 if c["add"] else 2) + 2 * c["n"], "flops": values * (5 if c["add"] else 4)}
