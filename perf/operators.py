"""Operators of a language model's serving path: attention over a paged key/value
cache (one new token per sequence, or a prompt's tokens), the cache's pages, and
products of a few rows with 4-bit weights.

``run`` computes them in elementary torch operations in 32 bits where ``own`` is
false, and through the package's entry points where it is true; ``exact`` computes
the attention and the products from their definition in 64 bits.  The head layout
16 / 8 / 128, the hidden width 1024 and the 28 layers are those of the Qwen3 shape
that this repository is built for; the others are generic.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # The next token of one answer over a prompt and a few passages: the
        # smallest call of a decoding loop, where latency counts.
        {"name": "decode_1x2049", "kind": "decode", "seqs": 1, "longest": 2049, "ragged": False, "heads": 16, "kv": 8,
         "dim": 128, "page": 16, "window": 0, "sinks": 0, "type": "bf16", "lse": False},
        # The next token of 64 answers that are at very different lengths, empty
        # slots among them: the ordinary step of a batch server.
        {"name": "decode_64_ragged", "kind": "decode", "seqs": 64, "longest": 8192, "ragged": True, "heads": 16,
         "kv": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "type": "bf16", "lse": True},
        # Four long sessions with a window and four first tokens kept; pages that
        # left the window have been given back, and there are few rows to fill
        # the GPU with.
        {"name": "decode_window_131072", "kind": "decode", "seqs": 4, "longest": 131072, "ragged": False, "heads": 32,
         "kv": 4, "dim": 64, "page": 64, "window": 32768, "sinks": 4, "type": "f16", "lse": False},
        # Three short questions of up to 77 tokens, each from an empty cache.
        {"name": "prompt_3x77", "kind": "prompt", "seqs": 3, "rows": 77, "before": 0, "ragged": True, "heads": 16,
         "kv": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "type": "bf16", "lse": False},
        # A 512-token chunk of four long prompts, through a window and sinks over
        # what the cache holds of the chunks before.
        {"name": "prompt_window_4x512", "kind": "prompt", "seqs": 4, "rows": 512, "before": 7681, "ragged": True,
         "heads": 32, "kv": 4, "dim": 64, "page": 64, "window": 2048, "sinks": 4, "type": "f16", "lse": True},
        # One whole prompt of retrieved passages, 8192 tokens, causal: the largest
        # product of the path.
        {"name": "prompt_8192", "kind": "prompt", "seqs": 1, "rows": 8192, "before": 0, "ragged": False, "heads": 16,
         "kv": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "type": "bf16", "lse": False},
        # The new keys and values of one token of 64 sequences, in one layer.
        {"name": "write_64x1", "kind": "write", "seqs": 64, "rows": 1, "before": 2000, "kv": 8, "dim": 128,
         "page": 16, "type": "bf16"},
        # A chunk of four prompts written into one layer's pages.
        {"name": "write_4x2048", "kind": "write", "seqs": 4, "rows": 2048, "before": 100, "kv": 8, "dim": 128,
         "page": 16, "type": "bf16"},
        # Eight candidate answers branch off each of two prompts in all 28 layers:
        # whole pages are shared, the last one is copied for each.
        {"name": "fork_2x8", "kind": "fork", "parents": 2, "each": 8, "length": 1001, "layers": 28, "kv": 8,
         "dim": 128, "page": 16, "type": "bf16"},
        # Half of the sequences end, the pages of the others move together, and
        # as many new ones are admitted.
        {"name": "compact_32", "kind": "compact", "seqs": 32, "length": 160, "layers": 28, "kv": 8, "dim": 128,
         "page": 16, "type": "bf16"},
        # The joint q/k/v projection of one new token.
        {"name": "w4_1x1024x4096", "kind": "w4", "m": 1, "k": 1024, "n": 4096, "group": 128, "zeros": False,
         "type": "bf16"},
        # The output head over the padded vocabulary for 16 answers.
        {"name": "w4_16x1024x155648", "kind": "w4", "m": 16, "k": 1024, "n": 155648, "group": 64, "zeros": True,
         "type": "f16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], uniform over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


HEADS = [(16, 8, 128), (16, 8, 128), (32, 4, 64), (8, 8, 64), (32, 8, 128), (12, 1, 96), (28, 4, 128)]


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "prompt", "write", "fork", "compact", "w4", "w4"])
    heads, kv, dim = rng.choice(HEADS)
    page, kind_of = rng.choice([16, 16, 32, 64, 128]), rng.choice(["bf16", "f16"])
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 4096), rng.randint(0, 8))])
    at = {"page": page, "type": kind_of, "kv": kv, "dim": dim}
    if kind == "decode":
        seqs = _log_int(rng, 1, 64)
        return {"kind": kind, "seqs": seqs, "longest": _log_int(rng, 1, min(131072, 153600 * 1024 // (seqs * kv * dim))),
                "ragged": rng.random() < 0.7, "heads": heads, "window": window, "sinks": sinks,
                "lse": rng.random() < 0.5, **at}
    if kind == "prompt":
        seqs, rows = _log_int(rng, 1, 8), _log_int(rng, 1, 4096)
        seqs = max(1, min(seqs, 8192 // rows))
        most = min(8192, 4096 * 8192 * 2048 // (seqs * rows * heads * dim) - rows // 2)
        return {"kind": kind, "seqs": seqs, "rows": rows, "before": rng.choice([0, _log_int(rng, 1, most)]),
                "ragged": rng.random() < 0.5, "heads": heads, "window": window, "sinks": sinks,
                "lse": rng.random() < 0.5, **at}
    if kind == "write":
        rows = _log_int(rng, 1, 2048)
        return {"kind": kind, "seqs": _log_int(rng, 1, max(1, min(64, 8192 // rows))), "rows": rows,
                "before": rng.randint(0, 2000), **at}
    if kind == "fork":
        return {"kind": kind, "parents": rng.randint(1, 3), "each": rng.randint(1, 8),
                "length": _log_int(rng, 1, 2000), "layers": rng.randint(1, 28), **at, "kv": 8, "dim": 128, "page": 16}
    if kind == "compact":
        return {"kind": kind, "seqs": 2 * rng.randint(1, 16), "length": _log_int(rng, 16, 160),
                "layers": rng.randint(1, 28), **at, "kv": 8, "dim": 128, "page": 16}
    return {"kind": kind, "m": _log_int(rng, 1, 32), "k": _log_int(rng, 64, 8192), "n": _log_int(rng, 16, 9000),
            "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "type": kind_of}


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, torch.Generator(device=DEV).manual_seed(seed))


def run(state):
    return state["run"](state)


def work(case):
    return globals()["_work_" + case["kind"]](case)


def exact(case, seed):
    made = globals().get("_exact_" + case["kind"])
    return made(prepare(case, seed)) if made else None


def _praghip():
    path = os.path.join(os.getcwd(), "privacy-rag_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import praghip
    return praghip


def _normal(g, *shape, type, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(type)


# ------------------------------------------------------------------ sequences
def _lengths(case):
    """Each sequence's tokens before and in the call: a function of the case."""
    rng = random.Random(case["seqs"] * 1000003 + case.get("longest", case.get("before", 0)))
    if case["kind"] == "decode":
        return [(rng.choice([0, 1, rng.randint(1, case["longest"]), rng.randint(1, case["longest"]),
                             rng.randint(1, case["longest"])]) if case["ragged"] and i else case["longest"], 1)
                for i in range(case["seqs"])]
    full = not case.get("ragged")
    return [(case["before"] if full or not i else rng.randint(0, case["before"]),
             case["rows"] if full or not i else rng.randint(1, case["rows"])) for i in range(case["seqs"])]


def _cache(case, g, lengths):
    """One layer's keys and values for sequences of these lengths, in pages at
    random places; pages that no later token can see are given back (entry -1)."""
    page, window, sinks = case["page"], case.get("window", 0), case.get("sinks", 0)
    width = max(1, max(-(-n // page) for n in lengths))
    first = [max(0, n - case.get("rows", 1) - window + 1) if window else 0 for n in lengths]
    held = [[c * page < n and (c * page < sinks or (c + 1) * page > lo) for c in range(width)]
            for n, lo in zip(lengths, first)]
    mask = torch.tensor(held, dtype=torch.bool)
    count = int(mask.sum())
    order = torch.randperm(count + 3, generator=g, device=DEV)[:count].to(torch.int32)
    tables = torch.full(mask.shape, -1, dtype=torch.int32)
    tables[mask] = order.cpu()
    shape = (count + 3, case["kv"], page, case["dim"])
    return (_normal(g, *shape, type=TYPES[case["type"]]), _normal(g, *shape, type=TYPES[case["type"]]),
            tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))


def _gather(pages, tables, at):
    """[seqs][positions][kv][dim] in 32 bits of the positions at[seqs][positions]."""
    size = pages.shape[2]
    entry = torch.gather(tables.long(), 1, (at // size).clamp(max=tables.shape[1] - 1)).clamp(min=0)
    return pages[entry, :, at % size].float()


def _softmax(scores, seen):
    """Probabilities over the last dim and the logarithm of their sum; rows that
    see nothing get zeros and -inf."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total), (top + torch.log(total))[..., 0]


# ---------------------------------------------------- one new token (decode)
def _prepare_decode(c, g):
    lengths = [n for n, _ in _lengths(c)]
    k, v, tables, held = _cache(c, g, lengths)
    q = _normal(g, c["seqs"], c["heads"], c["dim"], type=TYPES[c["type"]])
    return {"run": _run_decode, "q": q, "k": k, "v": v, "tables": tables, "lengths": held, "longest": max(lengths),
            "window": c["window"], "sinks": c["sinks"], "lse": c["lse"]}


def _run_decode(s):
    if own:
        return _praghip().paged_decode(s["q"], s["k"], s["v"], s["tables"], s["lengths"], window=s["window"],
                                       sinks=s["sinks"], max_length=s["longest"], lse=s["lse"])
    q, lengths, longest = s["q"], s["lengths"].long(), s["longest"]
    seqs, heads, dim = q.shape
    kv = s["k"].shape[1]
    # the positions that the window and the sinks leave, side by side
    lo = (lengths - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(lengths)
    few = lo.clamp(max=s["sinks"])
    span = min(longest, s["window"] + s["sinks"]) if s["window"] else longest
    i = torch.arange(max(span, 1), device=DEV)[None]
    at = torch.where(i < few[:, None], i, i - few[:, None] + lo[:, None])
    seen = at < lengths[:, None]
    at = torch.where(seen, at, torch.zeros_like(at))
    k, v = (_gather(s[x], s["tables"], at).masked_fill(~seen[..., None, None], 0) for x in "kv")
    scores = torch.matmul(q.float().view(seqs, kv, heads // kv, dim), k.permute(0, 2, 3, 1)) / math.sqrt(dim)
    p, lse = _softmax(scores, seen[:, None, None])
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(seqs, heads, dim).to(q.dtype)
    return (out, lse.reshape(seqs, heads)) if s["lse"] else out


def _exact_decode(s):
    return _exact_rows(s, list(range(len(s["q"]))) + [len(s["q"])])


def _work_decode(c):
    keys = sum(min(n, c["window"] + c["sinks"]) if c["window"] else n for n, _ in _lengths(c))
    return {"bytes": 4 * keys * c["kv"] * c["dim"] + 4 * c["seqs"] * c["heads"] * c["dim"],
            "flops": 4 * keys * c["heads"] * c["dim"]}


def _exact_rows(s, starts):
    """Attention of rows starts[i] .. starts[i+1] of q over sequence i, in 64 bits."""
    q, page = s["q"].double(), s["k"].shape[2]
    heads, dim, kv = q.shape[1], q.shape[2], s["k"].shape[1]
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lengths"].tolist()):
        a, b = starts[i], starts[i + 1]
        if not n or a == b:
            continue
        at = torch.arange(n, device=DEV)
        entry = s["tables"][i].long()[at // page]
        k, v = (s[x][entry.clamp(min=0), :, at % page].double() for x in "kv")
        place = torch.arange(n - (b - a), n, device=DEV)[:, None]
        seen = at[None] <= place
        if s["window"]:
            seen &= (at[None] > place - s["window"]) | (at[None] < s["sinks"])
        for h in range(heads):
            score = (q[a:b, h] @ k[:, h * kv // heads].T) * dim ** -0.5
            lse[a:b, h] = torch.logsumexp(score.masked_fill_(~seen, -math.inf), -1)
            out[a:b, h] = torch.exp(score - lse[a:b, h, None]) @ v[:, h * kv // heads]
    return (out, lse) if s["lse"] else out


# ------------------------------------------------------ many tokens (prompt)
def _prepare_prompt(c, g):
    rows = [m for _, m in _lengths(c)]
    lengths = [n + m for n, m in _lengths(c)]
    k, v, tables, held = _cache(c, g, lengths)
    starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
    q = _normal(g, starts[-1], c["heads"], c["dim"], type=TYPES[c["type"]])
    return {"run": _run_prompt, "q": q, "k": k, "v": v, "tables": tables, "lengths": held, "longest": max(lengths),
            "starts": torch.tensor(starts, dtype=torch.int32, device=DEV), "rows": max(rows), "window": c["window"],
            "sinks": c["sinks"], "lse": c["lse"], "starts_list": starts}


def _run_prompt(s):
    if own:
        return _praghip().paged_prompt(s["q"], s["k"], s["v"], s["tables"], s["lengths"], s["starts"], s["rows"],
                                       window=s["window"], sinks=s["sinks"], max_length=s["longest"], lse=s["lse"])
    q, lengths, starts = s["q"], s["lengths"].long(), s["starts"].long()
    total, heads, dim = q.shape
    kv, seqs = s["k"].shape[1], len(lengths)
    # one row of keys per sequence, one block of queries per sequence
    count = starts[1:] - starts[:-1]
    r = torch.arange(s["rows"], device=DEV)[None]
    mine = r < count[:, None]
    row = (starts[:-1, None] + r).clamp(max=total - 1)
    place = torch.where(mine, lengths[:, None] - count[:, None] + r, torch.full_like(row, -1))[..., None]
    at = torch.arange(s["longest"], device=DEV)[None]
    k, v = (_gather(s[x], s["tables"], at.expand(seqs, -1)).masked_fill(~(at < lengths[:, None])[..., None, None], 0)
            for x in "kv")
    seen = at[:, None] <= place
    if s["window"]:
        seen &= (at[:, None] > place - s["window"]) | (at[:, None] < s["sinks"])
    group = q[row].float().view(seqs, -1, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(group, k.permute(0, 2, 3, 1)[:, :, None]) / math.sqrt(dim)
    p, lse = _softmax(scores, seen[:, None, None])
    out = torch.matmul(p, v.permute(0, 2, 1, 3)[:, :, None])
    of = torch.repeat_interleave(torch.arange(seqs, device=DEV), count, output_size=total)
    i = torch.arange(total, device=DEV) - starts[of]
    out = out.permute(0, 3, 1, 2, 4)[of, i].reshape(total, heads, dim).to(q.dtype)
    return (out, lse.permute(0, 3, 1, 2)[of, i].reshape(total, heads)) if s["lse"] else out


def _exact_prompt(s):
    return _exact_rows(s, s["starts_list"])


def _work_prompt(c):
    pairs, keys, rows = 0, 0, 0
    for n, m in _lengths(c):
        w, few = c["window"], c["sinks"]
        if w:
            pairs += sum(min(p, w + min(few, max(0, p - w))) for p in range(n + 1, n + m + 1))
            keys += min(n + m, m - 1 + w + few)
        else:
            pairs += m * n + m * (m + 1) // 2
            keys += n + m
        rows += m
    return {"bytes": 4 * keys * c["kv"] * c["dim"] + 4 * rows * c["heads"] * c["dim"],
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------ the cache's pages
def _prepare_write(c, g):
    pairs = _lengths(c)
    k, v, tables, lengths = _cache(c, g, [n + m for n, m in pairs])
    rows = sum(m for _, m in pairs)
    starts = [sum(m for _, m in pairs[:i]) for i in range(len(pairs) + 1)]
    new = _normal(g, 2, rows, c["kv"], c["dim"], type=TYPES[c["type"]])
    return {"run": _run_write, "k": k, "v": v, "tables": tables, "lengths": lengths, "new": new,
            "starts": torch.tensor(starts, dtype=torch.int32, device=DEV)}


def _run_write(s):
    if own:
        _praghip().page_write(s["new"][0], s["new"][1], s["k"], s["v"], s["tables"], s["lengths"], s["starts"])
        return s["k"], s["v"]
    starts, lengths, size = s["starts"].long(), s["lengths"].long(), s["k"].shape[2]
    total = s["new"].shape[1]
    of = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), starts[1:] - starts[:-1], output_size=total)
    at = lengths[of] - starts[1:][of] + torch.arange(total, device=DEV)
    entry = s["tables"].long()[of, at // size]
    s["k"][entry, :, at % size] = s["new"][0]
    s["v"][entry, :, at % size] = s["new"][1]
    return s["k"], s["v"]


def _work_write(c):
    return {"bytes": 8 * c["seqs"] * c["rows"] * c["kv"] * c["dim"], "flops": 0}


def _pool(c, g, pages):
    """Every layer's keys and values: [layers][2][pages][kv][page][dim]."""
    out = torch.empty((c["layers"], 2, pages, c["kv"], c["page"], c["dim"]), dtype=TYPES[c["type"]], device=DEV)
    return out.normal_(generator=g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _prepare_fork(c, g):
    # the parents' pages at random places, the children as an earlier fork left them
    per, children = -(-c["length"] // c["page"]), c["parents"] * c["each"]
    pages, seqs = c["parents"] * per + children + 5, c["parents"] + children
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((seqs, per + 4), -1, dtype=torch.int32, device=DEV)
    tables[: c["parents"], :per] = order[: c["parents"] * per].view(c["parents"], per)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[order[: c["parents"] * per].long()] = 1
    lengths = _ints([c["length"]] * c["parents"] + [0] * children)
    s = {"run": _run_fork, "pool": _pool(c, g, pages), "tables": tables, "lengths": lengths, "refs": refs,
         "page": c["page"], "parents": _ints([i // c["each"] for i in range(children)]),
         "children": _ints([c["parents"] + i for i in range(children)])}
    _plain_fork(s, s["parents"].long(), s["children"].long())
    return s


def _plain_free(s, seqs):
    rows = s["tables"][seqs]
    s["refs"].index_add_(0, rows.clamp(min=0).long().flatten(), -(rows >= 0).to(torch.int32).flatten())
    s["tables"][seqs] = -1
    s["lengths"][seqs] = 0


def _plain_fork(s, parents, children):
    lengths, rows = s["lengths"][parents], s["tables"][parents]
    count = (lengths + s["page"] - 1) // s["page"]
    column = torch.arange(rows.shape[1], device=DEV)[None]
    rows = torch.where(column < count[:, None], rows, -1)
    last = (count - 1).clamp(min=0).long()[:, None]
    old = torch.gather(rows, 1, last)[:, 0]
    apart = (lengths % s["page"] > 0) & (old >= 0)  # a last page that is not full is copied
    free = torch.nonzero(s["refs"] == 0)[:, 0].to(torch.int32)
    new = free[(torch.cumsum(apart, 0) - 1).clamp(min=0)]
    rows = rows.scatter(1, last, torch.where(apart, new, old)[:, None])
    s["tables"][children] = rows
    s["lengths"][children] = lengths
    s["refs"].index_add_(0, rows.clamp(min=0).long().flatten(), (rows >= 0).to(torch.int32).flatten())
    s["pool"][:, :, new[apart].long()] = s["pool"][:, :, old[apart].long()]


def _run_fork(s):
    # the last answers end, and the next ones branch off the same prompts
    if own:
        p = _praghip()
        p.page_free(s["tables"], s["lengths"], s["refs"], s["children"])
        p.page_fork(s["pool"], s["tables"], s["lengths"], s["refs"], s["parents"], s["children"])
    else:
        _plain_free(s, s["children"].long())
        _plain_fork(s, s["parents"].long(), s["children"].long())
    return s["pool"], s["tables"], s["lengths"], s["refs"]


def _work_fork(c):
    children, per = c["parents"] * c["each"], -(-c["length"] // c["page"])
    copied = children if c["length"] % c["page"] else 0
    return {"bytes": 4 * copied * c["layers"] * 2 * c["kv"] * c["page"] * c["dim"] + 24 * children * per, "flops": 0}


def _prepare_compact(c, g):
    # the half that ends first sits in the lower pages, as the pass before left it
    per, half = -(-c["length"] // c["page"]), c["seqs"] // 2
    pages = c["seqs"] * per + 7
    low, high = (torch.randperm(half * per, generator=g, device=DEV).to(torch.int32) for _ in range(2))
    tables = torch.full((c["seqs"], per + 4), -1, dtype=torch.int32, device=DEV)
    tables[:, :per] = torch.cat([low, high + half * per]).view(c["seqs"], per)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[: c["seqs"] * per] = 1
    return {"run": _run_compact, "pool": _pool(c, g, pages), "tables": tables, "refs": refs, "page": c["page"],
            "lengths": _ints([c["length"]] * c["seqs"]), "turn": 0, "counts": _ints([c["length"]] * half),
            "halves": [_ints(list(range(half))), _ints(list(range(half, c["seqs"])))]}


def _plain_compact(s):
    held = s["refs"] > 0
    count = held.sum()
    index = torch.arange(len(held), device=DEV)
    moved = torch.nonzero(held & (index >= count))[:, 0]
    holes = torch.nonzero(~held & (index < count))[:, 0]
    place = index.to(torch.int32)
    place[moved] = holes.to(torch.int32)
    s["pool"][:, :, holes] = s["pool"][:, :, moved]
    s["refs"][holes] = s["refs"][moved]
    s["refs"][moved] = 0
    s["tables"].copy_(torch.where(s["tables"] >= 0, place[s["tables"].clamp(min=0).long()], -1))


def _plain_reserve(s, seqs, counts):
    old = s["lengths"][seqs]
    column = torch.arange(s["tables"].shape[1], device=DEV)[None]
    more = (column >= ((old + s["page"] - 1) // s["page"])[:, None]) \
        & (column < ((old + counts + s["page"] - 1) // s["page"])[:, None])
    free = torch.nonzero(s["refs"] == 0)[:, 0].to(torch.int32)
    new = free[(torch.cumsum(more.flatten(), 0) - 1).clamp(min=0)].view(more.shape)
    s["tables"][seqs] = torch.where(more, new, s["tables"][seqs])
    s["lengths"][seqs] = old + counts
    s["refs"].index_add_(0, torch.where(more, new, 0).long().flatten(), more.to(torch.int32).flatten())


def _run_compact(s):
    # each pass ends the half that the pass before kept
    seqs = s["halves"][s["turn"]]
    s["turn"] ^= 1
    if own:
        p = _praghip()
        p.page_free(s["tables"], s["lengths"], s["refs"], seqs)
        p.page_compact(s["pool"], s["tables"], s["refs"])
        p.page_reserve(s["tables"], s["lengths"], s["refs"], s["page"], seqs, s["counts"])
    else:
        _plain_free(s, seqs.long())
        _plain_compact(s)
        _plain_reserve(s, seqs.long(), s["counts"])
    return s["pool"], s["tables"], s["lengths"], s["refs"]


def _work_compact(c):
    moved = (c["seqs"] // 2) * -(-c["length"] // c["page"])
    return {"bytes": 4 * moved * c["layers"] * 2 * c["kv"] * c["page"] * c["dim"] + 24 * c["seqs"] * moved, "flops": 0}


# ------------------------------------------------------- 4-bit weights (w4)
def _prepare_w4(c, g):
    # rows of nibbles, the lower one first; a row ends on 16 bytes, groups of the
    # last row's length may be short
    width, groups = -(-c["k"] // 32) * 16, -(-c["k"] // c["group"])
    packed = torch.randint(0, 256, (c["n"], width), generator=g, device=DEV, dtype=torch.uint8)
    scales = (torch.rand((c["n"], groups), generator=g, device=DEV) * 0.02 + 0.001).to(TYPES[c["type"]])
    zeros = torch.randint(0, 16, (c["n"], groups), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None
    return {"run": _run_w4, "x": _normal(g, c["m"], c["k"], type=TYPES[c["type"]]), "w": packed, "scales": scales,
            "zeros": zeros, "group": c["group"]}


def _run_w4(s):
    if own:
        return _praghip().matvec_w4(s["x"], s["w"], s["scales"], s["zeros"], group=s["group"])
    k = s["x"].shape[1]
    w = torch.stack((s["w"] & 15, s["w"] >> 4), -1).flatten(1)[:, :k].float()
    group = torch.arange(k, device=DEV) // s["group"]
    zero = s["zeros"].float()[:, group] if s["zeros"] is not None else 8.0
    w = (w - zero) * s["scales"].float()[:, group]
    return torch.matmul(s["x"].float(), w.T).to(s["x"].dtype)


def _exact_w4(s):
    x = s["x"].double()
    y = torch.zeros((x.shape[0], s["w"].shape[0]), dtype=torch.float64, device=DEV)
    for g in range(s["scales"].shape[1]):
        lo, hi = g * s["group"], min((g + 1) * s["group"], x.shape[1])
        at = torch.arange(lo, hi, device=DEV)
        digit = (s["w"][:, at // 2].long() >> (4 * (at % 2))) % 16
        digit = digit - (s["zeros"][:, g, None].long() if s["zeros"] is not None else 8)
        y += (x[:, lo:hi] @ digit.double().T) * s["scales"][:, g].double()
    return y


def _work_w4(c):
    groups = -(-c["k"] // c["group"])
    return {"bytes": c["n"] * (-(-c["k"] // 2) + groups * (3 if c["zeros"] else 2)) + 2 * c["m"] * (c["k"] + c["n"]),
            "flops": 2 * c["m"] * c["k"] * c["n"]}
