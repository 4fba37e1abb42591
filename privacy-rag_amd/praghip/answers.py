"""Answers in the clear beside the protocol: a Qwen3-shaped model over a paged cache.

The reference computes its forward on shares; this serves the same shapes (model.hpp:63-64)
to a party that may see the text, and shows the serving calls together: 4-bit projections
(:func:`matvec_w4`), norms (:func:`add_norm`), a prompt into the cache (:func:`page_reserve`,
:func:`page_append`, :func:`paged_prompt`), several answers of one prompt (:func:`page_fork`),
their tokens (:func:`paged_shared` where they share enough, else :func:`paged_decode`), which
:func:`sample_tokens` draws, and their pages' way back (:func:`page_trim`, :func:`page_free`,
:func:`page_compact`).  Activations are torch's.

``python -m praghip.answers`` answers a synthetic prompt and prints its times.
"""
from __future__ import annotations

from .append import page_append, rotary_table
from .attention import paged_decode, paged_prompt, paged_shared
from .matvec import matvec_w4, quantize_w4
from .norm import add_norm
from .pages import page_check, page_compact, page_fork, page_free, page_reserve, page_trim
from .qwen3 import QWEN3_0_6B, Qwen3Shape
from .sample import sample_tokens

# Keys that a step reads once instead of once for each answer, from which on the attention of
# shared prefixes is the faster one, at 16 heads of 128 over 8: eight answers over 256 tokens
# (1,792 keys) take 14 us of 12, over 1,024 (7,168 keys) 14 of 15.5, over 8,192 18 of 51.  (Other
# shapes and numbers of answers have the same bound, unmeasured.)
_ENOUGH = 4096


def _runs(common):
    """Where to cut a list of answers into runs that read a prefix together, its end among them:
    common[i] tokens are the same for the i-th and the next, and for a run the fewest of its
    pairs', which all of its members but one need not read.  The cuts that save the most."""
    n = len(common) + 1
    saved, first = [0] * (n + 1), [0] * (n + 1)  # by the runs of what is before i; where the last of them begins
    for end in range(1, n + 1):
        most, begin, fewest = saved[end - 1], end - 1, 0
        for at in range(end - 2, -1, -1):
            fewest = min(fewest, common[at]) if fewest else common[at]
            if not fewest:
                break
            if saved[at] + (end - 1 - at) * fewest > most:
                most, begin = saved[at] + (end - 1 - at) * fewest, at
        saved[end], first[end] = most, begin
    cuts = [n]
    while cuts[-1]:
        cuts.append(first[cuts[-1]])
    return cuts[::-1]


class Qwen3Answers:
    """Weights, a cache of `pages` pages for every layer, and up to `slots` sequences of
    `capacity` tokens, rounded up to whole pages.

    weights: {"embed": [vocab][hidden], "norm": [hidden], "layers": [{"qkv", "o",
    "gate_up", "down": [out][in], "attention_norm", "mlp_norm": [hidden], "q_norm",
    "k_norm": [head_dim]}]} of one 16-bit type on one GPU; the projections are kept in
    4 bits, the output head is the embedding.  Norm weights of 32 bits that the type does not
    hold are kept, and their norms are torch's, which are slower.  With a window every layer sees the last
    `window` tokens and the first `sinks`, and pages that leave it are given back.  rotary:
    further arguments of :func:`rotary_table`, for contexts beyond those of the training.
    """

    def __init__(self, weights: dict, shape: Qwen3Shape = QWEN3_0_6B, *, slots: int = 16, pages: int = 1024,
                 page_size: int = 16, capacity: int = 8192, group: int = 128, window: int = 0, sinks: int = 0,
                 theta: float = 1e6, eps: float = 1e-6, rotary: dict | None = None):
        import torch
        self.shape, self.page_size, self.window, self.sinks, self.eps = shape, page_size, window, sinks, eps
        self.group, self.embed = group, weights["embed"].detach()
        self.device, self.type = self.embed.device, self.embed.dtype
        self.norm = self._norm(weights["norm"])
        self.head = quantize_w4(self.embed, group, zeros=True)
        self.layers = [{name: quantize_w4(w, group, zeros=True) if w.dim() == 2 else self._norm(w) for name, w in layer.items()}
                       for layer in weights["layers"]]
        self.pool = torch.zeros((shape.layers, 2, pages, shape.kv_heads, page_size, shape.head_dim), dtype=self.type,
                                device=self.device)
        ints = dict(dtype=torch.int32, device=self.device)
        self.tables = torch.full((slots, -(-capacity // page_size)), -1, **ints)
        self.lengths, self.refs = torch.zeros(slots, **ints), torch.zeros(pages, **ints)
        self.status = torch.zeros(1, **ints)
        self.held = [0] * slots  # the lengths, as the host knows them
        # what forks have left in common: a state's number and its tokens, of which a sequence's
        # first are the same as those of every other sequence with that number
        self.marks, self.states, self.changes = [[] for _ in range(slots)], 0, 0
        self.cos, self.sin = rotary_table(self.tables.shape[1] * page_size, shape.head_dim, theta=theta, device=self.device,
                                          **(rotary or {}))

    def _norm(self, weight):
        """A norm's weights as the calls take them: of the model's type, together, aligned; in
        32 bits (for :meth:`_normed`) where the type does not hold them."""
        import torch
        wide = weight.detach().float()
        w = wide.to(self.type).contiguous()
        if not torch.equal(w.float(), wide):
            return wide
        return w if w.data_ptr() % 16 == 0 else w.clone()

    def _held(self, weight):
        return weight.dtype is self.type

    def _normed(self, x, weight):
        x = x.float()
        return (x * (x.square().mean(-1, keepdim=True) + self.eps).rsqrt() * weight).to(self.type)

    def _added(self, x, weight, residual):
        """(the norm of the sum, the sum, in residual's place where that is one call)."""
        if self._held(weight):
            return add_norm(x, weight, residual, eps=self.eps, total=residual)
        total = x.float() + residual.float()
        return self._normed(total, weight), total.to(self.type)

    def _ints(self, values):
        import torch
        return torch.tensor(list(values), dtype=torch.int32).to(self.device)

    def _product(self, x, w):
        return matvec_w4(x, *w, group=self.group)

    _grouped = None  # the last list's groups, until a fork or an end

    def _groups(self, sequences):
        """(first of each run of neighbours that share a prefix, and the end; the tokens that
        each shares; keys that are read once instead of for each)."""
        key = self.changes, tuple(sequences)
        if self._grouped is None or self._grouped[0] != key:
            # (a sequence's marks are its parent's, in order, and its own: what a run has in common
            # is the least that two neighbours of it have)
            marks = [self.marks[s] for s in sequences]
            common = [max((n for state, n in a if (state, n) in b), default=0) for a, b in zip(marks, marks[1:])]
            groups = _runs(common)
            shared = [min(common[a: b - 1]) if b > a + 1 else max((n for _, n in marks[a]), default=0)
                      for a, b in zip(groups, groups[1:])]
            saved = sum((b - a - 1) * n for a, b, n in zip(groups, groups[1:], shared))
            self._grouped = key, (groups, shared, saved)
        return self._grouped[1]

    def _forward(self, sequences, rows):
        """Logits after the newest tokens, rows[i] of sequences[i], which have their pages already."""
        at = self._ints(sequences).long()
        ends = [sum(len(r) for r in rows[: i + 1]) for i in range(len(rows))]
        most, together = max(len(r) for r in rows), None
        if most == 1 and not self.window:
            groups, shared, saved = self._groups(sequences)
            if saved >= _ENOUGH:
                together = self._ints(groups), self._ints(shared)
        x = self._layers(self._ints(t for r in rows for t in r).long(), self.tables[at], self.lengths[at],
                         self._ints([0] + ends), most, max(self.held[s] for s in sequences), together)
        return self._logits(x[self._ints(e - 1 for e in ends).long()])

    def _layers(self, tokens, tables, lengths, starts, most: int, longest: int, together=None):
        """The last layer's output, under the last norm, of the tokens that are rows starts[s] ..
        of the sequences whose tables these are.  together: the groups and their shared tokens,
        where single tokens' attention reads prefixes once."""
        import torch
        shape = self.shape
        see = dict(window=self.window, sinks=self.sinks, max_length=longest)
        heads = shape.q_heads, shape.kv_heads, shape.kv_heads
        x = self.embed[tokens]
        norms = [layer["attention_norm"] for layer in self.layers] + [self.norm]
        h = add_norm(x, norms[0], eps=self.eps) if self._held(norms[0]) else self._normed(x, norms[0])
        for layer, norm, (keys, values) in zip(self.layers, norms[1:], self.pool):
            q, k, v = self._product(h, layer["qkv"]).unflatten(1, (-1, shape.head_dim)).split(heads, 1)
            q_norm, k_norm = layer["q_norm"], layer["k_norm"]
            if not self._held(q_norm):
                q, q_norm = self._normed(q, q_norm), None
            if not self._held(k_norm):
                k, k_norm = self._normed(k, k_norm), None
            q = page_append(q, k, v, keys, values, tables, lengths, starts, self.cos, self.sin, q_norm=q_norm, k_norm=k_norm,
                            eps=self.eps)
            if most > 1:
                o = paged_prompt(q, keys, values, tables, lengths, starts, most, **see)
            elif together:
                o = paged_shared(q, keys, values, tables, lengths, *together, max_length=longest)
            else:
                o = paged_decode(q, keys, values, tables, lengths, **see)
            h, x = self._added(self._product(o.flatten(1), layer["o"]), layer["mlp_norm"], x)
            gate, up = self._product(h, layer["gate_up"]).chunk(2, 1)
            h, x = self._added(self._product((torch.nn.functional.silu(gate.float()) * up.float()).to(self.type), layer["down"]), norm, x)
        return h

    def _logits(self, x):
        return self._product(x, self.head)

    def extend(self, sequences, rows):
        """Appends rows[i], a list of one token or more, to sequences[i]; returns the logits
        after each, [len(sequences)][vocab].  Raises, with nothing changed, where the pages
        or the capacity do not suffice.  (What fails later, for memory say, leaves the tokens
        without their keys: such sequences are to be ended.)"""
        sequences, rows = list(sequences), [list(r) for r in rows]
        if len(sequences) != len(rows) or not rows or not all(rows):
            raise ValueError("each sequence takes one token or more")
        if any(not 0 <= t < self.embed.shape[0] for r in rows for t in r):
            raise ValueError("a token outside the vocabulary")
        listed = self._ints(sequences)
        self._reserve(sequences, listed, self._ints(map(len, rows)), [len(r) for r in rows])
        logits = self._forward(sequences, rows)
        self._trim(listed)
        return logits

    def _reserve(self, sequences, listed, counts, more):
        page_reserve(self.tables, self.lengths, self.refs, self.page_size, listed, counts, self.status)
        page_check(self.status)
        for s, n in zip(sequences, more):
            self.held[s] += n

    def _trim(self, listed):
        if self.window:
            page_trim(self.tables, self.lengths, self.refs, self.page_size, listed, self.window, self.sinks, self.status)

    def steps(self, sequences):
        """A function that appends one token to each of these sequences, given as a list or a
        tensor of whole numbers (whose values outside the vocabulary count as its nearest), and
        returns the logits after them (in the same memory each time): the layers' calls, some
        14 a layer, as one captured graph.  The sequences may be forked, ended and extended
        between its calls.  Where they share enough when this is called, and there is no window,
        the graph reads what neighbours in the list share once, as it is at each step."""
        import torch
        sequences = list(sequences)
        if not sequences or any(not 0 <= s < len(self.held) for s in sequences):
            raise ValueError("no such sequence")
        n, capacity = len(sequences), self.tables.shape[1] * self.page_size
        listed, ones = self._ints(sequences), self._ints([1] * n)
        at, starts = listed.long(), self._ints(range(n + 1))
        tokens = torch.zeros(n, dtype=torch.int64, device=self.device)

        together, changes = None, self.changes
        if not self.window and self._groups(sequences)[2] >= _ENOUGH:
            together = self._ints([0] * (n + 1)), self._ints([0] * n)

        def share():
            groups, shared, _ = self._groups(sequences)
            together[0].copy_(self._ints(groups + [n] * (n + 1 - len(groups))))
            together[1].copy_(self._ints(shared + [0] * (n - len(shared))))

        if together:
            share()

        def forward():
            return self._logits(self._layers(tokens.clamp(0, self.embed.shape[0] - 1), self.tables[at], self.lengths[at], starts, 1,
                                             capacity, together))

        held = self.lengths.clone()
        try:
            self.lengths.zero_()  # (a first time outside, which loads code and writes nothing)
            forward()
        finally:
            self.lengths.copy_(held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = forward()

        whole = torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64

        def step(new):
            if not isinstance(new, torch.Tensor):
                if len(new) != n or any(not 0 <= t < self.embed.shape[0] for t in new):
                    raise ValueError("one token of the vocabulary for each sequence")
                new = torch.tensor(new)
            if new.shape != (n,) or new.dtype not in whole:
                raise ValueError("one whole number for each sequence")
            nonlocal changes
            self._reserve(sequences, listed, ones, [1] * n)
            tokens.copy_(new)
            if together and changes != self.changes:
                share()
                changes = self.changes
            graph.replay()
            self._trim(listed)
            return logits

        step.reads = at, starts, together  # (the graph's addresses: they live as long as it does)
        return step

    def fork(self, parent: int, children) -> None:
        """The empty sequences `children` go on from the parent's tokens, whose full pages they share."""
        children = list(children)
        page_fork(self.pool, self.tables, self.lengths, self.refs, self._ints([parent] * len(children)),
                  self._ints(children), self.status)
        page_check(self.status)
        self._forked(parent, children)

    def _forked(self, parent: int, children) -> None:
        marks = self.marks[parent]
        if not any(n == self.held[parent] for _, n in marks):
            marks.append((self.states, self.held[parent]))
            self.states += 1
        self.changes += 1
        for child in children:
            self.held[child], self.marks[child] = self.held[parent], list(marks)

    def end(self, sequences) -> None:
        """Empties sequences."""
        sequences = list(sequences)
        page_free(self.tables, self.lengths, self.refs, self._ints(sequences), self.status)
        page_check(self.status)
        self._ended(sequences)

    def _ended(self, sequences) -> None:
        self.changes += 1
        for s in sequences:
            self.held[s], self.marks[s] = 0, []

    def compact(self) -> None:
        """Moves the held pages to the pool's front."""
        page_compact(self.pool, self.tables, self.refs)


def random_weights(shape: Qwen3Shape = QWEN3_0_6B, vocab: int = 32768, *, seed: int = 0, type=None, device="cuda") -> dict:
    """Seeded weights of a shape, as :class:`Qwen3Answers` takes them."""
    import torch
    g = torch.Generator(device=device).manual_seed(seed)
    type = type or torch.bfloat16

    def normal(n, k):
        return torch.randn((n, k), generator=g, device=device).mul_(k ** -0.5).to(type)

    def ones(n):
        return torch.ones(n, dtype=type, device=device)

    layers = [{**{name: normal(n, k) for name, k, n in shape.products()}, "attention_norm": ones(shape.hidden),
               "mlp_norm": ones(shape.hidden), "q_norm": ones(shape.head_dim), "k_norm": ones(shape.head_dim)}
              for _ in range(shape.layers)]
    return {"embed": normal(vocab, shape.hidden), "norm": ones(shape.hidden), "layers": layers}


def main() -> None:
    import argparse
    import time

    import torch
    parser = argparse.ArgumentParser(description="Several answers of one synthetic prompt, in the clear.")
    parser.add_argument("--prompt", type=int, default=512, help="tokens of the prompt")
    parser.add_argument("--answers", type=int, default=8)
    parser.add_argument("--tokens", type=int, default=32, help="tokens of each answer")
    parser.add_argument("--window", type=int, default=0)
    parser.add_argument("--temperature", type=float, default=0.0, help="0: the likeliest token")
    parser.add_argument("--top-k", type=int, default=0)
    parser.add_argument("--top-p", type=float, default=1.0)
    parser.add_argument("--min-p", type=float, default=0.0)
    args = parser.parse_args()
    per = -(-(args.prompt + args.tokens) // 16)
    model = Qwen3Answers(random_weights(), slots=1 + args.answers, pages=per * (1 + args.answers), window=args.window,
                         sinks=4 if args.window else 0, capacity=16 * per)
    prompt = torch.randint(0, 32768, (args.prompt,), generator=torch.Generator().manual_seed(1)).tolist()
    times = {}

    def timed(name, call):
        torch.cuda.synchronize()
        start = time.perf_counter()
        got = call()
        torch.cuda.synchronize()
        times.setdefault(name, []).append(time.perf_counter() - start)
        return got

    for _ in range(2):  # the first time round loads code, and its capture gives torch's memory back
        model.extend([0], [prompt])
        model.end([0])
        times.clear()
        logits = timed("prompt", lambda: model.extend([0], [prompt]))
        answers = range(1, 1 + args.answers)
        timed("fork", lambda: model.fork(0, answers))
        draw = dict(temperature=args.temperature, top_k=args.top_k, top_p=args.top_p, min_p=args.min_p)
        numbers = torch.rand((args.tokens, args.answers), generator=torch.Generator().manual_seed(2)).to("cuda")
        if args.temperature:
            tokens = sample_tokens(logits[:1].expand(args.answers, -1), numbers[-1], **draw)
        else:
            tokens = logits[0].topk(args.answers).indices
        said = [tokens]
        step = timed("capture", lambda: model.steps(answers))
        for u in numbers[:-1]:
            tokens = timed("token", lambda: sample_tokens(step(tokens), u, **draw))
            said.append(tokens)
        timed("end", lambda: model.end(range(0, 1 + args.answers)))
    for name, t in times.items():
        print(f"{name:8s} {1e3 * sorted(t)[len(t) // 2]:8.3f} ms")
    print("answers begin", torch.stack(said, 1)[:, :4].tolist())


if __name__ == "__main__":
    main()
