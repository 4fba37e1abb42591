"""Answers in the clear beside the protocol: a Qwen3-shaped model over a paged cache.

The reference computes its forward on shares; this serves the same shapes (model.hpp:63-64)
to a party that may see the text, and shows the serving calls together: 4-bit projections
(:func:`matvec_w4`), a prompt into the cache (:func:`page_reserve`, :func:`page_write`,
:func:`paged_prompt`), several answers of one prompt (:func:`page_fork`), their tokens
(:func:`paged_decode`), and their pages' way back (:func:`page_trim`, :func:`page_free`,
:func:`page_compact`).  Norms, rotations and activations are torch's.

``python -m praghip.answers`` answers a synthetic prompt and prints its times.
"""
from __future__ import annotations

from .attention import page_write, paged_decode, paged_prompt
from .matvec import matvec_w4, quantize_w4
from .pages import page_check, page_compact, page_fork, page_free, page_reserve, page_trim
from .qwen3 import QWEN3_0_6B, Qwen3Shape


class Qwen3Answers:
    """Weights, a cache of `pages` pages for every layer, and up to `slots` sequences of
    `capacity` tokens, rounded up to whole pages.

    weights: {"embed": [vocab][hidden], "norm": [hidden], "layers": [{"qkv", "o",
    "gate_up", "down": [out][in], "attention_norm", "mlp_norm": [hidden], "q_norm",
    "k_norm": [head_dim]}]} of one 16-bit type on one GPU; the projections are kept in
    4 bits, the output head is the embedding.  With a window every layer sees the last
    `window` tokens and the first `sinks`, and pages that leave it are given back.
    """

    def __init__(self, weights: dict, shape: Qwen3Shape = QWEN3_0_6B, *, slots: int = 16, pages: int = 1024,
                 page_size: int = 16, capacity: int = 8192, group: int = 128, window: int = 0, sinks: int = 0,
                 theta: float = 1e6, eps: float = 1e-6):
        import torch
        self.shape, self.page_size, self.window, self.sinks, self.eps = shape, page_size, window, sinks, eps
        self.group, self.embed, self.norm = group, weights["embed"].detach(), weights["norm"].detach()
        self.device, self.type = self.embed.device, self.embed.dtype
        self.head = quantize_w4(self.embed, group, zeros=True)
        self.layers = [{name: quantize_w4(w, group, zeros=True) if w.dim() == 2 else w.detach() for name, w in layer.items()}
                       for layer in weights["layers"]]
        self.pool = torch.zeros((shape.layers, 2, pages, shape.kv_heads, page_size, shape.head_dim), dtype=self.type,
                                device=self.device)
        ints = dict(dtype=torch.int32, device=self.device)
        self.tables = torch.full((slots, -(-capacity // page_size)), -1, **ints)
        self.lengths, self.refs = torch.zeros(slots, **ints), torch.zeros(pages, **ints)
        self.status = torch.zeros(1, **ints)
        self.held = [0] * slots  # the lengths, as the host knows them
        half = torch.arange(0, shape.head_dim, 2, dtype=torch.float64, device=self.device)
        angle = torch.arange(self.tables.shape[1] * page_size, dtype=torch.float64, device=self.device)[:, None] * \
            theta ** (-half / shape.head_dim)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def _ints(self, values):
        import torch
        return torch.tensor(list(values), dtype=torch.int32).to(self.device)

    def _normed(self, x, weight):
        x = x.float()
        return (x * (x.square().mean(-1, keepdim=True) + self.eps).rsqrt() * weight.float()).to(self.type)

    def _turned(self, x, places):
        import torch
        a, b = x.float().chunk(2, -1)
        cos, sin = self.cos[places][:, None], self.sin[places][:, None]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(self.type)

    def _product(self, x, w):
        return matvec_w4(x, *w, group=self.group)

    def _forward(self, sequences, rows):
        """Logits after the newest tokens, rows[i] of sequences[i], which have their pages already."""
        at = self._ints(sequences).long()
        ends = [sum(len(r) for r in rows[: i + 1]) for i in range(len(rows))]
        places = self._ints(self.held[s] - len(r) + i for s, r in zip(sequences, rows) for i in range(len(r))).long()
        x = self._layers(self._ints(t for r in rows for t in r).long(), places, self.tables[at], self.lengths[at],
                         self._ints([0] + ends), max(len(r) for r in rows), max(self.held[s] for s in sequences))
        return self._logits(x[self._ints(e - 1 for e in ends).long()])

    def _layers(self, tokens, places, tables, lengths, starts, most: int, longest: int):
        """The last layer's output of tokens at `places`, rows starts[s] .. of the sequences whose tables these are."""
        import torch
        shape = self.shape
        see = dict(window=self.window, sinks=self.sinks, max_length=longest)
        q_out, kv_out = shape.q_heads * shape.head_dim, shape.kv_heads * shape.head_dim
        x = self.embed[tokens]
        for layer, (keys, values) in zip(self.layers, self.pool):
            qkv = self._product(self._normed(x, layer["attention_norm"]), layer["qkv"])
            q, k, v = (t.unflatten(1, (-1, shape.head_dim)) for t in qkv.split((q_out, kv_out, kv_out), 1))
            q = self._turned(self._normed(q, layer["q_norm"]), places)
            k = self._turned(self._normed(k, layer["k_norm"]), places)
            page_write(k, v, keys, values, tables, lengths, starts)
            if most == 1:
                o = paged_decode(q, keys, values, tables, lengths, **see)
            else:
                o = paged_prompt(q, keys, values, tables, lengths, starts, most, **see)
            x = x + self._product(o.flatten(1), layer["o"])
            gate, up = self._product(self._normed(x, layer["mlp_norm"]), layer["gate_up"]).chunk(2, 1)
            x = x + self._product((torch.nn.functional.silu(gate.float()) * up.float()).to(self.type), layer["down"])
        return x

    def _logits(self, x):
        return self._product(self._normed(x, self.norm), self.head)

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
        30 a layer, as one captured graph.  The sequences may be forked, ended and extended
        between its calls."""
        import torch
        sequences = list(sequences)
        if not sequences or any(not 0 <= s < len(self.held) for s in sequences):
            raise ValueError("no such sequence")
        n, capacity = len(sequences), self.tables.shape[1] * self.page_size
        listed, ones = self._ints(sequences), self._ints([1] * n)
        at, starts = listed.long(), self._ints(range(n + 1))
        tokens = torch.zeros(n, dtype=torch.int64, device=self.device)

        def forward():
            lengths = self.lengths[at]
            places = (lengths - 1).clamp(min=0).long()
            return self._logits(self._layers(tokens.clamp(0, self.embed.shape[0] - 1), places, self.tables[at], lengths,
                                             starts, 1, capacity))

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
            self._reserve(sequences, listed, ones, [1] * n)
            tokens.copy_(new)
            graph.replay()
            self._trim(listed)
            return logits

        step.reads = at, starts  # (the graph's addresses: they live as long as it does)
        return step

    def fork(self, parent: int, children) -> None:
        """The empty sequences `children` go on from the parent's tokens, whose full pages they share."""
        children = list(children)
        page_fork(self.pool, self.tables, self.lengths, self.refs, self._ints([parent] * len(children)),
                  self._ints(children), self.status)
        page_check(self.status)
        for child in children:
            self.held[child] = self.held[parent]

    def end(self, sequences) -> None:
        """Empties sequences."""
        sequences = list(sequences)
        page_free(self.tables, self.lengths, self.refs, self._ints(sequences), self.status)
        page_check(self.status)
        for s in sequences:
            self.held[s] = 0

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
        tokens = logits[0].topk(args.answers).indices.tolist()
        said = [[t] for t in tokens]
        step = timed("capture", lambda: model.steps(answers))
        for _ in range(args.tokens - 1):
            tokens = timed("token", lambda: step(tokens).argmax(-1).tolist())
            for s, t in zip(said, tokens):
                s.append(t)
        timed("end", lambda: model.end(range(0, 1 + args.answers)))
    for name, t in times.items():
        print(f"{name:8s} {1e3 * sorted(t)[len(t) // 2]:8.3f} ms")
    print("answers begin", [s[:4] for s in said])


if __name__ == "__main__":
    main()
