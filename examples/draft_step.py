"""Drafted tokens and long contexts, as a server runs them over two attention layers of GGUF weights:

    tables, slots, positions and masks of the step from its lengths -> residual + norm -> qkv + each row's adapter -> norm,
    rotation, store into the pages -> attention of all new tokens over the pages -> o_proj + adapter

Chunks of several prompts share a step; then each step checks a tree of drafted tokens for each sequence, of which one path
is taken (its keys move together, the others' places are written again); then sequences go on token by token, each token
attending to some of its sequence's pages.  The last two replay HIP graphs, the batch padded with a row that has no sequence.
Every output is checked against the same network in fp32 without a cache.  Run: python examples/draft_step.py"""
from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from decode_step import DIM, G, HEADS, K, KV_HEADS, PAGE, PARTS, Layer  # noqa: E402

EPS = 1e-6


class Model:
    def __init__(self, layers: int = 2, pages: int = 64, length: int = 256):
        gen = torch.Generator(device="cuda").manual_seed(3)
        self.layers = [Layer(gen) for _ in range(layers)]
        self.norms = [(1 + 0.1 * torch.randn(K, device="cuda", generator=gen)).bfloat16() for _ in range(layers + 1)]
        self.storage = torch.zeros((layers, 2, pages, KV_HEADS, PAGE, DIM), dtype=torch.bfloat16, device="cuda")
        self.bounds = torch.zeros((layers, pages, 2, KV_HEADS, DIM), dtype=torch.bfloat16, device="cuda")
        self.pool = G.PagePool(pages)
        self.rope = G.rope_table(DIM, length, base=1e6)
        self.length = length

    def pages(self, i: int):
        return self.storage[i, 0].transpose(1, 2), self.storage[i, 1].transpose(1, 2)

    def forward(self, x, adapters, t: G.StepTables, most: int, keep: int = 0):
        """x bf16 [rows, K], a row a new token; adapters [batch]; ``most`` new tokens of a sequence.  keep > 0: one new token each,
        which attends to that many pages; returns them too, [layers] of [batch, key heads, keep]."""
        rows, chosen = x.shape[0], []
        ids = torch.where(t.sequences < 0, -1, adapters[t.sequences.clamp_min(0).long()])
        h, stream = G.add_rms_norm(x, None, self.norms[0], eps=EPS)[0], x
        for i, w in enumerate(self.layers):
            k_pages, v_pages = self.pages(i)
            y = G.mul_mat_grouped(h, w.qkv)
            G.lora_add(y, h, w.lora[0], w.lora[1], ids, w.lora[2], PARTS, out=y)
            q, k, v = (p.view(rows, -1, DIM) for p in y.split(PARTS, 1))
            q, _ = G.qk_norm_rope(q, k, t.positions, self.rope, w.q_norm, w.k_norm, v=v, k_pages=k_pages, v_pages=v_pages, slots=t.slots)
            if keep:   # (row b is sequence b's: each brings a token, those without one are the last)
                batch = t.lengths.shape[0]
                G.page_bounds(k_pages, t.block_table, t.lengths, self.bounds[i])
                table, lengths = G.select_pages(q[:batch], self.bounds[i], t.block_table, t.lengths, keep, PAGE, max_length=self.length)
                o = G.paged_attention(q[:batch], k_pages, v_pages, table, lengths)
                chosen.append(table)
            else:
                o = G.tree_attention(q, k_pages, v_pages, t.block_table, t.lengths, t.starts, t.mask, max_length=self.length, max_tokens=most)
            o = o.view(rows, -1)
            z = G.mul_mat_grouped(o, w.o)
            G.lora_add(z, o, w.lora_o[0], w.lora_o[1], ids, w.lora_o[2], [K], out=z)
            h, stream = G.add_rms_norm(z, stream, self.norms[i + 1], eps=EPS)
        return h, chosen

    def plain(self, x, ids, seen):
        """The same network over one whole sequence in fp32: x [tokens, K], ids [tokens], seen bool [layers, key heads, tokens, tokens]."""
        x, n = x.float(), x.shape[0]
        cos, sin = self.rope[:n, None].chunk(2, 2)

        def update(h, lora, parts):
            a, b, scales = (t.float() for t in lora)
            at = ids.long().clamp_min(0)
            low = torch.matmul(a[at], h[:, None, :, None])[..., 0]
            out = torch.cat([torch.matmul(bp, low[:, p, :, None])[..., 0] for p, bp in enumerate(b[at].split(parts, 1))], 1)
            return out * (scales[at] * (ids >= 0))[:, None]

        def normed(x, weight):
            return torch.nn.functional.rms_norm(x, (x.shape[-1],), weight.float(), EPS)

        def heads(t, weight):
            s, c = normed(t.view(n, -1, DIM), weight).chunk(2, 2)
            return torch.cat([s * cos - c * sin, c * cos + s * sin], 2).transpose(0, 1)

        for w, norm, see in zip(self.layers, self.norms, seen):
            h = normed(x, norm)
            q, k, v = (h @ w.w_qkv.T + update(h, w.lora, PARTS)).split(PARTS, 1)
            q, k, v = heads(q, w.q_norm), heads(k, w.k_norm), v.reshape(n, -1, DIM).transpose(0, 1)
            k, v, see = (t.repeat_interleave(HEADS // KV_HEADS, 0) for t in (k, v, see))
            p = (torch.matmul(q, k.transpose(1, 2)) * DIM ** -0.5).masked_fill(~see, float("-inf")).softmax(2)
            o = torch.matmul(p, v).transpose(0, 1).reshape(n, -1)
            x = x + o @ w.w_o.T + update(o, w.lora_o, [K])
        return normed(x, self.norms[-1])


class Sequence:
    """A request: its row of the page lists, its pages, and what the check needs of its tokens."""

    def __init__(self, request: int, adapter: int):
        self.request, self.adapter, self.table = request, adapter, []
        self.inputs, self.chosen = [], []     # chosen: None, or a token's pages [layers, key heads, keep]
        self.checks = []                      # (tokens, output of the last one) of paths that were not taken, and of those that were

    def __len__(self):
        return len(self.inputs)


class Server:
    def __init__(self, model: Model, batch: int, requests: int, tree: int, keep: int):
        self.model, self.batch, self.tree = model, batch, tree
        ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.lists = ints(requests, model.length // PAGE)   # the pages of each request
        self.requests, self.lengths, self.counts, self.adapters = ints(batch), ints(batch), ints(batch), ints(batch)
        self.graphs = {}
        for name, rows, most, kept in (("tree", batch * tree, tree, 0), ("token", batch, 1, keep)):
            x, parents = torch.zeros((rows, K), dtype=torch.bfloat16, device="cuda"), ints(rows) if most > 1 else None
            self._write([], [])
            step = lambda: self._forward(x, parents, most, kept)  # noqa: E731, B023
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                step()   # a call before the capture
            torch.cuda.current_stream().wait_stream(stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            self.graphs[name] = (graph, x, parents, out)

    def _forward(self, x, parents, most: int, keep: int = 0):
        t = G.step_tables(self.lists, self.requests, self.lengths, self.counts, x.shape[0], PAGE, parents=parents, tree=most if parents is not None else 0)
        return self.model.forward(x, self.adapters, t, most, keep)

    def _write(self, sequences: list[Sequence], counts: list[int]) -> None:
        """The batch's rows; behind the sequences those that have none."""
        pad = self.batch - len(sequences)
        for t, values, fill in ((self.requests, [s.request for s in sequences], -1), (self.lengths, [len(s) for s in sequences], 0),
                                (self.counts, counts, 0), (self.adapters, [s.adapter for s in sequences], -1)):
            t.copy_(torch.tensor(values + [fill] * pad, dtype=torch.int32))
        for s, n in zip(sequences, counts):
            more = (len(s) + n - 1) // PAGE + 1 - len(s.table)
            if more > 0:
                s.table += self.model.pool.allocate(more)
                self.lists[s.request, :len(s.table)] = torch.tensor(s.table, dtype=torch.int32, device="cuda")

    def chunks(self, sequences: list[Sequence], parts: list[torch.Tensor]) -> None:
        """The next chunk of each one's prompt, in one step."""
        counts = [p.shape[0] for p in parts]
        self._write(sequences, counts)
        out = self._forward(torch.cat(parts), None, max(counts))[0]
        for s, part, y in zip(sequences, parts, out.split(counts)):
            for i in range(part.shape[0]):
                s.inputs.append(part[i])
                s.chosen.append(None)
                s.checks.append((list(s.inputs), list(s.chosen), y[i]))

    def trees(self, sequences: list[Sequence], drafts: list[tuple[torch.Tensor, list[int]]], taken: list[int]) -> None:
        """A tree of drafted tokens for each (its tokens and their parents); the path down to token taken[b] becomes b's next tokens."""
        graph, x, parents, (out, _) = self.graphs["tree"]
        counts = [len(p) for _, p in drafts]
        self._write(sequences, counts)
        x[:sum(counts)] = torch.cat([d for d, _ in drafts])
        parents[:sum(counts)] = torch.tensor([p for _, ps in drafts for p in ps], dtype=torch.int32, device="cuda")
        graph.replay()
        src, dst = [], []
        for s, (draft, ps), last, y in zip(sequences, drafts, taken, out[:sum(counts)].clone().split(counts)):
            paths = []
            for i, p in enumerate(ps):
                paths.append((paths[p] if p >= 0 else []) + [i])
                s.checks.append((s.inputs + [draft[j] for j in paths[i]], s.chosen + [None] * len(paths[i]), y[i]))
            n = len(s)
            src += [(s.table[(n + j) // PAGE], (n + j) % PAGE) for j in paths[last]]
            dst += [(s.table[(n + j) // PAGE], (n + j) % PAGE) for j in range(len(paths[last]))]
            s.inputs += [draft[j] for j in paths[last]]
            s.chosen += [None] * len(paths[last])
        (sp, st), (dp, dt) = (torch.tensor(t, device="cuda").unbind(1) for t in (src, dst))
        self.model.storage[:, :, dp, :, dt] = self.model.storage[:, :, sp, :, st]

    def bounds(self, sequences: list[Sequence]) -> None:
        """The bounds of all pages, before the sequences go on token by token."""
        tables = [s.table + [-1] * (self.lists.shape[1] - len(s.table)) for s in sequences]
        table = torch.tensor(tables, dtype=torch.int32, device="cuda")
        lengths = torch.tensor([len(s) for s in sequences], dtype=torch.int32, device="cuda")
        for i in range(len(self.model.layers)):
            G.page_bounds(self.model.pages(i)[0], table, lengths, self.model.bounds[i], count=self.model.length)

    def tokens(self, sequences: list[Sequence], new: torch.Tensor) -> None:
        graph, x, _, (out, chosen) = self.graphs["token"]
        self._write(sequences, [1] * len(sequences))
        x[:len(sequences)] = new
        graph.replay()
        for b, s in enumerate(sequences):
            s.inputs.append(new[b])
            s.chosen.append(torch.stack([c[b] for c in chosen]))
            s.checks.append((list(s.inputs), list(s.chosen), out[b].clone()))

    def error(self, s: Sequence) -> float:
        """The largest error of an output against the plain network's, relative to it."""
        worst = 0.0
        ids = torch.full((self.model.length,), s.adapter, device="cuda")
        page_of = torch.tensor(s.table, device="cuda")
        for inputs, chosen, got in s.checks:
            n = len(inputs)
            seen = torch.ones((len(self.model.layers), KV_HEADS, n, n), dtype=torch.bool, device="cuda").tril()
            for i, c in enumerate(chosen):
                if c is not None:
                    pages = page_of[torch.arange(n, device="cuda") // PAGE]
                    seen[:, :, i] &= (c[..., None] == pages).any(2)
            want = self.model.plain(torch.stack(inputs), ids[:n], seen)[-1]
            worst = max(worst, float((got.float() - want).norm() / want.norm()))
        return worst


def run(steps: int = 6) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(4)
    host = torch.Generator().manual_seed(5)
    tokens = lambda n: torch.randn((n, K), device="cuda", generator=gen).bfloat16()  # noqa: E731
    below = lambda n: int(torch.randint(0, n, (1,), generator=host))  # noqa: E731
    tree, keep = 8, 4
    server = Server(Model(), batch=4, requests=6, tree=tree, keep=keep)
    a, b, c = Sequence(4, 0), Sequence(0, -1), Sequence(5, 1)
    server.chunks([a, b, c], [tokens(50), tokens(3), tokens(41)])
    server.chunks([c, a], [tokens(30), tokens(17)])
    for _ in range(steps):
        drafts = []
        for _ in range(3):
            n = 1 + below(tree)
            drafts.append((tokens(n), [below(i + 1) - 1 for i in range(n)]))
        server.trees([b, a, c], drafts, [below(len(p)) for _, p in drafts])
    server.bounds([a, b, c])
    for _ in range(steps):
        server.tokens([a, c, b], tokens(3))
    errors = {name: server.error(s) for name, s in (("a", a), ("b", b), ("c", c))}
    times = {}
    for name, (graph, *_) in server.graphs.items():
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(100):
            graph.replay()
        torch.cuda.synchronize()
        times[name] = (time.perf_counter() - start) * 1e4
    return {"errors": errors, "outputs": sum(len(s.checks) for s in (a, b, c)), "us": times, "pages": max(len(s.table) for s in (a, b, c)), "keep": keep}


if __name__ == "__main__":
    got = run()
    print(f"largest error of {got['outputs']} outputs against fp32:", {n: f"{e:.4f}" for n, e in got["errors"].items()})
    print(f"a step of two layers (graph): trees of up to 8 tokens {got['us']['tree']:.0f} us, single tokens on {got['keep']} of up to "
          f"{got['pages']} pages {got['us']['token']:.0f} us")
