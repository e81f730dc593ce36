"""A decode step of two attention layers over GGUF weights, as a server runs it:

    qkv (Q8_0 shards, one launch) + each row's adapter -> norm, rotation, store into the pages -> attention over the
    pages -> o_proj + adapter

Prompts go through the same operators (each prompt token is a row of the batch that sees the keys before it); the steps
replay one HIP graph.  On the way a sequence is forked (the fork shares its pages and gets a page of its own where
it writes), one ends, and the cache is compacted.  Every output is checked against the same network in fp32 without
a cache.  Run: python examples/decode_step.py"""
from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hyperqwen-rtx4080s32_amd"))

import gguf_hip as G  # noqa: E402

Q8_0 = 8
K, HEADS, KV_HEADS, DIM, PAGE = 1024, 8, 2, 128, 16
PARTS = [HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM]


def q8_0(w: torch.Tensor) -> torch.Tensor:
    """fp32 [n, K] as GGUF's Q8_0 rows: blocks of an fp16 scale and 32 signed bytes."""
    blocks = w.reshape(w.shape[0], -1, 32)
    d = (blocks.abs().amax(2, keepdim=True) / 127).half()
    q = (blocks / d.float().clamp_min(1e-8)).round().clamp(-127, 127).to(torch.int8)
    return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], 2).reshape(w.shape[0], -1).contiguous()


class Layer:
    """Weights of one attention layer: the quantized projections, and adapters 0 and 1 for both (1 leaves k alone)."""

    def __init__(self, gen: torch.Generator):
        rand = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
        raw = [q8_0(rand(n, K) / K ** 0.5) for n in PARTS]
        raw_o = q8_0(rand(K, PARTS[0]) / PARTS[0] ** 0.5)
        self.w_qkv = torch.cat([G.dequantize(r, Q8_0, (n, K)) for r, n in zip(raw, PARTS)]).float()
        self.w_o = G.dequantize(raw_o, Q8_0, (K, PARTS[0])).float()
        self.qkv = G.pack_layer(raw, PARTS, [Q8_0] * 3)
        self.o = G.pack_layer([raw_o], [K], [Q8_0])
        self.q_norm, self.k_norm = ((1 + 0.1 * rand(DIM)).bfloat16() for _ in range(2))

        def adapter(rank, parts, k, leave=()):
            down = [None if p in leave else rand(rank, k) / k ** 0.5 for p in range(len(parts))]
            up = [None if p in leave else rand(n, rank) / rank ** 0.5 for p, n in enumerate(parts)]
            return down, up, 0.5

        self.lora = G.pack_adapters([adapter(16, PARTS, K), adapter(8, PARTS, K, leave=(1,))], PARTS, K)
        self.lora_o = G.pack_adapters([adapter(16, [K], PARTS[0]), adapter(8, [K], PARTS[0])], [K], PARTS[0])


class Model:
    def __init__(self, layers: int = 2, pages: int = 64, length: int = 256):
        gen = torch.Generator(device="cuda").manual_seed(1)
        self.layers = [Layer(gen) for _ in range(layers)]
        # a head's tokens side by side within a page; all layers' keys and values in one tensor for copy_pages
        self.storage = torch.zeros((layers, 2, pages, KV_HEADS, PAGE, DIM), dtype=torch.bfloat16, device="cuda")
        self.pool = G.PagePool(pages)
        self.rope = G.rope_table(DIM, length, base=1e6)
        self.length = length

    def pages(self, i: int):
        return self.storage[i, 0].transpose(1, 2), self.storage[i, 1].transpose(1, 2)

    def forward(self, x, ids, positions, slots, table, lengths):
        """x bf16 [rows, K], a row a new token: its adapter, position, slot in the cache, pages and number of keys."""
        rows = x.shape[0]
        for i, w in enumerate(self.layers):
            k_pages, v_pages = self.pages(i)
            h = torch.nn.functional.rms_norm(x, (K,))
            y = G.mul_mat_grouped(h, w.qkv)
            G.lora_add(y, h, w.lora[0], w.lora[1], ids, w.lora[2], PARTS, out=y)
            q, k, v = (t.view(rows, -1, DIM) for t in y.split(PARTS, 1))
            q, _ = G.qk_norm_rope(q, k, positions, self.rope, w.q_norm, w.k_norm, v=v, k_pages=k_pages, v_pages=v_pages,
                                  slots=slots)
            o = G.paged_attention(q, k_pages, v_pages, table, lengths, max_length=self.length).view(rows, -1)
            z = G.mul_mat_grouped(o, w.o)
            G.lora_add(z, o, w.lora_o[0], w.lora_o[1], ids, w.lora_o[2], [K], out=z)
            x = x + z
        return x

    def plain(self, x, ids):
        """The same network over one whole sequence in fp32: x [tokens, K], ids [tokens]."""
        x, n = x.float(), x.shape[0]
        cos, sin = self.rope[:n, None].chunk(2, 2)
        keep = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()

        def update(h, lora, parts):
            a, b, scales = (t.float() for t in lora)
            at = ids.long().clamp_min(0)
            low = torch.matmul(a[at], h[:, None, :, None])[..., 0]                             # [n, parts, rank]
            out = torch.cat([torch.matmul(bp, low[:, p, :, None])[..., 0] for p, bp in enumerate(b[at].split(parts, 1))], 1)
            return out * (scales[at] * (ids >= 0))[:, None]

        def heads(t, weight):
            t = torch.nn.functional.rms_norm(t.view(n, -1, DIM), (DIM,), weight.float(), 1e-6)
            s, c = t.chunk(2, 2)
            return torch.cat([s * cos - c * sin, c * cos + s * sin], 2).transpose(0, 1)

        for w in self.layers:
            h = torch.nn.functional.rms_norm(x, (K,))
            q, k, v = (h @ w.w_qkv.T + update(h, w.lora, PARTS)).split(PARTS, 1)
            q, k, v = heads(q, w.q_norm), heads(k, w.k_norm), v.reshape(n, -1, DIM).transpose(0, 1)
            k, v = (t.repeat_interleave(HEADS // KV_HEADS, 0) for t in (k, v))
            p = (torch.matmul(q, k.transpose(1, 2)) * DIM ** -0.5).masked_fill(~keep, float("-inf")).softmax(2)
            o = torch.matmul(p, v).transpose(0, 1).reshape(n, -1)
            x = x + o @ w.w_o.T + update(o, w.lora_o, [K])
        return x


class Sequence:
    """Its pages, and what the check needs: all inputs with their adapters, all outputs."""

    def __init__(self, adapter: int):
        self.adapter, self.table = adapter, []
        self.inputs, self.ids, self.outputs = [], [], []

    def __len__(self):
        return len(self.inputs)


class Server:
    def __init__(self, model: Model, batch: int):
        self.model, self.pool = model, model.pool
        width = model.length // PAGE
        ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        # a step's inputs: written before each replay; rows without a sequence have no key and no slot
        self.x = torch.zeros((batch, K), dtype=torch.bfloat16, device="cuda")
        self.args = [ints(batch), ints(batch), ints(batch), ints(batch, width), ints(batch)]
        self._write([], None)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            model.forward(self.x, *self.args)   # a call before the capture
        torch.cuda.current_stream().wait_stream(stream)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = model.forward(self.x, *self.args)

    def _slot(self, s: Sequence, at: int) -> int:
        """The cache's slot of s's token `at`, a page of its own under it."""
        if at // PAGE == len(s.table):
            s.table += self.pool.allocate(1)
        src, dst = self.pool.own(s.table, at // PAGE)
        if src:
            G.copy_pages(self.model.storage, src, dst, dim=2)
        return s.table[at // PAGE] * PAGE + at % PAGE

    def _rows(self, rows: list[tuple[Sequence, int]], total: int):
        """ids, positions, slots, tables and lengths of rows (sequence, token number), padded to `total`."""
        slots = [self._slot(s, at) for s, at in rows]
        pad = total - len(rows)
        width = self.model.length // PAGE
        tables = [s.table + [-1] * (width - len(s.table)) for s, _ in rows] + [[-1] * width] * pad
        return ([s.adapter for s, _ in rows] + [-1] * pad, [at for _, at in rows] + [0] * pad, slots + [-1] * pad, tables,
                [at + 1 for _, at in rows] + [0] * pad)

    def _write(self, rows, x) -> None:
        for t, values in zip(self.args, self._rows(rows, self.x.shape[0])):
            t.copy_(torch.tensor(values, dtype=torch.int32))
        if x is not None:
            self.x[:len(rows)] = x

    def _keep(self, s: Sequence, x, y) -> None:
        s.inputs.append(x)
        s.ids.append(s.adapter)
        s.outputs.append(y)

    def prompt(self, s: Sequence, x: torch.Tensor) -> None:
        n = x.shape[0]
        args = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in self._rows([(s, len(s) + i) for i in range(n)], n)]
        y = self.model.forward(x, *args)
        for i in range(n):
            self._keep(s, x[i], y[i])

    def step(self, sequences: list[Sequence], x: torch.Tensor) -> None:
        self._write([(s, len(s)) for s in sequences], x)
        self.graph.replay()
        for i, s in enumerate(sequences):
            self._keep(s, x[i].clone(), self.out[i].clone())

    def fork(self, s: Sequence, adapter: int) -> Sequence:
        t = Sequence(adapter)
        t.table = self.pool.fork(s.table)
        t.inputs, t.ids, t.outputs = list(s.inputs), list(s.ids), list(s.outputs)
        return t

    def error(self, s: Sequence) -> float:
        """The largest error of a token's output against the plain network's, relative to the token."""
        want = self.model.plain(torch.stack(s.inputs), torch.tensor(s.ids, device="cuda"))
        got = torch.stack(s.outputs).float()
        return float(((got - want).norm(dim=1) / want.norm(dim=1)).max())


def run(steps: int = 12) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(2)
    tokens = lambda n: torch.randn((n, K), device="cuda", generator=gen).bfloat16()  # noqa: E731
    server = Server(Model(), batch=4)
    errors = {}
    a, b, c = Sequence(0), Sequence(-1), Sequence(1)
    for s, n in ((a, 37), (b, 5), (c, 64)):
        server.prompt(s, tokens(n))
    for _ in range(steps):
        server.step([a, b, c], tokens(3))
    d = server.fork(a, 1)                       # a and d go on from the same pages
    for _ in range(steps):
        server.step([a, d, b, c], tokens(4))
    errors["a"] = server.error(a)               # a ends; the others move to the front of the cache
    server.pool.free(a.table)
    src, dst = server.pool.compact([b.table, c.table, d.table])
    G.copy_pages(server.model.storage, src, dst, dim=2)
    for _ in range(steps):
        server.step([c, d, b], tokens(3))
    for name, s in (("b", b), ("c", c), ("d", d)):
        errors[name] = server.error(s)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(100):
        server.graph.replay()
    torch.cuda.synchronize()
    return {"errors": errors, "moved": len(src), "us_per_step": (time.perf_counter() - start) * 1e4}


if __name__ == "__main__":
    got = run()
    print("largest error of a token against fp32:", {n: f"{e:.4f}" for n, e in got["errors"].items()})
    print(f"{got['moved']} pages moved by the compaction; {got['us_per_step']:.0f} us a step of two layers (graph)")
