"""A small stack of routed layers over the operators (tierstream_amd.ops): trained with its weights resident, then decoded with
its experts streamed through a device-gated context.

    python -m tierstream_amd.moe [--layers 4 --experts 16 --top-k 2 --d-model 256 --d-ff 512 --heads 0 --steps 60 --tokens 64]

A layer adds to its rows what their chosen experts give: logits = x R^T (linear), ids and weights (route), y = x + the
experts' gated blocks (ffn). A head (linear) scores the vocabulary. With --heads a layer attends first: queries, keys and values
are one product (linear), turned by their positions (attn.rotate) and attended to inside their sequence (attn.attend), x + what comes of it by another
product goes on to the experts. Decode is what an engine does with the library: the
ids that route wrote go to ss_dg_enqueue_export, the layer's ss_dg_enqueue_wait holds the stream until its experts are in
the arena, ffn reads them through the arena's slots, and the whole token is one captured graph. Its place in the 4-bit cache
(attn.plan, attn.store, attn.attend_cached) is the device's to find, so that the same graph goes on from token to token. Needs torch.
"""
from __future__ import annotations

import argparse
import tempfile
import time
from dataclasses import dataclass
from pathlib import Path

import numpy as np
import torch

from . import attn, lib, ops, ss
from . import workloads as wl

BF16 = torch.bfloat16


@dataclass
class Shape:
    layers: int = 4
    experts: int = 16
    top_k: int = 2
    d_model: int = 256
    d_ff: int = 512
    vocab: int = 512
    heads: int = 0      # query heads (0: no attention)
    kv_heads: int = 2
    head_dim: int = 64


def _empty(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _workspace(nbytes: int):
    return _empty(max(nbytes, 16), dtype=torch.uint8)


def _product(x, w, dtype=BF16, **kw):
    """x w^T by ops.linear, on the current stream."""
    x, w = x.contiguous(), w.contiguous()
    y = _empty(x.shape[0], w.shape[0], dtype=dtype)
    ops.linear(x, w, y, workspace=_workspace(ops.linear_workspace(x, w, y)), stream=torch.cuda.current_stream().cuda_stream, **kw)
    return y


class Packed:
    """Where the rows' sequences begin, and their positions: `lengths` rows each, or every row a sequence of its own."""

    def __init__(self, rows: int, lengths=None):
        lengths = torch.tensor([1] * rows if lengths is None else lengths)
        if int(lengths.sum()) != rows:
            raise ValueError(f"lengths: of {rows} rows together, not {int(lengths.sum())}")
        ends = lengths.cumsum(0)
        self.first = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).cuda()
        self.positions = (torch.arange(rows) - torch.repeat_interleave(ends - lengths, lengths)).to(torch.int32).cuda()


class Model:
    """Weights in 32 bits, and in 16 as the operators read them."""

    def __init__(self, s: Shape, seed: int = 0):
        self.s = s
        self.rotary = attn.Rotary(s.head_dim) if s.heads else None
        g = torch.Generator("cuda").manual_seed(seed)
        new = lambda *shape, sigma: torch.randn(shape, device="cuda", generator=g) * sigma  # noqa: E731
        n, d, f = s.experts, s.d_model, s.d_ff
        self.embedding = new(s.vocab, d, sigma=1.0).to(BF16)
        self.master = {"head": new(s.vocab, d, sigma=d ** -0.5)}
        for L in range(s.layers):
            self.master[f"router{L}"] = new(n, d, sigma=d ** -0.5)
            for part, shape in (("gate", (n, f, d)), ("up", (n, f, d)), ("down", (n, d, f))):
                self.master[f"{part}{L}"] = new(*shape, sigma=shape[-1] ** -0.5)
            if s.heads:
                self.master[f"qkv{L}"] = new((s.heads + 2 * s.kv_heads) * s.head_dim, d, sigma=d ** -0.5)
                self.master[f"mix{L}"] = new(d, s.heads * s.head_dim, sigma=(s.heads * s.head_dim) ** -0.5)
        self.round()

    def round(self):
        self.w = {k: v.to(BF16) for k, v in self.master.items()}
        self.experts = [ops.Experts.stacked(*(self.w[f"{p}{L}"] for p in ("gate", "up", "down"))) for L in range(self.s.layers)]

    def split(self, qkv):
        """Queries, keys and values of a product's rows."""
        s = self.s
        return qkv.view(len(qkv), -1, s.head_dim).split([s.heads, s.kv_heads, s.kv_heads], 1)

    def attend(self, L: int, x, packed: Packed):
        """x and what its rows attend to; (input, queries keys and values as they were attended to, output, log sums)."""
        h = torch.cuda.current_stream().cuda_stream
        qkv = _product(x, self.w[f"qkv{L}"])
        q, k, v = self.split(qkv)
        attn.rotate(self.rotary, packed.positions, q, k, stream=h)
        out, lse = _empty(*q.shape), _empty(q.shape[1], q.shape[0], dtype=torch.float32)
        attn.attend(q, k, v, out, lse=lse, first=packed.first, stream=h)
        return _product(out.view(len(x), -1), self.w[f"mix{L}"], residual=x), (x, qkv, out, lse)

    def attend_back(self, L: int, dy, kept, packed: Packed, grads):
        """The gradient of attend()'s input from its output's; its weights' go to grads."""
        h = torch.cuda.current_stream().cuda_stream
        x, qkv, out, lse = kept
        (q, k, v), dqkv = self.split(qkv), torch.empty_like(qkv)
        dq, dk, dv = self.split(dqkv)
        grads[f"mix{L}"] = _product(dy.T, out.view(len(x), -1).T, torch.float32)
        dout = _product(dy, self.w[f"mix{L}"].T).view(out.shape)
        attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, first=packed.first, workspace=_workspace(attn.attend_backward_workspace(q, k)), stream=h)
        attn.rotate(self.rotary, packed.positions, dq, dk, backward=True, stream=h)
        grads[f"qkv{L}"] = _product(dqkv.T, x.T, torch.float32)
        return _product(dqkv, self.w[f"qkv{L}"].T, residual=dy.contiguous())

    def forward(self, tokens, packed: Packed | None = None, attended: list | None = None):
        """The head's logits, and each layer's (input of its experts, router logits, ids, weights); what attend() kept goes to `attended`."""
        x, kept, h = self.embedding[tokens], [], torch.cuda.current_stream().cuda_stream
        rows, k = len(tokens), self.s.top_k
        if self.s.heads and packed is None:
            packed = Packed(rows)
        for L, e in enumerate(self.experts):
            if self.s.heads:
                x, held = self.attend(L, x, packed)
                if attended is not None:
                    attended.append(held)
            logits = _product(x, self.w[f"router{L}"], torch.float32)
            ids, weights, y = _empty(rows, k, dtype=torch.int32), _empty(rows, k, dtype=torch.float32), torch.empty_like(x)
            ops.route(logits, ids, weights, stream=h)
            ops.ffn(e, x, y, ids=ids, weights=weights, residual=x, workspace=_workspace(ops.ffn_workspace(e, rows, k)), stream=h)
            kept.append((x, logits, ids, weights))
            x = y
        return _product(x, self.w["head"], torch.float32), x, kept

    def step(self, tokens, targets, rate: float, lengths=None) -> float:
        """One step down the mean cross-entropy of the targets (a gradient longer than 1 is shortened to it); the loss before it. lengths: of
        the tokens' sequences (where layers attend; None: each token by itself)."""
        attended, packed = [], Packed(len(tokens), lengths) if self.s.heads else None
        logits, top, kept = self.forward(tokens, packed, attended)
        loss = torch.nn.functional.cross_entropy(logits, targets)
        dlogits = torch.softmax(logits, 1)
        dlogits[torch.arange(len(tokens), device="cuda"), targets] -= 1
        dlogits = (dlogits / len(tokens)).to(BF16)
        grads = {"head": _product(dlogits.T, top.T, torch.float32)}
        dy, h = _product(dlogits, self.w["head"].T), torch.cuda.current_stream().cuda_stream
        for L in reversed(range(self.s.layers)):
            e, (x, logits, ids, weights) = self.experts[L], kept[L]
            dx, dweights = torch.empty_like(x), torch.empty_like(weights)
            parts = [torch.empty_like(self.w[f"{p}{L}"]) for p in ("gate", "up", "down")]
            ops.ffn_backward(e, x, dy, dx, ids=ids, weights=weights, dweights=dweights, dgate=parts[0], dup=parts[1], ddown=parts[2],
                             workspace=_workspace(ops.ffn_backward_workspace(e, *ids.shape)), stream=h)
            dlogits = torch.empty_like(logits)
            ops.route_backward(logits, ids, dweights, dlogits, stream=h)
            dlogits = dlogits.to(BF16)
            grads[f"router{L}"] = _product(dlogits.T, x.T, torch.float32)
            dy = _product(dlogits, self.w[f"router{L}"].T, residual=dy + dx)
            if self.s.heads:
                dy = self.attend_back(L, dy, attended[L], packed, grads)
            grads.update((f"{p}{L}", t) for p, t in zip(("gate", "up", "down"), parts))
        norm = float(sum(t.float().square().sum() for t in grads.values()).sqrt())
        for name, t in grads.items():
            self.master[name].add_(t, alpha=-rate / max(1.0, norm))
        self.round()
        return float(loss)

    def workload(self, resident: float = 0.4) -> wl.Workload:
        s = self.s
        return wl.Workload("routed-layers", s.layers, s.experts, [s.d_model * s.d_ff * wl.BF16] * 3, top_k=s.top_k, gen=1,
                           resident_fraction=resident, tier_mode=1, forward=1)

    def write(self, path) -> str:
        """The experts as one source file; its descriptor."""
        w, hashes = self.workload(), []
        with open(path, "wb") as out:
            for L in range(self.s.layers):
                parts = [self.w[f"{p}{L}"].view(torch.int16).cpu().numpy() for p in ("gate", "up", "down")]
                for u in range(self.s.experts):
                    unit = np.concatenate([p[u].reshape(-1) for p in parts])
                    hashes.append(int(lib().tsa_xxh64_host(unit.ctypes.data, unit.nbytes)))
                    out.write(unit.tobytes().ljust(w.unit_stride_file, b"\0"))
        return wl.desc_json(w, path, hashes)


class Decoder:
    """Tokens one at a time, the experts of `model` read from a device-gated context over its written source. The model may be
    trained on: the decoder keeps the weights it was made with, as the source does (a step gives the model new tensors, and
    the captured graph goes on reading these). With attention, a token attends to those behind it since forget(), up to `context` of them
    (in whole pages)."""

    def __init__(self, model: Model, desc_json: str, context: int = 1024):
        s, shape = model.s, wl.dg_shape(model.workload())
        parts = ("router", "qkv", "mix") if s.heads else ("router",)
        self.embedding, self.w = model.embedding, {"head": model.w["head"], **{f"{p}{L}": model.w[f"{p}{L}"] for p in parts for L in range(s.layers)}}
        self.model = model
        self.desc, budget = ss.Desc(desc_json), ss.budget(**shape.budget)
        self.plan = ss.Plan(self.desc, budget)
        self.ctx = ss.Ctx(self.desc, budget, self.plan, ss.options(**shape.options, verify_hash=2, dg_wait_timeout_ms=5000))
        self.experts = [ops.Experts.in_arena(self.ctx.dg_view(), self.ctx.dg_gated_index(L), s.experts, s.d_model, s.d_ff, "bf16")
                        for L in range(s.layers)]
        self.x = [_empty(1, s.d_model) for _ in range(s.layers + 1)]
        self.scores = _empty(1, s.experts, dtype=torch.float32)
        self.ids = [_empty(1, s.top_k, dtype=torch.int32) for _ in range(s.layers)]
        self.weights = _empty(1, s.top_k, dtype=torch.float32)
        self.logits = _empty(1, s.vocab, dtype=torch.float32)
        self.room = _workspace(max(ops.ffn_workspace(self.experts[0], 1, s.top_k),
                                   ops.linear_workspace(self.x[0], self.w["head"], self.logits),
                                   ops.linear_workspace(self.x[0], self.w["router0"], self.scores)))
        if s.heads:
            self._attention(s, context)
        self.stream, self.graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        # (the library's threads go on with their own calls while this one captures)
        with torch.cuda.graph(self.graph, stream=self.stream, capture_error_mode="thread_local"):
            self._enqueue(torch.cuda.current_stream().cuda_stream)

    def _attention(self, s: Shape, context: int):
        """One request's pages, and the buffers of its tokens."""
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
        n = -(-context // attn.PAGE)
        self.caches = [attn.Cache(_empty(n, s.kv_heads, attn.page_bytes(s.head_dim), dtype=torch.uint8), s.kv_heads, s.head_dim) for _ in range(s.layers)]
        self.length, self.fresh, self.table, self.free, self.n_free = ints(1), ints(1), ints(1, n), torch.arange(n, dtype=torch.int32, device="cuda"), ints(1)
        self.first, self.position, self.slot, self.status = ints(2), ints(1), ints(1), ints(1)
        self.fresh += 1
        self.n_free += n
        self.qkv, self.mixed = _empty(1, (s.heads + 2 * s.kv_heads) * s.head_dim), _empty(1, s.heads, s.head_dim)
        self.mid = [_empty(1, s.d_model) for _ in range(s.layers)]
        q = self.model.split(self.qkv)[0]
        need = [attn.attend_cached_workspace(self.caches[0], q, self.table), ops.linear_workspace(self.x[0], self.w["qkv0"], self.qkv),
                ops.linear_workspace(self.mixed.view(1, -1), self.w["mix0"], self.mid[0])]
        self.room = _workspace(max(self.room.numel(), *need))

    def _attend(self, L: int, h):
        """mid[L] = x[L] and what it attends to."""
        q, k, v = self.model.split(self.qkv)
        ops.linear(self.x[L], self.w[f"qkv{L}"], self.qkv, workspace=self.room, stream=h)
        attn.rotate(self.model.rotary, self.position, q, k, stream=h)
        attn.store(self.caches[L], k, v, self.slot, stream=h)
        attn.attend_cached(self.caches[L], q, self.mixed, self.table, self.length, self.first, workspace=self.room, stream=h)
        ops.linear(self.mixed.view(1, -1), self.w[f"mix{L}"], self.mid[L], residual=self.x[L], workspace=self.room, stream=h)
        return self.mid[L]

    def forget(self):
        """The next token is the first one."""
        with torch.cuda.stream(self.stream):
            ended = torch.full_like(self.fresh, -1)
            attn.plan(self.length, ended, self.table, self.free, self.n_free, self.first, self.position, self.slot, self.status, stream=self.stream.cuda_stream)

    def _enqueue(self, h):
        w, x = self.w, list(self.x)
        self.ctx.dg_enqueue_begin(h)
        if self.model.s.heads:
            attn.plan(self.length, self.fresh, self.table, self.free, self.n_free, self.first, self.position, self.slot, self.status, stream=h)
        for L, e in enumerate(self.experts):
            if self.model.s.heads:
                x[L] = self._attend(L, h)
            ops.linear(x[L], w[f"router{L}"], self.scores, workspace=self.room, stream=h)
            ops.route(self.scores, self.ids[L], self.weights, stream=h)
            self.ctx.dg_enqueue_export(e.s.gated, self.ids[L].data_ptr(), self.ids[L].numel(), h)
            self.ctx.dg_enqueue_wait(e.s.gated, h)
            ops.ffn(e, x[L], x[L + 1], ids=self.ids[L], weights=self.weights, residual=x[L], workspace=self.room, stream=h)
        self.ctx.dg_enqueue_end(h)
        ops.linear(x[-1], w["head"], self.logits, workspace=self.room, stream=h)

    def token(self, token: int) -> int:
        """The likeliest token behind `token`."""
        # What a caller left on the null stream ends first: the library's streams wait for it, and where it shares the graph's hardware queue
        # their wait would stand behind the token's own waits, which wait for them.
        torch.cuda.default_stream().synchronize()
        with torch.cuda.stream(self.stream):
            self.x[0].copy_(self.embedding[token:token + 1])
            self.ctx.begin()
            try:
                self.graph.replay()
            finally:
                self.ctx.end()
            if self.model.s.heads and int(self.status):
                raise RuntimeError(f"the token has no place in the cache (status {int(self.status)}): forget() gives it back")
            return int(self.logits.argmax())

    def close(self):
        self.stream.synchronize()
        self.ctx.close()


def main(argv=None) -> None:
    p = argparse.ArgumentParser(prog="python -m tierstream_amd.moe", description="Trains a small stack of routed layers, then decodes it.")
    for name, value in (("layers", 4), ("experts", 16), ("top-k", 2), ("d-model", 256), ("d-ff", 512), ("vocab", 512), ("steps", 60),
                        ("tokens", 64), ("heads", 0)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = vars(p.parse_args(argv))
    steps, tokens = a.pop("steps"), a.pop("tokens")
    model = Model(Shape(**a))
    after = torch.randperm(model.s.vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(1))  # what it learns
    everything = torch.arange(model.s.vocab, device="cuda")
    lengths = [min(16, model.s.vocab - at) for at in range(0, model.s.vocab, 16)]  # (of the sequences that they are, where layers attend)
    for i in range(steps):
        loss = model.step(everything, after, model.s.vocab / 1024, lengths)
        if i % 10 == 0 or i + 1 == steps:
            print(f"step {i}: loss {loss:.4f}", flush=True)
    with tempfile.TemporaryDirectory() as folder:
        decoder = Decoder(model, model.write(Path(folder) / "experts.bin"))
        try:
            at, right, began = 0, 0, time.perf_counter()
            for _ in range(tokens):
                got = decoder.token(at)
                right += got == int(after[at])
                at = got
            took = time.perf_counter() - began
            stats = decoder.ctx.dg_stats()
            print(f"{tokens} tokens, {right} as trained, {tokens / took:.0f} a second; experts looked up {stats['lookups']}, "
                  f"fetched {stats['fetched']}, evicted {stats['evicted']}, failed checks {decoder.ctx.verify_failures()}")
        finally:
            decoder.close()


if __name__ == "__main__":
    main()
