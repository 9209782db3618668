"""Best of n: one prompt, n sampled continuations, scored and thinned out as they grow.

A small Llama-architecture model with quantized matrices (seeded synthetic
weights: there are no model files here) serves them as one batch.  The
sequences share the prompt's pages in a cache held in 4 bits:

  prompt    cache.append writes it, cache.attention with `begin` attends its rows
  fork      every candidate continues the prompt; whole pages are shared
  step      one row per candidate: append, attention, token_scores
  thin out  fork with the survivors as sources: the others' pages are free
  compact   the pages in use move to the front of the pool

    python examples/best_of_n.py [--n 8] [--prompt 200] [--steps 32]
"""
from __future__ import annotations

import argparse
import ctypes
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cllm_inference_b200 import _lib, gguf, synth  # noqa: E402
from cllm_inference_b200.kv4 import KV4Cache  # noqa: E402
from cllm_inference_b200.scoring import token_scores  # noqa: E402


class Model:
    """The layers of a Llama-architecture model on device buffers, through the C ABI's operators."""

    def __init__(self, shape: gguf.LlamaShape, seed: int = 0):
        self.s, self.lib = shape, _lib.load()
        _lib.check(self.lib.cllm_cuda_init(0))
        n, kv = shape.n_embd, shape.n_head_kv * shape.head_dim
        sizes = {"qkv": (n + 2 * kv, n), "o": (n, n), "gate": (shape.n_ff, n), "up": (shape.n_ff, n),
                 "down": (n, shape.n_ff)}
        self.layers = [{k: self._matrix(*v, seed + 10 * i + j) for j, (k, v) in enumerate(sizes.items())}
                       for i in range(shape.n_layers)]
        self.output = self._matrix(shape.vocab, n, seed + 9)
        gen = torch.Generator("cuda").manual_seed(seed)
        self.embed = torch.randn(shape.vocab, n, device="cuda", generator=gen)
        self.ones = torch.ones(n, device="cuda")
        table = np.empty((shape.n_ctx, shape.head_dim // 2, 2), np.float32)
        _lib.check(self.lib.cllm_cuda_rope_table(shape.rope_theta, shape.head_dim, shape.n_ctx,
                                                 table.ctypes.data_as(ctypes.c_void_p)))
        self.rope = torch.from_numpy(table).cuda()

    @staticmethod
    def _matrix(rows: int, cols: int, seed: int):
        """Q4_K blocks whose product with a unit vector is about a unit vector."""
        d = 1 / np.sqrt(cols) / (36 * 4.6)
        w = synth.make_weights(synth.Q4_K, rows, cols, seed, centered=True, d_range=(0.5 * d, 1.5 * d))
        return torch.from_numpy(w).cuda(), rows, cols

    def _mm(self, x: torch.Tensor, matrix) -> torch.Tensor:
        w, rows, cols = matrix
        y = torch.empty((x.shape[0], rows), device="cuda")
        _lib.check(self.lib.cllm_cuda_matmul_quant(x.data_ptr(), w.data_ptr(), synth.Q4_K, None, cols, rows, x.shape[0],
                                                   y.data_ptr(), 0, torch.cuda.current_stream().cuda_stream))
        return y

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        y = torch.empty_like(x)
        _lib.check(self.lib.cllm_cuda_rms_norm(x.data_ptr(), self.ones.data_ptr(), x.shape[1], x.shape[0],
                                               self.s.norm_eps, y.data_ptr(), torch.cuda.current_stream().cuda_stream))
        return y

    def rows(self, cache: KV4Cache, tokens, seq, pos, begin=None, last=None) -> torch.Tensor:
        """Logits of new tokens (int64) of the sequences `seq` at the positions `pos` (int32), whose lengths in the
        cache include them; `last`: of these rows only."""
        n, kv = self.s.n_embd, self.s.n_head_kv * self.s.head_dim
        x = self.embed[tokens]
        for i, w in enumerate(self.layers):
            qkv = self._mm(self._norm(x), w["qkv"])
            q = cache.append(i, qkv[:, n:n + kv], qkv[:, n + kv:], seq, pos, q=qkv[:, :n], rope=self.rope)
            x = x + self._mm(cache.attention(i, q, begin=begin), w["o"])
            h = self._norm(x)
            gate, up = self._mm(h, w["gate"]), self._mm(h, w["up"])
            _lib.check(self.lib.cllm_cuda_silu_mul(gate.data_ptr(), up.data_ptr(), gate.numel(),
                                                   torch.cuda.current_stream().cuda_stream))
            x = x + self._mm(gate, w["down"])
        return self._mm(self._norm(x if last is None else x[last].contiguous()), self.output)


def ints(*values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def best_of_n(model: Model, prompt, n: int = 8, steps: int = 32, keep: int = 2, top_k: int = 20, page_len: int = 16,
              seed: int = 0):
    """(tokens [keep][steps], their log probabilities [keep][steps], pages in use at the end, the cache)."""
    s, length = model.s, len(prompt)
    slots = -(-(length + steps) // page_len)
    cache = KV4Cache.empty(s.n_layers, slots + n * (slots - length // page_len), page_len, s.n_head_kv, s.head_dim, 1,
                           slots)
    gen = torch.Generator("cuda").manual_seed(seed)

    # the prompt, in one piece
    cache = cache.fork(ints(-1), ints(length))
    logits = model.rows(cache, torch.tensor(prompt, device="cuda"), torch.zeros(length, dtype=torch.int32, device="cuda"),
                        torch.arange(length, dtype=torch.int32, device="cuda"), begin=ints(0, length), last=[length - 1])

    cache = cache.fork(torch.zeros(n, dtype=torch.int32, device="cuda"),
                       torch.full((n,), length, dtype=torch.int32, device="cuda"))
    logits = logits.expand(n, -1)
    tokens, scores = [], []
    for step in range(steps):
        top = token_scores(logits, None, top_k)
        pick = torch.multinomial(top.top_logprobs.exp(), 1, generator=gen)
        token = top.top_ids.gather(1, pick)[:, 0].contiguous()
        tokens.append(token)
        scores.append(token_scores(logits, token).logprob)
        live = cache.n_seqs
        source = torch.arange(live, dtype=torch.int32, device="cuda")
        if step == steps // 2:  # half way: the best go on
            best = torch.stack(scores).sum(0).topk(keep).indices
            source, live = best.int(), keep
            tokens, scores = [t[best] for t in tokens], [t[best] for t in scores]
        cache = cache.fork(source, torch.full((live,), length + step + 1, dtype=torch.int32, device="cuda"))
        if step + 1 < steps:
            logits = model.rows(cache, tokens[-1].long(), torch.arange(live, dtype=torch.int32, device="cuda"),
                                cache.lens - 1)
    cache, in_use = cache.compact()
    _lib.check(model.lib.cllm_cuda_check_device_status())
    return torch.stack(tokens, 1), torch.stack(scores, 1), int(in_use[0]), cache


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--n", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--keep", type=int, default=2)
    a = ap.parse_args()
    model = Model(gguf.SMALL)
    prompt = np.random.default_rng(0).integers(0, model.s.vocab, a.prompt).tolist()
    tokens, scores, in_use, cache = best_of_n(model, prompt, a.n, a.steps, a.keep)
    for t, lp in zip(tokens.tolist(), scores.sum(1).tolist()):
        print(f"{lp:9.3f}  {t}")
    print(f"{in_use} of {cache.n_pages} pages in use, {cache.page_bytes * cache.n_layers} bytes each")


if __name__ == "__main__":
    main()
