"""Sampled generation over an 8-bit paged KV cache.

The loop of examples/serve_kv4.py (page bookkeeping on the GPU, prompts in chunks, one CUDA
graph per decode step) with the cache in 8 bits, one scale per page and head
(lc_qk_norm_rope_append_kv8, lc_unpack_kv8, lc_paged_decode_kv8), and tokens drawn by
lc_sample: every request has its own temperature, top-k, top-p and min-p, and the random
numbers are a device tensor that the step's graph reads and moves on.

    python examples/serve_kv8.py [--steps 64]
"""
from __future__ import annotations

import argparse
import time

import torch

import serve_kv4 as base
from serve_kv4 import PAGE, L, generate


class Stack(base.Stack):
    """With a small embedding, so that the tied head's logits leave a draw a choice."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.embed *= 0.07


class Engine(base.Engine):
    """Up to `slots` sequences over one 8-bit pool; request i samples with entry i of the
    parameters (None: temperature 1 and no filter). The random numbers begin anew after
    max_steps choices."""

    def __init__(self, stack, slots=8, max_len=1024, num_blocks=256, temperature=None, top_k=None,
                 top_p=None, min_p=None, seed=0, max_steps=4096):
        super().__init__(stack, slots, max_len, num_blocks)

        def row(values, dtype):
            return None if values is None else torch.tensor(values, dtype=dtype, device="cuda")
        self.params = dict(temperature=row(temperature, torch.float32),
                           top_k=row(top_k, torch.int32), top_p=row(top_p, torch.float32),
                           min_p=row(min_p, torch.float32))
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.numbers = torch.rand(max_steps, slots, generator=gen, device="cuda")
        self.step_no = torch.zeros(1, dtype=torch.int64, device="cuda")

    def _alloc_pool(self):
        s = self.stack
        return L.alloc_kv8_pool(self.num_blocks, s.layers, s.hkv, s.hd)

    def _alloc_workspace(self, batch):
        s = self.stack
        return L.alloc_decode_kv8_workspace(batch, s.hq, s.hkv, s.hd)

    def _append(self, qkv, positions, slot_map, layer):
        s = self.stack
        q = torch.empty(qkv.shape[0], s.hq * s.hd, dtype=torch.bfloat16, device="cuda")
        L.qk_norm_rope_append_kv8(q, qkv, positions, slot_map, s.cos, s.sin, self.pool,
                                  self.num_blocks, s.layers, layer, s.hq, s.hkv, s.hd,
                                  q_norm=s.q_norm[layer], k_norm=s.k_norm[layer],
                                  dev_status=self.status)
        return q

    def _unpack(self, tables, lens, longest, layer):
        s = self.stack
        L.unpack_kv8(self.k16, self.v16, self.pool, self.num_blocks, s.layers, layer, s.hkv, s.hd,
                     tables, lens, longest, dev_status=self.status)

    def _attend(self, out, q, layer):
        s = self.stack
        L.paged_decode_kv8(out, q, self.pool, self.num_blocks, s.layers, layer, s.hq, s.hkv, s.hd,
                           self.step_rows, self.batch_lens, max_context_len=self.width * PAGE,
                           workspace=self.ws, dev_status=self.status)

    def choose(self, out, logits, first=0):
        rows = slice(first, first + logits.shape[0])
        rand = self.numbers.index_select(0, self.step_no)[0, rows]
        L.sample(out, logits, rand,
                 **{k: None if v is None else v[rows] for k, v in self.params.items()})
        self.step_no.add_(1).remainder_(self.numbers.shape[0])


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=64)
    steps = ap.parse_args().steps
    stack = Stack()
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, stack.embed.shape[0], (n,), generator=gen, device="cuda")
               for n in (7, 100, 300, 513)]
    engine = Engine(stack, temperature=[0.0, 0.7, 1.0, 1.3] * 2, top_k=[0, 50, 0, 200] * 2,
                    top_p=[1.0, 0.9, 0.95, 1.0] * 2, min_p=[0.0, 0.0, 0.05, 0.0] * 2)
    generate(engine, prompts, 4)  # sets up the library's kernels
    engine.release(list(range(len(prompts))))
    torch.cuda.synchronize()
    t = time.perf_counter()
    tokens = generate(engine, prompts, steps)
    torch.cuda.synchronize()
    dt = time.perf_counter() - t
    print(f"{len(prompts)} prompts, {steps} sampled tokens each in {dt * 1e3:.1f} ms; "
          f"{int(engine.free_count.item())} of {engine.num_blocks} pages free")
    print("last tokens:", tokens[-1].tolist())
    engine.release(list(range(len(prompts))))
    print("after release:", int(engine.free_count.item()), "pages free")


if __name__ == "__main__":
    main()
