"""Greedy generation over a 4-bit paged KV cache, with the page bookkeeping on the GPU.

An attention-only stack (random weights, the shapes of Qwen2.5-0.5B's attention with
per-head norms of q and k) serves a few prompts:

  * prompts: lc_step_tables (pages, positions, slots), then per layer the QKV
    projection, lc_qk_norm_rope_append_kv4, lc_unpack_kv4 + lc_paged_prefill over
    the sequences' cached pages, and o_proj with the residual; long prompts come
    in chunks that continue the cached context;
  * decode: the whole step (bookkeeping, layers, logits, token choice) is one CUDA
    graph. Lengths, free pages and tables live on the device and advance by
    themselves, so a step is one graph launch and no host copy;
  * finished sequences give their pages back with lc_step_release.

    python examples/serve_kv4.py [--steps 64]
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "lucciola-rs_b200"))
import lucciola as L  # noqa: E402

PAGE = 16


class Stack:
    """Weights of `layers` attention blocks and a tied embedding."""

    def __init__(self, layers=2, hidden=896, hq=14, hkv=2, hd=64, vocab=2048, max_pos=4096, seed=0):
        self.layers, self.hidden, self.hq, self.hkv, self.hd = layers, hidden, hq, hkv, hd
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def w(*shape, std):
            return (torch.randn(*shape, generator=gen, device="cuda") * std).bfloat16()
        row = (hq + 2 * hkv) * hd
        self.embed = w(vocab, hidden, std=1.0)
        self.w_qkv = [w(row, hidden, std=hidden ** -0.5) for _ in range(layers)]
        self.w_o = [w(hidden, hq * hd, std=(hq * hd) ** -0.5) for _ in range(layers)]
        self.q_norm = [1 + w(hd, std=0.1) for _ in range(layers)]
        self.k_norm = [1 + w(hd, std=0.1) for _ in range(layers)]
        cos, sin = L.rope_table_host(max_pos, hd, 1e6)
        self.cos, self.sin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()


class Engine:
    """Up to `slots` sequences of at most `max_len` tokens over one 4-bit pool."""

    K_SCALE, V_SCALE = 1.0, 0.25

    def __init__(self, stack, slots=8, max_len=1024, num_blocks=256):
        s = self.stack = stack
        self.slots, self.num_blocks = slots, num_blocks
        self.width = -(-max_len // PAGE)  # pages of one sequence at most
        self.pool = L.alloc_kv4_pool(num_blocks, s.layers, s.hkv, s.hd)

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device="cuda")
        # page bookkeeping: the stack hands out pages 0, 1, 2, ...
        self.free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device="cuda")
        self.free_count = ints(1, fill=num_blocks)
        self.tables = ints(slots, self.width, fill=-1)
        self.lens = ints(slots)  # cached tokens, by slot
        self.step_ws = L.alloc_step_workspace()
        self.status = ints(1)
        self.ints = ints
        # bf16 pages of one layer, for a prompt's attention
        shape = (self.width, 1, s.hkv, PAGE, s.hd)
        self.k16, self.v16 = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.own_pages = torch.arange(self.width, dtype=torch.int32, device="cuda").view(1, -1)

    def _project(self, x, layer):
        s = self.stack
        qkv = torch.empty(x.shape[0], (s.hq + 2 * s.hkv) * s.hd, dtype=torch.bfloat16, device="cuda")
        L.proj_gemm(qkv, x, s.w_qkv[layer])
        return qkv

    def _append(self, qkv, positions, slot_map, layer):
        s = self.stack
        q = torch.empty(qkv.shape[0], s.hq * s.hd, dtype=torch.bfloat16, device="cuda")
        L.qk_norm_rope_append_kv4(q, qkv, positions, slot_map, s.cos, s.sin, self.pool,
                                  self.num_blocks, s.layers, layer, s.hq, s.hkv, s.hd,
                                  k_scale=self.K_SCALE, v_scale=self.V_SCALE,
                                  q_norm=s.q_norm[layer], k_norm=s.k_norm[layer],
                                  dev_status=self.status)
        return q

    def prompt(self, slot, tokens, start=0):
        """Feeds `tokens` (1-d int tensor) of the sequence in `slot`, `start` of whose tokens
        are cached; returns the hidden rows [tokens, hidden]."""
        s, n = self.stack, tokens.shape[0]
        slots, new = self.ints(1, fill=slot), self.ints(1, fill=n)
        lens = self.lens[slot:slot + 1]
        step, pos, slot_map = self.ints(1, self.width), self.ints(n), self.ints(n)
        before = lens.clone()
        L.step_tables(self.tables, lens, new, self.free, self.free_count, pos, slot_map,
                      self.ints(2), lens, self.free_count, self.step_ws, slots=slots,
                      step_tables=step, dev_status=self.status)
        x = s.embed[tokens.long()]
        for layer in range(s.layers):
            q = self._append(self._project(x, layer), pos, slot_map, layer)
            L.unpack_kv4(self.k16, self.v16, self.pool, self.num_blocks, s.layers, layer, s.hkv,
                         s.hd, step, lens, start + n, k_scale=self.K_SCALE, v_scale=self.V_SCALE,
                         dev_status=self.status)
            out = torch.empty_like(q)
            L.paged_prefill(out, q, self.k16, self.v16, self.width, 1, 0, s.hq, s.hkv, s.hd,
                            self.own_pages, before, n, start, dev_status=self.status)
            L.proj_gemm(x, out, s.w_o[layer], residual=x)
        return x

    def start_decode(self, slots, first_tokens):
        """The decode step of `slots` (list) as a function to call; keeps their next tokens."""
        self.live = torch.tensor(slots, dtype=torch.int32, device="cuda")
        b = len(slots)
        self.batch_lens = self.lens[self.live.long()].contiguous()  # advances by itself
        self.token = first_tokens.int().clone()
        self.ones = self.ints(b, fill=1)
        self.step_rows = self.ints(b, self.width, fill=-1)
        self.pos, self.slot_map, self.starts = self.ints(b), self.ints(b), self.ints(b + 1)
        s = self.stack
        self.ws = L.alloc_decode_kv4_workspace(b, s.hq, s.hkv, s.hd)

        def step():
            L.step_tables(self.tables, self.batch_lens, self.ones, self.free, self.free_count,
                          self.pos, self.slot_map, self.starts, self.batch_lens, self.free_count,
                          self.step_ws, slots=self.live, step_tables=self.step_rows,
                          dev_status=self.status)
            x = s.embed.index_select(0, self.token)
            for layer in range(s.layers):
                q = self._append(self._project(x, layer), self.pos, self.slot_map, layer)
                out = torch.empty_like(q)
                L.paged_decode_kv4(out, q, self.pool, self.num_blocks, s.layers, layer, s.hq, s.hkv,
                                   s.hd, self.step_rows, self.batch_lens,
                                   max_context_len=self.width * PAGE, k_scale=self.K_SCALE,
                                   v_scale=self.V_SCALE, workspace=self.ws, dev_status=self.status)
                L.proj_gemm(x, out, s.w_o[layer], residual=x)
            logits = torch.empty(b, s.embed.shape[0], dtype=torch.bfloat16, device="cuda")
            L.proj_gemm(logits, x, s.embed)
            L.argmax(self.token, logits)
            return x
        return step

    def end_decode(self):
        """Lengths back by slot, and a check of what the device saw."""
        self.lens[self.live.long()] = self.batch_lens
        status = L.lib.lc_status_from_device_word(int(self.status.item()))
        if status:
            raise L.LucciolaError(status, "decode")

    def release(self, slots):
        which = torch.tensor(slots, dtype=torch.int32, device="cuda")
        L.step_release(self.free, self.free_count, self.tables, self.lens[which.long()].contiguous(),
                       self.free_count, self.step_ws, slots=which, dev_status=self.status)
        self.lens[which.long()] = 0


def first_token(engine, hidden):
    s = engine.stack
    logits = torch.empty(1, s.embed.shape[0], dtype=torch.bfloat16, device="cuda")
    L.proj_gemm(logits, hidden[-1:].contiguous(), s.embed)
    out = torch.zeros(1, dtype=torch.int32, device="cuda")
    L.argmax(out, logits)
    return out


def generate(engine, prompts, steps, chunk=256, graph=True):
    """Greedy tokens [steps, len(prompts)] for a list of 1-d token tensors."""
    nxt = []
    for slot, p in enumerate(prompts):
        for at in range(0, p.shape[0], chunk):
            hidden = engine.prompt(slot, p[at:at + chunk], at)
        nxt.append(first_token(engine, hidden))
    step = engine.start_decode(list(range(len(prompts))), torch.cat(nxt))
    got = [engine.token.clone()]
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()  # the first step sets up the library's kernels
        torch.cuda.current_stream().wait_stream(side)
        got.append(engine.token.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        run = g.replay
    else:
        run = step
    while len(got) < steps:
        run()
        got.append(engine.token.clone())
    engine.end_decode()
    return torch.stack(got[:steps])


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=64)
    steps = ap.parse_args().steps
    stack = Stack()
    engine = Engine(stack)
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, stack.embed.shape[0], (n,), generator=gen, device="cuda")
               for n in (7, 100, 300, 513)]
    generate(engine, prompts, 4)  # sets up the library's kernels
    engine.release(list(range(len(prompts))))
    torch.cuda.synchronize()
    t = time.perf_counter()
    tokens = generate(engine, prompts, steps)
    torch.cuda.synchronize()
    dt = time.perf_counter() - t
    print(f"{len(prompts)} prompts, {steps} greedy tokens each in {dt * 1e3:.1f} ms; "
          f"{int(engine.free_count.item())} of {engine.num_blocks} pages free")
    print("last tokens:", tokens[-1].tolist())
    engine.release(list(range(len(prompts))))
    print("after release:", int(engine.free_count.item()), "pages free")


if __name__ == "__main__":
    main()
