"""Workloads of the 4-bit cache operators: a step's block tables and slot map
built on the GPU, per-head norm + RoPE + append, the 4-bit cache's round trip,
and single-token attention over it.

run() computes each operator in a plain form (elementary torch operations in
fp32) or, where `own` is set, through lucciola's entry points. Shapes are those
of the Qwen2 family (0.5B: 14/2 heads of 64; 1.5B: 12/2 of 128; 7B: 28/4 of 128;
72B: 64/8 of 128).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 16          # tokens per page
ROPE_ROWS = 32768  # rows of the cos/sin tables
EPS = 1e-6


def listed():
    return [
        # --- tables: what a serving loop does first in every step
        # one decode step of 64 sequences, 256 .. 4096 tokens each: the smallest call
        dict(name="tables_decode64", op="tables", batch=64, slots=64, max_ctx=4096, prompts=0,
             max_new=1, stride=257, done=0, spare=300),
        # decoding sequences and arriving prompts in one step, finished ones released;
        # too few free pages for all of them
        dict(name="tables_mixed256", op="tables", batch=256, slots=300, max_ctx=8192, prompts=24,
             max_new=2048, stride=640, done=17, spare=400),
        # a large engine: 1024 sequences of up to 32768 tokens, prompts of up to 8192
        dict(name="tables_wide1024", op="tables", batch=1024, slots=1200, max_ctx=24576,
             prompts=37, max_new=8191, stride=2048, done=64, spare=20000),
        # --- nra: norm + RoPE + append into the bf16 pools
        # decode step of a 7B-shaped batch
        dict(name="nra_decode32", op="nra", rows=32, hq=28, hkv=4, hd=128, bias=False, norm=True,
             layers=2, pad=0, idle=0),
        # odd row count, heads of 64, biases as well, padded rows, rows without a slot
        dict(name="nra_odd5001", op="nra", rows=5001, hq=14, hkv=2, hd=64, bias=True, norm=True,
             layers=1, pad=8, idle=23),
        # four prompts of 4096 tokens, 1.5B shape
        dict(name="nra_prompt16k", op="nra", rows=16384, hq=12, hkv=2, hd=128, bias=False,
             norm=True, layers=1, pad=0, idle=0),
        # --- kv4: a prompt appended to the 4-bit cache and its context unpacked for the
        # prefill attention
        # one short ragged prompt chunk after 77 cached tokens
        dict(name="kv4_chunk", op="kv4", batch=1, start=77, tokens=179, hq=14, hkv=2, hd=64,
             bias=True, norm=False, layers=2, k_scale=1.0, v_scale=0.25),
        # prompts of 2048 tokens, 7B shape
        dict(name="kv4_prompt8k", op="kv4", batch=4, start=0, tokens=2048, hq=28, hkv=4, hd=128,
             bias=False, norm=True, layers=1, k_scale=0.5, v_scale=0.0625),
        # --- dec: attention of the newest tokens over the 4-bit cache
        # one sequence, 1024 cached tokens: latency
        dict(name="dec_single1k", op="dec", batch=1, lo=1024, hi=1024, hq=14, hkv=2, hd=64,
             tokens=1, layers=2, k_scale=1.0, v_scale=0.25),
        # 64 ragged sequences of 256 .. 4096 tokens, one of them empty
        dict(name="dec_ragged64", op="dec", batch=64, lo=256, hi=4096, hq=14, hkv=2, hd=64,
             tokens=1, layers=1, k_scale=1.0, v_scale=0.25),
        # 32 sequences of 8192 tokens, 7B shape
        dict(name="dec_batch32", op="dec", batch=32, lo=8192, hi=8192, hq=28, hkv=4, hd=128,
             tokens=1, layers=1, k_scale=0.5, v_scale=0.0625),
        # three drafted tokens checked at once over long ragged contexts, 72B shape
        dict(name="dec_verify8", op="dec", batch=8, lo=1024, hi=32768, hq=64, hkv=8, hd=128,
             tokens=3, layers=1, k_scale=0.5, v_scale=0.0625),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, hd = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (64, 8, 128), (16, 1, 64),
                              (8, 8, 128), (40, 8, 128)])
    op = rng.choice(["tables", "nra", "kv4", "dec", "dec"])
    if op == "tables":
        batch = _log(rng, 1, 1024)
        prompts = rng.randint(0, max(1, batch // 8))
        max_ctx = _log(rng, 64, 16384)
        max_new = _log(rng, 2, 4096)
        return dict(op=op, batch=batch, slots=batch + rng.randint(0, batch) + 8, max_ctx=max_ctx,
                    prompts=prompts, max_new=max_new,
                    stride=(max_ctx + max_new) // PAGE + rng.randint(2, 9),
                    done=rng.randint(0, 8), spare=_log(rng, 16, 20000))
    if op == "nra":
        return dict(op=op, rows=_log(rng, 1, 33000000 // ((hq + 2 * hkv) * hd)), hq=hq, hkv=hkv, hd=hd,
                    bias=rng.random() < 0.5, norm=rng.random() < 0.8, layers=rng.randint(1, 2),
                    pad=8 * rng.randint(0, 3), idle=rng.randint(0, 5))
    scales = dict(k_scale=rng.choice([0.5, 1.0, 2.0]), v_scale=rng.choice([0.0625, 0.25, 1.0]))
    if op == "kv4":
        batch = rng.randint(1, 6)
        return dict(op=op, batch=batch, start=rng.choice([0, rng.randint(1, 900)]),
                    tokens=_log(rng, 1, 14000000 // (batch * (hq + 2 * hkv) * hd)), hq=hq, hkv=hkv, hd=hd,
                    bias=rng.random() < 0.5, norm=rng.random() < 0.7, layers=rng.randint(1, 2),
                    **scales)
    batch = _log(rng, 1, 128)
    tokens = rng.choice([1, 1, 1, 2, 4])
    hi = _log(rng, 1, min(32768, 2 ** 20 // (batch * hkv), 3 * 10 ** 9 // (batch * tokens * hq * hd)))
    return dict(op=op, batch=batch, lo=rng.choice([hi, max(1, hi // 8)]), hi=hi, hq=hq, hkv=hkv,
                hd=hd, tokens=tokens, layers=rng.randint(1, 2), **scales)


# ------------------------------------------------------------------ inputs --

def _ceil(a, b):
    return (a + b - 1) // b


def _page_bytes(hd):
    """Bytes of one page's K (or V): 16 rows of hd/2 code bytes, 16 rows of hd/16 scales."""
    return PAGE * hd // 2 + PAGE * hd // 16


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


def _rope_tables(hd):
    inv = 1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = torch.arange(ROPE_ROWS, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float(), ang.sin().float()


def _assign(pages, stride, num_blocks, gen):
    """[N, stride] tables of distinct shuffled pages (-1 padded) and the pages left over."""
    perm = torch.randperm(num_blocks, generator=gen, device="cuda").int()
    start = pages.cumsum(0) - pages
    j = torch.arange(stride, device="cuda")
    at = (start[:, None] + j[None, :]).clamp(max=num_blocks - 1)
    tables = torch.where(j[None, :] < pages[:, None], perm[at], torch.tensor(-1, device="cuda").int())
    return tables.int().contiguous(), perm[int(pages.sum()):]


def _prepare_tables(c, gen):
    b, n = c["batch"], c["slots"]
    order = torch.randperm(n, generator=gen, device="cuda").int()
    slots, done = order[:b].contiguous(), order[b:b + min(c["done"], n - b)].contiguous()
    ctx = torch.randint(0, c["max_ctx"] + 1, (n,), generator=gen, device="cuda").int()
    new = torch.ones(b, dtype=torch.int32, device="cuda")
    if c["prompts"]:
        at = torch.randperm(b, generator=gen, device="cuda")[:c["prompts"]]
        new[at] = torch.randint(0, c["max_new"] + 1, (c["prompts"],), generator=gen,
                                device="cuda").int()
        ctx[slots[at[::2]].long()] = 0  # half of the prompts are new, the others continue
    pages = _ceil(ctx, PAGE).long()
    # a pool of the expected size and six deviations; `spare` of its pages are free
    num_blocks = int(n * (c["max_ctx"] / (2 * PAGE) + 1)
                     + 6 * math.sqrt(n / 12) * c["max_ctx"] / PAGE) + c["spare"]
    tables, left = _assign(pages, c["stride"], num_blocks, gen)
    free = torch.full((num_blocks,), -1, dtype=torch.int32, device="cuda")
    free[:c["spare"]] = left[:c["spare"]]
    cap = b + c["prompts"] * c["max_new"]  # rows of the step's buffers

    def ints(*shape):
        return torch.zeros(*shape, dtype=torch.int32, device="cuda")
    return dict(tables=tables, slots=slots, ctx=ctx[slots.long()].contiguous(), new=new,
                done=done, done_ctx=ctx[done.long()].contiguous(), free=free,
                free_count=torch.tensor([c["spare"]], dtype=torch.int32, device="cuda"),
                num_blocks=num_blocks, cap=cap, mid=ints(1), count=ints(1),
                step=ints(b, c["stride"]), positions=ints(cap), slot_map=ints(cap),
                row_starts=ints(b + 1), ctx_out=ints(b))


def _prepare_rows(c, rows, gen):
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    row = (hq + 2 * hkv) * hd + c.get("pad", 0)
    qkv = _normal(gen, rows, row)
    # a few channels of K much larger than the rest, as trained models have
    big = torch.randint(0, hd, (3,), generator=gen, device="cuda")
    k = qkv[:, hq * hd:(hq + hkv) * hd].view(rows, hkv, hd)
    k[:, :, big] *= 8.0
    qkv[:, (hq + hkv) * hd:] *= 0.3

    def vec(n, mean, std):
        return (mean + _normal(gen, n, scale=std)).bfloat16()
    cos, sin = _rope_tables(hd)
    return dict(qkv=qkv.bfloat16(), cos=cos, sin=sin,
                q_bias=vec(hq * hd, 0, 0.5) if c["bias"] else None,
                k_bias=vec(hkv * hd, 0, 2.0) if c["bias"] else None,
                v_bias=vec(hkv * hd, 0, 0.05) if c["bias"] else None,
                q_norm=vec(hd, 1, 0.1) if c["norm"] else None,
                k_norm=vec(hd, 1, 0.1) if c["norm"] else None,
                q_out=torch.zeros(rows, hq * hd, dtype=torch.bfloat16, device="cuda"))


def _prepare_nra(c, gen):
    rows = c["rows"]
    s = _prepare_rows(c, rows, gen)
    pages = _ceil(rows, PAGE) + 3  # the last page belongs to no sequence
    order = torch.randperm((pages - 1) * PAGE, generator=gen, device="cuda")[:rows].int()
    pos = torch.randint(0, ROPE_ROWS, (rows,), generator=gen, device="cuda").int()
    if c["idle"]:
        off = torch.randperm(rows, generator=gen, device="cuda")[:min(c["idle"], rows)]
        order[off] = -1
        pos[off[::2]] = -1  # half of them are padding, the others only want their q
    shape = (pages, c["layers"], c["hkv"], PAGE, c["hd"])
    s.update(positions=pos, slot_map=order, num_blocks=pages,
             k_pool=_normal(gen, *shape).bfloat16(), v_pool=_normal(gen, *shape).bfloat16())
    return s


def _plain_quantise(x, scale):
    """x [..., 16k] fp32 -> (codes 0..15, uint8 e4m3 scales): blocks of 16, the scale
    e4m3(amax / (6 * scale)), the value x / (its scale) to the nearest of
    0 .5 1 1.5 2 3 4 6 (ties to the even code). A block with an inf or NaN gets a NaN scale."""
    b = x.reshape(*x.shape[:-1], -1, 16)
    amax = b.abs().amax(-1)
    s8 = (amax / torch.full_like(amax, 6.0 * scale)).clamp(max=448.0)
    s8 = torch.where(amax.isfinite(), s8, float("nan")).to(torch.float8_e4m3fn)
    s = (s8.float() * scale)[..., None]
    y = torch.where(s > 0, b / s, torch.copysign(torch.zeros_like(b), b))
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
            + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    code = code + 8 * y.signbit().int()
    return code.reshape(x.shape), s8.view(torch.uint8)


def _grid(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0,
                         -3.0, -4.0, -6.0], device=device)


def _pack(x, scale):
    """fp32 [..., 16 tokens, hd] -> uint8 [..., page bytes]."""
    code, s8 = _plain_quantise(x, scale)
    code = code.to(torch.uint8)
    data = code[..., 0::2] | (code[..., 1::2] << 4)
    return torch.cat([data.flatten(-2), s8.flatten(-2)], -1)


def _plain_values(pages, hd, scale):
    """uint8 [..., page bytes] -> fp32 [..., 16 tokens, hd]."""
    data, s8 = pages.split([PAGE * hd // 2, PAGE * hd // 16], -1)
    code = torch.stack([data & 15, data >> 4], -1).reshape(*data.shape[:-1], PAGE, hd // 16, 16)
    s = s8.contiguous().view(torch.float8_e4m3fn).float().reshape(*s8.shape[:-1], PAGE, hd // 16, 1)
    return (_grid(pages.device)[code.int()] * (s * scale)).reshape(*data.shape[:-1], PAGE, hd)


def _filled_pool(c, num_blocks, gen):
    """A pool [blocks, layers, hkv, 2, page bytes] of quantised K and V."""
    hkv, hd = c["hkv"], c["hd"]
    pool = torch.empty(num_blocks, c["layers"], hkv, 2, _page_bytes(hd), dtype=torch.uint8,
                       device="cuda")
    gain = torch.ones(hd, device="cuda")
    gain[torch.randint(0, hd, (3,), generator=gen, device="cuda")] = 6.0
    step = max(1, (1 << 25) // (c["layers"] * hkv * PAGE * hd))
    for at in range(0, num_blocks, step):
        n = min(step, num_blocks - at)
        shape = (n, c["layers"], hkv, PAGE, hd)
        pool[at:at + n, :, :, 0] = _pack(_normal(gen, *shape) * gain, c["k_scale"])
        pool[at:at + n, :, :, 1] = _pack(_normal(gen, *shape, scale=0.3), c["v_scale"])
    return pool


def _spoil(pool, tables, lens, hd):
    """Slots past each sequence's last token hold whatever the page held before: NaN scales here."""
    part = torch.nonzero(lens % PAGE)[:, 0]
    if part.numel():
        page = tables[part, (lens[part] // PAGE).long()].long()
        at = torch.arange(PAGE, device="cuda")[None, :] >= (lens[part] % PAGE)[:, None]
        view = pool[..., PAGE * hd // 2:].reshape(*pool.shape[:-1], PAGE, hd // 16)
        old = view[page]
        old.masked_fill_(at[:, None, None, None, :, None], 0x7f)
        pool[page, ..., PAGE * hd // 2:] = old.flatten(-2)


def _prepare_kv4(c, gen):
    b, t, start = c["batch"], c["tokens"], c["start"]
    s = _prepare_rows(c, b * t, gen)
    per = _ceil(start + t, PAGE)
    num_blocks = b * per + 2
    tables, _ = _assign(torch.full((b,), per, device="cuda"), per, num_blocks - 1, gen)
    pool = _filled_pool(c, num_blocks, gen)
    lens = torch.full((b,), start + t, dtype=torch.int32, device="cuda")
    pos = torch.arange(start, start + t, device="cuda").int().repeat(b)
    seq = torch.arange(b, device="cuda").repeat_interleave(t)
    slot = tables[seq, (pos // PAGE).long()] * PAGE + pos % PAGE
    _spoil(pool, tables, lens, c["hd"])
    shape = (b * per, 1, c["hkv"], PAGE, c["hd"])
    s.update(positions=pos, slot_map=slot.int().contiguous(), tables=tables, lens=lens, pool=pool,
             num_blocks=num_blocks, per=per,
             k16=torch.zeros(shape, dtype=torch.bfloat16, device="cuda"),
             v16=torch.zeros(shape, dtype=torch.bfloat16, device="cuda"))
    return s


def _prepare_dec(c, gen):
    b, hq, hd, t = c["batch"], c["hq"], c["hd"], c["tokens"]
    lens = torch.randint(c["lo"], c["hi"] + 1, (b,), generator=gen, device="cuda").int()
    lens[0] = c["hi"]
    if b > 8:
        lens[b // 2] = 0  # a slot without a sequence
    pages = _ceil(lens, PAGE).long()
    num_blocks = int(pages.sum()) + 2
    tables, _ = _assign(pages, int(pages.max()) + 1, num_blocks, gen)
    pool = _filled_pool(c, num_blocks, gen)
    _spoil(pool, tables, lens, hd)
    return dict(q=_normal(gen, b * t, hq * hd, scale=1.5).bfloat16(), lens=lens, tables=tables,
                pool=pool, num_blocks=num_blocks, longest=c["hi"],
                out=torch.zeros(b * t, hq * hd, dtype=torch.bfloat16, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(tables=_prepare_tables, nra=_prepare_nra, kv4=_prepare_kv4,
                 dec=_prepare_dec)[case["op"]](case, gen)
    state["case"] = case
    return state


# ------------------------------------------------------------- plain forms --

def _plain_tables(s):
    c, tables, dev = s["case"], s["tables"], s["tables"].device
    stride, nb = tables.shape[1], s["num_blocks"]
    j = torch.arange(stride, device=dev)
    # release: the finished requests' pages onto the stack, each one's last page first
    np_ = _ceil(s["done_ctx"], PAGE).long()
    first = s["free_count"].long() + np_.cumsum(0) - np_
    at = torch.where(j[None, :] < np_[:, None], first[:, None] + np_[:, None] - 1 - j[None, :], nb)
    stack = torch.cat([s["free"], s["free"][:1]])
    stack.scatter_(0, at.flatten(), tables[s["done"].long()].flatten())
    s["free"].copy_(stack[:nb])
    count = s["free_count"] + np_.sum().int()
    # the step: pages from the top of the stack in request order, all or nothing per request
    ctx, new = s["ctx"].long(), s["new"].long()
    have, want = _ceil(ctx, PAGE), _ceil(ctx + new, PAGE)
    need = want - have
    upto = need.cumsum(0)
    served = (need == 0) | (upto <= count)
    take = torch.where(served, need, 0)
    before = (upto - need)[:, None] + (j[None, :] - have[:, None])
    fresh = (j[None, :] >= have[:, None]) & (j[None, :] < want[:, None]) & served[:, None]
    rows = tables[s["slots"].long()]
    rows = torch.where(fresh, s["free"][(count - 1 - before).clamp(0, nb - 1)], rows)
    tables[s["slots"].long()] = rows
    ctx_out = torch.where(served, ctx + new, ctx)
    step = torch.where(j[None, :] < _ceil(ctx_out, PAGE)[:, None], rows, -1)
    ends = new.cumsum(0)
    starts = torch.cat([ends[:1] * 0, ends])
    tok = torch.arange(s["cap"], device=dev)
    req = torch.searchsorted(ends, tok, right=True).clamp(max=c["batch"] - 1)
    live = tok < ends[-1]
    pos = ctx[req] + tok - starts[req]
    page = rows[req, (pos // PAGE).clamp(0, stride - 1)].long()
    slot = torch.where(live & served[req], page * PAGE + pos % PAGE, -1)
    return dict(tables=tables, step=step.int(), positions=torch.where(live, pos, -1).int(),
                slot_map=slot.int(), row_starts=starts.int(), ctx_out=ctx_out.int(),
                free=s["free"], count=(count - take.sum()).int())


def _plain_norm(x, w):
    """RMS norm over the last axis; the squares are added pairwise, halves first."""
    hd = x.shape[-1]
    q = (x * x).unflatten(-1, (2, hd // 16, 8)).sum(-3)
    q = q.unflatten(-1, (2, 4)).sum(-2).unflatten(-1, (2, 2)).sum(-2).sum(-1)
    q = q.unflatten(-1, (2, -1)).sum(-2).unflatten(-1, (2, -1)).sum(-2).sum(-1, keepdim=True)
    return x * (q * (1.0 / hd) + EPS).sqrt().reciprocal() * w.float()


def _plain_rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_rows(s):
    """q, k (normed and rotated) and v of every row, fp32 [rows, heads, hd]."""
    c = s["case"]
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    x = s["qkv"][:, :(hq + 2 * hkv) * hd].float()
    if c["bias"]:
        x = x + torch.cat([s["q_bias"], s["k_bias"], s["v_bias"]]).float()
    q, k, v = x.unflatten(-1, (-1, hd)).split([hq, hkv, hkv], 1)
    if c["norm"]:
        q, k = _plain_norm(q, s["q_norm"]), _plain_norm(k, s["k_norm"])
    at = s["positions"].long().clamp(min=0)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    return _plain_rotate(q, cos, sin), _plain_rotate(k, cos, sin), v


def _plain_nra(s):
    c = s["case"]
    q, k, v = _plain_rows(s)
    live = (s["positions"] >= 0)[:, None]
    s["q_out"].copy_(torch.where(live, q.flatten(1).bfloat16(), s["q_out"]))
    # rows without a slot go to the page that no sequence has, which is then put back
    slot = torch.where(s["slot_map"] < 0, (s["num_blocks"] - 1) * PAGE, s["slot_map"]).long()
    layer = c["layers"] - 1
    for pool, rows in ((s["k_pool"], k), (s["v_pool"], v)):
        kept = pool[-1].clone()
        pool[slot // PAGE, layer, :, slot % PAGE] = rows.bfloat16()
        pool[-1] = kept
    return dict(q=s["q_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _plain_kv4(s):
    c = s["case"]
    layer, hd, b, per = c["layers"] - 1, c["hd"], c["batch"], s["per"]
    q, k, v = _plain_rows(s)
    s["q_out"].copy_(q.flatten(1).bfloat16())
    seq = torch.arange(b, device=q.device).repeat_interleave(c["tokens"])
    page, row = seq * per + s["positions"].long() // PAGE, s["positions"].long() % PAGE
    past = torch.arange(per * PAGE, device=q.device)[None, :] >= s["lens"][:, None]
    outs = []
    for i, (new, scale, out) in enumerate(((k, c["k_scale"], s["k16"]), (v, c["v_scale"], s["v16"]))):
        old = s["pool"][s["tables"].long().flatten(), layer, :, i]
        vals = _plain_values(old, hd, scale)
        code, s8 = _plain_quantise(new, scale)
        step = s8.view(torch.float8_e4m3fn).float() * scale
        vals[page, :, row] = _grid(q.device)[code.int()] * step.repeat_interleave(16, -1)
        vals.masked_fill_(past.reshape(b * per, 1, PAGE, 1), 0.0)
        out[:, 0] = vals.bfloat16()
        outs.append(out)
    return dict(q=s["q_out"], k=outs[0], v=outs[1])


def _plain_dec(s):
    c = s["case"]
    b, t, hkv, hd = c["batch"], c["tokens"], c["hkv"], c["hd"]
    group, layer = c["hq"] // hkv, c["layers"] - 1
    pages = s["pool"][s["tables"].long().clamp(min=0), layer]  # [b, pages, hkv, 2, bytes]
    n = pages.shape[1] * PAGE
    at = torch.arange(n, device=pages.device)
    k = _plain_values(pages[:, :, :, 0], hd, c["k_scale"]).transpose(1, 2).reshape(b, hkv, n, hd)
    v = _plain_values(pages[:, :, :, 1], hd, c["v_scale"]).transpose(1, 2).reshape(b, hkv, n, hd)
    held = (at[None, :] < s["lens"][:, None])[:, None, :, None]
    v = torch.where(held, v, 0.0)
    q = s["q"].float().reshape(b, t, hkv, group, hd).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * group, hd)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    # query i of t sees the tokens up to its own
    seen = s["lens"][:, None] - (t - 1 - torch.arange(t, device=pages.device))[None, :]
    seen = seen.repeat_interleave(group, 1)[:, None, :, None]
    x = torch.where(at < seen, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0.0)
    o = o.reshape(b, hkv, t, group, hd).permute(0, 2, 1, 3, 4).reshape(b * t, c["hq"] * hd)
    s["out"].copy_(o.bfloat16())
    return s["out"]


# ------------------------------------------------------- the framework's own --

def _lucciola():
    path = os.path.abspath("lucciola-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import lucciola
    return lucciola


def _own_tables(s):
    L = _lucciola()
    if "ws" not in s:
        s["ws"] = L.alloc_step_workspace()
    count = s["free_count"]
    if s["done"].numel():
        L.step_release(s["free"], count, s["tables"], s["done_ctx"], slots=s["done"],
                       free_count_out=s["mid"], workspace=s["ws"])
        count = s["mid"]
    L.step_tables(s["tables"], s["ctx"], s["new"], s["free"], count, s["positions"],
                  s["slot_map"], row_starts=s["row_starts"], context_out=s["ctx_out"],
                  free_count_out=s["count"], slots=s["slots"], step_tables=s["step"],
                  workspace=s["ws"])
    return dict(tables=s["tables"], step=s["step"], positions=s["positions"],
                slot_map=s["slot_map"], row_starts=s["row_starts"], ctx_out=s["ctx_out"],
                free=s["free"], count=s["count"])


def _own_nra(s):
    L, c = _lucciola(), s["case"]
    L.qk_norm_rope_append(s["q_out"], s["qkv"], s["positions"], s["slot_map"], s["cos"], s["sin"],
                          s["k_pool"], s["v_pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                          c["hq"], c["hkv"], c["hd"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                          eps=EPS, q_bias=s["q_bias"], k_bias=s["k_bias"], v_bias=s["v_bias"])
    return dict(q=s["q_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _own_kv4(s):
    L, c = _lucciola(), s["case"]
    L.qk_norm_rope_append_kv4(s["q_out"], s["qkv"], s["positions"], s["slot_map"], s["cos"],
                              s["sin"], s["pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                              c["hq"], c["hkv"], c["hd"], k_scale=c["k_scale"],
                              v_scale=c["v_scale"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                              eps=EPS, q_bias=s["q_bias"], k_bias=s["k_bias"], v_bias=s["v_bias"])
    L.unpack_kv4(s["k16"], s["v16"], s["pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                 c["hkv"], c["hd"], s["tables"], s["lens"], c["start"] + c["tokens"],
                 k_scale=c["k_scale"], v_scale=c["v_scale"])
    return dict(q=s["q_out"], k=s["k16"], v=s["v16"])


def _own_dec(s):
    L, c = _lucciola(), s["case"]
    if "ws" not in s:
        s["ws"] = L.alloc_decode_kv4_workspace(c["batch"], c["hq"], c["hkv"], c["hd"],
                                               tokens_per_seq=c["tokens"])
    L.paged_decode_kv4(s["out"], s["q"], s["pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                       c["hq"], c["hkv"], c["hd"], s["tables"], s["lens"],
                       max_context_len=s["longest"], tokens_per_seq=c["tokens"],
                       k_scale=c["k_scale"], v_scale=c["v_scale"], workspace=s["ws"])
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(tables=_own_tables, nra=_own_nra, kv4=_own_kv4, dec=_own_dec)[op](state)
    return dict(tables=_plain_tables, nra=_plain_nra, kv4=_plain_kv4, dec=_plain_dec)[op](state)


# -------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["op"] == "tables":
        # expected sizes of the seeded lengths
        mean_pages = c["max_ctx"] / 2 / PAGE
        tokens = c["batch"] - c["prompts"] + c["prompts"] * c["max_new"] / 2
        fresh = tokens / PAGE
        return dict(bytes=4.0 * (c["batch"] * (3 + 2)  # lengths, slots; starts and new lengths
                                 + 2 * (c["batch"] + c["prompts"] * c["max_new"])  # positions, slots
                                 + 2 * fresh   # stack -> tables
                                 + c["batch"] * (mean_pages + c["stride"])  # rows read, step rows
                                 + 2 * c["done"] * mean_pages), flops=0)
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    if c["op"] == "nra":
        rows = c["rows"]
        return dict(bytes=rows * (2 * 2 * (hq + 2 * hkv) * hd + 2 * 4 * hd // 2 + 8),
                    flops=rows * ((hq + hkv) * hd * 8 + hkv * hd))
    code = hd / 2 + hd / 16  # bytes of one token's K (or V) of one head
    if c["op"] == "kv4":
        rows, seen = c["batch"] * c["tokens"], c["batch"] * (c["start"] + c["tokens"])
        return dict(bytes=rows * (2 * (2 * hq + 2 * hkv) * hd + 2 * 4 * hd // 2 + 8
                                  + 2 * hkv * code)
                    + seen * 2 * hkv * (code + 2 * hd),
                    flops=rows * ((hq + hkv) * hd * 8 + 2 * hkv * hd * 4) + seen * 2 * hkv * hd)
    seen = c["batch"] * (c["lo"] + c["hi"]) / 2
    return dict(bytes=seen * (2 * hkv * code + 4 / PAGE) + 2 * 2 * c["batch"] * c["tokens"] * hq * hd,
                flops=4 * seen * c["tokens"] * hq * hd)


# ------------------------------------------------------------------- exact --

_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_e4m3(x):
    """Nearest e4m3 value (ties to even) of non-negative float64, at most 448."""
    x = np.minimum(x, 448.0)
    e = np.floor(np.log2(np.maximum(x, 2.0 ** -9)))
    step = 2.0 ** (np.maximum(e, -6.0) - 3.0)
    return np.rint(x / step) * step


def _exact_round4(x, scale):
    """The value that each element of float64 x [..., hd] stands for once it is held in 4 bits."""
    b = x.reshape(x.shape[:-1] + (-1, 16))
    s = _exact_e4m3(np.abs(b).max(-1, keepdims=True) / (6.0 * scale)) * scale
    y = np.abs(b) / np.where(s > 0, s, 1.0)
    out = np.zeros_like(y)
    for i in range(7):
        mid = (_MAGNITUDES[i] + _MAGNITUDES[i + 1]) / 2
        over = (y > mid) if i % 2 == 0 else (y >= mid)
        out = np.where(over, _MAGNITUDES[i + 1], out)
    return (np.sign(b) * out * s).reshape(x.shape)


def _np(t):
    if t is None:
        return None
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _exact_rows(s):
    c = s["case"]
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    x = _np(s["qkv"])
    parts = []
    at = 0
    pos = np.maximum(_np(s["positions"]), 0)
    cos, sin = _np(s["cos"])[pos][:, None, :], _np(s["sin"])[pos][:, None, :]
    for name, heads in (("q", hq), ("k", hkv), ("v", hkv)):
        y = x[:, at:at + heads * hd]
        at += heads * hd
        if c["bias"]:
            y = y + _np(s[name + "_bias"])
        y = y.reshape(len(y), heads, hd)
        if name != "v":
            if c["norm"]:
                y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + EPS) * _np(s[name + "_norm"])
            lo, hi = y[..., :hd // 2], y[..., hd // 2:]
            y = np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], -1)
        parts.append(y)
    return parts


def _exact_unpack(pages, hd, scale):
    """float64 [..., 16, hd] of uint8 pages [..., bytes] (a NaN scale gives NaN)."""
    half = PAGE * hd // 2
    data = pages[..., :half].reshape(pages.shape[:-1] + (PAGE, hd // 2))
    s = pages[..., half:].reshape(pages.shape[:-1] + (PAGE, hd // 16)).astype(np.int64)
    e, m = (s >> 3) & 15, s & 7
    val = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    val = np.where((s & 127) == 127, np.nan, val) * scale
    table = np.array(_MAGNITUDES + tuple(-x for x in _MAGNITUDES))
    out = np.empty(data.shape[:-1] + (hd,))
    out[..., 0::2] = table[data & 15]
    out[..., 1::2] = table[data >> 4]
    return out * np.repeat(val, 16, -1)


def _exact_tables(s):
    tables, free = _np(s["tables"]).copy(), _np(s["free"]).copy()
    count = int(s["free_count"].item())
    for slot, n in zip(_np(s["done"]), _np(s["done_ctx"])):
        for page in tables[slot, :_ceil(int(n), PAGE)][::-1]:
            free[count] = page
            count += 1
    slots, ctx, new = _np(s["slots"]), _np(s["ctx"]), _np(s["new"])
    step = np.full((len(slots), tables.shape[1]), -1)
    pos, slot_map = np.full(s["cap"], -1), np.full(s["cap"], -1)
    starts, ctx_out = [0], []
    wanted, avail = 0, count
    for b, (slot, n, m) in enumerate(zip(slots, ctx, new)):
        have, want = _ceil(int(n), PAGE), _ceil(int(n + m), PAGE)
        wanted += want - have
        served = want == have or wanted <= avail
        if served and want > have:
            for j in range(have, want):
                count -= 1
                tables[slot, j] = free[count]
        ctx_out.append(n + m if served else n)
        k = _ceil(int(ctx_out[-1]), PAGE)
        step[b, :k] = tables[slot, :k]
        at = np.arange(n, n + m)
        pos[starts[-1]:starts[-1] + m] = at
        if served:
            slot_map[starts[-1]:starts[-1] + m] = tables[slot, at // PAGE] * PAGE + at % PAGE
        starts.append(starts[-1] + m)
    return dict(tables=tables, step=step, positions=pos, slot_map=slot_map,
                row_starts=np.array(starts), ctx_out=np.array(ctx_out), free=free,
                count=np.array([count]))


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "tables":
        return _exact_tables(s)
    hkv, hd, layer = c["hkv"], c["hd"], c["layers"] - 1
    if c["op"] in ("nra", "kv4"):
        q, k, v = _exact_rows(s)
        q = q.reshape(len(q), -1)
    if c["op"] == "nra":
        slot, pos = _np(s["slot_map"]), _np(s["positions"])
        q[pos < 0] = 0.0
        pools = [_np(s["k_pool"]), _np(s["v_pool"])]
        on = slot >= 0
        for pool, rows in zip(pools, (k, v)):
            pool[slot[on] // PAGE, layer, :, slot[on] % PAGE] = rows[on]
        return dict(q=q, k_pool=pools[0], v_pool=pools[1])
    if c["op"] == "kv4":
        b, per, n = c["batch"], s["per"], c["start"] + c["tokens"]
        tables, packed = _np(s["tables"]), _np(s["pool"])
        out = dict(q=q)
        for i, (name, rows, scale) in enumerate((("k", k, c["k_scale"]), ("v", v, c["v_scale"]))):
            vals = _exact_unpack(packed[tables.reshape(-1), layer, :, i], hd, scale)
            vals = vals.reshape(b, per, hkv, PAGE, hd).transpose(0, 1, 3, 2, 4)
            vals = vals.reshape(b, per * PAGE, hkv, hd)
            vals[:, c["start"]:n] = _exact_round4(rows, scale).reshape(b, c["tokens"], hkv, hd)
            vals[:, n:] = 0.0
            out[name] = vals.reshape(b, per, PAGE, hkv, hd).transpose(0, 1, 3, 2, 4).reshape(
                b * per, 1, hkv, PAGE, hd)
        return out
    t, group = c["tokens"], c["hq"] // hkv
    lens, tables = _np(s["lens"]), s["tables"].long()
    q = s["q"].double().view(c["batch"], t, hkv, group, hd)
    out = torch.zeros_like(q)
    table = torch.tensor(_MAGNITUDES + tuple(-x for x in _MAGNITUDES), dtype=torch.float64,
                         device="cuda")
    half = PAGE * hd // 2
    for b in range(c["batch"]):
        n = int(lens[b])
        if n == 0:
            continue
        pages = s["pool"][tables[b, :_ceil(n, PAGE)], layer]
        kv = []
        for i, scale in enumerate((c["k_scale"], c["v_scale"])):
            data = pages[:, :, i, :half].reshape(-1, hkv, PAGE, hd // 2)
            step = pages[:, :, i, half:].contiguous().view(torch.float8_e4m3fn).double()
            step = step.reshape(-1, hkv, PAGE, hd // 16).repeat_interleave(16, -1) * scale
            val = torch.empty(*data.shape[:-1], hd, dtype=torch.float64, device="cuda")
            val[..., 0::2] = table[(data & 15).int()]
            val[..., 1::2] = table[(data >> 4).int()]
            kv.append((val * step).transpose(0, 1).reshape(hkv, -1, hd)[:, :n])
        for i in range(t):
            m = n - (t - 1 - i)
            if m <= 0:
                continue
            x = torch.einsum("hgd,hnd->hgn", q[b, i], kv[0][:, :m]) / math.sqrt(hd)
            out[b, i] = torch.softmax(x, -1) @ kv[1][:, :m]
    return out.reshape(c["batch"] * t, -1).cpu().numpy()
