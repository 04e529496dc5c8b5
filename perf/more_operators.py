"""Workloads of a serving step over an 8-bit cache: norm + RoPE + append with a scale per page
and head, the cache's round trip, attention over it, and the choice of the next tokens.

run() computes each operator in a plain form (elementary torch operations in fp32, the
choice of tokens in 64 bits) or, where `own` is set, through lucciola's entry points. Shapes
are those of the Qwen2 family (0.5B: 14/2 heads of 64; 1.5B: 12/2 of 128; 7B: 28/4 of 128;
72B: 64/8 of 128; 151936 logits).
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
E_MIN, E_MAX = -40, 40  # exponents of a page's scale
VOCAB = 151936


def listed():
    return [
        # --- kv8: a prompt appended to the 8-bit cache and its context read back for the
        # prefill attention
        # one short ragged prompt chunk after 77 cached tokens, biases: the smallest call
        dict(name="kv8_chunk", op="kv8", batch=1, start=77, tokens=179, hq=14, hkv=2, hd=64,
             bias=True, norm=False, layers=2, pad=8),
        # prompts of 2048 tokens, 7B shape
        dict(name="kv8_prompt8k", op="kv8", batch=4, start=0, tokens=2048, hq=28, hkv=4, hd=128,
             bias=False, norm=True, layers=1, pad=0),
        # --- step8: a decode step's cache work, the new tokens appended and attended over
        # one sequence, 1024 cached tokens: latency
        dict(name="step8_single1k", op="step8", batch=1, lo=1024, hi=1024, hq=14, hkv=2, hd=64,
             tokens=1, bias=True, norm=False, layers=2, pad=0),
        # 64 ragged sequences of 256 .. 4096 tokens, one slot of the batch empty
        dict(name="step8_ragged64", op="step8", batch=64, lo=256, hi=4096, hq=14, hkv=2, hd=64,
             tokens=1, bias=False, norm=True, layers=1, pad=0),
        # three drafted tokens checked at once over long ragged contexts, 72B shape
        dict(name="step8_verify8", op="step8", batch=8, lo=1024, hi=32000, hq=64, hkv=8, hd=128,
             tokens=3, bias=False, norm=True, layers=1, pad=8),
        # --- dec8: attention alone over the 8-bit cache
        # one short context: the smallest call
        dict(name="dec8_short", op="dec8", batch=1, lo=203, hi=203, hq=12, hkv=2, hd=128, tokens=1,
             layers=1),
        # 32 sequences of 8192 tokens, 7B shape
        dict(name="dec8_batch32", op="dec8", batch=32, lo=8192, hi=8192, hq=28, hkv=4, hd=128,
             tokens=1, layers=1),
        # two documents of 131072 tokens, 7B shape
        dict(name="dec8_long", op="dec8", batch=2, lo=131072, hi=131072, hq=28, hkv=4, hd=128,
             tokens=1, layers=1),
        # --- sample: the next tokens from the logits
        # one sequence, as a chat decodes
        dict(name="sample_one", op="sample", batch=1, vocab=VOCAB, pad=0),
        # a small odd vocabulary with rows that are not aligned
        dict(name="sample_odd7", op="sample", batch=7, vocab=32003, pad=5),
        # a decode batch whose requests have parameters of their own
        dict(name="sample_batch64", op="sample", batch=64, vocab=VOCAB, pad=0),
        # a large engine's step
        dict(name="sample_batch256", op="sample", batch=256, vocab=VOCAB, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, hd = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (64, 8, 128), (16, 1, 64),
                              (8, 8, 128), (40, 8, 128)])
    op = rng.choice(["kv8", "step8", "step8", "dec8", "dec8", "sample", "sample"])
    if op == "sample":
        vocab = rng.choice([VOCAB, _log(rng, 100, VOCAB)])
        return dict(op=op, batch=_log(rng, 1, 256), vocab=vocab, pad=rng.choice([0, 0, 8, 3]))
    rows = dict(bias=rng.random() < 0.5, norm=rng.random() < 0.7, pad=8 * rng.randint(0, 3))
    shape = dict(hq=hq, hkv=hkv, hd=hd, layers=rng.randint(1, 2))
    if op == "kv8":
        batch = rng.randint(1, 6)
        return dict(op=op, batch=batch, start=rng.choice([0, rng.randint(1, 900)]),
                    tokens=_log(rng, 1, 14000000 // (batch * (hq + 2 * hkv) * hd)), **shape, **rows)
    batch = _log(rng, 1, 128)
    tokens = rng.choice([1, 1, 1, 2, 4])
    most = min(2 ** 20 // (batch * hkv), 3 * 10 ** 9 // (batch * tokens * hq * hd))
    hi = _log(rng, tokens, min(most, 32000 if op == "step8" else 131072))
    case = dict(op=op, batch=batch, lo=rng.choice([hi, max(tokens, hi // 8)]), hi=hi, tokens=tokens,
                **shape)
    return dict(case, **rows) if op == "step8" else case


# ------------------------------------------------------------------ inputs --

def _ceil(a, b):
    return (a + b - 1) // b


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


def _rope_tables(hd):
    inv = 1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = torch.arange(ROPE_ROWS, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float(), ang.sin().float()


def _assign(pages, stride, num_blocks, gen):
    """[N, stride] tables of distinct shuffled pages, -1 padded."""
    perm = torch.randperm(num_blocks, generator=gen, device="cuda").int()
    start = pages.cumsum(0) - pages
    j = torch.arange(stride, device="cuda")
    at = (start[:, None] + j[None, :]).clamp(max=num_blocks - 1)
    tables = torch.where(j[None, :] < pages[:, None], perm[at], torch.tensor(-1, device="cuda").int())
    return tables.int().contiguous()


def _prepare_rows(c, rows, gen):
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    qkv = _normal(gen, rows, (hq + 2 * hkv) * hd + c["pad"])
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


def _page_bytes(hd):
    """Bytes of a page of one head: 16 rows of hd bytes for K, for V, two fp32 scales, 8 unused."""
    return 2 * PAGE * hd + 16


def _places(hd):
    """Byte of (token, dim) within a page's K or V: the 16-dim pieces of token t are at
    c ^ ((t * hd / 64) & (hd / 16 - 2)). [16, hd]"""
    t = torch.arange(PAGE, device="cuda")[:, None]
    d = torch.arange(hd, device="cuda")[None, :]
    return t * hd + ((d // 16) ^ ((t * (hd // 64)) & (hd // 16 - 2))) * 16 + d % 16


def _plain_exponent(amax):
    """Smallest e with amax <= 448 * 2^e, within the scales' range."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).int(), E_MIN)
    return e.clamp(E_MIN, E_MAX)


def _pack(x):
    """fp32 [..., 16 tokens, hd] -> (uint8 [..., 16 * hd] in page order, fp32 scales [...])."""
    scale = torch.exp2(_plain_exponent(x.abs().amax((-1, -2))).float())
    code = (x / scale[..., None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    out = torch.empty(*x.shape[:-2], PAGE * x.shape[-1], dtype=torch.uint8, device=x.device)
    out[..., _places(x.shape[-1]).flatten()] = code.view(torch.uint8).flatten(-2)
    return out, scale


def _scales(pages):
    """fp32 [..., 2] scales (K, V) of uint8 [..., page bytes]."""
    return pages[..., -16:-8].contiguous().view(torch.float32)


def _plain_values(pages, hd, i):
    """uint8 [..., page bytes] -> fp32 [..., 16 tokens, hd] of K (i = 0) or V (1)."""
    code = pages[..., i * PAGE * hd:(i + 1) * PAGE * hd][..., _places(hd)]
    return code.view(torch.float8_e4m3fn).float() * _scales(pages)[..., i, None, None]


def _filled_pool(c, num_blocks, gen):
    """A pool [blocks, layers, hkv, page bytes] of quantised K and V."""
    hkv, hd = c["hkv"], c["hd"]
    pool = torch.zeros(num_blocks, c["layers"], hkv, _page_bytes(hd), dtype=torch.uint8, device="cuda")
    gain = torch.ones(hd, device="cuda")
    gain[torch.randint(0, hd, (3,), generator=gen, device="cuda")] = 6.0
    step = max(1, (1 << 25) // (c["layers"] * hkv * PAGE * hd))
    for at in range(0, num_blocks, step):
        n = min(step, num_blocks - at)
        shape = (n, c["layers"], hkv, PAGE, hd)
        k, ks = _pack(_normal(gen, *shape) * gain)
        v, vs = _pack(_normal(gen, *shape, scale=0.3))
        part = pool[at:at + n]
        part[..., :PAGE * hd] = k
        part[..., PAGE * hd:2 * PAGE * hd] = v
        part[..., -16:-8] = torch.stack([ks, vs], -1).view(torch.uint8)
    return pool


def _spoil(pool, tables, lens, hd):
    """Tokens past each sequence's last hold whatever the page held before: NaN here."""
    part = torch.nonzero(lens % PAGE)[:, 0]
    if part.numel():
        page = tables[part, (lens[part] // PAGE).long()].long()
        at = torch.arange(PAGE, device="cuda")[None, :] >= (lens[part] % PAGE)[:, None]
        view = pool[..., :2 * PAGE * hd].unflatten(-1, (2, PAGE, hd))
        old = view[page]
        old.masked_fill_(at[:, None, None, None, :, None], 0x7f)
        pool[page, ..., :2 * PAGE * hd] = old.flatten(-3)


def _prepare_kv8(c, gen):
    b, t, start = c["batch"], c["tokens"], c["start"]
    s = _prepare_rows(c, b * t, gen)
    per = _ceil(start + t, PAGE)
    num_blocks = b * per + 2
    tables = _assign(torch.full((b,), per, device="cuda"), per, num_blocks - 1, gen)
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


def _prepare_dec8(c, gen):
    b, hq, hd, t = c["batch"], c["hq"], c["hd"], c["tokens"]
    lens = torch.randint(c["lo"], c["hi"] + 1, (b,), generator=gen, device="cuda").int()
    lens[0] = c["hi"]
    if b > 8:
        lens[b // 2] = 0  # a slot without a sequence
    pages = _ceil(lens, PAGE).long()
    num_blocks = int(pages.sum()) + 2
    tables = _assign(pages, int(pages.max()) + 1, num_blocks, gen)
    pool = _filled_pool(c, num_blocks, gen)
    _spoil(pool, tables, lens, hd)
    return dict(q=_normal(gen, b * t, hq * hd, scale=1.5).bfloat16(), lens=lens, tables=tables,
                pool=pool, num_blocks=num_blocks, longest=c["hi"],
                out=torch.zeros(b * t, hq * hd, dtype=torch.bfloat16, device="cuda"))


def _prepare_step8(c, gen):
    """The cache holds lens - tokens of each sequence; the step's rows are the last tokens."""
    b, t = c["batch"], c["tokens"]
    s = _prepare_dec8(c, gen)
    s.update(_prepare_rows(c, b * t, gen))
    lens = s["lens"]
    pos = (lens[:, None] - t + torch.arange(t, device="cuda").int()[None, :])
    page = s["tables"].gather(1, (pos // PAGE).clamp(min=0).long())
    live = lens[:, None] > 0
    s["positions"] = torch.where(live, pos, -1).int().flatten()
    s["slot_map"] = torch.where(live, page * PAGE + pos % PAGE, -1).int().flatten()
    return s


def _prepare_sample(c, gen):
    b, v = c["batch"], c["vocab"]
    wide = torch.zeros(b, v + c["pad"], dtype=torch.bfloat16, device="cuda")
    x = _normal(gen, b, v, scale=2.0) - 1.0
    # some tokens fit well, in a few rows one much better than all others
    fit = torch.rand(b, v, generator=gen, device="cuda") < 40.0 / v
    x += fit * (4.0 + 3.0 * _normal(gen, b, 1).abs() + 2.0 * _normal(gen, b, v).abs())
    # a token may be forbidden in every row, a sixteenth of a vocabulary in some rows
    x[:, torch.randint(0, v, (3,), generator=gen, device="cuda")] = float("-inf")
    barred = torch.rand(b, v, generator=gen, device="cuda") < 1.0 / 16
    x.masked_fill_(barred & (torch.rand(b, 1, generator=gen, device="cuda") < 0.25),
                   torch.finfo(torch.bfloat16).min)
    wide[:, :v] = x.bfloat16()

    def pick(*values):
        at = torch.randint(0, len(values), (b,), generator=gen, device="cuda")
        return torch.tensor(values, device="cuda")[at]
    return dict(logits=wide[:, :v], temperature=pick(0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.3),
                top_k=pick(0, 0, 20, 50, 1000).int(), top_p=pick(0.8, 0.9, 0.95, 1.0),
                min_p=pick(0.0, 0.0, 0.05, 0.1),
                rand=torch.rand(b, generator=gen, device="cuda"),
                out=torch.zeros(b, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(kv8=_prepare_kv8, step8=_prepare_step8, dec8=_prepare_dec8,
                 sample=_prepare_sample)[case["op"]](case, gen)
    state["case"] = case
    return state


# ------------------------------------------------------------- plain forms --

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


def _plain_append(vals, scales, rows, page, off):
    """vals [N, hkv, 16, hd] (what the pages hold) with rows [R, hkv, hd] written to token
    `off` of page `page`, held in 8 bits: a page written from its first token on gets the scale
    of its new rows, another one the larger of that and its old one."""
    n, hkv = vals.shape[:2]
    amax = torch.zeros(n, hkv, device=vals.device)
    amax.scatter_reduce_(0, page[:, None].expand(-1, hkv), rows.abs().amax(-1), "amax")
    fresh = torch.zeros(n, dtype=torch.bool, device=vals.device)
    fresh[page[off == 0]] = True
    touched = torch.zeros_like(fresh)
    touched[page] = True
    scale = torch.exp2(_plain_exponent(amax).float())
    scale = torch.where(fresh[:, None], scale, torch.maximum(scale, scales))
    scale = torch.where(touched[:, None], scale, scales)[..., None, None]
    vals = vals.clone()
    vals[page, :, off] = rows
    held = (vals / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float() * scale
    return torch.where(touched[:, None, None, None], held, vals)


def _plain_kv8(s):
    c = s["case"]
    layer, hd, b, per = c["layers"] - 1, c["hd"], c["batch"], s["per"]
    q, k, v = _plain_rows(s)
    s["q_out"].copy_(q.flatten(1).bfloat16())
    seq = torch.arange(b, device=q.device).repeat_interleave(c["tokens"])
    page, off = seq * per + s["positions"].long() // PAGE, s["positions"].long() % PAGE
    past = torch.arange(per * PAGE, device=q.device)[None, :] >= s["lens"][:, None]
    old = s["pool"][s["tables"].long().flatten(), layer]
    for i, (new, out) in enumerate(((k, s["k16"]), (v, s["v16"]))):
        vals = _plain_append(_plain_values(old, hd, i), _scales(old)[..., i], new, page, off)
        out[:, 0] = vals.masked_fill(past.reshape(b * per, 1, PAGE, 1), 0.0).bfloat16()
    return dict(q=s["q_out"], k=s["k16"], v=s["v16"])


def _plain_attention(s, q, k, v):
    """q [b * t, hq * hd], k and v [b, pages, hkv, 16, hd] fp32."""
    c = s["case"]
    b, t, hkv, hd = c["batch"], c["tokens"], c["hkv"], c["hd"]
    group, n = c["hq"] // hkv, k.shape[1] * PAGE
    at = torch.arange(n, device=q.device)
    k, v = (x.transpose(1, 2).reshape(b, hkv, n, hd) for x in (k, v))
    v = torch.where((at[None, :] < s["lens"][:, None])[:, None, :, None], v, 0.0)
    q = q.float().reshape(b, t, hkv, group, hd).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * group, hd)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    # query i of t sees the tokens up to its own
    seen = s["lens"][:, None] - (t - 1 - torch.arange(t, device=q.device))[None, :]
    seen = seen.repeat_interleave(group, 1)[:, None, :, None]
    x = torch.where(at < seen, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0.0)
    o = o.reshape(b, hkv, t, group, hd).permute(0, 2, 1, 3, 4).reshape(b * t, c["hq"] * hd)
    s["out"].copy_(o.bfloat16())
    return s["out"]


def _plain_dec8(s):
    c = s["case"]
    pages = s["pool"][s["tables"].long().clamp(min=0), c["layers"] - 1]  # [b, pages, hkv, bytes]
    return _plain_attention(s, s["q"], _plain_values(pages, c["hd"], 0),
                            _plain_values(pages, c["hd"], 1))


def _plain_step8(s):
    c = s["case"]
    b, hd = c["batch"], c["hd"]
    q, k, v = _plain_rows(s)
    live = s["slot_map"] >= 0
    s["q_out"].copy_(torch.where(live[:, None], q.flatten(1).bfloat16(), s["q_out"]))
    pages = s["pool"][s["tables"].long().clamp(min=0), c["layers"] - 1]
    per = pages.shape[1]
    seq = torch.arange(b, device=q.device).repeat_interleave(c["tokens"])[live]
    pos = s["positions"].long()[live]
    old = pages.flatten(0, 1)
    kv = []
    for i, new in enumerate((k, v)):
        vals = _plain_append(_plain_values(old, hd, i), _scales(old)[..., i], new[live],
                             seq * per + pos // PAGE, pos % PAGE)
        kv.append(vals.unflatten(0, (b, per)))
    return dict(q=s["q_out"], out=_plain_attention(s, s["q_out"], *kv))


def _plain_sample(s):
    x = s["logits"].double()
    v = x.shape[1]
    x = torch.where(x > -1e30, x, float("-inf"))
    top, order = torch.sort(x, dim=-1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    warm = t > 0
    w = torch.exp((top - top[:, :1]) / torch.where(warm, t, 1.0))
    c = w.cumsum(-1)
    k = s["top_k"].long()[:, None]
    keep = torch.where((k > 0) & (k < v), k, v)
    total = c.gather(1, keep - 1)
    p = s["top_p"].double()[:, None]
    keep = torch.where(p < 1, torch.minimum(keep, (c < p * total).sum(-1, keepdim=True) + 1), keep)
    keep = torch.minimum(keep, (w >= s["min_p"].double()[:, None]).sum(-1, keepdim=True))
    keep = torch.minimum(keep, (top > float("-inf")).sum(-1, keepdim=True)).clamp(min=1)
    target = s["rand"].double()[:, None] * c.gather(1, keep - 1)
    rank = torch.minimum((c <= target).sum(-1, keepdim=True), keep - 1)
    s["out"].copy_(order.gather(1, torch.where(warm, rank, 0))[:, 0])
    return s["out"]


# ------------------------------------------------------- the framework's own --

def _lucciola():
    path = os.path.abspath("lucciola-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import lucciola
    return lucciola


def _own_append(L, s):
    c = s["case"]
    L.qk_norm_rope_append_kv8(s["q_out"], s["qkv"], s["positions"], s["slot_map"], s["cos"],
                              s["sin"], s["pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                              c["hq"], c["hkv"], c["hd"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                              eps=EPS, q_bias=s["q_bias"], k_bias=s["k_bias"], v_bias=s["v_bias"])


def _own_attention(L, s, q):
    c = s["case"]
    if "ws" not in s:
        s["ws"] = L.alloc_decode_kv8_workspace(c["batch"], c["hq"], c["hkv"], c["hd"],
                                               tokens_per_seq=c["tokens"])
    L.paged_decode_kv8(s["out"], q, s["pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                       c["hq"], c["hkv"], c["hd"], s["tables"], s["lens"],
                       max_context_len=s["longest"], tokens_per_seq=c["tokens"],
                       workspace=s["ws"])
    return s["out"]


def _own_kv8(s):
    L, c = _lucciola(), s["case"]
    _own_append(L, s)
    L.unpack_kv8(s["k16"], s["v16"], s["pool"], s["num_blocks"], c["layers"], c["layers"] - 1,
                 c["hkv"], c["hd"], s["tables"], s["lens"], c["start"] + c["tokens"])
    return dict(q=s["q_out"], k=s["k16"], v=s["v16"])


def _own_step8(s):
    L = _lucciola()
    _own_append(L, s)
    return dict(q=s["q_out"], out=_own_attention(L, s, s["q_out"]))


def _own_dec8(s):
    return _own_attention(_lucciola(), s, s["q"])


def _own_sample(s):
    _lucciola().sample(s["out"], s["logits"], s["rand"], temperature=s["temperature"],
                       top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(kv8=_own_kv8, step8=_own_step8, dec8=_own_dec8, sample=_own_sample)[op](state)
    return dict(kv8=_plain_kv8, step8=_plain_step8, dec8=_plain_dec8,
                sample=_plain_sample)[op](state)


# -------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["op"] == "sample":
        return dict(bytes=c["batch"] * (2 * c["vocab"] + 24), flops=2 * c["batch"] * c["vocab"])
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    token = 2 * hkv * (hd + 4 / PAGE)  # bytes of one token's K and V, the page's scales shared

    def append(rows):  # q, k, v in, q out; cos and sin; position and slot; the cache
        return rows * (2 * (2 * hq + 2 * hkv) * hd + 2 * 4 * hd // 2 + 8 + token)
    if c["op"] == "kv8":
        rows, seen = c["batch"] * c["tokens"], c["batch"] * (c["start"] + c["tokens"])
        return dict(bytes=append(rows) + seen * (token + 2 * hkv * 2 * hd),
                    flops=rows * ((hq + hkv) * hd * 8 + 2 * hkv * hd * 4) + seen * 2 * hkv * hd)
    rows, seen = c["batch"] * c["tokens"], c["batch"] * (c["lo"] + c["hi"]) / 2
    need = dict(bytes=seen * (token + 4 / PAGE) + 2 * 2 * rows * hq * hd,
                flops=4 * seen * c["tokens"] * hq * hd)
    if c["op"] == "step8":  # the appended q is read where it was written
        need["bytes"] += append(rows)
        need["flops"] += rows * ((hq + hkv) * hd * 8 + 2 * hkv * hd * 4)
    return need


# ------------------------------------------------------------------- exact --

def _np(t):
    if t is None:
        return None
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _exact_e4m3(x):
    """Nearest e4m3 value (ties to even) of float64."""
    a = np.minimum(np.abs(x), 448.0)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -9)))
    step = 2.0 ** (np.maximum(e, -6.0) - 3.0)
    return np.sign(x) * np.minimum(np.rint(a / step) * step, 448.0)


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


_E4M3 = np.array([(-1) ** (i >> 7) * (np.nan if i & 127 == 127 else (i & 7) * 2.0 ** -9 if i & 120 == 0
                                      else (8 + (i & 7)) * 2.0 ** ((i >> 3 & 15) - 10))
                  for i in range(256)])


def _exact_pages(pages, hd):
    """float64 K and V [2, n, hkv, 16, hd] and scales [2, n, hkv] of uint8 numpy [n, hkv, bytes]."""
    scale = np.moveaxis(np.ascontiguousarray(pages[..., 32 * hd:32 * hd + 8]).view(np.float32), -1, 0)
    scale = scale.astype(np.float64)
    rows = pages[..., :32 * hd].reshape(pages.shape[:2] + (2, PAGE, hd // 16, 16))
    out = np.empty(rows.shape)
    for t in range(PAGE):
        for piece in range(hd // 16):
            out[:, :, :, t, piece] = _E4M3[rows[:, :, :, t, piece ^ (t * hd // 64 & (hd // 16 - 2))]]
    out = np.moveaxis(out.reshape(pages.shape[:2] + (2, PAGE, hd)), 2, 0)
    return out * scale[..., None, None], scale


def _exact_append(s, k, v, pages):
    """K and V [2, n, hkv, 16, hd] of `pages` (physical numbers) after the rows are appended."""
    c = s["case"]
    vals, scale = _exact_pages(_np(s["pool"][pages, c["layers"] - 1]), c["hd"])
    where = {int(p): i for i, p in enumerate(pages.tolist())}
    into = {}
    for row, slot in enumerate(_np(s["slot_map"])):
        if slot >= 0:
            into.setdefault(where[int(slot) // PAGE], []).append((row, int(slot) % PAGE))
    for page, rows in into.items():
        at, off = [r for r, _ in rows], [o for _, o in rows]
        for i, x in enumerate((k, v)):
            new = x[at]  # [rows, hkv, hd]
            top = np.abs(new).max((0, 2))
            e = np.clip(np.ceil(np.log2(np.maximum(top, 1e-300) / 448.0)), E_MIN, E_MAX)
            step = 2.0 ** e if 0 in off else np.maximum(2.0 ** e, scale[i, page])
            vals[i, page][:, off] = new.transpose(1, 0, 2)
            vals[i, page] = _exact_e4m3(vals[i, page] / step[:, None, None]) * step[:, None, None]
    return vals


def _exact_attention(s, q, kv_of):
    c = s["case"]
    t, hkv, hd, group = c["tokens"], c["hkv"], c["hd"], c["hq"] // c["hkv"]
    q = q.double().reshape(c["batch"], t, hkv, group, hd)
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        k, v = (x.transpose(0, 1).reshape(hkv, -1, hd)[:, :n] for x in kv_of(b, n))
        for i in range(t):
            m = n - (t - 1 - i)
            if m > 0:
                x = torch.einsum("hgd,hnd->hgn", q[b, i], k[:, :m]) / math.sqrt(hd)
                out[b, i] = torch.softmax(x, -1) @ v[:, :m]
    return out.reshape(c["batch"] * t, -1).cpu().numpy()


def _exact_sample(s):
    got = []
    par = [_np(s[n]) for n in ("temperature", "top_k", "top_p", "min_p", "rand")]
    logits = s["logits"].float().cpu().numpy()
    for row, t, k, p, least, u in zip(logits, *par):
        value, count = np.unique(row[row > -1e30], return_counts=True)
        value, count = value[::-1].astype(np.float64), count[::-1]
        rank, j = 0, 0
        if t > 0:
            w = np.exp((value - value[0]) / t)
            before = np.concatenate([[0], np.cumsum(count)])
            mass = np.concatenate([[0.0], np.cumsum(count * w)])

            def weight(n):  # of the n first tokens
                g = np.searchsorted(before, n, side="right") - 1
                return mass[-1] if g >= len(w) else mass[g] + (n - before[g]) * w[g]
            keep = min(int(k), int(before[-1])) if k > 0 else int(before[-1])
            if p < 1:
                need = p * weight(keep)
                g = np.searchsorted(mass, need, side="left") - 1  # the group that reaches it
                if g >= 0:
                    keep = min(keep, int(before[g] + np.ceil((need - mass[g]) / w[g])))
                else:
                    keep = 1
            keep = max(1, min(keep, int(count[w >= least].sum())))
            goal = u * weight(keep)
            j = min(int(np.searchsorted(mass, goal, side="right")) - 1, len(w) - 1)
            rank = min(before[j] + int((goal - mass[j]) // w[j]), keep - 1)
            j = int(np.searchsorted(before, rank, side="right")) - 1
            rank -= before[j]
        got.append(np.nonzero(row == np.float32(value[j]))[0][rank])
    return np.array(got)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "sample":
        return _exact_sample(s)
    layer, hd, hkv = c["layers"] - 1, c["hd"], c["hkv"]
    if c["op"] == "kv8":
        q, k, v = _exact_rows(s)
        b, per = c["batch"], s["per"]
        vals = _exact_append(s, k, v, s["tables"].long().flatten())
        vals = vals.reshape(2, b, per, hkv, PAGE, hd).transpose(0, 1, 2, 4, 3, 5)
        vals = vals.reshape(2, b, per * PAGE, hkv, hd)
        vals[:, :, c["start"] + c["tokens"]:] = 0.0
        vals = vals.reshape(2, b, per, PAGE, hkv, hd).transpose(0, 1, 2, 4, 3, 5)
        vals = vals.reshape(2, b * per, 1, hkv, PAGE, hd)
        return dict(q=q.reshape(len(q), -1), k=vals[0], v=vals[1])
    lut = torch.tensor(_E4M3, device="cuda")
    place = _places(hd)

    def cached(b, n):
        pages = s["pool"][s["tables"][b, :_ceil(n, PAGE)].long(), layer]
        scale = pages[..., -16:-8].contiguous().view(torch.float32).double()
        return [lut[pages[..., i * PAGE * hd:][..., place].int()] * scale[..., i, None, None]
                for i in range(2)]
    if c["op"] == "dec8":
        return _exact_attention(s, s["q"], cached)
    q, k, v = _exact_rows(s)
    slot = s["slot_map"][s["slot_map"] >= 0].long()
    touched = torch.unique(slot // PAGE)
    vals = torch.from_numpy(_exact_append(s, k, v, touched)).cuda()

    def stepped(b, n):
        pages = s["tables"][b, :_ceil(n, PAGE)].long()
        at = torch.searchsorted(touched, pages).clamp(max=len(touched) - 1)
        new = (touched[at] == pages)[:, None, None, None]
        return [torch.where(new, vals[i, at], old) for i, old in enumerate(cached(b, n))]
    # the attention takes q as it was stored, rounded to bf16
    rows = torch.from_numpy(q.reshape(len(q), -1)).cuda()
    live = (s["slot_map"] >= 0)[:, None]
    out = _exact_attention(s, torch.where(live, rows, 0.0).bfloat16(), stepped)
    return dict(q=torch.where(live, rows, 0.0).cpu().numpy(), out=out)
