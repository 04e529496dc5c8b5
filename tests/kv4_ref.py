"""float64 references of the step tables, the per-head norm + RoPE and the 4-bit
cache (numpy only, written from the formulas in include/lucciola_attn.h)."""
from __future__ import annotations

import numpy as np

PAGE = 16
MAG = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E2M1 = np.concatenate([MAG, -MAG])


def ceil16(n):
    return -(-int(n) // PAGE)


def half_bytes(hd):
    return PAGE * hd // 2 + PAGE * hd // 16


def bf16_round(x):
    """float64 -> nearest bf16 (ties to even), as float64."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)
    e = np.maximum(e, -125)
    return np.ldexp(np.rint(np.ldexp(x, 8 - e)), e - 8)


def bf16_f64(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounds_to(got, want, slack):
    """Whether each `got` is the bf16 rounding of something within `slack` of `want`."""
    return (bf16_round(want - slack) <= got) & (got <= bf16_round(want + slack))


def e4m3_value(byte):
    s = np.asarray(byte, np.int64)
    e, m = (s >> 3) & 15, s & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    return np.where((s & 127) == 127, np.nan, v)


def e4m3_byte(x):
    """Nearest e4m3 byte of non-negative x, at most 448; NaN for what is not finite."""
    grid = e4m3_value(np.arange(0, 127))
    y = np.minimum(np.where(np.isfinite(x), x, 0.0), 448.0)
    hi = np.clip(np.searchsorted(grid, y), 1, 126)
    lo = hi - 1
    dl, dh = y - grid[lo], grid[hi] - y
    byte = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.where(np.isfinite(x), byte, 0x7f).astype(np.uint8)


def quantise(x, g):
    """x [..., hd] -> (codes [..., hd] 0..15, scale bytes [..., hd/16], x / step [..., hd])."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[:-1] + (-1, 16))
    amax = np.abs(b).max(-1)  # NaN and infinity carry through
    s8 = e4m3_byte(amax / (6.0 * g))
    step = (e4m3_value(s8) * g)[..., None]
    with np.errstate(all="ignore"):
        y = np.where(step > 0, b / step, 0.0)
    a = np.abs(y)
    code = np.zeros(b.shape, np.int64)
    for i in range(7):
        mid = (MAG[i] + MAG[i + 1]) / 2
        code += (a > mid) if i % 2 == 0 else (a >= mid)
    code += 8 * np.signbit(b)
    return code.reshape(x.shape), s8, y.reshape(x.shape)


def pack(x, g):
    """x [..., 16, hd] -> uint8 [..., half page bytes]."""
    code, s8, _ = quantise(x, g)
    data = (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)
    lead = x.shape[:-2]
    return np.concatenate([data.reshape(lead + (-1,)), s8.reshape(lead + (-1,))], -1)


def unpack(pages, hd, g):
    """uint8 [..., half page bytes] -> float64 [..., 16, hd]."""
    n = PAGE * hd // 2
    data = pages[..., :n].reshape(pages.shape[:-1] + (PAGE, hd // 2))
    s = e4m3_value(pages[..., n:].reshape(pages.shape[:-1] + (PAGE, hd // 16))) * g
    out = np.empty(data.shape[:-1] + (hd,))
    out[..., 0::2], out[..., 1::2] = E2M1[data & 15], E2M1[data >> 4]
    return out * np.repeat(s, 16, -1)


def norm_rope(x, bias, w, eps, cos, sin):
    """float64 [rows, heads, hd] with cos, sin [rows, hd/2]: (result, |y1| + |y2| per dim)."""
    u = x if bias is None else x + bias
    y = u if w is None else u / np.sqrt((u ** 2).mean(-1, keepdims=True) + eps) * w
    a, b = np.split(y, 2, -1)
    c, s = cos[:, None, :], sin[:, None, :]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, a * s + b * c], -1), np.concatenate([size, size], -1)


def make_pool(rng, num_blocks, layers, hkv, hd, k_scale, v_scale, k_std=1.0, v_std=0.3):
    shape = (num_blocks, layers, hkv, PAGE, hd)
    gain = np.ones(hd)
    gain[rng.integers(0, hd, 2)] = 6.0
    k = pack(rng.standard_normal(shape) * k_std * gain, k_scale)
    v = pack(rng.standard_normal(shape) * v_std, v_scale)
    return np.concatenate([k, v], -1)


def decode(q, pool, layer, tables, lens, hkv, hd, tokens, k_scale, v_scale, sm_scale=None):
    """q float64 [batch * tokens, hq, hd]. Returns (out, slack): the float64 attention and,
    per element, how far fp16 probabilities (2^-11 of the mass, 2^-25 of the largest
    probability where they are subnormal) and fp32 products (2^-21 of sum |q k|) may take a
    kernel from it before its one rounding to bf16."""
    sm_scale = sm_scale or hd ** -0.5
    rows, hq, _ = q.shape
    group = hq // hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    num_blocks = pool.shape[0]
    hb = half_bytes(hd)
    for r in range(rows):
        b, i = divmod(r, tokens)
        n = int(lens[b]) - (tokens - 1 - i)
        if n <= 0:
            continue
        ids = tables[b, :ceil16(n)]
        ok = (ids >= 0) & (ids < num_blocks)
        pages = pool[np.where(ok, ids, 0), layer]
        kv = []
        for part, g in ((pages[..., :hb], k_scale), (pages[..., hb:], v_scale)):
            val = unpack(part, hd, g)
            val[~ok] = 0.0
            kv.append(val.transpose(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :n])
        for h in range(hq):
            k, v = kv[0][h // group], kv[1][h // group]
            with np.errstate(all="ignore"):
                x = k @ q[r, h] * sm_scale
                dx = (np.abs(k) @ np.abs(q[r, h])).max() * sm_scale * 2.0 ** -21
                p = np.exp(x - x.max())
                p /= p.sum()
                out[r, h] = p @ v
                mass = p @ np.abs(v)
                top = np.abs(v).max(0) * p.max() * n * 2.0 ** -25
                bound[r, h] = mass * (2.0 ** -11 + 2 * dx) + top
    return out, bound


def quantise_codes(y):
    """Magnitude codes 0..7 of y (negative y: 0)."""
    code = np.zeros(np.shape(y), np.int64)
    for i in range(7):
        mid = (MAG[i] + MAG[i + 1]) / 2
        code += (y > mid) if i % 2 == 0 else (y >= mid)
    return code
