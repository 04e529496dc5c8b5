"""float64 references of the 8-bit cache (numpy only, written from the formulas in
include/lucciola_attn.h)."""
from __future__ import annotations

import numpy as np

from kv4_ref import PAGE, bf16_f64, bf16_round, ceil16, norm_rope, rounds_to  # noqa: F401

E_MIN, E_MAX = -40, 40
_I = np.arange(256)
VALUES = np.where((_I >> 3) & 15 == 0, (_I & 7) * 2.0 ** -9, (8 + (_I & 7)) * 2.0 ** (((_I >> 3) & 15) - 10.0))
VALUES = np.where(_I & 127 == 127, np.nan, VALUES) * np.where(_I & 128, -1.0, 1.0)


def page_bytes(hd):
    return 32 * hd + 16


def places(hd):
    """[16, hd]: byte of (token, dim) within a page's K or V."""
    t, d = np.mgrid[:PAGE, :hd]
    return t * hd + ((d // 16) ^ ((t * hd // 64) & (hd // 16 - 2))) * 16 + d % 16


def round8(x):
    """Nearest e4m3 value (ties to even), at most 448 in magnitude; not finite: NaN."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.where(np.isfinite(x), x, 0.0)), 448.0)
    _, e = np.frexp(a)  # a = m 2^e, m in [.5, 1)
    step = 2.0 ** (np.maximum(e - 1, -6) - 3.0)
    y = np.copysign(np.minimum(np.rint(a / step) * step, 448.0), x)
    return np.where(np.isfinite(x), y, np.nan)


def exponent(amax):
    """Smallest e with amax <= 448 * 2^e, within the scales' range."""
    m, e = np.frexp(np.asarray(amax, np.float64))
    return np.clip(np.where(np.asarray(amax) > 0, e - 9 + (m > 0.875), E_MIN), E_MIN, E_MAX)


def code_of(y):
    """Bytes of values that are e4m3's."""
    grid = VALUES[:127]
    at = np.searchsorted(grid, np.where(np.isnan(y), 0.0, np.abs(y)))
    byte = np.where(np.isnan(y), 0x7f, at | np.where(np.signbit(y), 128, 0))
    return byte.astype(np.uint8)


def pack(k, v):
    """K and V [..., 16, hd] -> uint8 [..., page bytes], each page at its own scale."""
    hd = k.shape[-1]
    out = np.zeros(k.shape[:-2] + (page_bytes(hd),), np.uint8)
    where = places(hd).ravel()
    for i, x in enumerate((k, v)):
        scale = 2.0 ** exponent(np.abs(x).max((-1, -2)))
        code = code_of(round8(x / scale[..., None, None]))
        out[..., i * PAGE * hd:(i + 1) * PAGE * hd][..., where] = code.reshape(code.shape[:-2] + (-1,))
        at = 32 * hd + 4 * i
        out[..., at:at + 4] = scale.astype(np.float32)[..., None].view(np.uint8)
    return out


def scales(pages, hd):
    """float64 [..., 2] (K's and V's) of uint8 [..., page bytes]."""
    return np.ascontiguousarray(pages[..., 32 * hd:32 * hd + 8]).view(np.float32).astype(np.float64)


def codes(pages, hd, i):
    """Code bytes [..., 16, hd] in the order of tokens and dims."""
    return pages[..., i * PAGE * hd:(i + 1) * PAGE * hd][..., places(hd)]


def unpack(pages, hd, i):
    """float64 [..., 16, hd] of K (i = 0) or V (1)."""
    return VALUES[codes(pages, hd, i)] * scales(pages, hd)[..., i, None, None]


def put_code(pool, page, layer, head, i, token, dim, hd, byte):
    pool[page, layer, head, i * PAGE * hd + places(hd)[token, dim]] = byte


def make_pool(rng, num_blocks, layers, hkv, hd, k_std=1.0, v_std=0.3, spread=0):
    """Random pages; `spread`: their magnitudes vary by 2^-spread .. 2^spread."""
    shape = (num_blocks, layers, hkv, PAGE, hd)
    gain = np.ones(hd)
    gain[rng.integers(0, hd, 2)] = 6.0

    def size():
        return 2.0 ** rng.integers(-spread, spread + 1, shape[:3])[..., None, None]
    return pack(rng.standard_normal(shape) * k_std * gain * size(),
                rng.standard_normal(shape) * v_std * size())


def spoil(pool, tables, lens, hkv, hd):
    """NaN behind each sequence's last token."""
    for b, n in enumerate(lens):
        if n % PAGE:
            page = pool[tables[b, n // PAGE]]
            rows = page[..., :32 * hd].reshape(page.shape[:-1] + (2, PAGE, hd))
            rows[..., n % PAGE:, :] = 0x7f


def decode(q, pool, layer, tables, lens, hkv, hd, tokens, sm_scale=None):
    """q float64 [batch * tokens, hq, hd]. Returns (out, slack): the float64 attention and, per
    element, how far fp16 probabilities (2^-11 of the mass; 2^-25 of the largest probability
    times V scale where they are subnormal) and fp32 products (2^-21 of sum |q k|) may take a
    kernel from it before its one rounding to bf16."""
    sm_scale = sm_scale or hd ** -0.5
    rows, hq, _ = q.shape
    group = hq // hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(rows):
        b, i = divmod(r, tokens)
        n = int(lens[b]) - (tokens - 1 - i)
        if n <= 0:
            continue
        ids = tables[b, :ceil16(n)]
        ok = (ids >= 0) & (ids < pool.shape[0])
        pages = pool[np.where(ok, ids, 0), layer]
        kv = []
        for part in range(2):
            val = unpack(pages, hd, part)
            val[~ok] = 0.0
            kv.append(val.transpose(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :n])
        vs = scales(pages, hd)[..., 1].T.repeat(PAGE, 1)[:, :n]
        for h in range(hq):
            k, v = kv[0][h // group], kv[1][h // group]
            with np.errstate(all="ignore"):
                x = k @ q[r, h] * sm_scale
                dx = (np.abs(k) @ np.abs(q[r, h])).max() * abs(sm_scale) * 2.0 ** -21
                p = np.exp(x - x.max())
                p /= p.sum()
                out[r, h] = p @ v
                mass = p @ np.abs(v)
                s = vs[h // group]
                top = np.abs(v / s[:, None]).max(0) * (p * s).max() * n * 2.0 ** -25
                bound[r, h] = mass * (2.0 ** -11 + 2 * dx) + top
    return out, bound
