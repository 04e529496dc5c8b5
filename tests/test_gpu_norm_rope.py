"""Per-head norm + RoPE + append into the bf16 pools (lc_qk_norm_rope_append)
against float64, and against lc_rope_append where both apply."""
import numpy as np
import pytest

import kv4_ref as R
import lucciola as L
import oracle.oracle as O
from workloads import from_device, randn_bf16, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def run(rng, hq, hkv, hd, rows, norm, bias, pad=8, scale=1.0, in_place=False, eps=1e-6, layers=2,
        layer=1):
    nb = rows // 16 + 2
    row = (hq + 2 * hkv) * hd + pad
    qkv = O.f32_to_bf16(rng.standard_normal((rows, row)).astype(np.float32) * scale)
    vec = {k: randn_bf16(rng, n * hd) if on else None for k, n, on in (
        ("q_bias", hq, bias), ("k_bias", hkv, bias), ("v_bias", hkv, bias),
        ("q_norm", 1, norm), ("k_norm", 1, norm))}
    cos, sin = O.rope_table(700, hd, 1e6)
    pos = rng.integers(0, 700, rows).astype(np.int32)
    slot = rng.permutation(nb * 16)[:rows].astype(np.int32)
    k0, v0 = (randn_bf16(rng, (nb, layers, hkv, 16, hd)) for _ in range(2))
    dk, dv, dq = to_device(k0), to_device(v0), to_device(qkv)
    q_out = dq if in_place else torch.zeros(rows, hq * hd, dtype=torch.bfloat16, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    L.qk_norm_rope_append(q_out, dq, to_device(pos), to_device(slot), to_device(cos),
                          to_device(sin), dk, dv, nb, layers, layer, hq, hkv, hd, eps=eps,
                          dev_status=st, **{k: None if v is None else to_device(v)
                                            for k, v in vec.items()})
    assert int(st.item()) == 0
    got_q = R.bf16_f64(from_device(q_out))[:, :hq * hd].reshape(rows, hq, hd)
    got_k, got_v = (R.bf16_f64(from_device(t)) for t in (dk, dv))
    if not in_place:
        assert np.array_equal(from_device(dq), qkv)  # only read
    else:
        assert np.array_equal(from_device(dq)[:, hq * hd:], qkv[:, hq * hd:])

    f = {k: None if v is None else R.bf16_f64(v) for k, v in vec.items()}
    x = R.bf16_f64(qkv)[:, :(hq + 2 * hkv) * hd].reshape(rows, -1, hd)
    c64, s64 = cos.astype(np.float64)[pos], sin.astype(np.float64)[pos]

    def bias_of(name):
        b = f[name + "_bias"]
        return None if b is None else b.reshape(-1, hd)
    q, qs = R.norm_rope(x[:, :hq], bias_of("q"), f["q_norm"], eps, c64, s64)
    k, ks = R.norm_rope(x[:, hq:hq + hkv], bias_of("k"), f["k_norm"], eps, c64, s64)
    v = x[:, hq + hkv:]
    if bias:
        v = (v + bias_of("v")).astype(np.float32).astype(np.float64)

    def close(got, want, size):
        # one bf16 rounding after about a dozen fp32 ones of the terms
        assert R.rounds_to(got, want, 16 * 2.0 ** -24 * size).all()
    close(got_q, q, qs)
    stored = np.zeros((nb, 16), bool)
    stored[slot // 16, slot % 16] = True
    for got, before, want, size in ((got_k, k0, k, ks), (got_v, v0, v, None)):
        rows_got = got[slot // 16, layer, :, slot % 16]
        if size is None:
            assert np.array_equal(rows_got, R.bf16_round(want))
        else:
            close(rows_got, want, size)
        same = got == R.bf16_f64(before)
        same[:, layer] |= stored[:, None, :, None]
        assert same.all()


@pytest.mark.parametrize("hq,hkv,hd", [(14, 2, 64), (28, 4, 128), (1, 1, 64), (1, 1, 128),
                                       (3, 3, 128), (64, 8, 128), (9, 1, 64), (40, 8, 64)])
@pytest.mark.parametrize("rows", [1, 3, 130])
def test_norm_rope_append(hq, hkv, hd, rows):
    rng = np.random.default_rng(hq * rows + hd)
    run(rng, hq, hkv, hd, rows, norm=True, bias=rows == 3)
    run(rng, hq, hkv, hd, rows, norm=False, bias=rows != 3)


def test_norm_rope_append_many_rows():
    rng = np.random.default_rng(1)
    run(rng, 4, 2, 64, 3001, norm=True, bias=True, pad=0, layers=1, layer=0)
    run(rng, 2, 2, 128, 2049, norm=True, bias=False, pad=16, layers=1, layer=0)


@pytest.mark.parametrize("hd", [64, 128])
def test_norm_rope_append_in_place_and_scales(hd):
    rng = np.random.default_rng(2)
    run(rng, 6, 2, hd, 20, norm=True, bias=True, in_place=True)
    run(rng, 6, 2, hd, 20, norm=True, bias=False, scale=1e-4)  # eps matters
    run(rng, 6, 2, hd, 20, norm=True, bias=False, scale=1e4, eps=0.0)


def test_zero_heads_and_special_values():
    hq, hkv, hd = 2, 1, 64
    x = np.zeros((3, 4 * hd), np.float32)
    x[1] = 1.0
    x[1, 3] = np.nan       # head 0 of q
    x[2, hd + 1] = np.inf  # head 1 of q: inf / inf
    cos, sin = O.rope_table(8, hd, 1e6)
    pool = [torch.zeros(1, 1, 1, 16, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    q = torch.zeros(3, hq * hd, dtype=torch.bfloat16, device="cuda")
    rows = torch.arange(3, dtype=torch.int32, device="cuda")
    w = torch.ones(hd, dtype=torch.bfloat16, device="cuda")
    L.qk_norm_rope_append(q, torch.from_numpy(x).cuda().bfloat16(), rows, rows, to_device(cos),
                          to_device(sin), *pool, 1, 1, 0, hq, hkv, hd, q_norm=w, k_norm=w)
    got = q.float().cpu().numpy().reshape(3, hq, hd)
    assert not got[0].any()
    assert np.isnan(got[1, 0]).all() and np.isfinite(got[1, 1]).all()
    assert np.isfinite(got[2, 0]).all() and np.isnan(got[2, 1, [1, 33]]).all()
    assert np.isfinite(pool[0].float().cpu().numpy()).all()


def test_agrees_with_rope_append():
    """Without norms the pools and q are those of lc_rope_append, up to the one fp32
    rounding in which a fused and an unfused rotation differ."""
    hq, hkv, hd, rows = 14, 2, 64, 48
    rng = np.random.default_rng(3)
    qkv = randn_bf16(rng, (rows, (hq + 2 * hkv) * hd))
    qb, kb, vb = (to_device(randn_bf16(rng, n * hd)) for n in (hq, hkv, hkv))
    cos, sin = (to_device(t) for t in O.rope_table(64, hd, 1e6))
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    slot = (tables[0][(pos // 16).long()] * 16 + pos % 16).int()
    a, b = ([torch.zeros(3, 1, hkv, 16, hd, dtype=torch.bfloat16, device="cuda")
             for _ in range(2)] for _ in range(2))
    d1, d2 = to_device(qkv), to_device(qkv)
    L.rope_append(d1, pos, qb, kb, vb, cos, sin, *a, 3, 1, 0, hq, hkv, hd, tables,
                  tokens_per_seq=rows)
    q = torch.zeros(rows, hq * hd, dtype=torch.bfloat16, device="cuda")
    L.qk_norm_rope_append(q, d2, pos, slot, cos, sin, *b, 3, 1, 0, hq, hkv, hd, q_bias=qb,
                          k_bias=kb, v_bias=vb)
    assert torch.equal(a[1], b[1])
    for x, y in ((d1[:, :hq * hd], q), (a[0], b[0])):
        x, y = x.float(), y.float()
        # the rotation's terms are below 16; one bf16 step where the last fp32 bit decides
        assert ((x - y).abs() <= torch.maximum(x.abs() * 2.0 ** -7, torch.tensor(16 * 2.0 ** -23))).all()
        assert (x != y).float().mean() < 1e-3


def separately_rounded(x, bias, w, eps, cos, sin):
    """float32 in, float32 out: every product and sum rounded by itself, the squares added
    in halves (d with d + hd/2, within 8 dims, across the 8-dim chunks)."""
    f = np.float32
    u = x if bias is None else x + bias
    hd = u.shape[-1]
    if w is not None:
        q = (u * u).reshape(u.shape[:-1] + (2, hd // 16, 8))
        q = q[..., 0, :, :] + q[..., 1, :, :]
        while q.shape[-1] > 1:
            n = q.shape[-1] // 2
            q = q[..., :n] + q[..., n:]
        q = q[..., 0]
        while q.shape[-1] > 1:
            n = q.shape[-1] // 2
            q = q[..., :n] + q[..., n:]
        u = u * (f(1) / np.sqrt(q * f(1 / hd) + f(eps))) * w
    a, b = np.split(u, 2, -1)
    c, s = cos[:, None, :], sin[:, None, :]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("norm,bias", [(True, False), (True, True), (False, True), (False, False)])
def test_bits_do_not_depend_on_the_kernel(hd, norm, bias):
    """Compilers like to contract a * b + c * d: a last bit here can be a whole step once a
    value is held in 4 bits, so the bits are pinned."""
    hq, hkv, rows = 6, 2, 70
    rng = np.random.default_rng(hd)
    qkv = randn_bf16(rng, (rows, (hq + 2 * hkv) * hd))
    vec = {k: randn_bf16(rng, n * hd) if on else None for k, n, on in (
        ("q_bias", hq, bias), ("k_bias", hkv, bias), ("v_bias", hkv, bias),
        ("q_norm", 1, norm), ("k_norm", 1, norm))}
    cos, sin = O.rope_table(rows, hd, 1e6)
    pool = [torch.zeros(5, 1, hkv, 16, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    q = torch.zeros(rows, hq * hd, dtype=torch.bfloat16, device="cuda")
    ids = torch.arange(rows, dtype=torch.int32, device="cuda")
    L.qk_norm_rope_append(q, to_device(qkv), ids, ids, to_device(cos), to_device(sin), *pool, 5, 1,
                          0, hq, hkv, hd, **{k: None if v is None else to_device(v)
                                             for k, v in vec.items()})
    f = {k: None if v is None else R.bf16_f64(v).astype(np.float32).reshape(-1, hd)
         for k, v in vec.items()}
    x = R.bf16_f64(qkv).astype(np.float32).reshape(rows, -1, hd)
    for got, lo, n, part in ((from_device(q).reshape(rows, hq, hd), 0, hq, "q"),
                             (from_device(pool[0])[:, 0].transpose(0, 2, 1, 3)
                              .reshape(80, hkv, hd)[:rows], hq, hkv, "k")):
        w = f[part + "_norm"]
        want = separately_rounded(x[:, lo:lo + n], f[part + "_bias"], None if w is None else w[0],
                                  1e-6, cos, sin)
        assert np.array_equal(got, O.f32_to_bf16(want))
