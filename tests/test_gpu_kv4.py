"""The 4-bit cache on the GPU: append (lc_qk_norm_rope_append_kv4), unpack
(lc_unpack_kv4) and decode attention (lc_paged_decode_kv4) against float64."""
import numpy as np
import pytest

import kv4_ref as R
import lucciola as L
import oracle.oracle as O
from workloads import from_device, make_tables, randn_bf16, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------- append --

@pytest.mark.parametrize("hq,hkv,hd,rows,norm,bias,g", [
    (14, 2, 64, 1, True, False, (1.0, 1.0)), (14, 2, 64, 37, False, True, (0.5, 0.0625)),
    (28, 4, 128, 33, True, True, (1.0, 0.25)), (1, 1, 128, 5, True, False, (2.0, 1.0)),
    (40, 8, 128, 16, False, False, (0.3, 0.7)), (9, 3, 64, 50, True, True, (1.0, 1e-3)),
])
def test_append_kv4_matches_the_formula(hq, hkv, hd, rows, norm, bias, g):
    rng = np.random.default_rng(hq * 100 + rows)
    layers, layer, nb = 3, 1, rows // 16 + 3
    row = (hq + 2 * hkv) * hd + 8
    qkv = randn_bf16(rng, (rows, row))
    vec = {k: randn_bf16(rng, n * hd) if on else None for k, n, on in (
        ("q_bias", hq, bias), ("k_bias", hkv, bias), ("v_bias", hkv, bias),
        ("q_norm", 1, norm), ("k_norm", 1, norm))}
    cos, sin = O.rope_table(512, hd, 1e6)
    pos = rng.integers(0, 512, rows).astype(np.int32)
    slot = rng.permutation(nb * 16)[:rows].astype(np.int32)
    before = rng.integers(0, 256, (nb, layers, hkv, 18 * hd), dtype=np.uint8)
    pool = to_device(before)
    q_out = torch.zeros(rows, hq * hd + 16, dtype=torch.bfloat16, device="cuda")
    st = status_word()
    L.qk_norm_rope_append_kv4(
        q_out, to_device(qkv), to_device(pos), to_device(slot), to_device(cos), to_device(sin),
        pool, nb, layers, layer, hq, hkv, hd, k_scale=g[0], v_scale=g[1], eps=1e-6, dev_status=st,
        **{k: None if v is None else to_device(v) for k, v in vec.items()})
    got, word = from_device(pool), int(st.item())
    assert word == 0

    f = {k: None if v is None else R.bf16_f64(v) for k, v in vec.items()}
    x = R.bf16_f64(qkv)[:, :(hq + 2 * hkv) * hd].reshape(rows, -1, hd)

    def part(a, b, name):
        bb = f[name + "_bias"]
        return x[:, a:b], None if bb is None else bb.reshape(-1, hd)
    c64, s64 = cos.astype(np.float64)[pos], sin.astype(np.float64)[pos]
    qx, qb = part(0, hq, "q")
    kx, kb = part(hq, hq + hkv, "k")
    vx, vb = part(hq + hkv, hq + 2 * hkv, "v")
    q, q_size = R.norm_rope(qx, qb, f["q_norm"], 1e-6, c64, s64)
    k, k_size = R.norm_rope(kx, kb, f["k_norm"], 1e-6, c64, s64)
    # v + bias is one fp32 sum
    v = vx if vb is None else (vx + vb).astype(np.float32).astype(np.float64)

    # q: one bf16 rounding after fp32 steps (16 of 2^-24 of the terms)
    got_q = R.bf16_f64(from_device(q_out))[:, :hq * hd].reshape(q.shape)
    assert R.rounds_to(got_q, q, 16 * 2.0 ** -24 * q_size).all()
    assert not from_device(q_out)[:, hq * hd:].any()

    hb = R.half_bytes(hd)
    untouched = np.ones(before.shape[:1] + (16,), bool)
    untouched[slot // 16, slot % 16] = False
    n = 16 * hd // 2

    def rows_of(pages, is_v):
        half = pages[:, layer, :, is_v * hb:(is_v + 1) * hb]
        data = half[..., :n].reshape(nb, hkv, 16, hd // 2)
        sc = half[..., n:].reshape(nb, hkv, 16, hd // 16)
        return data, sc
    for is_v, val, size in ((0, k, k_size), (1, v, None)):
        data, sc = rows_of(got, is_v)
        data0, sc0 = rows_of(before, is_v)
        keep = untouched[:, None, :, None]
        assert (np.where(keep, data == data0, True)).all()
        assert (np.where(keep, sc == sc0, True)).all()
        d, s8 = data[slot // 16, :, slot % 16], sc[slot // 16, :, slot % 16]
        code = np.empty(val.shape, np.int64)
        code[..., 0::2], code[..., 1::2] = d & 15, d >> 4
        want, want_s8, y = R.quantise(val, np.float64(np.float32(g[is_v])))
        if is_v:
            # 6 g and the steps are exact here only for a power of two
            if np.log2(g[1]) % 1 == 0:
                assert np.array_equal(s8, want_s8)
                assert np.array_equal(code, want)
                continue
            slack = 4 * 2.0 ** -24 * np.abs(val)
        else:
            slack = 16 * 2.0 ** -24 * size + 4 * 2.0 ** -24 * np.abs(val)
        # a value within `slack` of where two scales or codes meet may go to either
        near = np.abs(s8.astype(int) - want_s8.astype(int))
        assert near.max() <= 1 and (near > 0).mean() <= 1e-3
        step = (R.e4m3_value(s8) * g[is_v]).repeat(16, -1)
        y = np.where(step > 0, val / np.where(step > 0, step, 1), 0.0)
        lo = R.quantise_codes(np.abs(y) - slack / np.where(step > 0, step, 1))
        hi = R.quantise_codes(np.abs(y) + slack / np.where(step > 0, step, 1))
        assert ((code & 7) >= lo).all() and ((code & 7) <= hi).all()
        assert (((code >> 3) == np.signbit(val)) | (np.abs(val) <= slack)).all()
    other = [i for i in range(layers) if i != layer]
    assert np.array_equal(got[:, other], before[:, other])


def test_append_kv4_of_special_values():
    """Zeros, tiny and huge groups, infinities and NaN."""
    hq, hkv, hd = 1, 1, 64
    x = np.zeros((6, 3 * hd), np.float32)
    x[1, 2 * hd:] = 1e-6          # below the smallest scale: zeros
    x[2, 2 * hd:] = 1e6           # above the largest: 6 * 448
    x[3, 2 * hd + 5] = np.inf     # group 0 of row 3
    x[4, 2 * hd + 20] = np.nan    # group 1 of row 4
    x[5, 2 * hd:] = -0.0
    qkv = torch.from_numpy(x).cuda().bfloat16()
    cos, sin = O.rope_table(16, hd, 1e6)
    pool = L.alloc_kv4_pool(1, 1, 1, hd)
    q_out = torch.zeros(6, hd, dtype=torch.bfloat16, device="cuda")
    rows = torch.arange(6, dtype=torch.int32, device="cuda")
    L.qk_norm_rope_append_kv4(q_out, qkv, rows, rows, to_device(cos), to_device(sin), pool, 1, 1,
                              0, hq, hkv, hd)
    got = R.unpack(from_device(pool)[0, 0, 0, R.half_bytes(hd):], hd, 1.0)
    assert not got[[0, 1, 5]].any()
    assert (got[2] == 2688.0).all()
    assert np.isnan(got[3, :16]).all() and not got[3, 16:].any()
    assert np.isnan(got[4, 16:32]).all() and not got[4, :16].any() and not got[4, 32:].any()


def test_append_kv4_skips_padding_and_reports_bad_rows():
    hq, hkv, hd, nb = 2, 1, 64, 2
    rng = np.random.default_rng(4)
    qkv = to_device(randn_bf16(rng, (6, 4 * hd)))
    cos, sin = O.rope_table(32, hd, 1e6)
    cos, sin = to_device(cos), to_device(sin)

    def run(pos, slot):
        pool = L.alloc_kv4_pool(nb, 1, 1, hd)
        q_out = torch.full((6, hq * hd), 7.0, dtype=torch.bfloat16, device="cuda")
        st = status_word()
        L.qk_norm_rope_append_kv4(q_out, qkv, to_device(np.array(pos, np.int32)),
                                  to_device(np.array(slot, np.int32)), cos, sin, pool, nb, 1, 0,
                                  hq, hkv, hd, dev_status=st)
        data = from_device(pool)[:, 0, 0, :16 * hd // 2].reshape(nb * 16, hd // 2)
        return (q_out == 7.0).all(1).cpu().numpy(), data.any(1), int(st.item())
    kept, stored, word = run([0, 1, 2, -1, 4, 5], [3, -1, 4, 5, 6, 31])
    assert word == 0
    assert kept.tolist() == [False, False, False, True, False, False]
    assert np.flatnonzero(stored).tolist() == [3, 4, 6, 31]
    kept, stored, word = run([0, 32, -2, 3, 4, 5], [3, 4, 5, 32, -2, 6])
    assert word == L.LC_DEV_BAD_POS | L.LC_DEV_BAD_BLOCK
    assert kept.tolist() == [False, True, True, False, False, False]
    assert np.flatnonzero(stored).tolist() == [3, 6]


# ----------------------------------------------------------------- unpack --

@pytest.mark.parametrize("hkv,hd,g", [(2, 64, (1.0, 0.25)), (4, 128, (0.5, 0.3)), (1, 128, (1, 1))])
def test_unpack_kv4(hkv, hd, g):
    rng = np.random.default_rng(hd + hkv)
    lens = np.array([0, 1, 15, 16, 17, 100, 63], np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng, table_stride=9)
    layers, layer = 2, 1
    pool = R.make_pool(rng, nb, layers, hkv, hd, *g)
    pool[:, :, :, R.half_bytes(hd) - 1] = 0x7f  # token 15 of K: a NaN scale
    bad = 5
    tables[bad, 2] = nb + 7
    P = R.ceil16(100)
    out = [torch.full((len(lens) * P, 1, hkv, 16, hd), 3.0, dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    st = status_word()
    L.unpack_kv4(*out, to_device(pool), nb, layers, layer, hkv, hd, to_device(tables),
                 to_device(lens), 100, k_scale=g[0], v_scale=g[1], dev_status=st)
    assert int(st.item()) == L.LC_DEV_BAD_BLOCK
    hb = R.half_bytes(hd)
    for half, (o, s) in enumerate(zip(out, g)):
        got = R.bf16_f64(from_device(o)).reshape(len(lens), P, hkv, 16, hd)
        for b, n in enumerate(lens):
            for j in range(P):
                if j * 16 >= n:
                    assert (got[b, j] == 3.0).all()
                    continue
                if b == bad and j == 2:
                    assert not got[b, j].any()
                    continue
                want = R.unpack(pool[tables[b, j], layer, :, half * hb:(half + 1) * hb], hd,
                                np.float64(np.float32(s)))
                want[:, max(0, n - j * 16):] = 0.0
                want = R.bf16_round(want.astype(np.float32))
                assert np.array_equal(got[b, j], want, equal_nan=True)


# ----------------------------------------------------------------- decode --

def run_decode(q, pool, layer, tables, lens, hkv, hd, tokens=1, g=(1.0, 1.0), hint=0, pad=(0, 0),
               offset=0, ws=None, sm_scale=None, st=None):
    rows, hq, _ = q.shape
    batch = rows // tokens
    qd = torch.zeros(rows, hq * hd + pad[0], dtype=torch.bfloat16, device="cuda")
    qd[:, :hq * hd] = to_device(q.reshape(rows, -1))
    # `offset` elements in: an output that is only 2-byte aligned
    flat = torch.full((rows * (hq * hd + pad[1]) + offset,), 9.0, dtype=torch.bfloat16,
                      device="cuda")
    out = flat[offset:].view(rows, hq * hd + pad[1])
    ws = ws if ws is not None else L.alloc_decode_kv4_workspace(batch, hq, hkv, hd, tokens)
    L.paged_decode_kv4(out, qd, to_device(pool) if isinstance(pool, np.ndarray) else pool,
                       pool.shape[0], pool.shape[1], layer, hq, hkv, hd, to_device(tables),
                       to_device(lens), hint, tokens, *g, sm_scale=sm_scale, workspace=ws,
                       dev_status=st)
    torch.cuda.synchronize()
    assert (out[:, hq * hd:] == 9.0).all()
    return R.bf16_f64(from_device(out[:, :hq * hd].contiguous())).reshape(rows, hq, hd)


def check_decode(hq, hkv, hd, lens, tokens=1, g=(1.0, 0.25), seed=0, q_std=1.0, hint=0, **kw):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    pages = np.array([R.ceil16(n) for n in lens])
    tables, nb = make_tables(pages, rng, table_stride=max(1, pages.max()) + 1)
    pool = R.make_pool(rng, nb, 2, hkv, hd, *g)
    for b, n in enumerate(lens):  # what lies past the last token is not a number
        if n % 16:
            half = pool[tables[b, n // 16]].reshape(2, hkv, 2, -1)
            half[..., 16 * hd // 2 + n % 16 * (hd // 16):] = 0x7f
    q = O.f32_to_bf16((rng.standard_normal((len(lens) * tokens, hq, hd)) * q_std).astype(np.float32))
    st = status_word()
    got = run_decode(q, pool, 1, tables, lens, hkv, hd, tokens, g, hint, st=st, **kw)
    assert int(st.item()) == 0
    want, bound = R.decode(R.bf16_f64(q), pool, 1, tables, lens, hkv, hd, tokens, *g)
    bad = ~R.rounds_to(got, want, bound)
    assert not bad.any(), f"{bad.sum()} off, first at {np.argwhere(bad)[0]}"


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (14, 2), (8, 8), (5, 1), (16, 1), (27, 3), (40, 2)])
def test_decode_head_layouts(hq, hkv, hd):
    check_decode(hq, hkv, hd, [1, 16, 17, 0, 200, 77], seed=hq + hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 129, 255, 513, 1000, 2049])
def test_decode_single_sequence_lengths(n, hd):
    check_decode(14, 2, hd, [n], seed=n)
    check_decode(14, 2, hd, [n], seed=n, hint=n)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [2, 3, 5, 9])
def test_decode_several_tokens(tokens, hd):
    # contexts shorter than the tokens leave rows empty
    check_decode(14, 2, hd, [0, 1, 2, tokens - 1, tokens, 40, 300, 16 * 9], tokens=tokens, seed=tokens)
    check_decode(6, 6, hd, [tokens, 130], tokens=tokens, seed=tokens, hint=130)


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_ragged_batch_and_hints(hd):
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 900, 70)
    lens[::9] = 0
    check_decode(14, 2, hd, lens, seed=6)
    check_decode(14, 2, hd, lens, seed=6, hint=int(lens.max()))
    check_decode(14, 2, hd, lens, seed=6, hint=8)  # a hint that is too short is only a hint
    check_decode(14, 2, hd, np.zeros(3), seed=7)


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_sharp_and_large_scores(hd):
    check_decode(14, 2, hd, [700, 33, 5], seed=8, q_std=30.0)
    check_decode(14, 2, hd, [300], seed=9, q_std=1e-3)
    check_decode(14, 2, hd, [300], seed=10, g=(0.37, 1e-3))


def test_decode_strides_and_alignment():
    for pad, offset in (((8, 8), 0), ((0, 3), 1), ((64, 2), 2), ((8, 1), 0)):
        check_decode(14, 2, 64, [100, 17, 0], seed=11, pad=pad, offset=offset)
        check_decode(12, 2, 128, [100, 17, 0], seed=11, tokens=2, pad=pad, offset=offset)


def test_decode_rising_scores():
    """Scores that grow along the context, so that every later page raises the maximum."""
    hq, hkv, hd, n = 8, 1, 64, 640
    rng = np.random.default_rng(12)
    tables, nb = make_tables(np.array([n // 16]), rng)
    k = np.zeros((nb, 1, hkv, 16, hd))
    for j, page in enumerate(tables[0]):
        k[page, 0, 0, :, 0] = (np.arange(16) + 16 * j) * 0.75
    v = rng.standard_normal(k.shape)
    pool = np.concatenate([R.pack(k, 1.0), R.pack(v, 1.0)], -1)
    q = np.zeros((1, hq, hd), np.float32)
    q[0, :, 0] = [8.0, 4.0, 1.0, 0.0, -1.0, -4.0, -8.0, 0.25]
    q = O.f32_to_bf16(q)
    lens = np.array([n], np.int32)
    got = run_decode(q, pool, 0, tables, lens, hkv, hd)
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1, 1.0, 1.0)
    assert R.rounds_to(got, want, bound).all()


def test_decode_of_what_is_not_finite():
    """A NaN key or value reaches exactly the rows that see it."""
    hq, hkv, hd, tokens = 4, 2, 64, 3
    rng = np.random.default_rng(13)
    lens = np.array([40, 40, 40], np.int32)
    tables, nb = make_tables(np.array([3, 3, 3]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0)
    hb, n = R.half_bytes(hd), 16 * hd // 2
    # sequence 0: K of its last token (39), head 1: only the last query row sees it
    pool[tables[0, 2], 0, 1, n + 7 * (hd // 16)] = 0x7f
    # sequence 1: V group 2 of token 20, head 0: every row; V group 0 of token 38, head 1:
    # not the first query row
    pool[tables[1, 1], 0, 0, hb + n + 4 * (hd // 16) + 2] = 0x7f
    pool[tables[1, 2], 0, 1, hb + n + 6 * (hd // 16)] = 0x7f
    q = randn_bf16(rng, (9, hq, hd))
    q[6, 0, 3] = 0x7f80  # an infinite query element of sequence 2
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, tokens)
    nan = np.isnan(got)
    want = np.zeros_like(nan)
    want[2, 2:] = True
    want[3:6, :2, 32:48] = True
    want[4:6, 2:, :16] = True
    want[6, 0] = True
    assert np.array_equal(nan, want)


def test_decode_reports_bad_pages_and_lengths():
    hq, hkv, hd = 14, 2, 64
    rng = np.random.default_rng(14)
    lens = np.array([100, 50], np.int32)
    tables, nb = make_tables(np.array([7, 4]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0)
    tables[0, 3], tables[1, 0] = nb, -5
    q = randn_bf16(rng, (2, hq, hd))
    st = status_word()
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, st=st)
    assert int(st.item()) == L.LC_DEV_BAD_BLOCK
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1, 1.0, 1.0)
    assert R.rounds_to(got, want, bound).all()
    st = status_word()
    run_decode(q, pool, 0, tables, np.array([100, 7 * 16 + 1], np.int32), hkv, hd, st=st)
    assert int(st.item()) & L.LC_DEV_BAD_POS


def test_decode_repeats_bit_for_bit_and_leaves_the_workspace_zero():
    hq, hkv, hd = 14, 2, 128
    rng = np.random.default_rng(15)
    lens = rng.integers(1, 3000, 9).astype(np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    pool = to_device(R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0))
    q = randn_bf16(rng, (9, hq, hd))
    ws = L.alloc_decode_kv4_workspace(9, hq, hkv, hd)
    first = run_decode(q, pool, 0, tables, lens, hkv, hd, ws=ws)
    for _ in range(5):
        assert np.array_equal(run_decode(q, pool, 0, tables, lens, hkv, hd, ws=ws), first)


def test_decode_pool_beyond_32_bit_offsets():
    """Pages past 4 GiB of the pool; only those are written."""
    hq, hkv, hd, n = 8, 8, 128, 70
    rng = np.random.default_rng(16)
    layers = 4
    nb = (5 << 30) // (layers * hkv * 18 * hd)
    pool = torch.empty(nb, layers, hkv, 18 * hd, dtype=torch.uint8, device="cuda")
    small = R.make_pool(rng, 5, layers, hkv, hd, 1.0, 0.25)
    pool[nb - 5:] = to_device(small)
    tables = np.array([[nb - 1, nb - 3, nb - 5, nb - 2, nb - 4]], np.int32)
    lens = np.array([n], np.int32)
    q = randn_bf16(rng, (1, hq, hd))
    got = run_decode(q, pool, 3, tables, lens, hkv, hd, g=(1.0, 0.25))
    want, bound = R.decode(R.bf16_f64(q), small, 3, tables - (nb - 5), lens, hkv, hd, 1, 1.0, 0.25)
    assert R.rounds_to(got, want, bound).all()


def test_decode_on_another_stream_and_in_a_graph():
    hq, hkv, hd = 14, 2, 64
    rng = np.random.default_rng(17)
    lens = np.array([500, 20, 333], np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0)
    q = randn_bf16(rng, (3, hq, hd))
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1, 1.0, 1.0)
    d = [to_device(a) for a in (q.reshape(3, -1), pool, tables, lens)]
    out = torch.zeros(3, hq * hd, dtype=torch.bfloat16, device="cuda")
    ws = L.alloc_decode_kv4_workspace(3, hq, hkv, hd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def call(stream=None):
        L.paged_decode_kv4(out, d[0], d[1], nb, 1, 0, hq, hkv, hd, d[2], d[3], 500, workspace=ws,
                           stream=stream)
    call(side)
    torch.cuda.current_stream().wait_stream(side)
    got = R.bf16_f64(from_device(out)).reshape(3, hq, hd)
    assert R.rounds_to(got, want, bound).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(R.bf16_f64(from_device(out)).reshape(3, hq, hd), got)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hq,hkv,tokens", [(14, 2, 1), (16, 2, 2), (8, 1, 3), (16, 2, 5), (3, 3, 11)])
def test_decode_long_contexts_over_many_ctas(hq, hkv, tokens, hd):
    """Segments split over CTAs, for 8, 16 and 24 columns at a time and several slices."""
    check_decode(hq, hkv, hd, [2500, 0, 700, 33, 1601], tokens=tokens, seed=hq + tokens)
    check_decode(hq, hkv, hd, [3333], tokens=tokens, seed=hq + tokens, hint=3333)


def test_decode_many_short_sequences():
    """CTAs with many segments each."""
    rng = np.random.default_rng(21)
    check_decode(4, 2, 64, rng.integers(0, 40, 600), seed=22)
    check_decode(8, 1, 128, rng.integers(1, 20, 900), seed=23, hint=19)


@pytest.mark.parametrize("n", [2304, 2305, 4608, 4609, 7003, 9216, 9217])
def test_decode_one_sequence_in_several_rounds(n):
    """Around the lengths from which each CTA works through one more round of pages."""
    check_decode(32, 32, 64, [n], seed=n)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [2300, 4100, 4352, 8300, 8704, 20000])
def test_decode_one_sequence_of_many_pieces(n, hd):
    """9 to 79 pieces per head, around the 16 and 32 that are joined at a time."""
    check_decode(4, 2, hd, [n], seed=n)


def test_decode_one_sequence_of_more_heads_than_ctas():
    check_decode(300, 300, 64, [41], seed=5)


@pytest.mark.parametrize("mode", [1, 2])
def test_decode_with_dependent_launch(mode):
    """An append and the decode over it, back to back: the same bits in every launch mode."""
    hq, hkv, hd, b = 14, 2, 64, 6
    rng = np.random.default_rng(24)
    lens = rng.integers(200, 900, b).astype(np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    base = to_device(R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0))
    cos, sin = (to_device(t) for t in O.rope_table(1024, hd, 1e6))
    qkv = to_device(randn_bf16(rng, (b, (hq + 2 * hkv) * hd)))
    pos = lens - 1
    slot = to_device((tables[np.arange(b), pos // 16] * 16 + pos % 16).astype(np.int32))
    pos, lens_d, tables_d = to_device(pos), to_device(lens), to_device(tables)
    ws = L.alloc_decode_kv4_workspace(b, hq, hkv, hd)

    def run():
        pool = base.clone()
        q = torch.zeros(b, hq * hd, dtype=torch.bfloat16, device="cuda")
        outs = []
        for _ in range(4):
            L.qk_norm_rope_append_kv4(q, qkv, pos, slot, cos, sin, pool, nb, 1, 0, hq, hkv, hd)
            outs.append(torch.zeros_like(q))
            L.paged_decode_kv4(outs[-1], q, pool, nb, 1, 0, hq, hkv, hd, tables_d, lens_d, 900,
                               workspace=ws)
        torch.cuda.synchronize()
        return outs
    want = run()
    old = L.set_dependent_launch(mode)
    try:
        got = run()
    finally:
        L.set_dependent_launch(old)
    for x in got + want:
        assert torch.equal(x, want[0])
