"""The 8-bit cache on the GPU: append (lc_qk_norm_rope_append_kv8), unpack (lc_unpack_kv8)
and decode attention (lc_paged_decode_kv8) against float64."""
import numpy as np
import pytest

import kv8_ref as R
import lucciola as L
import oracle.oracle as O
from workloads import from_device, make_tables, randn_bf16, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------- append --

def run_append(qkv, pos, slot, pool, layer, hq, hkv, hd, vec, cos, sin, q_out=None):
    """(q bits [rows, hq * hd + 16], pool bytes, status word) after the call."""
    st = status_word()
    pool_d = to_device(pool)
    if q_out is None:
        q_out = torch.zeros(len(pos), hq * hd + 16, dtype=torch.bfloat16, device="cuda")
    L.qk_norm_rope_append_kv8(
        q_out, to_device(qkv), to_device(pos), to_device(slot), to_device(cos), to_device(sin),
        pool_d, pool.shape[0], pool.shape[1], layer, hq, hkv, hd, eps=1e-6, dev_status=st,
        **{k: None if v is None else to_device(v) for k, v in vec.items()})
    return from_device(q_out), from_device(pool_d), int(st.item())


def reference_rows(qkv, pos, hq, hkv, hd, vec, cos, sin):
    """float64 q, k (with |y1| + |y2| per dim) and v of every row; negative positions as 0."""
    f = {k: None if v is None else R.bf16_f64(v) for k, v in vec.items()}
    x = R.bf16_f64(qkv)[:, :(hq + 2 * hkv) * hd].reshape(len(pos), -1, hd)
    at = np.clip(pos, 0, len(cos) - 1)
    c, s = cos.astype(np.float64)[at], sin.astype(np.float64)[at]

    def bias(name):
        return None if f[name] is None else f[name].reshape(-1, hd)
    q = R.norm_rope(x[:, :hq], bias("q_bias"), f["q_norm"], 1e-6, c, s)
    k = R.norm_rope(x[:, hq:hq + hkv], bias("k_bias"), f["k_norm"], 1e-6, c, s)
    v = x[:, hq + hkv:]
    if f["v_bias"] is not None:  # one fp32 sum
        v = (v + bias("v_bias")).astype(np.float32).astype(np.float64)
    return q, k, v


def check_append(hq, hkv, hd, runs, norm=False, bias=False, seed=0, nb=None, before=None,
                 edit=None, layers=2, layer=1, pads=0):
    """`runs`: (page, first token, tokens) in row order. Returns what the pool holds after."""
    rng = np.random.default_rng(seed)
    nb = nb or max(p for p, _, _ in runs) + 2
    slot = np.concatenate([[p * 16 + t + i for i in range(n)] for p, t, n in runs]).astype(np.int32)
    rows = len(slot)
    pos = rng.integers(0, 512, rows).astype(np.int32)
    for _ in range(pads):  # padding rows and rows that are not stored, behind the runs
        slot, pos = np.append(slot, [-1, -1]).astype(np.int32), np.append(pos, [-1, 3]).astype(np.int32)
    qkv = randn_bf16(rng, (len(slot), (hq + 2 * hkv) * hd + 8))
    if edit:
        edit(qkv)
    vec = {k: randn_bf16(rng, n * hd) if on else None for k, n, on in (
        ("q_bias", hq, bias), ("k_bias", hkv, bias), ("v_bias", hkv, bias),
        ("q_norm", 1, norm), ("k_norm", 1, norm))}
    cos, sin = O.rope_table(512, hd, 1e6)
    if before is None:
        before = R.make_pool(rng, nb, layers, hkv, hd, spread=3)
    got_q, got, word = run_append(qkv, pos, slot, before, layer, hq, hkv, hd, vec, cos, sin)
    assert word == 0
    (q, q_size), (k, k_size), v = reference_rows(qkv, pos, hq, hkv, hd, vec, cos, sin)
    live = pos >= 0
    # q: one bf16 rounding after fp32 steps (16 of 2^-24 of the terms)
    q64 = R.bf16_f64(got_q)[:, :hq * hd].reshape(q.shape)
    assert R.rounds_to(q64, q, 16 * 2.0 ** -24 * q_size)[live].all()
    assert not got_q[:, hq * hd:].any() and not got_q[~live].any()

    want = before.copy()
    at = 0
    order = R.places(hd)
    for page, first, n in runs:
        offs = np.arange(first, first + n)
        for i, (x, slack) in enumerate(((k, 16 * 2.0 ** -24 * k_size), (v, np.zeros_like(v)))):
            new, d = x[at:at + n].transpose(1, 0, 2), slack[at:at + n].transpose(1, 0, 2)
            old = R.scales(before[page, layer], hd)[:, i]
            after = R.scales(got[page, layer], hd)[:, i]
            finite = np.where(np.isfinite(new), np.abs(new), 0.0)
            lo = 2.0 ** R.exponent(np.maximum(finite - d, 0).max((1, 2)))
            hi = 2.0 ** R.exponent((finite + d).max((1, 2)))
            if first:
                lo, hi = np.maximum(lo, old), np.maximum(hi, old)
            assert ((lo <= after) & (after <= hi)).all()
            step = after[:, None, None]
            values = R.VALUES[R.codes(got[page, layer], hd, i)][:, offs]
            with np.errstate(invalid="ignore"):
                low, high = R.round8((new - d) / step), R.round8((new + d) / step)
                good = (low <= values) & (values <= high)
            good |= ~np.isfinite(new) & np.isnan(values)
            assert good.all(), (page, i, np.argwhere(~good)[:4])
            # the page's other tokens: as they were, or rounded to the larger scale
            rest = np.setdiff1d(np.arange(16), offs)
            was = R.codes(before[page, layer], hd, i)[:, rest]
            now = R.codes(got[page, layer], hd, i)[:, rest]
            same = (was == now).all((1, 2))
            if first:
                moved = R.round8(R.VALUES[was] * old[:, None, None] / step)
                assert np.array_equal(R.VALUES[now], moved, equal_nan=True)
                assert same[after == old].all()
            else:  # a page begun anew: nothing but the run and the scale is written
                assert same.all()
            # all that the call may have written
            flat = want[page, layer, :, i * 16 * hd:(i + 1) * 16 * hd]
            flat[:] = got[page, layer, :, i * 16 * hd:(i + 1) * 16 * hd]
            want[page, layer, :, 32 * hd + 4 * i:32 * hd + 4 * i + 4] = \
                got[page, layer, :, 32 * hd + 4 * i:32 * hd + 4 * i + 4]
        at += n
    assert np.array_equal(got, want) and order.size
    return got


@pytest.mark.parametrize("hq,hkv,hd", [(14, 2, 64), (28, 4, 128), (1, 1, 128), (9, 3, 64), (8, 8, 128)])
@pytest.mark.parametrize("norm,bias", [(True, False), (False, True), (True, True), (False, False)])
def test_append_head_layouts(hq, hkv, hd, norm, bias):
    check_append(hq, hkv, hd, [(3, 0, 16), (1, 5, 11), (0, 0, 3), (5, 7, 1)], norm, bias, seed=hq, pads=2)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("runs", [
    [(0, 0, 1)], [(2, 15, 1)], [(0, 0, 16)], [(1, 3, 13)], [(0, 8, 4)],
    [(p, 0, 16) for p in range(9)],                                  # a prompt
    [(7, 9, 7)] + [(p, 0, 16) for p in (3, 0, 5)] + [(6, 0, 2)],     # a chunk of one
    [(p, p % 16, 1) for p in range(70)],                             # a decode step
    [(p, 3 * p % 14, 1 + p % 3) for p in range(50)],                 # drafted tokens
    [(0, 14, 2), (1, 0, 16), (2, 0, 1), (9, 4, 1), (8, 0, 5), (4, 1, 15), (5, 0, 16), (6, 0, 9)],
], ids=lambda r: f"{len(r)}-{sum(n for _, _, n in r)}")
def test_append_runs(runs, hd):
    check_append(6, 2, hd, runs, norm=True, seed=len(runs))


@pytest.mark.parametrize("hd", [64, 128])
def test_append_many_rows(hd):
    """Enough rows for the widest windows, prompts and decoding sequences mixed."""
    rng = np.random.default_rng(4)
    runs, page = [], 0
    while sum(n for _, _, n in runs) < 6000:
        first = int(rng.integers(0, 16))
        n = int(rng.integers(1, 17 - first)) if rng.random() < 0.5 else 16 - first
        runs.append((page, first, n))
        page += 1
    check_append(4, 4, hd, runs, seed=5)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_moves_a_page_to_a_larger_scale(hd):
    """A large row after small ones, small ones after a large row, zeros, and a first token."""
    nb, hkv = 6, 2
    rng = np.random.default_rng(6)
    before = R.make_pool(rng, nb, 2, hkv, hd, k_std=1e-3, v_std=1e-5)
    runs = [(0, 4, 1), (1, 0, 2), (2, 15, 1), (3, 6, 9), (4, 1, 1)]
    got = check_append(4, hkv, hd, runs, seed=7, before=before, nb=nb)
    assert (R.scales(got[0, 1], hd) > R.scales(before[0, 1], hd)).all()
    large = R.make_pool(rng, nb, 2, hkv, hd, k_std=1e4, v_std=1e6)
    got = check_append(4, hkv, hd, runs, seed=8, before=large, nb=nb)
    assert np.array_equal(R.scales(got[0, 1], hd), R.scales(large[0, 1], hd))
    assert (R.scales(got[1, 1], hd) < R.scales(large[1, 1], hd)).all()  # begun anew

    def zeros(qkv):
        qkv[:] = 0
    got = check_append(4, hkv, hd, runs, seed=9, before=before, nb=nb, edit=zeros)
    assert (R.scales(got[1, 1], hd) == 2.0 ** R.E_MIN).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_what_is_not_finite_and_of_the_largest(hd):
    hq, hkv = 2, 2

    def edit(qkv):
        row = qkv[:, hq * hd:(hq + 2 * hkv) * hd]
        row[3, 5], row[4, hd // 2 + 9], row[20, 2 * hd + 1] = 0x7f80, 0xffc0, 0xff80  # K, K, V
        row[9, 3 * hd:] = 0x7f7f  # a head of V at bf16's largest value
        row[10, 3 * hd + 1] = 0xff7f
    runs = [(0, 0, 6), (2, 3, 8), (1, 0, 16)]

    def no_rotation(qkv):
        edit(qkv)
    # K: an infinite pair of dims becomes NaN through the rotation as well; only V's are
    # compared element by element here
    rng = np.random.default_rng(3)
    nb = 4
    slot = np.concatenate([[p * 16 + t + i for i in range(n)] for p, t, n in runs]).astype(np.int32)
    pos = np.zeros(len(slot), np.int32)
    qkv = randn_bf16(rng, (len(slot), (hq + 2 * hkv) * hd))
    no_rotation(qkv)
    vec = dict.fromkeys(("q_bias", "k_bias", "v_bias", "q_norm", "k_norm"))
    cos, sin = np.ones((1, hd // 2), np.float32), np.zeros((1, hd // 2), np.float32)
    before = R.make_pool(rng, nb, 1, hkv, hd)
    _, got, word = run_append(qkv, pos, slot, before, 0, hq, hkv, hd, vec, cos, sin)
    assert word == 0
    x = R.bf16_f64(qkv).reshape(len(slot), -1, hd)
    for i in range(2):
        for h in range(hkv):
            rows = x[:, hq + i * hkv + h]
            vals = R.VALUES[R.codes(got[slot // 16, 0, h], hd, i)][np.arange(len(slot)), slot % 16]
            scale = R.scales(got[slot // 16, 0, h], hd)[:, i]
            want = R.round8(rows / scale[:, None])
            if i == 0:  # an infinite or NaN dim makes its partner inf * 0 = NaN
                odd = ~np.isfinite(rows)
                want[odd | np.roll(odd, hd // 2, -1)] = np.nan
            assert np.array_equal(vals, want, equal_nan=True)
    # 0x7f7f: above 448 * 2^40, held at the largest scale
    assert R.scales(got[2, 0, 1], hd)[1] == 2.0 ** 40


def test_append_in_place_padding_and_bad_rows():
    """q_out over the qkv rows; rows that are not stored, positions and slots out of range."""
    hq, hkv, hd, nb = 6, 2, 64, 4
    rng = np.random.default_rng(11)
    cos, sin = O.rope_table(64, hd, 1e6)
    pos = np.array([0, 1, 5, -1, 64, 7, -3, 63], np.int32)
    slot = np.array([16, 17, -1, 40, 18, nb * 16, 20, 48], np.int32)
    qkv = randn_bf16(rng, (8, (hq + 2 * hkv) * hd))
    vec = dict.fromkeys(("q_bias", "k_bias", "v_bias", "q_norm", "k_norm"))
    before = R.make_pool(rng, nb, 1, hkv, hd)
    st = status_word()
    rows, pool = to_device(qkv), to_device(before)
    L.qk_norm_rope_append_kv8(rows, rows, to_device(pos), to_device(slot), to_device(cos),
                              to_device(sin), pool, nb, 1, 0, hq, hkv, hd, dev_status=st)
    assert int(st.item()) == L.LC_DEV_BAD_POS | L.LC_DEV_BAD_BLOCK
    got, got_q = from_device(pool), from_device(rows)
    (q, size), _, v = reference_rows(qkv, pos, hq, hkv, hd, vec, cos, sin)
    done = (pos >= 0) & (pos < 64)
    q64 = R.bf16_f64(got_q)[:, :hq * hd].reshape(q.shape)
    assert R.rounds_to(q64, q, 16 * 2.0 ** -24 * size)[done].all()
    assert np.array_equal(got_q[~done], qkv[~done])
    assert np.array_equal(got_q[:, hq * hd:], qkv[:, hq * hd:])
    # pages 1 (rows 0 and 1) and 3 (row 7) are written, nothing else
    assert np.array_equal(got[[0, 2]], before[[0, 2]])
    for row, s in ((0, 16), (1, 17), (7, 48)):
        page = got[s // 16, 0]
        step = R.scales(page, hd)[:, 1]
        vals = R.VALUES[R.codes(page, hd, 1)][:, s % 16]
        assert np.array_equal(vals, R.round8(v[row] / step[:, None]))
    assert np.array_equal(R.codes(got[1, 0], hd, 1)[:, 2:], R.codes(before[1, 0], hd, 1)[:, 2:])


@pytest.mark.parametrize("hd", [64, 128])
def test_append_with_bad_positions_inside_a_page(hd):
    """Rows without a place in the RoPE tables are left alone; their page's other rows are
    held as if they were not there, at one scale."""
    hq, hkv, nb = 2, 2, 8
    rng = np.random.default_rng(14)
    cos, sin = O.rope_table(64, hd, 1e6)
    vec = dict.fromkeys(("q_bias", "k_bias", "v_bias", "q_norm", "k_norm"))
    slot = np.array([32, 33, 34, 35, 36, 69, 70, 71, 100, 101, 7, 112, 48, 49], np.int32)
    pos = np.array([0, 64, 2, 99, 4, -7, 6, 7, 64, 64, 3, 70, 64, 1], np.int32)
    qkv = randn_bf16(rng, (len(slot), (hq + 2 * hkv) * hd))
    qkv[[1, 3, 5, 8, 9, 11, 12]] = 0x5000  # large, and not looked at
    before = R.make_pool(rng, nb, 1, hkv, hd)
    _, got, word = run_append(qkv, pos, slot, before, 0, hq, hkv, hd, vec, cos, sin)
    assert word == L.LC_DEV_BAD_POS
    keep = (pos >= 0) & (pos < 64)
    _, want, word = run_append(qkv[keep], pos[keep], slot[keep], before, 0, hq, hkv, hd, vec, cos, sin)
    assert word == 0 and np.array_equal(got, want)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_leaves_out_rows_that_do_not_rise(hd):
    """The same slot twice, and a falling one: the page keeps the rows before."""
    hq, hkv, nb = 2, 1, 8
    rng = np.random.default_rng(12)
    cos, sin = O.rope_table(64, hd, 1e6)
    vec = dict.fromkeys(("q_bias", "k_bias", "v_bias", "q_norm", "k_norm"))
    slot = np.array([32, 33, 33, 34, 16, 70, 69, 71] + list(range(96, 112)) + [111, 0], np.int32)
    pos = np.arange(len(slot)).astype(np.int32)
    qkv = randn_bf16(rng, (len(slot), (hq + 2 * hkv) * hd))
    before = R.make_pool(rng, nb, 1, hkv, hd)
    _, got, word = run_append(qkv, pos, slot, before, 0, hq, hkv, hd, vec, cos, sin)
    assert word == L.LC_DEV_BAD_BLOCK
    keep = np.ones(len(slot), bool)
    keep[[2, 3, 6, 7, 24]] = False
    _, want, word = run_append(qkv[keep], pos[keep], slot[keep], before, 0, hq, hkv, hd, vec, cos, sin)
    assert word == 0 and np.array_equal(got, want)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_token_by_token_holds_what_a_prompt_holds(hd):
    """A page filled by decode steps has the prompt's scale; its codes differ by a second
    rounding of what was small at most."""
    hq, hkv, nb = 2, 2, 2
    rng = np.random.default_rng(13)
    cos, sin = O.rope_table(64, hd, 1e6)
    vec = dict.fromkeys(("q_bias", "k_bias", "v_bias", "q_norm", "k_norm"))
    qkv = randn_bf16(rng, (16, (hq + 2 * hkv) * hd))
    slot, pos = np.arange(16, 32).astype(np.int32), np.arange(16).astype(np.int32)
    empty = np.full((nb, 1, hkv, R.page_bytes(hd)), 0xff, np.uint8)  # what a page held before
    _, whole, _ = run_append(qkv, pos, slot, empty, 0, hq, hkv, hd, vec, cos, sin)
    pool = empty
    for r in range(16):
        _, pool, word = run_append(qkv[r:r + 1], pos[r:r + 1], slot[r:r + 1], pool, 0, hq, hkv, hd,
                                   vec, cos, sin)
        assert word == 0
    assert np.array_equal(R.scales(pool[1], hd), R.scales(whole[1], hd))
    for i in range(2):
        a, b = R.unpack(pool[1], hd, i), R.unpack(whole[1], hd, i)
        step = R.scales(whole[1], hd)[..., i, None, None] * 2.0 ** -9  # e4m3's smallest
        assert (np.abs(a - b) <= step).all()


# ----------------------------------------------------------------- unpack --

@pytest.mark.parametrize("hkv,hd", [(2, 64), (4, 128), (1, 64)])
@pytest.mark.parametrize("offset", [0, 1])
def test_unpack_kv8(hkv, hd, offset):
    rng = np.random.default_rng(31)
    lens = np.array([0, 1, 15, 16, 33, 90], np.int32)
    pages = np.array([R.ceil16(n) for n in lens])
    tables, nb = make_tables(pages, rng, table_stride=8)
    pool = R.make_pool(rng, nb, 3, hkv, hd, spread=6)
    R.spoil(pool, tables, lens, hkv, hd)
    longest = 100
    per = R.ceil16(longest)
    out = [torch.full((len(lens) * per, 1, hkv, 16, hd), 5.0, dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    st = status_word()
    tables[5, 2] = nb  # reads as zeros
    L.unpack_kv8(*out, to_device(pool), nb, 3, 2, hkv, hd, to_device(tables),
                 to_device(lens - offset), longest, len_offset=offset, dev_status=st)
    assert int(st.item()) == L.LC_DEV_BAD_BLOCK
    for i in range(2):
        got = R.bf16_f64(from_device(out[i])).reshape(len(lens), per, hkv, 16, hd)
        for b, n in enumerate(lens):
            want = np.full((per, hkv, 16, hd), 5.0)
            if pages[b]:
                ids = tables[b, :pages[b]]
                vals = R.unpack(pool[np.where(ids < nb, ids, 0), 2], hd, i)
                vals[ids >= nb] = 0.0
                if n % 16:
                    vals[-1, :, n % 16:] = 0.0
                want[:pages[b]] = vals
            assert np.array_equal(got[b], want)


def test_unpack_kv8_lengths_beyond_the_output():
    hkv, hd = 2, 64
    rng = np.random.default_rng(32)
    tables, nb = make_tables(np.array([4]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)
    out = [torch.zeros(2, 1, hkv, 16, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    st = status_word()
    L.unpack_kv8(*out, to_device(pool), nb, 1, 0, hkv, hd, to_device(tables),
                 to_device(np.array([60], np.int32)), 32, dev_status=st)
    assert int(st.item()) == L.LC_DEV_BAD_POS
    for i in range(2):
        assert np.array_equal(R.bf16_f64(from_device(out[i]))[:, 0], R.unpack(pool[tables[0, :2], 0], hd, i))


# ----------------------------------------------------------------- decode --

def run_decode(q, pool, layer, tables, lens, hkv, hd, tokens=1, hint=0, pad=(0, 0), offset=0,
               ws=None, sm_scale=None, st=None):
    rows, hq, _ = q.shape
    batch = rows // tokens
    qd = torch.zeros(rows, hq * hd + pad[0], dtype=torch.bfloat16, device="cuda")
    qd[:, :hq * hd] = to_device(q.reshape(rows, -1))
    # `offset` elements in: an output that is only 2-byte aligned
    flat = torch.full((rows * (hq * hd + pad[1]) + offset,), 9.0, dtype=torch.bfloat16,
                      device="cuda")
    out = flat[offset:].view(rows, hq * hd + pad[1])
    ws = ws if ws is not None else L.alloc_decode_kv8_workspace(batch, hq, hkv, hd, tokens)
    L.paged_decode_kv8(out, qd, to_device(pool) if isinstance(pool, np.ndarray) else pool,
                       pool.shape[0], pool.shape[1], layer, hq, hkv, hd, to_device(tables),
                       to_device(lens), hint, tokens, sm_scale=sm_scale, workspace=ws,
                       dev_status=st)
    torch.cuda.synchronize()
    assert (out[:, hq * hd:] == 9.0).all()
    return R.bf16_f64(from_device(out[:, :hq * hd].contiguous())).reshape(rows, hq, hd)


def check_decode(hq, hkv, hd, lens, tokens=1, seed=0, q_std=1.0, hint=0, spread=2, sm_scale=None, **kw):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    pages = np.array([R.ceil16(n) for n in lens])
    tables, nb = make_tables(pages, rng, table_stride=max(1, pages.max()) + 1)
    pool = R.make_pool(rng, nb, 2, hkv, hd, spread=spread, k_std=2.0 ** -spread)
    R.spoil(pool, tables, lens, hkv, hd)
    q = O.f32_to_bf16((rng.standard_normal((len(lens) * tokens, hq, hd)) * q_std).astype(np.float32))
    st = status_word()
    got = run_decode(q, pool, 1, tables, lens, hkv, hd, tokens, hint, st=st, sm_scale=sm_scale, **kw)
    assert int(st.item()) == 0
    want, bound = R.decode(R.bf16_f64(q), pool, 1, tables, lens, hkv, hd, tokens, sm_scale)
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
    check_decode(14, 2, hd, [300, 40], seed=10, sm_scale=-0.3)


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_of_pages_with_very_different_scales(hd):
    """V scales from 2^-20 to 2^20 about their middle: small values beside large ones."""
    check_decode(14, 2, hd, [700, 33, 5, 64], seed=10, spread=20)
    check_decode(24, 2, hd, [500, 48], tokens=2, seed=11, spread=20)


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
    pool = R.pack(k, rng.standard_normal(k.shape))
    q = np.zeros((1, hq, hd), np.float32)
    q[0, :, 0] = [8.0, 4.0, 1.0, 0.0, -1.0, -4.0, -8.0, 0.25]
    q = O.f32_to_bf16(q)
    lens = np.array([n], np.int32)
    got = run_decode(q, pool, 0, tables, lens, hkv, hd)
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1)
    assert R.rounds_to(got, want, bound).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_of_what_is_not_finite(hd):
    """A NaN key or value reaches exactly the rows (and of a value, the dims) that see it."""
    hq, hkv, tokens = 4, 2, 3
    rng = np.random.default_rng(13)
    lens = np.array([40, 40, 40], np.int32)
    tables, nb = make_tables(np.array([3, 3, 3]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)

    def put(b, token, head, i, dim):
        R.put_code(pool, tables[b, token // 16], 0, head, i, token % 16, dim, hd, 0x7f if dim % 2 else 0xff)
    # sequence 0: K of its last token (39), head 1: only the last query row sees it
    put(0, 39, 1, 0, 5)
    # sequence 1: V of token 20, head 0: every row; V of tokens 38 and 39, head 1: not the
    # first query row, and the last one alone
    for dim in (0, 33, 63):
        put(1, 20, 0, 1, dim)
    for dim in (7, 8, hd - 1):
        put(1, 38, 1, 1, dim)
    put(1, 39, 1, 1, 20)
    q = randn_bf16(rng, (9, hq, hd))
    q[6, 0, 3] = 0x7f80  # an infinite query element of sequence 2
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, tokens)
    nan = np.isnan(got)
    want = np.zeros_like(nan)
    want[2, 2:] = True
    want[3:6, :2, [0, 33, 63]] = True
    want[4:6, 2:, [7, 8, hd - 1]] = True
    want[5, 2:, 20] = True
    want[6, 0] = True
    assert np.array_equal(nan, want)
    clean, bound = R.decode(R.bf16_f64(q), np.where(pool & 0x7f == 0x7f, 0, pool), 0, tables, lens,
                            hkv, hd, tokens)
    assert R.rounds_to(got, clean, bound)[3][:, 1:32].all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,tokens", [(1, 4), (8, 2), (8, 3), (5, 7)])
def test_nan_values_reach_the_drafted_rows_that_see_them(group, tokens, hd):
    """For 8, 16 and 24 columns at a time and several slices: V is NaN in one dim of each of the
    newest tokens."""
    hkv, n = 2, 85
    rng = np.random.default_rng(group + tokens)
    lens = np.array([n, 3, 32], np.int32)
    tables, nb = make_tables(np.array([R.ceil16(k) for k in lens]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)
    R.spoil(pool, tables, lens, hkv, hd)
    q = randn_bf16(rng, (3 * tokens, group * hkv, hd))
    want = np.zeros((3 * tokens, group * hkv, hd), bool)
    for b, held in enumerate(lens):
        for k in range(min(tokens, held)):  # token held - 1 - k
            token, dim = held - 1 - k, (11 * k + 7 * b) % hd
            R.put_code(pool, tables[b, token // 16], 0, k % 2, 1, token % 16, dim, hd, 0xff if k % 3 else 0x7f)
            rows = b * tokens + np.arange(tokens - k - 1, tokens)
            want[rows, k % 2 * group:(k % 2 + 1) * group, dim] = True
    # a row sees `token` if it lies before its end; rows before the first token are zeros
    for b, held in enumerate(lens):
        for i in range(tokens):
            if held - (tokens - 1 - i) <= 0:
                want[b * tokens + i] = False
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, tokens)
    assert np.array_equal(np.isnan(got), want)
    clean = np.where(pool & 0x7f == 0x7f, 0, pool)
    clean[..., 32 * hd:] = pool[..., 32 * hd:]
    ref, bound = R.decode(R.bf16_f64(q), clean, 0, tables, lens, hkv, hd, tokens)
    assert R.rounds_to(got, ref, bound)[~want].all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,first,last", [(1, 0, 1), (33, 32, 33), (700, 96, 128), (700, 0, 256),
                                          (700, 0, 700), (6000, 0, 2000), (6000, 0, 6000)])
def test_nan_keys_reach_every_row_that_sees_them(n, first, last, hd):
    """All that one warp, eight warps, some CTAs or the row sees is NaN."""
    hq, hkv = 4, 2
    rng = np.random.default_rng(n + last)
    lens = np.array([n], np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n)]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)
    for token in range(first, last):
        R.put_code(pool, tables[0, token // 16], 0, 1, 0, token % 16, token % hd, hd, 0x7f)
    q = randn_bf16(rng, (1, hq, hd))
    got = run_decode(q, pool, 0, tables, lens, hkv, hd)
    assert np.isnan(got[0, 2:]).all()
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1)
    assert R.rounds_to(got, want, bound)[0, :2].all()


def test_decode_of_a_scale_that_is_not_a_number():
    """A NaN sm_scale gives NaN, but zeros where a row has no tokens."""
    hq, hkv, hd = 6, 2, 64
    rng = np.random.default_rng(18)
    lens = np.array([50, 0, 3], np.int32)
    tables, nb = make_tables(np.array([4, 0, 1]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)
    got = run_decode(randn_bf16(rng, (3, hq, hd)), pool, 0, tables, lens, hkv, hd,
                     sm_scale=float("nan"))
    assert np.isnan(got[[0, 2]]).all() and not got[1].any()


def test_decode_reports_bad_pages_and_lengths():
    hq, hkv, hd = 14, 2, 64
    rng = np.random.default_rng(14)
    lens = np.array([100, 50], np.int32)
    tables, nb = make_tables(np.array([7, 4]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)
    tables[0, 3], tables[1, 0] = nb, -5
    q = randn_bf16(rng, (2, hq, hd))
    st = status_word()
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, st=st)
    assert int(st.item()) == L.LC_DEV_BAD_BLOCK
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1)
    assert R.rounds_to(got, want, bound).all()
    st = status_word()
    run_decode(q, pool, 0, tables, np.array([100, 7 * 16 + 1], np.int32), hkv, hd, st=st)
    assert int(st.item()) & L.LC_DEV_BAD_POS


def test_decode_repeats_bit_for_bit():
    hq, hkv, hd = 14, 2, 128
    rng = np.random.default_rng(15)
    lens = rng.integers(1, 3000, 9).astype(np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    pool = to_device(R.make_pool(rng, nb, 1, hkv, hd))
    q = randn_bf16(rng, (9, hq, hd))
    ws = L.alloc_decode_kv8_workspace(9, hq, hkv, hd)
    first = run_decode(q, pool, 0, tables, lens, hkv, hd, ws=ws)
    for _ in range(5):
        assert np.array_equal(run_decode(q, pool, 0, tables, lens, hkv, hd, ws=ws), first)


def test_pool_beyond_32_bit_offsets():
    """Pages past 4 GiB of the pool; only those are written."""
    hq, hkv, hd, n = 8, 8, 128, 70
    rng = np.random.default_rng(16)
    layers = 4
    nb = (5 << 30) // (layers * hkv * R.page_bytes(hd))
    pool = torch.empty(nb, layers, hkv, R.page_bytes(hd), dtype=torch.uint8, device="cuda")
    small = R.make_pool(rng, 5, layers, hkv, hd)
    pool[nb - 5:] = to_device(small)
    tables = np.array([[nb - 1, nb - 3, nb - 5, nb - 2, nb - 4]], np.int32)
    lens = np.array([n], np.int32)
    q = randn_bf16(rng, (1, hq, hd))
    got = run_decode(q, pool, 3, tables, lens, hkv, hd)
    want, bound = R.decode(R.bf16_f64(q), small, 3, tables - (nb - 5), lens, hkv, hd, 1)
    assert R.rounds_to(got, want, bound).all()
    # an append and its unpacking out there
    cos, sin = O.rope_table(8, hd, 1e6)
    qkv = to_device(randn_bf16(rng, (1, (hq + 2 * hkv) * hd)))
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    slot = one + (nb - 1) * 16
    L.qk_norm_rope_append_kv8(torch.zeros(1, hq * hd, dtype=torch.bfloat16, device="cuda"), qkv,
                              one, slot, to_device(cos), to_device(sin), pool, nb, layers, 3, hq,
                              hkv, hd)
    out = [torch.zeros(1, 1, hkv, 16, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    L.unpack_kv8(*out, pool, nb, layers, 3, hkv, hd, to_device(tables), one + 1, 16)
    v = qkv[0, (hq + hkv) * hd:].float().view(hkv, hd)
    assert ((out[1][0, 0, :, 0].float() - v).abs() <= v.abs() * 2.0 ** -4 + 2.0 ** -8).all()


def test_decode_on_another_stream_and_in_a_graph():
    hq, hkv, hd = 14, 2, 64
    rng = np.random.default_rng(17)
    lens = np.array([500, 20, 333], np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd)
    q = randn_bf16(rng, (3, hq, hd))
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1)
    d = [to_device(a) for a in (q.reshape(3, -1), pool, tables, lens)]
    out = torch.zeros(3, hq * hd, dtype=torch.bfloat16, device="cuda")
    ws = L.alloc_decode_kv8_workspace(3, hq, hkv, hd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def call(stream=None):
        L.paged_decode_kv8(out, d[0], d[1], nb, 1, 0, hq, hkv, hd, d[2], d[3], 500, workspace=ws,
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


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [2300, 4100, 4352, 8300, 8704, 20000])
def test_decode_one_sequence_of_many_pieces(n, hd):
    check_decode(4, 2, hd, [n], seed=n)


def test_decode_one_sequence_of_more_heads_than_ctas():
    check_decode(300, 300, 64, [41], seed=5)


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_append_and_decode_back_to_back(mode):
    """An append and the decode over it, in every launch mode and twice on two streams: the
    same bits, and those of a fresh decode over the pool that came out."""
    hq, hkv, hd, b = 14, 2, 64, 6
    rng = np.random.default_rng(24)
    lens = rng.integers(200, 900, b).astype(np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    base = to_device(R.make_pool(rng, nb, 1, hkv, hd))
    cos, sin = (to_device(t) for t in O.rope_table(1024, hd, 1e6))
    qkv = to_device(randn_bf16(rng, (b, (hq + 2 * hkv) * hd)))
    pos = lens - 1
    slot = to_device((tables[np.arange(b), pos // 16] * 16 + pos % 16).astype(np.int32))
    pos, lens_d, tables_d = to_device(pos), to_device(lens), to_device(tables)

    def run(ws):
        pool = base.clone()
        q = torch.zeros(b, hq * hd, dtype=torch.bfloat16, device="cuda")
        outs = []
        for _ in range(4):
            L.qk_norm_rope_append_kv8(q, qkv, pos, slot, cos, sin, pool, nb, 1, 0, hq, hkv, hd)
            outs.append(torch.zeros_like(q))
            L.paged_decode_kv8(outs[-1], q, pool, nb, 1, 0, hq, hkv, hd, tables_d, lens_d, 900,
                               workspace=ws)
        return outs, q, pool
    ws = [L.alloc_decode_kv8_workspace(b, hq, hkv, hd) for _ in range(2)]
    old = L.set_dependent_launch(mode)
    try:
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s, w in zip(streams, ws):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(w))
        torch.cuda.synchronize()
    finally:
        L.set_dependent_launch(old)
    q64 = from_device(got[0][1]).reshape(b, hq, hd)
    want, bound = R.decode(R.bf16_f64(q64), from_device(got[0][2]), 0, tables, lens, hkv, hd, 1)
    for outs, q, pool in got:
        assert torch.equal(q, got[0][1]) and torch.equal(pool, got[0][2])
        for x in outs:
            assert torch.equal(x, got[0][0][0])
    assert R.rounds_to(R.bf16_f64(from_device(got[0][0][0])).reshape(b, hq, hd), want, bound).all()
