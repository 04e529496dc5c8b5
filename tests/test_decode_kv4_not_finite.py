"""What is not a number stays visible in lc_paged_decode_kv4's rows, also where all
that one warp, one CTA or the whole row sees is NaN or minus infinity."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import run_decode
from workloads import make_tables, randn_bf16

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HQ, HKV = 4, 2


def make(lens, hd, seed):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    tables, nb = make_tables(np.array([R.ceil16(n) for n in lens]), rng)
    return rng, lens, tables, R.make_pool(rng, nb, 1, HKV, hd, 1.0, 1.0)


def nan_key(pool, tables, b, token, head, hd):
    """A NaN scale in the first group of one key."""
    pool[tables[b, token // 16], 0, head, 8 * hd + token % 16 * (hd // 16)] = 0x7f


def check(q, pool, tables, lens, hd, tokens, nan):
    """NaN rows are NaN all through; the others are the finite formula's."""
    got = run_decode(q, pool, 0, tables, lens, HKV, hd, tokens)
    assert np.array_equal(np.isnan(got), np.repeat(nan[..., None], hd, -1))
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, HKV, hd, tokens, 1.0, 1.0)
    assert R.rounds_to(got, want, bound)[~nan].all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 3, 5, 11])
def test_a_nan_in_q_reaches_its_whole_row(tokens, hd):
    """Rows of one warp, of eight warps and of several CTAs."""
    rng, lens, tables, pool = make([1, 20, 300, 0, 5000], hd, tokens)
    q = randn_bf16(rng, (len(lens) * tokens, HQ, hd))
    nan = np.zeros(q.shape[:2], bool)
    for b, n in enumerate(lens):
        row, head = b * tokens + tokens - 1, b % HQ  # the newest token: sees all n
        q[row, head, 7 * b] = 0x7fc0
        nan[row, head] = n > 0
    check(q, pool, tables, lens, hd, tokens, nan)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,first,last", [
    (1, 0, 1),         # the only token
    (33, 32, 33),      # the newest one, alone in its warp's pages
    (700, 96, 128),    # all that one warp reads
    (700, 0, 256),     # all that eight warps read in one turn
    (700, 0, 700),     # everything
    (6000, 0, 2000),   # all that some CTAs read
    (6000, 0, 6000),
])
def test_nan_keys_reach_every_row_that_sees_them(n, first, last, hd):
    rng, lens, tables, pool = make([n], hd, n + last)
    for token in range(first, last):
        nan_key(pool, tables, 0, token, 1, hd)
    q = randn_bf16(rng, (1, HQ, hd))
    check(q, pool, tables, lens, hd, 1, np.array([[False, False, True, True]]))


@pytest.mark.parametrize("hd", [64, 128])
def test_nan_keys_leave_rows_alone_that_do_not_see_them(hd):
    """The newest of three tokens has a NaN key, alone in its page, or is all there is."""
    rng, lens, tables, pool = make([33, 2, 1], hd, 9)
    q = randn_bf16(rng, (9, HQ, hd))
    nan = np.zeros((9, HQ), bool)
    for b, n in enumerate(lens):
        nan_key(pool, tables, b, n - 1, 0, hd)
        nan[3 * b + 2, :2] = True
    check(q, pool, tables, lens, hd, 3, nan)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 40, 5000])
def test_scores_of_minus_infinity_only_are_not_an_empty_row(n, hd):
    """softmax over scores that are all -inf is 0 / 0, as lc_paged_decode has it; a row
    without tokens is zeros."""
    rng, lens, tables, pool = make([n, 0], hd, n)
    k = R.unpack(pool[..., :R.half_bytes(hd)], hd, 1.0)
    k[..., 5] = -np.abs(k[..., 5]) - 0.5 * np.abs(k).max(-1)
    pool[..., :R.half_bytes(hd)] = R.pack(k, 1.0)
    q = randn_bf16(rng, (2, HQ, hd))
    q[0, 1, 5] = 0x7f80
    q[1, :, 5] = 0x7f80
    nan = np.zeros((2, HQ), bool)
    nan[0, 1] = True
    check(q, pool, tables, lens, hd, 1, nan)


def test_a_scale_that_is_not_a_number():
    """A NaN factor gives NaN, not the mean of the values; rows without tokens stay zeros."""
    rng, lens, tables, pool = make([50, 0], 64, 3)
    q = randn_bf16(rng, (2, HQ, 64))
    got = run_decode(q, pool, 0, tables, lens, HKV, 64, sm_scale=float("nan"))
    assert np.isnan(got[0]).all() and not got[1].any()
    rng, lens, tables, pool = make([50, 1], 64, 4)
    q = randn_bf16(rng, (6, HQ, 64))
    got = run_decode(q, pool, 0, tables, lens, HKV, 64, 3, sm_scale=float("nan"))
    assert np.isnan(got[[0, 1, 2, 5]]).all() and not got[3:5].any()
