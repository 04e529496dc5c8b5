"""lc_paged_decode_kv4 over rows of q and over probabilities of a wide range: both go
through fp16, whose ends must not show."""
import numpy as np
import pytest

import kv4_ref as R
import oracle.oracle as O
from test_gpu_kv4 import run_decode
from workloads import make_tables

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** -12, 2.0 ** -17, 2.0 ** -21, 2.0 ** -25])
def test_small_elements_of_q_beside_a_large_one(ratio, hd):
    """One dim of q is large where all keys are zero; the scores come from the others,
    `ratio` as large. Nothing but q's own rounding could tell: the bound is the ordinary one."""
    hq, hkv, n = 4, 1, 150
    rng = np.random.default_rng(hd)
    tables, nb = make_tables(np.array([R.ceil16(n)]), rng)
    k = rng.standard_normal((nb, 1, hkv, 16, hd)) * 64.0
    k[..., 3] = 0.0
    v = rng.standard_normal(k.shape)
    pool = np.concatenate([R.pack(k, 1.0), R.pack(v, 1.0)], -1)
    q = rng.standard_normal((1, hq, hd)).astype(np.float32)
    q[..., 3] = 1.0 / ratio
    q = O.f32_to_bf16(q)
    lens = np.array([n], np.int32)
    # scores of a few units
    sm_scale = 2.0 / (64.0 * hd ** 0.5)
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, sm_scale=sm_scale)
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1, 1.0, 1.0, sm_scale)
    assert R.rounds_to(got, want, bound).all()


@pytest.mark.parametrize("exponent", [-125, -110, -60, 60, 110, 127])
def test_q_of_any_exponent(exponent):
    """Rows whose largest element lies anywhere in bf16's normal numbers."""
    hq, hkv, hd, n = 4, 2, 64, 90
    rng = np.random.default_rng(exponent + 200)
    tables, nb = make_tables(np.array([R.ceil16(n)]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0)
    q = rng.uniform(-0.99, 0.99, (1, hq, hd))
    q[..., 0] = 0.99
    q = O.f32_to_bf16(np.ldexp(q, exponent + 1).astype(np.float32))
    lens = np.array([n], np.int32)
    sm_scale = 2.0 ** -min(max(exponent, -120), 120)
    got = run_decode(q, pool, 0, tables, lens, hkv, hd, sm_scale=sm_scale)
    want, bound = R.decode(R.bf16_f64(q), pool, 0, tables, lens, hkv, hd, 1, 1.0, 1.0, sm_scale)
    assert R.rounds_to(got, want, bound).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bits", [0.3, 9.7, 14.4, 16.6, 18.3, 19.7, 20.7])
def test_small_probabilities_beside_a_large_one(bits, hd):
    """31 tokens 2^-bits as probable as the first, whose value is zero: the row is what
    these bring. fp16 keeps 11 bits of them (2^-12 after rounding to nearest); fp32 scores
    of 20 and their ex2 add under 2^-17, the quotient and the sums under 2^-20."""
    n, rng = 32, np.random.default_rng(1)
    tables, nb = make_tables(np.array([2]), rng)
    k = np.zeros((nb, 1, 1, 16, hd))
    k[tables[0, 0], 0, 0, 0, :] = 6.0
    v = np.full(k.shape, 6.0)
    v[tables[0, 0], 0, 0, 0, :] = 0.0
    pool = np.concatenate([R.pack(k, 1.0), R.pack(v, 1.0)], -1)
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 5] = 1.0
    sm_scale = bits * np.log(2.0) / 6.0
    got = run_decode(O.f32_to_bf16(q), pool, 0, tables, np.array([n], np.int32), 1, hd,
                     sm_scale=sm_scale)
    want = 31 * 6.0 * 2.0 ** -bits / (1 + 31 * 2.0 ** -bits)
    slack = want * (2.0 ** -12 + 2.0 ** -16)
    assert R.rounds_to(got, np.full(got.shape, want), slack).all(), (got[0, 0, 0], want)
