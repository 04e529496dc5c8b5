"""The bytes of the 4-bit cache around every boundary between two codes, in both signs:
the kernel's corrected quotient against a division rounded once."""
import numpy as np
import pytest

import kv4_ref as R
import lucciola as L
import oracle.oracle as O
from workloads import from_device, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def fp32_quantise(x, g):
    """x float32 [rows, 16] -> (codes, scale bytes) from the header's formula, every
    quotient and product rounded to fp32."""
    g = np.float32(g)
    amax = np.abs(x).max(-1)
    s8 = R.e4m3_byte((amax / (np.float32(6) * g)).astype(np.float64))
    step = (R.e4m3_value(s8).astype(np.float32) * g)[:, None]
    with np.errstate(all="ignore"):
        y = np.where(step > 0, x / step, np.float32(0))
    assert y.dtype == np.float32
    return R.quantise_codes(np.abs(y)) + 8 * np.signbit(x), s8


def append_v(x, g):
    """Groups of 16 as the V rows of an append: (codes, scale bytes)."""
    rows = x.shape[0] // 4
    nb, hd = rows // 16 + 1, 64
    qkv = np.zeros((rows, 3 * hd), np.uint16)
    qkv[:, 2 * hd:] = x.reshape(rows, hd)
    cos, sin = (to_device(t) for t in O.rope_table(4, hd, 1e6))
    pool = L.alloc_kv4_pool(nb, 1, 1, hd)
    q_out = torch.zeros(rows, hd, dtype=torch.bfloat16, device="cuda")
    slot = torch.arange(rows, dtype=torch.int32, device="cuda")
    L.qk_norm_rope_append_kv4(q_out, to_device(qkv), slot % 4, slot, cos, sin, pool, nb, 1, 0, 1, 1,
                              hd, v_scale=float(g))
    half = from_device(pool)[:, 0, 0, R.half_bytes(hd):]
    n = 8 * hd
    data = half[:, :n].reshape(nb * 16, hd // 2)[:rows]
    code = np.stack([data & 15, data >> 4], -1).reshape(rows * 4, 16)
    return code, half[:, n:].reshape(-1)[:rows * 4]


def groups(g):
    """For each scale byte, groups whose largest value is 6 steps and whose others lie
    on and beside the seven boundaries, positive and negative, with both zeros."""
    out = []
    for byte in range(1, 127):
        step = R.e4m3_value(byte) * float(np.float32(g))
        top = R.bf16_round(6 * step)
        if abs(top) > 3e38 or step < 2.0 ** -100:
            continue
        mids = np.array([(R.MAG[i] + R.MAG[i + 1]) / 2 for i in range(7)]) * step
        m = R.bf16_round(mids)
        ulp = 2.0 ** (np.floor(np.log2(m)) - 7)
        for d in (-2, -1, 0, 1, 2):
            for sign in (1.0, -1.0):
                v = np.concatenate([[top], sign * (m + d * ulp), [0.0, -0.0, 1e-30 * sign],
                                    sign * R.MAG[1:6] * step])
                out.append(v)
    x = np.array(out)
    x = O.f32_to_bf16(x.astype(np.float32))
    return np.concatenate([x, np.zeros((-len(x) % 4, 16), np.uint16)])


@pytest.mark.parametrize("g", [1.0, 0.25, 2.0 ** -40, 2.0 ** 60, 0.3, 1e-3, 1.7])
def test_codes_around_every_boundary(g):
    x = groups(g)
    code, s8 = append_v(x, g)
    want, want_s8 = fp32_quantise((x.astype(np.uint32) << 16).view(np.float32), g)
    assert np.array_equal(s8, want_s8)
    bad = code != want
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:3], code[bad][:3], want[bad][:3])


def test_negative_zero_has_one_code():
    """-0 is code 8 in a group of values, of zeros, and beside what is not finite."""
    x = np.zeros((4, 16), np.float32)
    x[:, 1::2] = -0.0
    x[0, 0], x[1, 0], x[2, 0] = 3.0, 1e6, np.inf
    code, _ = append_v(O.f32_to_bf16(x), 1.0)
    assert (code[:, 1::2] == 8).all()
    assert (code[:, 2::2] == 0).all()
