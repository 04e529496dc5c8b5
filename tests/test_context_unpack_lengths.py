"""lc_unpack_kv4 says so when it leaves tokens of a sequence out."""
import numpy as np
import pytest

import kv4_ref as R
import lucciola as L
from workloads import from_device, make_tables, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("longest,lens,word", [
    (100, (100, 3, 0), 0),
    (100, (111, 5, 50), 0),               # in the pages of 100 tokens, and written
    (96, (97, 96, 1), L.LC_DEV_BAD_POS),  # a seventh page
    (1, (400, 0, 0), L.LC_DEV_BAD_POS),
])
def test_lengths_past_the_pages_of_the_output(longest, lens, word, offset):
    hkv, hd = 2, 64
    rng = np.random.default_rng(longest)
    lens = np.array(lens, np.int32)
    tables, nb = make_tables(np.array([26, 26, 26]), rng)
    pool = R.make_pool(rng, nb, 1, hkv, hd, 1.0, 1.0)
    P = R.ceil16(longest)
    out = [torch.full((3 * P, 1, hkv, 16, hd), 3.0, dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    L.unpack_kv4(*out, to_device(pool), nb, 1, 0, hkv, hd, to_device(tables),
                 to_device(lens - offset), longest, len_offset=offset, dev_status=st)
    assert st.item() == word
    for part, o in zip((pool[..., :R.half_bytes(hd)], pool[..., R.half_bytes(hd):]), out):
        got = R.bf16_f64(from_device(o)).reshape(3, P, hkv, 16, hd)
        for b, n in enumerate(lens):
            for j in range(P):
                held = min(16, n - 16 * j)
                if held <= 0:
                    assert (got[b, j] == 3.0).all()
                    continue
                want = R.unpack(part[tables[b, j], 0], hd, 1.0)
                want[:, held:] = 0.0
                assert np.array_equal(got[b, j], want)
