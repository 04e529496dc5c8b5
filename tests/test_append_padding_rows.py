"""What the rows with position -1 hold in qkv does not matter, and nothing is written for
them: as many tokens with and without padding rows of NaN, the same bits."""
import numpy as np
import pytest

import lucciola as L
import oracle.oracle as O
from workloads import randn_bf16, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,rows,padded", [
    (14, 2, 64, 5, 64), (28, 4, 128, 33, 2000), (1, 1, 64, 1, 9), (3, 3, 128, 2500, 20000)])
def test_rows_past_the_last_token(hq, hkv, hd, rows, padded, kv4):
    rng = np.random.default_rng(rows)
    nb = rows // 16 + 1
    qkv = torch.full((padded, (hq + 2 * hkv) * hd), float("nan"), dtype=torch.bfloat16,
                     device="cuda")
    qkv[:rows] = to_device(randn_bf16(rng, (rows, (hq + 2 * hkv) * hd)))
    cos, sin = (to_device(t) for t in O.rope_table(64, hd, 1e6))
    w = to_device(randn_bf16(rng, hd))

    def run(count):
        pos = torch.full((count,), -1, dtype=torch.int32, device="cuda")
        slot = pos.clone()
        pos[:rows] = torch.arange(rows, device="cuda") % 64
        slot[:rows] = torch.arange(rows, device="cuda")
        q_out = torch.full((count, hq * hd), 5.0, dtype=torch.bfloat16, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        if kv4:
            pools = [L.alloc_kv4_pool(nb, 1, hkv, hd)]
            L.qk_norm_rope_append_kv4(q_out, qkv, pos, slot, cos, sin, *pools, nb, 1, 0, hq, hkv, hd,
                                      q_norm=w, k_norm=w, dev_status=status)
        else:
            pools = [torch.zeros(nb, 1, hkv, 16, hd, dtype=torch.bfloat16, device="cuda")
                     for _ in range(2)]
            L.qk_norm_rope_append(q_out, qkv, pos, slot, cos, sin, *pools, nb, 1, 0, hq, hkv, hd,
                                  q_norm=w, k_norm=w, dev_status=status)
        assert status.item() == 0
        assert (q_out[rows:] == 5.0).all()
        return [q_out[:rows]] + pools
    for a, b in zip(run(rows), run(padded)):
        assert torch.equal(a, b)
