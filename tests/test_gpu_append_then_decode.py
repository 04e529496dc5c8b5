"""lc_qk_norm_rope_append_kv8 and the decode that reads what it wrote, with nothing between them on
the stream, so that in launch modes 1 and 2 the decode is there before the append has ended. Every
pass appends new rows at the next tokens: a decode that read too early would see other q rows, pages
and scales than in mode 0, whose bits every pass has to have."""
import numpy as np
import pytest

import kv8_ref as R
import lucciola as L
import oracle.oracle as O
from workloads import make_tables, randn_bf16, to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

PASSES = 5


class Passes:
    """PASSES appends of `rows` tokens to each of `batch` sequences, and what comes with each. The
    decode attends with each sequence's last `tokens` of them."""

    def __init__(self, batch, rows, hq, hkv, hd, seed, pad=8, tokens=1):
        self.shape, self.batch, self.rows, self.tokens = (hq, hkv, hd), batch, rows, tokens
        rng = np.random.default_rng(seed)
        start = rng.integers(0, 300, batch)
        total = start + PASSES * rows
        tables, self.nb = make_tables(np.array([R.ceil16(n) for n in total]), rng)
        self.tables, self.longest = to_device(tables), int(total.max())
        some = R.make_pool(rng, 32, 1, hkv, hd)
        self.pool = to_device(some[rng.integers(0, len(some), self.nb)])
        self.cos, self.sin = (to_device(t) for t in O.rope_table(self.longest, hd, 1e6))
        self.norm = to_device(randn_bf16(rng, hd))
        self.qkv, self.pos, self.slot, self.lens = [], [], [], []
        for i in range(PASSES):
            pos = (start[:, None] + i * rows + np.arange(rows)).astype(np.int32)
            slot = np.take_along_axis(tables, pos // 16, 1) * 16 + pos % 16
            # each pass of another magnitude, so that scales grow too
            qkv = rng.standard_normal((batch * rows, (hq + 2 * hkv) * hd + pad)) * 2.0 ** (i - 2)
            self.qkv.append(to_device(O.f32_to_bf16(qkv.astype(np.float32))))
            self.pos.append(to_device(pos.ravel()))
            self.slot.append(to_device(slot.astype(np.int32).ravel()))
            self.lens.append(to_device((start + (i + 1) * rows).astype(np.int32)))

    def run(self, mode, in_place):
        """(q rows and outputs of every pass, the pool) in launch mode `mode`."""
        hq, hkv, hd = self.shape
        width = hq * hd
        pool, qkv = self.pool.clone(), [x.clone() for x in self.qkv]
        q = qkv if in_place else [torch.full((self.batch * self.rows, width), float("nan"),
                                             dtype=torch.bfloat16, device="cuda") for _ in qkv]
        if self.tokens == 1:  # the last row of each sequence
            newest = [x.view(self.batch, self.rows, -1)[:, -1] for x in q]
        else:
            assert self.tokens == self.rows
            newest = q
        out = [torch.full((self.batch * self.tokens, width), float("nan"), dtype=torch.bfloat16,
                          device="cuda") for _ in qkv]
        ws = L.alloc_decode_kv8_workspace(self.batch, hq, hkv, hd, self.tokens)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        old = L.set_dependent_launch(mode)
        try:
            for i in range(PASSES):
                L.qk_norm_rope_append_kv8(q[i], qkv[i], self.pos[i], self.slot[i], self.cos, self.sin,
                                          pool, self.nb, 1, 0, hq, hkv, hd, q_norm=self.norm,
                                          k_norm=self.norm, dev_status=status)
                L.paged_decode_kv8(out[i], newest[i], pool, self.nb, 1, 0, hq, hkv, hd, self.tables,
                                   self.lens[i], self.longest, self.tokens, workspace=ws,
                                   dev_status=status)
            torch.cuda.synchronize()
        finally:
            L.set_dependent_launch(old)
        assert int(status.item()) == 0
        assert not any(torch.isnan(x).any() for x in out)
        return q + out, pool

    def check(self, mode, in_place):
        want, want_pool = self.run(0, in_place)
        for _ in range(3):
            got, pool = self.run(mode, in_place)
            for a, b in zip(got, want):
                assert torch.equal(a.view(torch.int16), b.view(torch.int16))
            assert torch.equal(pool, want_pool)


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("batch,rows,hq,hkv,hd", [
    (1, 1, 14, 2, 64), (6, 1, 28, 4, 128),
    (96, 70, 28, 4, 128),  # an append of several waves of CTAs
])
def test_q_over_the_qkv_rows(batch, rows, hq, hkv, hd, mode):
    """In place, with rows an odd number of 16 bytes apart: neighbouring heads, which different
    warps read and write, share 32-byte sectors."""
    Passes(batch, rows, hq, hkv, hd, seed=batch + rows, pad=8).check(mode, True)


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("batch,rows,hq,hkv,hd,tokens", [
    (1, 1, 14, 2, 64, 1), (6, 1, 28, 4, 128, 1), (64, 1, 14, 2, 64, 1), (300, 1, 8, 8, 64, 1),
    (3, 40, 12, 2, 128, 1), (96, 70, 28, 4, 128, 1),
    (8, 3, 64, 8, 128, 3), (5, 2, 14, 2, 64, 2),  # drafted tokens
])
def test_new_rows_in_every_pass(batch, rows, hq, hkv, hd, tokens, mode):
    Passes(batch, rows, hq, hkv, hd, seed=batch + rows + tokens, tokens=tokens).check(mode, False)


@pytest.mark.parametrize("mode", [1, 2])
def test_new_rows_in_every_pass_of_a_graph(mode):
    """The same as one captured graph, replayed from the pool's first state."""
    hq, hkv, hd, batch = 14, 2, 64, 7
    p = Passes(batch, 1, hq, hkv, hd, seed=3)
    want, want_pool = p.run(0, False)
    pool = p.pool.clone()
    q = [torch.zeros(batch, hq * hd, dtype=torch.bfloat16, device="cuda") for _ in p.qkv]
    out = [torch.zeros_like(x) for x in q]
    ws = L.alloc_decode_kv8_workspace(batch, hq, hkv, hd)
    graph = torch.cuda.CUDAGraph()
    old = L.set_dependent_launch(mode)
    try:
        with torch.cuda.graph(graph):
            for i in range(PASSES):
                L.qk_norm_rope_append_kv8(q[i], p.qkv[i], p.pos[i], p.slot[i], p.cos, p.sin, pool,
                                          p.nb, 1, 0, hq, hkv, hd, q_norm=p.norm, k_norm=p.norm)
                L.paged_decode_kv8(out[i], q[i], pool, p.nb, 1, 0, hq, hkv, hd, p.tables, p.lens[i],
                                   p.longest, workspace=ws)
    finally:
        L.set_dependent_launch(old)
    for _ in range(3):
        pool.copy_(p.pool)
        for x in q + out:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(q + out, want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        assert torch.equal(pool, want_pool)
