"""One workspace of lc_paged_decode_kv8 for calls of different shapes, eager and in two graphs:
every call finds and leaves the counters at zero, in the same bytes whatever its shape."""
import numpy as np
import pytest

import lucciola as L

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

COUNTERS = 288  # bytes per SM


class Decode:
    """Calls of one shape over a pool of random codes and scales. Sequences may share pages:
    they are only read."""

    def __init__(self, hq, hkv, hd, lens, tokens=1, hint=0, seed=0, pages=1500):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.shape, self.tokens, self.hint, self.pages = (hq, hkv, hd), tokens, hint, pages
        lens = np.asarray(lens, np.int32)
        pool = torch.randint(0, 256, (pages, 1, hkv, 32 * hd + 16), generator=gen, device="cuda",
                             dtype=torch.uint8)
        pool[..., :32 * hd][pool[..., :32 * hd] & 0x7f == 0x7f] = 0  # no NaN
        scales = torch.randint(-9, -4, (pages, 1, hkv, 2), generator=gen, device="cuda")
        pool[..., 32 * hd:32 * hd + 8] = torch.exp2(scales.float()).view(torch.uint8)
        self.pool = pool
        stride = -(-int(lens.max()) // 16)
        self.tables = torch.randint(0, pages, (len(lens), stride), generator=gen, device="cuda",
                                    dtype=torch.int32)
        self.lens = torch.from_numpy(lens).cuda()
        self.q = torch.randn(len(lens) * tokens, hq * hd, generator=gen, device="cuda").bfloat16()
        self.out = torch.full_like(self.q, 9.0)

    def own_workspace(self):
        return L.alloc_decode_kv8_workspace(len(self.lens), *self.shape, self.tokens)

    def __call__(self, ws):
        L.paged_decode_kv8(self.out, self.q, self.pool, self.pages, 1, 0, *self.shape, self.tables,
                           self.lens, self.hint, self.tokens, workspace=ws)
        return self.out.clone()


def check_shared(calls):
    """The calls in turn, twice, on one workspace: the bits of separate ones, and the
    counters zero after each."""
    want = [c(c.own_workspace()) for c in calls]
    assert all(w.isfinite().all() for w in want)
    ws = max((c.own_workspace() for c in calls), key=lambda w: w.numel())
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for _ in range(2):
        for c, w in zip(calls, want):
            assert torch.equal(c(ws), w), (len(c.lens), c.tokens)
            assert not ws[:COUNTERS * sms].any().item()
    return ws, want


def test_batches_and_drafted_tokens_share_a_workspace():
    shape = (64, 8, 128)
    check_shared([Decode(*shape, [2500] * 64), Decode(*shape, [4096] * 4, seed=1),
                  Decode(*shape, [1500] * 16, tokens=3, seed=2), Decode(*shape, [900] * 20, tokens=2, seed=3),
                  Decode(*shape, [2500] * 64, seed=4)])


@pytest.mark.parametrize("hd", [64, 128])
def test_long_single_sequences_and_batches_share_a_workspace(hd):
    """Segments of more than 32 pieces, which are joined in groups, between batches."""
    lens = np.random.default_rng(3).integers(0, 3000, 40)
    check_shared([Decode(14, 2, hd, lens), Decode(14, 2, hd, [33000], hint=33000, seed=1),
                  Decode(28, 4, hd, [9000], seed=2), Decode(14, 2, hd, lens, tokens=5, seed=3),
                  Decode(14, 2, hd, [20000], tokens=2, seed=4)])


def test_two_graphs_share_a_workspace():
    calls = [Decode(14, 2, 64, [3000, 17, 0, 900]), Decode(28, 4, 128, [20000], hint=20000, seed=1)]
    ws, want = check_shared(calls)
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c(ws)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    for c, w in zip(calls, want):
        c.out.fill_(9.0)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert torch.equal(c.out, w)


@pytest.mark.parametrize("hd", [64, 128])
def test_many_pieces_join_the_same_way_every_time(hd):
    calls = [Decode(4, 2, hd, [n], seed=n) for n in (2400, 8400, 20000)]
    calls.append(Decode(8, 1, hd, [15000, 15000, 1], seed=1))
    ws = max((c.own_workspace() for c in calls), key=lambda w: w.numel())
    want = [c(ws) for c in calls]
    for _ in range(40):
        for c, w in zip(calls, want):
            assert torch.equal(c(ws), w)
