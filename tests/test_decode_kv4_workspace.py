"""One workspace of lc_paged_decode_kv4 for calls of different shapes: every call finds
and leaves the counters at zero, in the same bytes whatever its shape."""
import numpy as np
import pytest

import lucciola as L

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

COUNTERS = 288  # bytes per SM


class Decode:
    """Calls of one shape over a pool of random codes. Sequences may share pages: they
    are only read."""

    def __init__(self, hq, hkv, hd, lens, tokens=1, hint=0, seed=0, pages=1500):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.shape, self.tokens, self.hint, self.pages = (hq, hkv, hd), tokens, hint, pages
        lens = np.asarray(lens, np.int32)
        pool = torch.randint(0, 256, (pages, 1, hkv, 2, 9 * hd), generator=gen, device="cuda",
                             dtype=torch.uint8)
        pool[..., 8 * hd:] = pool[..., 8 * hd:] % 24 + 40  # scales 2^-2 .. 2^1
        self.pool = pool.view(pages, 1, hkv, 18 * hd)
        stride = -(-int(lens.max()) // 16)
        self.tables = torch.randint(0, pages, (len(lens), stride), generator=gen, device="cuda",
                                    dtype=torch.int32)
        self.lens = torch.from_numpy(lens).cuda()
        self.q = torch.randn(len(lens) * tokens, hq * hd, generator=gen, device="cuda").bfloat16()

    def own_workspace(self):
        return L.alloc_decode_kv4_workspace(len(self.lens), *self.shape, self.tokens)

    def __call__(self, ws):
        out = torch.full_like(self.q, 9.0)
        L.paged_decode_kv4(out, self.q, self.pool, self.pages, 1, 0, *self.shape, self.tables,
                           self.lens, self.hint, self.tokens, k_scale=0.5, v_scale=0.25,
                           workspace=ws)
        return out


def check_shared(calls):
    """The calls in turn, twice, on one workspace: the bits of separate ones, and the
    counters zero after each."""
    want = [c(c.own_workspace()) for c in calls]
    ws = max((c.own_workspace() for c in calls), key=lambda w: w.numel())
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for _ in range(2):
        for c, w in zip(calls, want):
            got = c(ws)
            assert torch.equal(got, w), (len(c.lens), c.tokens, (got != w).any(1).sum().item())
            assert not ws[:COUNTERS * sms].any().item()


def test_batches_of_several_sizes_share_a_workspace():
    shape = (64, 8, 128)
    check_shared([Decode(*shape, [4096] * 64), Decode(*shape, [4096] * 8, seed=1),
                  Decode(*shape, [4096] * 4, seed=2), Decode(*shape, [4096] * 64, seed=3)])


def test_drafted_and_single_tokens_share_a_workspace():
    shape = (64, 8, 128)
    check_shared([Decode(*shape, [2500] * 64, tokens=t, seed=t) for t in (1, 3, 1, 2)])


@pytest.mark.parametrize("hd", [64, 128])
def test_long_single_sequences_and_batches_share_a_workspace(hd):
    """Segments of more than 32 pieces, which are joined in groups, between batches."""
    lens = np.random.default_rng(3).integers(0, 3000, 40)
    check_shared([Decode(14, 2, hd, lens), Decode(14, 2, hd, [33000], hint=33000, seed=1),
                  Decode(28, 4, hd, [9000], seed=2), Decode(14, 2, hd, lens, tokens=5, seed=3),
                  Decode(14, 2, hd, [20000], tokens=2, seed=4)])


@pytest.mark.parametrize("hd", [64, 128])
def test_many_pieces_join_the_same_way_every_time(hd):
    """9 to 80 pieces per column, whichever CTA is last, 40 times."""
    calls = [Decode(4, 2, hd, [n], seed=n) for n in (2400, 5000, 8400, 20000)]
    calls.append(Decode(8, 1, hd, [15000, 15000, 1], seed=1))
    ws = max((c.own_workspace() for c in calls), key=lambda w: w.numel())
    want = [c(ws) for c in calls]
    for _ in range(40):
        for c, w in zip(calls, want):
            assert torch.equal(c(ws), w)
