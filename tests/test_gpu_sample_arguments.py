"""lucciola.sample on the GPU: what its checks let through is read as it is."""
import pytest

import lucciola as L

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_more_entries_than_rows_unsigned_types_and_host_memory():
    gen = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn(6, 3008, generator=gen, device="cuda").bfloat16()
    logits = wide[:5, 3:3000]
    rand = torch.rand(8, generator=gen, device="cuda")
    par = dict(temperature=torch.full((8,), 0.8, device="cuda"),
               top_k=torch.tensor([0, 50, 3, 1, 700, 9, 9, 9], device="cuda").int(),
               top_p=torch.full((8,), 0.9, device="cuda"), min_p=torch.zeros(8, device="cuda"))
    want = torch.full((8,), -7, dtype=torch.int32, device="cuda")
    L.sample(want, logits, rand, **par)
    assert (want[:5] >= 0).all() and (want[5:] == -7).all()
    got = torch.zeros(5, 1, dtype=torch.uint32, device="cuda")
    L.sample(got, logits, rand.cpu().pin_memory(),
             **dict(par, top_k=par["top_k"].to(torch.uint32)))
    assert torch.equal(got.view(torch.int32)[:, 0], want[:5])


def test_refusals():
    logits = torch.zeros(4, 100, dtype=torch.bfloat16, device="cuda")
    rand, out = torch.zeros(4, device="cuda"), torch.full((4,), 5, dtype=torch.int32, device="cuda")
    with pytest.raises(L.LucciolaError, match="top_k"):
        L.sample(out, logits, rand, top_k=torch.tensor([0, 50, 1, 2], device="cuda"))  # int64
    with pytest.raises(L.LucciolaError, match="temperature"):
        L.sample(out, logits, rand, temperature=torch.ones(1, device="cuda").expand(4))
    with pytest.raises(L.LucciolaError, match="on the GPU"):
        L.sample(out, logits, rand.cpu())
    with pytest.raises(L.LucciolaError, match="logits"):
        L.sample(out, logits.float(), rand)
    torch.cuda.synchronize()
    assert (out == 5).all()
