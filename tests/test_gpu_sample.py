"""lc_sample on the GPU against the float64 choice, and against lc_argmax."""
import numpy as np
import pytest

import lucciola as L
from kv4_ref import bf16_f64
from sample_ref import NONE, choose
from oracle.oracle import f32_to_bf16
from workloads import to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

VOCAB = 151936


def randn_bf16(rng, shape, scale=1.0):
    return f32_to_bf16((rng.standard_normal(shape) * scale).astype(np.float32))


NAMES = ("temperature", "top_k", "top_p", "min_p")


def run(bits, rand, stride=None, offset=0, **par):
    """Tokens of the rows of bf16 bits [batch, vocab] (uint32 values)."""
    batch, vocab = bits.shape
    stride = stride or vocab
    flat = torch.full((offset + batch * stride,), 300.0, dtype=torch.bfloat16, device="cuda")
    rows = flat[offset:].view(batch, stride)[:, :vocab]
    rows.copy_(to_device(np.ascontiguousarray(bits)))
    out = torch.full((batch,), 77, dtype=torch.int32, device="cuda")
    dev = {k: None if v is None else to_device(np.asarray(
        v, np.int32 if k == "top_k" else np.float32)) for k, v in par.items()}
    L.sample(out, rows, to_device(np.asarray(rand, np.float32)), **dev)
    return out.cpu().numpy().view(np.uint32)


def check(bits, rand, stride=None, offset=0, **par):
    got = run(bits, rand, stride, offset, **par)
    x = bf16_f64(bits)
    for b in range(len(x)):
        one = {k: float(np.float32(v[b])) if k != "top_k" else int(v[b]) for k, v in par.items()
               if v is not None}
        want, margin = choose(x[b], float(np.float32(rand[b])), **one)
        # sums of 64-bit weights differ by 1e-12 of the whole at most
        assert got[b] == want or margin < 1e-12, (b, got[b], want, one, margin)
    return got


def params(rng, batch):
    return dict(temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5, 10.0], batch),
                top_k=rng.choice([0, 1, 2, 40, 1000, 10 ** 9, -3], batch),
                top_p=rng.choice([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 2.0], batch),
                min_p=rng.choice([0.0, 0.01, 0.3, 1.0, -1.0], batch))


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 33, 255, 1000, 4097, 32003, VOCAB])
@pytest.mark.parametrize("scale", [0.5, 3.0, 20.0])
def test_vocabularies_and_parameters(vocab, scale):
    rng = np.random.default_rng(vocab)
    batch = 9 if vocab == VOCAB else 40
    bits = randn_bf16(rng, (batch, vocab), scale=scale)
    check(bits, rng.random(batch), **params(rng, batch))


@pytest.mark.parametrize("batch", [1, 2, 3, 17, 60, 150, 200])
def test_batches(batch):
    """However many rows there are, the choices are the same, one row's too."""
    rng = np.random.default_rng(batch)
    bits = randn_bf16(rng, (batch, 5000), scale=2.0)
    rand, par = rng.random(batch), params(rng, batch)
    got = check(bits, rand, **par)
    for b in range(0, batch, 29):
        one = run(bits[b:b + 1], rand[b:b + 1], **{k: v[b:b + 1] for k, v in par.items()})
        assert one[0] == got[b]


@pytest.mark.parametrize("batch", [1, 5, 40, 80, 160])
def test_whole_vocabulary_batches(batch):
    rng = np.random.default_rng(batch)
    bits = np.tile(randn_bf16(rng, (8, VOCAB), scale=2.0), (batch // 8 + 1, 1))[:batch]
    check(bits, rng.random(batch), **params(rng, batch))


@pytest.mark.parametrize("name", NAMES)
def test_each_parameter_alone(name):
    rng = np.random.default_rng(3)
    bits = randn_bf16(rng, (60, 2000), scale=2.0)
    check(bits, rng.random(60), **{name: params(rng, 60)[name]})


def test_no_parameters_at_all():
    rng = np.random.default_rng(4)
    check(randn_bf16(rng, (30, 700)), rng.random(30))


@pytest.mark.parametrize("stride,offset", [(1000, 0), (1001, 0), (1003, 3), (1008, 8), (1004, 1)])
def test_strides_and_alignment(stride, offset):
    rng = np.random.default_rng(stride)
    bits = randn_bf16(rng, (12, 1000), scale=2.0)
    check(bits, rng.random(12), stride=stride, offset=offset, **params(rng, 12))


def test_ties_go_to_the_lower_index():
    """Rows of few different values: the draw counts along the index within one value."""
    rng = np.random.default_rng(5)
    levels = np.array([0x3f80, 0x4000, 0x4040, 0x0000, 0x8000, 0xbf80], np.uint16)
    for vocab in (50, 3001, 70000):
        bits = levels[rng.integers(0, 6, (20, vocab))]
        par = params(rng, 20)
        par["top_k"] = rng.integers(0, vocab, 20)
        check(bits, rng.random(20), **par)
        got = run(bits, rng.random(20), temperature=np.zeros(20))
        assert np.array_equal(got, (bits == 0x4040).argmax(1))
    same = np.full((4, VOCAB), 0x3f80, np.uint16)  # all tokens alike
    rand = np.array([0.0, 0.25, 0.5, 1 - 2.0 ** -24], np.float32)
    got = run(same, rand)
    assert np.array_equal(got, np.floor(rand.astype(np.float64) * VOCAB).astype(np.uint32))
    assert np.array_equal(run(same, rand, top_k=[10, 10, 10, 10]), [0, 2, 5, 9])
    assert np.array_equal(run(same[:, :1000], rand, top_p=[0.5] * 4), [0, 125, 250, 499])


def test_masked_logits():
    """Minus infinity, the type's lowest value and NaN are never chosen; a row of them gives
    no token."""
    rng = np.random.default_rng(6)
    for bar in (0xff80, 0xff7f, 0x7fc0, 0xffc0):
        bits = randn_bf16(rng, (16, 3000), scale=2.0)
        barred = rng.random(bits.shape) < 0.7
        bits[barred] = bar
        bits[3] = bar
        bits[4] = bar
        bits[4, 2999] = 0xc2c8  # one token, of a low logit
        got = check(bits, rng.random(16), **params(rng, 16))
        assert got[3] == NONE and got[4] == 2999
        got = check(bits, np.full(16, 1 - 2.0 ** -24))
        live = np.arange(16) != 3
        assert not barred[np.arange(16), np.minimum(got, 2999)][live & (np.arange(16) != 4)].any()


def test_infinite_and_extreme_logits():
    """Plus infinity takes all the weight; large, tiny and zero logits keep their order."""
    rng = np.random.default_rng(7)
    bits = randn_bf16(rng, (24, 5000), scale=2.0)
    bits[0, 77] = 0x7f80
    bits[1, [5, 900, 4000]] = 0x7f80
    bits[2] = randn_bf16(rng, 5000, scale=1e5)
    bits[3] = randn_bf16(rng, 5000, scale=1e30)
    bits[4] = randn_bf16(rng, 5000, scale=1e-9)
    bits[5] = randn_bf16(rng, 5000, scale=1e-38)
    bits[6, ::2] = randn_bf16(rng, 2500, scale=1e-12)
    bits[7, ::3] = 0x8000
    bits[8] = 0x8000
    bits[9] = rng.integers(0, 65536, 5000)  # any bits at all
    bits[10] = rng.integers(0, 65536, 5000)
    bits[11, ::7] = 0x4f00
    bits[12, ::7] = 0xcf00
    bits[13] = 0xc800  # all alike, large and negative
    bits[14] = np.where(np.arange(5000) % 2, 0x3380, 0x337f)
    bits[15] = np.where(np.arange(5000) % 2, 0x4480, 0x447f)
    for seed in range(3):
        rng = np.random.default_rng(seed)
        par = params(rng, 24)
        if seed == 0:
            par = dict(temperature=np.full(24, 1.0))
        got = check(bits, rng.random(24), **par)
        assert got[0] == 77 and got[1] in (5, 900, 4000)


@pytest.mark.parametrize("batch", [1, 30, 100])
def test_extreme_logits_of_rows_over_several_ctas(batch):
    """One token in each range beside the histogram's, in different slices of the row, and more
    than one: the slow way, for the whole cluster."""
    rng = np.random.default_rng(batch)
    vocab = 70000 if batch < 100 else 40000
    bits = randn_bf16(rng, (batch, vocab), scale=2.0)
    for row in range(batch):
        at = rng.integers(0, vocab, 40)
        kind = row % 5 if batch > 1 else 0
        if kind == 0:
            bits[row, at[:4]] = (0x4500, 0x0123, 0x8123, 0xc500)  # one each
        elif kind == 1:
            bits[row, at[:2]] = (0x0123, 0x0124)
        elif kind == 2:
            bits[row, at[:4]] = (0x4500, 0x4501, 0x4500, 0x7f80)
        elif kind == 3:
            bits[row] = randn_bf16(rng, vocab, scale=1e-9)
        else:
            bits[row, at] = 0xc501
    for seed in range(3):
        rng = np.random.default_rng(seed)
        par = params(rng, batch)
        if seed == 0:
            par = dict(temperature=np.full(batch, 300.0))  # the tails count
        check(bits, rng.random(batch), **par)


def test_ends_of_the_draw_and_odd_parameters():
    rng = np.random.default_rng(8)
    bits = randn_bf16(rng, (10, 400), scale=2.0)
    x = bf16_f64(bits)
    order = np.argsort(-x, axis=1, kind="stable")
    assert np.array_equal(run(bits, np.zeros(10)), order[:, 0])
    got = run(bits, np.full(10, 1 - 2.0 ** -24), top_k=np.full(10, 7))
    assert np.array_equal(got, order[:, 6])
    nan = np.full(10, np.nan)
    rand = rng.random(10)
    # NaN: no filter, the first of the order
    assert np.array_equal(run(bits, rand, top_p=nan, min_p=nan), run(bits, rand))
    assert np.array_equal(run(bits, rand, temperature=nan), order[:, 0])
    assert np.array_equal(run(bits, rand, temperature=-np.ones(10)), order[:, 0])
    assert np.array_equal(run(bits, nan), order[:, 0])
    assert np.array_equal(run(bits, np.full(10, 1.5), top_k=np.full(10, 3)), order[:, 2])
    # a temperature so low that one token has all the weight, and one so high that none has
    assert np.array_equal(run(bits, rand, temperature=np.full(10, 1e-30)), order[:, 0])
    got = run(bits, np.full(10, 0.5), temperature=np.full(10, np.inf))
    assert np.array_equal(got, order[:, 200])


def test_greedy_rows_equal_argmax_without_ties():
    rng = np.random.default_rng(9)
    bits = np.stack([rng.permutation(30000)[:20000] for _ in range(6)]).astype(np.uint16)  # distinct
    out = torch.zeros(6, dtype=torch.int32, device="cuda")
    L.argmax(out, to_device(bits))
    got = run(bits, rng.random(6), temperature=np.zeros(6))
    assert np.array_equal(got, out.cpu().numpy().view(np.uint32))


def test_stream_graph_and_repeats():
    rng = np.random.default_rng(10)
    bits = randn_bf16(rng, (33, 9000), scale=2.0)
    rand, par = rng.random(33).astype(np.float32), params(rng, 33)
    want = check(bits, rand, **par)
    rows, rnd = to_device(bits), to_device(rand)
    dev = {k: to_device(v.astype(np.int32 if k == "top_k" else np.float32)) for k, v in par.items()}
    outs = [torch.zeros(33, dtype=torch.int32, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    L.sample(outs[0], rows, rnd, **dev, stream=side)  # two calls at once
    L.sample(outs[1], rows, rnd, **dev)
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.cpu().numpy().view(np.uint32), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.sample(outs[0], rows, rnd, **dev)
    for shift in (1, 2):  # other inputs through the same graph
        rnd.copy_(to_device(np.roll(rand, shift)))
        rows.copy_(to_device(np.roll(bits, shift, 0)))
        for v, d in zip(par.values(), dev.values()):
            d.copy_(to_device(np.roll(v, shift)).to(d.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(outs[0].cpu().numpy().view(np.uint32), np.roll(want, shift))


def test_draws_follow_the_weights():
    """Evenly spaced numbers draw each token as often as its share of the weight says."""
    rng = np.random.default_rng(11)
    n, vocab = 4096, 60
    bits = np.tile(randn_bf16(rng, (1, vocab), scale=1.5), (n, 1))
    got = run(bits, (np.arange(n) + 0.5) / n, temperature=np.full(n, 0.8))
    x = bf16_f64(bits[0])
    p = np.exp((x - x.max()) / np.float32(0.8))
    p /= p.sum()
    counts = np.bincount(got, minlength=vocab)
    assert (np.abs(counts - n * p) <= 1.0).all()
