"""Draws at borders between two tokens. lc_sample's weights and sums are in 64 bits, so where the
draw, the top-p cut or the min-p threshold lies within 1e-12 of a border either side may be taken;
the token is then one of the few that the formula gives with them moved that far, never another."""
import numpy as np
import pytest

import lucciola as L
from kv4_ref import bf16_f64
from oracle.oracle import f32_to_bf16
from workloads import to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

SLACK = 1e-12  # of the weight in question, as the header says
VOCAB = 151936
EXTENDED = np.longdouble  # 64 bits of mantissa


def allowed(x, rand, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens that the formula gives for the logits x with its three comparisons moved by up to
    SLACK of the weight compared; one where none lies that close to a border. By the formula's
    definition, in extended precision; written apart from sample_ref."""
    live = np.nonzero(x > -1e30)[0]
    order = live[np.argsort(-x[live], kind="stable")]
    if not temperature > 0:
        return {int(order[0])}
    top = x[order].astype(EXTENDED)
    with np.errstate(invalid="ignore", over="ignore"):
        gap = np.where(top == top[0], EXTENDED(0), top - top[0])
        w = np.exp(gap / EXTENDED(temperature))
    if top_k > 0:
        w = w[:top_k]
    run = np.cumsum(w)
    keeps = {len(w)}
    if top_p <= 0:
        keeps = {1}
    elif top_p < 1:
        need = EXTENDED(top_p) * run[-1]
        lo, hi = (int(np.searchsorted(run, need + d * run[-1], side="left")) + 1 for d in (-SLACK, SLACK))
        keeps = {min(max(k, 1), len(w)) for k in range(lo, hi + 1)}
    if min_p > 0:
        lo, hi = (int((w >= min_p * (1 + d)).sum()) for d in (SLACK, -SLACK))
        keeps = {min(k, max(1, n)) for k in keeps for n in {lo, hi}}
    tokens = set()
    for keep in keeps:
        total = run[keep - 1]
        goal = EXTENDED(rand) * total
        # the first token past the goal moved down, the first one past it moved up
        lo, hi = (int(np.searchsorted(run[:keep], goal + d * total, side="right")) for d in (-SLACK, SLACK))
        for at in range(lo, hi + 1):
            at = min(at, keep - 1)
            while at > 0 and w[at] == 0:
                at -= 1
            tokens.add(int(order[at]))
    return tokens


def check(bits, rand, least_alone=0.9, **par):
    """Every row's token is allowed, and at least that share of the rows allows one only."""
    batch = len(bits)
    rand = np.asarray(rand, np.float32)
    par = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in par.items()}
    out = torch.full((batch,), -1, dtype=torch.int32, device="cuda")
    L.sample(out, to_device(np.ascontiguousarray(bits)), to_device(rand),
             **{k: to_device(v) for k, v in par.items()})
    got = out.cpu().numpy()
    alone = 0
    for b, x in enumerate(bf16_f64(bits)):
        may = allowed(x, float(rand[b]), **{k: v[b].item() for k, v in par.items()})
        assert int(got[b]) in may, (b, int(got[b]), sorted(may)[:8], {k: v[b] for k, v in par.items()})
        alone += len(may) == 1
    assert alone >= least_alone * batch, (alone, batch)


def randn_bf16(rng, shape, scale):
    return f32_to_bf16((rng.standard_normal(shape) * scale).astype(np.float32))


@pytest.mark.parametrize("vocab", [5, 100, 4097, 32003, VOCAB])
@pytest.mark.parametrize("scale", [0.5, 3.0, 20.0])
def test_draws_away_from_borders_have_one_answer(vocab, scale):
    rng = np.random.default_rng(vocab)
    batch = 8 if vocab == VOCAB else 40
    check(randn_bf16(rng, (batch, vocab), scale), rng.random(batch),
          temperature=rng.choice([0.0, 0.3, 0.8, 1.0, 2.0], batch),
          top_k=rng.choice([0, 1, 40, 1000], batch), top_p=rng.choice([0.1, 0.9, 0.999, 1.0], batch),
          min_p=rng.choice([0.0, 0.01, 0.3], batch))


def test_draws_on_exact_borders():
    """Equal logits: rand and top_p at k / n of the tokens, where sums are whole numbers and the
    comparison itself decides: running weight > rand * weight, running weight >= top_p * weight."""
    n = 1024
    bits = np.full((64, n), 0x3f80, np.uint16)
    k = np.arange(64) * 16
    check(bits, k / n, least_alone=0.0)
    out = torch.zeros(64, dtype=torch.int32, device="cuda")
    L.sample(out, to_device(bits), to_device((k / n).astype(np.float32)))
    assert np.array_equal(out.cpu().numpy(), k)
    p = to_device(((k + 16) / n).astype(np.float32))  # keeps k + 16 tokens; the draw takes the last
    L.sample(out, to_device(bits), to_device(np.full(64, 1 - 2.0 ** -24, np.float32)), top_p=p)
    assert np.array_equal(out.cpu().numpy(), k + 15)


@pytest.mark.parametrize("vocab", [9, 700, 20000])
def test_draws_beside_borders(vocab):
    """rand and top_p as near to the running sums as fp32 comes: rounded to either side of one."""
    rng = np.random.default_rng(vocab)
    bits = randn_bf16(rng, (48, vocab), 2.0)
    x = -np.sort(-bf16_f64(bits), 1)
    w = np.exp(x - x[:, :1])
    share = np.cumsum(w, 1) / w.sum(1, keepdims=True)
    at = rng.integers(0, min(vocab - 1, 40), 48)
    border = share[np.arange(48), at].astype(np.float32)
    side = np.where(rng.random(48) < 0.5, 0, 2).astype(np.float32)
    near = np.minimum(np.nextafter(border, side), np.float32(1 - 2.0 ** -24))
    check(bits, near, least_alone=0.8)
    check(bits, rng.random(48), least_alone=0.8, top_p=near)
    check(bits, near, least_alone=0.8, temperature=np.full(48, 1.0), top_k=np.full(48, vocab))


@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.0, 3.0])
def test_min_p_beside_a_weight(temperature):
    """min_p is fp32's neighbour of a token's weight, on either side."""
    rng = np.random.default_rng(int(temperature * 10))
    bits = randn_bf16(rng, (48, 3000), 2.0)
    x = -np.sort(-bf16_f64(bits), 1)
    w = np.exp((x - x[:, :1]) / np.float64(np.float32(temperature)))
    at = rng.integers(0, 60, 48)
    weight = w[np.arange(48), at].astype(np.float32)
    near = np.where(rng.random(48) < 0.5, weight, np.nextafter(weight, np.float32(0)))
    check(bits, rng.random(48), least_alone=0.8, temperature=np.full(48, temperature), min_p=near)


def test_tails_without_weight():
    """Logits so far below the best that their weights underflow: never chosen, wherever rand is."""
    rng = np.random.default_rng(8)
    bits = randn_bf16(rng, (32, 5000), 1.0)
    bits[:, 100] = 0x447a  # 1000
    bits[:16, 4000] = 0x447a
    rand = np.where(np.arange(32) % 2, 1 - 2.0 ** -24, rng.random(32)).astype(np.float32)
    for t in (1e-3, 0.5, 1.0):
        check(bits, rand, temperature=np.full(32, t))
        check(bits, rand, temperature=np.full(32, t), top_p=np.full(32, 0.99), top_k=np.full(32, 3000))
