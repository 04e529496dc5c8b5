"""The step tables, the 8-bit append, unpack + prefill, the 8-bit decode and the sampling as
one serving loop (examples/serve_kv8.py)."""
import sys
from pathlib import Path

import numpy as np
import pytest

import kv8_ref as R
import lucciola as L
from conftest import ATTN_ATOL
from sample_ref import choose
from workloads import from_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EXAMPLES = Path(__file__).resolve().parents[1] / "examples"
if str(EXAMPLES) not in sys.path:
    sys.path.insert(0, str(EXAMPLES))

PARAMS = dict(temperature=[0.0, 0.7, 1.0, 1.3], top_k=[0, 50, 0, 200], top_p=[1.0, 0.9, 0.95, 1.0],
              min_p=[0.0, 0.0, 0.05, 0.0])


def prompts_of(stack, lengths):
    gen = torch.Generator(device="cuda").manual_seed(3)
    return [torch.randint(0, stack.embed.shape[0], (n,), generator=gen, device="cuda")
            for n in lengths]


def test_graph_steps_equal_eager_steps_and_pages_come_back():
    import serve_kv8 as S
    stack = S.Stack()
    lengths, steps = (5, 33, 64, 200), 40
    tokens, pools = [], []
    for graph in (True, False):
        e = S.Engine(stack, slots=4, num_blocks=64, **PARAMS)
        tokens.append(S.generate(e, prompts_of(stack, lengths), steps, graph=graph))
        held = sum(-(-(n + steps - 1) // 16) for n in lengths)
        assert int(e.free_count.item()) == 64 - held
        assert e.lens[:4].tolist() == [n + steps - 1 for n in lengths]
        pools.append(e.pool)
        e.release([0, 1, 2, 3])
        assert int(e.free_count.item()) == 64
        # a second round over recycled pages, whose old scales no longer count
        again = S.Engine(stack, slots=4, num_blocks=64, **PARAMS)
        e.step_no.zero_()
        tokens.append(S.generate(e, prompts_of(stack, lengths), 9, graph=graph))
        assert torch.equal(tokens[-1], S.generate(again, prompts_of(stack, lengths), 9, graph=graph))
    assert torch.equal(tokens[0], tokens[2]) and torch.equal(tokens[1], tokens[3])
    assert torch.equal(pools[0], pools[1])


@pytest.mark.parametrize("max_steps", [4096, 5])
def test_the_chosen_tokens_are_the_formulas(max_steps):
    """Each step's tokens from that step's logits and numbers, a prompt's first token with its own
    request's parameters; the numbers begin anew after the last."""
    import serve_kv8 as S
    stack = S.Stack(layers=1)
    e = S.Engine(stack, slots=4, max_steps=max_steps, **PARAMS)
    seen = []
    chosen = e.choose

    def record(out, logits, first=0):
        n = int(e.step_no.item())
        chosen(out, logits, first)
        seen.append((n, first, from_device(logits), out.cpu().numpy().copy()))
    e.choose = record
    S.generate(e, prompts_of(stack, (5, 33, 64, 200)), 12, graph=False)
    assert len(seen) == 4 + 11
    assert [first for _, first, _, _ in seen] == [0, 1, 2, 3] + [0] * 11
    assert [n for n, _, _, _ in seen] == [i % max_steps for i in range(15)]
    numbers = e.numbers.cpu().numpy()
    drawn = np.array([out - np.argmax(R.bf16_f64(logits), 1) for _, _, logits, out in seen[4:]])
    # row 0 is greedy, and the others' draws are draws (one row may take its likeliest each time)
    assert not drawn[:, 0].any() and drawn[:, 1:].any()
    for n, first, logits, out in seen:
        for row, bits in enumerate(logits, first):
            par = {k: v[row] if k == "top_k" else float(np.float32(v[row])) for k, v in PARAMS.items()}
            want, margin = choose(R.bf16_f64(bits), float(numbers[n, row]), **par)
            assert out[row - first] == want or margin < 1e-12


def test_prompt_chunks_and_decode_agree():
    """A prompt in chunks gives what it gives at once (its pages' scales are those of all their
    tokens in the end), and its last token's attention over the 8-bit cache is the same through
    unpack + prefill and through decode."""
    import serve_kv8 as S
    stack = S.base.Stack(layers=1)
    tokens = prompts_of(stack, (150,))[0]
    whole, parts = S.Engine(stack), S.Engine(stack)
    a = whole.prompt(0, tokens)
    b = torch.cat([parts.prompt(0, tokens[:70], 0), parts.prompt(0, tokens[70:149], 70),
                   parts.prompt(0, tokens[149:], 149)])
    assert (a.float() - b.float()).abs().max().item() <= ATTN_ATOL * 4  # through o_proj
    s = stack
    x = s.embed[tokens[-1:].long()]
    q = torch.empty(1, s.hq * s.hd, dtype=torch.bfloat16, device="cuda")
    pos = torch.full((1,), 149, dtype=torch.int32, device="cuda")
    slot = torch.full((1,), -1, dtype=torch.int32, device="cuda")  # cached already
    L.qk_norm_rope_append_kv8(q, whole._project(x, 0), pos, slot, s.cos, s.sin, whole.pool,
                              whole.num_blocks, 1, 0, s.hq, s.hkv, s.hd, q_norm=s.q_norm[0],
                              k_norm=s.k_norm[0])
    out = torch.empty_like(q)
    L.paged_decode_kv8(out, q, whole.pool, whole.num_blocks, 1, 0, s.hq, s.hkv, s.hd, whole.tables,
                       whole.lens[:1], 150, workspace=L.alloc_decode_kv8_workspace(1, s.hq, s.hkv, s.hd))
    y = x.clone()
    L.proj_gemm(y, out, s.w_o[0], residual=x)
    assert (y.float() - a[-1:].float()).abs().max().item() <= ATTN_ATOL * 4
    assert int(whole.status.item()) == 0 and int(parts.status.item()) == 0


def test_running_out_of_pages_is_reported():
    import serve_kv8 as S
    stack = S.Stack(layers=1)
    e = S.Engine(stack, num_blocks=4)
    with pytest.raises(L.LucciolaError) as err:
        S.generate(e, prompts_of(stack, (40, 14)), 12)
    assert err.value.status == 9  # LC_ERR_OUT_OF_BLOCKS
