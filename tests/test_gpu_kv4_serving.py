"""The step tables, the 4-bit append, unpack + prefill and the 4-bit decode as one
serving loop (examples/serve_kv4.py)."""
import sys
from pathlib import Path

import numpy as np
import pytest

import lucciola as L
from conftest import ATTN_ATOL

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EXAMPLES = Path(__file__).resolve().parents[1] / "examples"
if str(EXAMPLES) not in sys.path:
    sys.path.insert(0, str(EXAMPLES))


def prompts_of(stack, lengths):
    gen = torch.Generator(device="cuda").manual_seed(3)
    return [torch.randint(0, stack.embed.shape[0], (n,), generator=gen, device="cuda")
            for n in lengths]


def test_graph_steps_equal_eager_steps_and_pages_come_back():
    import serve_kv4 as S
    stack = S.Stack()
    lengths, steps = (5, 33, 64, 200), 40
    tokens, pages = [], []
    for graph in (True, False):
        e = S.Engine(stack, num_blocks=64)
        tokens.append(S.generate(e, prompts_of(stack, lengths), steps, graph=graph))
        # a sequence holds the pages of its prompt and of every token but the last chosen one
        held = sum(-(-(n + steps - 1) // 16) for n in lengths)
        assert int(e.free_count.item()) == 64 - held
        assert e.lens[:4].tolist() == [n + steps - 1 for n in lengths]
        pages.append(e.tables.cpu().numpy())
        used = [pages[-1][i, :-(-(n + steps - 1) // 16)] for i, n in enumerate(lengths)]
        flat = np.concatenate(used)
        assert len(set(flat.tolist())) == len(flat) and flat.min() >= 0 and flat.max() < 64
        e.release([0, 1, 2, 3])
        assert int(e.free_count.item()) == 64
        assert sorted(e.free.tolist()) == list(range(64))
    assert torch.equal(tokens[0], tokens[1])
    assert np.array_equal(pages[0], pages[1])


def test_prompt_chunks_and_decode_agree():
    """A prompt in chunks gives what it gives at once, and its last token's attention over
    the 4-bit cache is the same through unpack + prefill and through decode."""
    import serve_kv4 as S
    stack = S.Stack(layers=1)
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
    L.qk_norm_rope_append_kv4(q, whole._project(x, 0), pos, slot, s.cos, s.sin, whole.pool,
                              whole.num_blocks, 1, 0, s.hq, s.hkv, s.hd, q_norm=s.q_norm[0],
                              k_norm=s.k_norm[0])
    out = torch.empty_like(q)
    L.paged_decode_kv4(out, q, whole.pool, whole.num_blocks, 1, 0, s.hq, s.hkv, s.hd,
                       whole.tables, whole.lens[:1], 150, k_scale=whole.K_SCALE,
                       v_scale=whole.V_SCALE, workspace=L.alloc_decode_kv4_workspace(1, s.hq, s.hkv, s.hd))
    y = x.clone()
    L.proj_gemm(y, out, s.w_o[0], residual=x)
    assert (y.float() - a[-1:].float()).abs().max().item() <= ATTN_ATOL * 4
    assert int(whole.status.item()) == 0 and int(parts.status.item()) == 0


def test_running_out_of_pages_is_reported():
    import serve_kv4 as S
    stack = S.Stack(layers=1)
    e = S.Engine(stack, num_blocks=4)
    with pytest.raises(L.LucciolaError) as err:
        S.generate(e, prompts_of(stack, (40, 14)), 12)
    assert err.value.status == 9  # LC_ERR_OUT_OF_BLOCKS
    assert e.lens[:2].tolist()[0] == 48  # full pages only
