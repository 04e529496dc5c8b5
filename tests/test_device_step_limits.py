"""lc_step_tables and lc_step_release up to their stated 8192 requests: around the sizes
whose shared memory, with the kernels' own static part, passes the 48 KB that a launch
has without asking. Each size runs first in a process of its own: a larger call asks for
all later ones."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TESTS = Path(__file__).resolve().parent

CHILD = """
import sys
sys.path[:0] = [{tests!r}, {package!r}]
import test_device_step_limits as T
T.{name}({n})
"""


def in_a_process(name, n):
    code = CHILD.format(tests=str(TESTS), package=str(TESTS.parent / "lucciola-rs_b200"), name=name,
                        n=n)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def reserve(batch):
    """Every request adds 17 tokens to none: two pages each."""
    import lucciola as L
    blocks, stride = 2 * batch + 5, 2
    tables = torch.full((batch, stride), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device="cuda")
    count = ints(blocks)
    ctx, new = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.full(
        (batch,), 17, dtype=torch.int32, device="cuda")
    pos, slot = (torch.full((17 * batch,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    starts = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    status = ints(0)
    L.step_tables(tables, ctx, new, free, count, pos, slot, starts, ctx, count,
                  L.alloc_step_workspace(), dev_status=status)
    assert status.item() == 0 and count.item() == 5
    assert torch.equal(tables.flatten().cpu(), torch.arange(2 * batch, dtype=torch.int32))
    rows = torch.arange(17 * batch)
    assert torch.equal(pos.cpu().long(), rows % 17)
    assert torch.equal(slot.cpu().long(), rows // 17 * 32 + rows % 17)
    assert torch.equal(starts.cpu().long(), torch.arange(batch + 1) * 17)
    assert (ctx == 17).all()


def release(requests):
    """Every request gives its two pages back, the last one first."""
    import lucciola as L
    blocks = 2 * requests + 5
    tables = torch.arange(2 * requests, dtype=torch.int32, device="cuda").view(requests, 2)
    free = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
    free[:5] = torch.arange(2 * requests, blocks)
    count, status = ints(5), ints(0)
    ctx = torch.full((requests,), 20, dtype=torch.int32, device="cuda")
    L.step_release(free, count, tables, ctx, count, L.alloc_step_workspace(), dev_status=status)
    assert status.item() == 0 and count.item() == blocks
    assert torch.equal(free[5:].cpu().view(requests, 2), tables.cpu().flip(1))


@pytest.mark.parametrize("batch", [3062, 3063, 3067, 3071, 3081, 8191, 8192])
def test_step_tables_of_many_requests(batch):
    in_a_process("reserve", batch)


@pytest.mark.parametrize("requests", [6128, 6129, 6137, 6143, 6145, 8192])
def test_step_release_of_many_requests(requests):
    in_a_process("release", requests)
