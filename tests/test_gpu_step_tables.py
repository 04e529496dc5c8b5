"""Block tables, positions and slot maps built on the GPU (lc_step_tables,
lc_step_release) against the host bookkeeping and a plain restatement."""
import numpy as np
import pytest

import kv4_ref as R
import lucciola as L
from workloads import to_device

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def ints(*shape, fill=0):
    return torch.full(shape, fill, dtype=torch.int32, device="cuda")


def plain(tables, slots, ctx, new, free, count, cap, width, num_blocks):
    """What lc_step_tables does, one request at a time."""
    tables = tables.copy()
    step = np.full((len(ctx), width), -1)
    pos, slot_map = np.full(cap, -1), np.full(cap, -1)
    starts, out, used, want_sum, word = [0], [], 0, 0, 0
    for b, (s, c, m) in enumerate(zip(slots, ctx, new)):
        room = tables.shape[1] * 16
        ok_slot = 0 <= s < len(tables)
        if not (0 <= c <= room and 0 <= m and c + m <= room and ok_slot):
            word |= L.LC_DEV_BAD_POS
            c = c if 0 <= c <= room and ok_slot else 0
            m = 0
        have, want = R.ceil16(c), R.ceil16(c + m)
        want_sum += want - have
        served = have == want or want_sum <= count
        if not served:
            word |= L.LC_DEV_OUT_OF_BLOCKS
        elif ok_slot:
            for j in range(have, want):
                used += 1
                tables[s, j] = free[count - used]
        out.append(c + m if served else c)
        if ok_slot:
            k = R.ceil16(out[-1])
            if k > width:
                word |= L.LC_DEV_BAD_POS
            step[b, :k] = tables[s, :min(k, width)]
        for i in range(m):
            r = starts[-1] + i
            if r < cap:
                pos[r] = c + i
                if served:
                    slot_map[r] = tables[s, (c + i) // 16] * 16 + (c + i) % 16
        starts.append(starts[-1] + m)
    if starts[-1] > cap:
        word |= L.LC_DEV_BAD_POS
    return tables, step, pos, slot_map, np.array(starts), np.array(out), count - used, word


def run(tables, slots, ctx, new, free, count, cap, width=None, alias=False):
    b = len(ctx)
    width = width or tables.shape[1]
    num_blocks = len(free)
    want = plain(tables, range(b) if slots is None else slots, ctx, new, free, count, cap, width,
                 num_blocks)
    d = [to_device(np.asarray(a, np.int32)) for a in (tables, ctx, new, free, [count])]
    ctx_out, count_out = (d[1], d[4]) if alias else (ints(b), ints(1))
    pos, slot_map, starts, step = ints(cap, fill=7), ints(cap, fill=7), ints(b + 1), ints(b, width)
    st, ws = ints(1), L.alloc_step_workspace()
    L.step_tables(d[0], d[1], d[2], d[3], d[4], pos, slot_map, starts, ctx_out, count_out, ws,
                  slots=None if slots is None else to_device(np.asarray(slots, np.int32)),
                  step_tables=step, dev_status=st)
    got = [t.cpu().numpy() for t in (d[0], step, pos, slot_map, starts, ctx_out)]
    for name, g, w in zip(("tables", "step", "positions", "slots", "starts", "ctx"), got, want):
        assert np.array_equal(g, w), name
    assert int(count_out.item()) == want[6]
    assert int(st.item()) == want[7]
    assert not ws.any()
    return got, want


def make(rng, slots, max_ctx, stride, spare, batch, max_new, shuffle=True):
    ctx_all = rng.integers(0, max_ctx + 1, slots)
    pages = np.array([R.ceil16(c) for c in ctx_all])
    num_blocks = int(pages.sum()) + spare + 3
    perm = rng.permutation(num_blocks)
    tables = np.full((slots, stride), -1)
    at = 0
    for s, n in enumerate(pages):
        tables[s, :n] = perm[at:at + n]
        at += n
    free = np.full(num_blocks, -1)
    free[:spare] = perm[at:at + spare]
    order = rng.permutation(slots)[:batch] if shuffle else np.arange(batch)
    new = rng.integers(0, max_new + 1, batch)
    return tables, order, ctx_all[order], new, free


@pytest.mark.parametrize("batch,slots,max_ctx,max_new,spare", [
    (1, 1, 0, 1, 4), (1, 3, 100, 33, 9), (7, 9, 64, 40, 100), (64, 64, 500, 1, 64),
    (300, 311, 300, 90, 2500), (513, 600, 40, 3, 700), (1030, 1030, 900, 17, 3000),
])
def test_step_tables(batch, slots, max_ctx, max_new, spare):
    rng = np.random.default_rng(batch)
    stride = (max_ctx + max_new) // 16 + 2
    t, order, ctx, new, free = make(rng, slots, max_ctx, stride, spare, batch, max_new)
    total = int(new.sum())
    run(t, order, ctx, new, free, spare, total)
    run(t, order, ctx, new, free, spare, total + 9, alias=True)        # padding rows
    run(t, order, ctx, new, free, spare, max(1, total // 2), width=stride + 3)  # too few rows
    run(t, order, ctx, new, free, min(3, spare), total)               # out of pages
    run(t, order, ctx, new, free, 0, total)
    ident = make(rng, slots, max_ctx, stride, spare, batch, max_new, shuffle=False)
    run(ident[0], None, *ident[2:], spare, total + 1)


def test_long_rows_and_many_tokens():
    """Rows of several segments, token counts above one CTA's share."""
    rng = np.random.default_rng(3)
    t, order, ctx, new, free = make(rng, 40, 30000, 4100, 30000, 33, 20000)
    new[::3] = 1
    run(t, order, ctx, new, free, 30000, int(new.sum()) + 1)


def test_invalid_requests_get_nothing():
    rng = np.random.default_rng(4)
    t, order, ctx, new, free = make(rng, 8, 100, 9, 50, 8, 20)
    ctx[1], new[2], order[3], new[4], ctx[5] = -3, -1, 8, 9 * 16, 9 * 16 + 1
    order[6] = -1
    got, want = run(t, order, ctx, new, free, 50, 80)
    assert want[7] & L.LC_DEV_BAD_POS
    run(t, order, ctx, new, free, 50, 80, width=2)  # step rows too short for some


def test_bad_state_is_reported():
    rng = np.random.default_rng(5)
    t, order, ctx, new, free = make(rng, 4, 50, 9, 10, 4, 40)
    new[:] = 33
    d = [to_device(np.asarray(a, np.int32)) for a in (t, ctx, new, free)]

    def word(count, free_t):
        st = ints(1)
        pos, slot = ints(140), ints(140)
        L.step_tables(d[0].clone(), d[1], d[2], free_t, to_device(np.array([count], np.int32)), pos,
                      slot, ints(5), ints(4), ints(1), L.alloc_step_workspace(),
                      slots=to_device(order.astype(np.int32)), dev_status=st)
        return int(st.item()), slot.cpu().numpy()
    assert word(-4, d[3])[0] == L.LC_DEV_BAD_BLOCK | L.LC_DEV_OUT_OF_BLOCKS
    bad = d[3].clone()
    bad[9] = len(free)  # the first page to come off the stack
    w, slot = word(10, bad)
    assert w & L.LC_DEV_BAD_BLOCK and slot.max() < 16 * len(free)


def test_follows_the_host_bookkeeping():
    """Random steps of arriving, growing and finishing sequences: the same pages in the
    same order as lc_block_alloc gives them."""
    rng = np.random.default_rng(6)
    num_blocks, max_seqs, stride = 300, 12, 24
    host = L.BlockAlloc(num_blocks, max_seqs, stride)
    free = to_device(np.arange(num_blocks - 1, -1, -1, dtype=np.int32))
    count, tables = to_device(np.array([num_blocks], np.int32)), ints(max_seqs, stride, fill=-1)
    ws, st = L.alloc_step_workspace(), ints(1)
    lens = {}
    for step in range(40):
        done = [s for s in lens if rng.random() < 0.15]
        for s in done:
            host.release(s)
        if done:
            L.step_release(free, count, tables,
                           to_device(np.array([lens.pop(s) for s in done], np.int32)), count, ws,
                           slots=to_device(np.array(done, np.int32)), dev_status=st)
        while len(lens) < max_seqs and rng.random() < 0.6:
            lens[host.add()] = 0
        if not lens:
            continue
        batch = [int(s) for s in rng.permutation(list(lens))]
        new = [int(rng.integers(1, 60)) if lens[s] == 0 else 1 for s in batch]
        new = [min(m, stride * 16 - lens[s]) for s, m in zip(batch, new)]
        ctx = to_device(np.array([lens[s] for s in batch], np.int32))
        total = sum(new)
        rows, slot_map, starts = ints(total + 1), ints(total + 1), ints(len(batch) + 1)
        L.step_tables(tables, ctx, to_device(np.array(new, np.int32)), free, count, rows, slot_map,
                      starts, ctx, count, ws, slots=to_device(np.array(batch, np.int32)),
                      dev_status=st)
        for s, m in zip(batch, new):
            lens[s] += m
            host.reserve(s, lens[s])
        got = tables.cpu().numpy()
        for s in lens:
            pages = host.pages(s)
            assert got[s, :len(pages)].tolist() == pages
        assert int(count.item()) == host.num_free
        assert ctx.cpu().tolist() == [lens[s] for s in batch]
    assert int(st.item()) == 0


def test_release():
    rng = np.random.default_rng(7)
    t, order, ctx, _, free = make(rng, 700, 900, 60, 10, 650, 1)
    num_blocks = len(free)
    ctx[3] = 0
    want, at = free.copy(), 10
    for s, c in zip(order, ctx):
        for page in t[s, :R.ceil16(c)][::-1]:
            want[at] = page
            at += 1
    d = [to_device(np.asarray(a, np.int32)) for a in (t, order, ctx, free, [10])]
    st, out, ws = ints(1), ints(1), L.alloc_step_workspace()
    L.step_release(d[3], d[4], d[0], d[2], out, ws, slots=d[1], dev_status=st)
    assert np.array_equal(d[3].cpu().numpy(), want) and int(out.item()) == at
    assert int(st.item()) == 0 and int(d[4].item()) == 10
    # more pages than the stack has room for: dropped and reported
    full = to_device(np.array([num_blocks - 1], np.int32))
    L.step_release(d[3], full, d[0], d[2], full, ws, slots=d[1], dev_status=st)
    assert int(st.item()) == L.LC_DEV_BAD_BLOCK and int(full.item()) == num_blocks
    st.zero_()
    bad = d[2].clone()
    bad[0], bad[1] = -1, 60 * 16 + 1
    L.step_release(d[3].clone(), d[4], d[0], bad, out, ws, slots=d[1], dev_status=st)
    assert int(st.item()) == L.LC_DEV_BAD_POS
    assert int(out.item()) == at - R.ceil16(ctx[0]) - R.ceil16(ctx[1])
