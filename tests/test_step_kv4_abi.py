"""Argument checks of the step tables, the per-head norm + RoPE and the 4-bit
cache: refused on the host, before anything is launched. No GPU needed."""
import pytest

import lucciola as L

FAKE = 0x10000  # aligned non-null pointer value; never dereferenced by host validation


def caller(name, order, defaults):
    def call(**kw):
        a = dict(defaults)
        assert set(kw) <= set(a)
        a.update(kw)
        return getattr(L.lib, name)(*[a[k] for k in order.split()])
    return call


STEP = caller(
    "lc_step_tables",
    "tables stride slots_n slots ctx new batch free count blocks step step_stride pos slot "
    "max_tokens starts ctx_out count_out ws ws_bytes status stream",
    dict(tables=FAKE, stride=64, slots_n=8, slots=None, ctx=FAKE, new=FAKE, batch=0, free=FAKE,
         count=FAKE, blocks=100, step=None, step_stride=0, pos=FAKE, slot=FAKE, max_tokens=0,
         starts=FAKE, ctx_out=FAKE, count_out=FAKE, ws=FAKE, ws_bytes=256, status=None,
         stream=None))
RELEASE = caller(
    "lc_step_release",
    "free count blocks tables stride slots_n slots ctx n count_out ws ws_bytes status stream",
    dict(free=FAKE, count=FAKE, blocks=100, tables=FAKE, stride=64, slots_n=8, slots=None,
         ctx=FAKE, n=0, count_out=FAKE, ws=FAKE, ws_bytes=256, status=None, stream=None))
ROWS = dict(q_out=FAKE, q_out_stride=14 * 64, qkv=FAKE, row=18 * 64, rows=0, pos=FAKE, slot=FAKE,
            qb=None, kb=None, vb=None, qn=None, kn=None, eps=1e-6, cos=FAKE, sin=FAKE,
            rope_rows=4096, blocks=64, layers=2, layer=1, hq=14, hkv=2, hd=64, status=None,
            stream=None)
_HEAD = "q_out q_out_stride qkv row rows pos slot qb kb vb qn kn eps cos sin rope_rows "
_TAIL = " blocks layers layer hq hkv hd status stream"
APPEND = caller("lc_qk_norm_rope_append", _HEAD + "k v" + _TAIL, dict(ROWS, k=FAKE, v=FAKE))
APPEND4 = caller("lc_qk_norm_rope_append_kv4", _HEAD + "kv ks vs" + _TAIL,
                 dict(ROWS, kv=FAKE, ks=1.0, vs=1.0))
UNPACK = caller(
    "lc_unpack_kv4",
    "k v kv blocks layers layer hkv hd tables stride lens offset batch longest ks vs status stream",
    dict(k=FAKE, v=FAKE, kv=FAKE, blocks=64, layers=2, layer=1, hkv=2, hd=64, tables=FAKE,
         stride=8, lens=FAKE, offset=0, batch=0, longest=100, ks=1.0, vs=1.0, status=None,
         stream=None))
DECODE = caller(
    "lc_paged_decode_kv4",
    "out out_stride q q_stride kv blocks layers layer hq hkv hd tables stride lens offset batch "
    "tokens longest ks vs scale ws ws_bytes status stream",
    dict(out=FAKE, out_stride=14 * 64, q=FAKE, q_stride=14 * 64, kv=FAKE, blocks=64, layers=2,
         layer=1, hq=14, hkv=2, hd=64, tables=FAKE, stride=64, lens=FAKE, offset=0, batch=0,
         tokens=1, longest=0, ks=1.0, vs=1.0, scale=0.125, ws=FAKE, ws_bytes=1 << 40,
         status=None, stream=None))

INVALID, HEAD_DIM, SHAPE, WORKSPACE, ALIGN = 1, 2, 3, 4, 5


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("tables", "ctx", "new", "free", "count", "pos", "slot",
                                     "starts", "ctx_out", "count_out")],
    (INVALID, dict(batch=-1)), (INVALID, dict(stride=0)), (INVALID, dict(slots_n=0)),
    (INVALID, dict(blocks=0)), (INVALID, dict(blocks=1 << 27)), (INVALID, dict(max_tokens=-1)),
    (INVALID, dict(step=FAKE, step_stride=0)), (INVALID, dict(batch=9)),
    (SHAPE, dict(batch=8193, slots_n=10000)), (SHAPE, dict(batch=8192, slots_n=8192, stride=1 << 15)),
    (SHAPE, dict(stride=1 << 28)), (WORKSPACE, dict(ws_bytes=255)), (WORKSPACE, dict(ws=None)),
    (ALIGN, dict(ws=FAKE + 2)), (0, dict()),
])
def test_step_tables_refusals(status, kw):
    assert STEP(**kw) == status


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("free", "count", "tables", "ctx", "count_out")],
    (INVALID, dict(n=-1)), (INVALID, dict(n=9)), (INVALID, dict(stride=0)),
    (INVALID, dict(blocks=0)), (SHAPE, dict(n=8193, slots_n=10000)), (WORKSPACE, dict(ws=None)),
    (ALIGN, dict(ws=FAKE + 1)), (0, dict()),
])
def test_step_release_refusals(status, kw):
    assert RELEASE(**kw) == status


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("q_out", "qkv", "pos", "slot", "cos", "sin")],
    (HEAD_DIM, dict(hd=96)), (HEAD_DIM, dict(hd=0)), (SHAPE, dict(hkv=4)),
    (INVALID, dict(rows=-1)), (INVALID, dict(layer=2)), (INVALID, dict(layer=-1)),
    (INVALID, dict(layers=0)), (INVALID, dict(hkv=0)), (INVALID, dict(blocks=0)),
    (INVALID, dict(blocks=1 << 27)), (INVALID, dict(rope_rows=0)), (INVALID, dict(eps=-1e-6)),
    (INVALID, dict(eps=float("nan"))), (INVALID, dict(eps=float("inf"))),
    (INVALID, dict(row=17 * 64)), (INVALID, dict(q_out_stride=13 * 64)),
    (ALIGN, dict(row=18 * 64 + 4)), (ALIGN, dict(q_out_stride=14 * 64 + 2)),
    *[(ALIGN, {k: FAKE + 8}) for k in ("q_out", "qkv", "qb", "kb", "vb", "qn", "kn", "cos", "sin")],
    (0, dict()),
])
def test_norm_rope_append_refusals(status, kw):
    assert APPEND(**kw) == status
    assert APPEND4(**kw) == status


def test_pool_and_scale_refusals():
    assert APPEND(k=None) == INVALID and APPEND(v=None) == INVALID
    assert APPEND(k=FAKE + 2) == ALIGN and APPEND(v=FAKE + 8) == ALIGN
    for call in (APPEND4, UNPACK, DECODE):
        assert call(kv=None) == INVALID and call(kv=FAKE + 8) == ALIGN
        for bad in (0.0, -1.0, float("nan"), float("inf"), 2.0 ** 65, 2.0 ** -65):
            assert call(ks=bad) == INVALID and call(vs=bad) == INVALID


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("k", "v", "tables", "lens")],
    (HEAD_DIM, dict(hd=32)), (INVALID, dict(batch=-1)), (INVALID, dict(longest=-1)),
    (INVALID, dict(offset=2)), (INVALID, dict(layer=2)), (INVALID, dict(stride=0)),
    (INVALID, dict(batch=1, longest=129)), (ALIGN, dict(k=FAKE + 8)), (0, dict()),
    (0, dict(batch=3, longest=0)),
])
def test_unpack_refusals(status, kw):
    assert UNPACK(**kw) == status


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("out", "q", "tables", "lens")],
    (HEAD_DIM, dict(hd=96)), (SHAPE, dict(hkv=3)), (INVALID, dict(batch=-1)),
    (INVALID, dict(tokens=0)), (INVALID, dict(layer=2)), (INVALID, dict(blocks=0)),
    (INVALID, dict(stride=0)), (INVALID, dict(stride=1 << 28)), (INVALID, dict(offset=2)),
    (INVALID, dict(longest=-1)), (INVALID, dict(q_stride=13 * 64)),
    (INVALID, dict(out_stride=13 * 64)), (INVALID, dict(batch=1 << 20, tokens=1 << 12)),
    (ALIGN, dict(q=FAKE + 8)), (ALIGN, dict(q_stride=14 * 64 + 4)), (ALIGN, dict(out=FAKE + 1)),
    (WORKSPACE, dict(batch=2, ws=None)), (WORKSPACE, dict(batch=2, ws_bytes=16)),
    (ALIGN, dict(batch=2, ws=FAKE + 8)), (0, dict()),
])
def test_decode_refusals(status, kw):
    assert DECODE(**kw) == status


def test_sizes():
    assert L.kv4_page_bytes(64) == 18 * 64 and L.kv4_page_bytes(128) == 18 * 128
    assert L.kv4_page_bytes(96) == 0
    size = L.lib.lc_paged_decode_kv4_workspace_size
    assert size(4, 14, 2, 64, 1) > 0
    for bad in ((0, 14, 2, 64, 1), (4, 14, 3, 64, 1), (4, 14, 2, 96, 1), (4, 14, 2, 64, 0),
                (4, 0, 2, 64, 1)):
        assert size(*bad) == 0
    assert size(64, 14, 2, 64, 4) >= size(64, 14, 2, 64, 1)
    assert L.lib.lc_status_from_device_word(L.LC_DEV_OUT_OF_BLOCKS) == 9
    assert L.lib.lc_status_from_device_word(L.LC_DEV_OUT_OF_BLOCKS | L.LC_DEV_BAD_POS) == 7


def test_wrappers_raise():
    with pytest.raises(L.LucciolaError) as e:
        L.alloc_kv4_pool(1, 1, 1, 96, device="cpu")
    assert e.value.status == 2
