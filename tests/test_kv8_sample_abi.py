"""Argument checks of the 8-bit cache and of lc_sample: refused on the host, before anything
is launched. No GPU needed."""
import pytest

import lucciola as L
from test_step_kv4_abi import _HEAD, _TAIL, ALIGN, FAKE, HEAD_DIM, INVALID, ROWS, SHAPE, WORKSPACE, caller

APPEND = caller("lc_qk_norm_rope_append_kv8", _HEAD + "kv" + _TAIL, dict(ROWS, kv=FAKE))
UNPACK = caller(
    "lc_unpack_kv8",
    "k v kv blocks layers layer hkv hd tables stride lens offset batch longest status stream",
    dict(k=FAKE, v=FAKE, kv=FAKE, blocks=64, layers=2, layer=1, hkv=2, hd=64, tables=FAKE,
         stride=8, lens=FAKE, offset=0, batch=0, longest=100, status=None, stream=None))
DECODE = caller(
    "lc_paged_decode_kv8",
    "out out_stride q q_stride kv blocks layers layer hq hkv hd tables stride lens offset batch "
    "tokens longest scale ws ws_bytes status stream",
    dict(out=FAKE, out_stride=14 * 64, q=FAKE, q_stride=14 * 64, kv=FAKE, blocks=64, layers=2,
         layer=1, hq=14, hkv=2, hd=64, tables=FAKE, stride=64, lens=FAKE, offset=0, batch=0,
         tokens=1, longest=0, scale=0.125, ws=FAKE, ws_bytes=1 << 40, status=None, stream=None))
SAMPLE = caller(
    "lc_sample", "logits stride vocab batch temperature top_k top_p min_p rand out stream",
    dict(logits=FAKE, stride=1000, vocab=1000, batch=0, temperature=FAKE, top_k=FAKE, top_p=FAKE,
         min_p=FAKE, rand=FAKE, out=FAKE, stream=None))


def test_nothing_to_do_is_accepted():
    assert [f() for f in (APPEND, UNPACK, DECODE, SAMPLE)] == [0, 0, 0, 0]
    assert SAMPLE(temperature=None, top_k=None, top_p=None, min_p=None) == 0
    assert UNPACK(batch=3, longest=0) == 0


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("q_out", "qkv", "pos", "slot", "cos", "sin", "kv")],
    (INVALID, dict(rows=-1)), (INVALID, dict(layer=2)), (INVALID, dict(layer=-1)),
    (INVALID, dict(layers=0)), (INVALID, dict(hq=0)), (INVALID, dict(hkv=0)),
    (INVALID, dict(blocks=0)), (INVALID, dict(blocks=1 << 27)), (INVALID, dict(rope_rows=0)),
    (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=float("nan"))), (INVALID, dict(eps=float("inf"))),
    (INVALID, dict(row=17 * 64)), (INVALID, dict(q_out_stride=13 * 64)),
    (HEAD_DIM, dict(hd=96)), (SHAPE, dict(hq=15, q_out_stride=1 << 12, row=1 << 12)),
    *[(ALIGN, {k: FAKE + 8}) for k in ("q_out", "qkv", "cos", "sin", "kv", "qb", "kb", "vb", "qn", "kn")],
    (ALIGN, dict(row=18 * 64 + 4)), (ALIGN, dict(q_out_stride=14 * 64 + 4)),
    (SHAPE, dict(rows=2 ** 30)),  # more heads than a 32-bit count holds
])
def test_append_refusals(status, kw):
    assert APPEND(**kw) == status


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("k", "v", "kv", "tables", "lens")],
    (INVALID, dict(batch=-1)), (INVALID, dict(layers=0)), (INVALID, dict(layer=2)),
    (INVALID, dict(hkv=0)), (INVALID, dict(blocks=0)), (INVALID, dict(stride=0)),
    (INVALID, dict(longest=-1)), (INVALID, dict(offset=2)), (INVALID, dict(offset=-1)),
    (INVALID, dict(batch=1, longest=129)), (HEAD_DIM, dict(hd=32)),
    (INVALID, dict(batch=2 ** 31 - 1, stride=1 << 20, longest=1 << 24)),
    (INVALID, dict(batch=1 << 20, stride=1 << 20, longest=1 << 24, hkv=2 ** 30)),
    *[(ALIGN, {k: FAKE + 8}) for k in ("k", "v", "kv")],
])
def test_unpack_refusals(status, kw):
    assert UNPACK(**kw) == status


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("out", "q", "kv", "tables", "lens")],
    (INVALID, dict(batch=-1)), (INVALID, dict(tokens=0)), (INVALID, dict(layers=0)),
    (INVALID, dict(layer=2)), (INVALID, dict(blocks=0)), (INVALID, dict(stride=0)),
    (INVALID, dict(stride=1 << 28)), (INVALID, dict(blocks=1 << 31)), (INVALID, dict(longest=-1)),
    (INVALID, dict(offset=2)), (INVALID, dict(q_stride=13 * 64)), (INVALID, dict(out_stride=13 * 64)),
    (INVALID, dict(batch=1 << 22)), (HEAD_DIM, dict(hd=256)),
    (SHAPE, dict(hq=15, q_stride=1 << 12, out_stride=1 << 12)),
    (ALIGN, dict(q=FAKE + 8)), (ALIGN, dict(kv=FAKE + 8)), (ALIGN, dict(out=FAKE + 1)),
    (ALIGN, dict(q_stride=14 * 64 + 4)), (ALIGN, dict(batch=1, ws=FAKE + 8)),
    (WORKSPACE, dict(batch=1, ws=None)), (WORKSPACE, dict(batch=1, ws_bytes=100)),
])
def test_decode_refusals(status, kw):
    assert DECODE(**kw) == status


@pytest.mark.parametrize("status,kw", [
    *[(INVALID, {k: None}) for k in ("logits", "rand", "out")],
    (INVALID, dict(vocab=0)), (INVALID, dict(vocab=1001)), (INVALID, dict(batch=-1)),
    (ALIGN, dict(logits=FAKE + 1)),
])
def test_sample_refusals(status, kw):
    assert SAMPLE(**kw) == status


def test_sizes():
    assert [L.kv8_page_bytes(d) for d in (64, 128, 32)] == [2064, 4112, 0]
    with pytest.raises(L.LucciolaError):
        L.alloc_kv8_pool(4, 1, 2, 96, device="cpu")
    size = L.lib.lc_paged_decode_kv8_workspace_size
    assert size(4, 14, 2, 64, 1) > 0
    assert [size(0, 14, 2, 64, 1), size(4, 15, 2, 64, 1), size(4, 14, 2, 96, 1),
            size(4, 14, 2, 64, 0), size(4, 0, 2, 64, 1)] == [0] * 5


def test_packed_calls():
    """Arguments in one block: the same refusals, and the block's own."""
    import struct
    call = L.lib.lc_call_packed
    words = struct.pack("QqqqQQQQQQQ", FAKE, 1000, 1000, 0, 0, 0, 0, 0, FAKE, FAKE, 0)
    assert call(3, words, 11) == 0
    assert call(3, words, 10) == INVALID and call(4, words, 11) == INVALID
    assert call(-1, words, 11) == INVALID and call(3, None, 11) == INVALID
    assert call(3, struct.pack("QqqqQQQQQQQ", FAKE, 999, 1000, 0, 0, 0, 0, 0, FAKE, FAKE, 0), 11) == INVALID
    assert call(3, struct.pack("QqqqQQQQQQQ", FAKE, 1000, 1000, -1, 0, 0, 0, 0, FAKE, FAKE, 0), 11) == INVALID
    eps = [FAKE, 14 * 64, FAKE, 18 * 64, 0, FAKE, FAKE, 0, 0, 0, 0, 0, float("nan"), FAKE, FAKE, 4096,
           FAKE, 64, 2, 1, 14, 2, 64, 0, 0]
    fmt = "QqQqqQQQQQQQdQQqQqqqqqqQQ"
    assert call(0, struct.pack(fmt, *eps), 25) == INVALID
    eps[12] = 1e-6
    assert call(0, struct.pack(fmt, *eps), 25) == 0
