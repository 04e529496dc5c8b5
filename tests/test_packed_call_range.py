"""lc_call_packed: a word that its int parameter cannot hold is refused, not cut to its low half.
No GPU needed: the calls have no rows."""
import struct

import pytest

import lucciola as L
from test_step_kv4_abi import FAKE, INVALID

SAMPLE = [FAKE, 1000, 1000, 0, 0, 0, 0, 0, FAKE, FAKE, 0]
DECODE = [FAKE, 14 * 64, FAKE, 14 * 64, FAKE, 64, 2, 1, 14, 2, 64, FAKE, 64, FAKE, 0, 0, 1, 0, 0.125, FAKE,
          1 << 40, 0, 0]
# index of an int parameter -> its name
SAMPLE_INTS = {2: "vocab", 3: "batch"}
DECODE_INTS = {6: "num_layers", 7: "layer", 8: "num_q_heads", 9: "num_kv_heads", 10: "head_dim",
               12: "table_stride", 14: "len_offset", 15: "batch", 16: "tokens_per_seq",
               17: "max_context_len"}


def call(entry, fmt, words):
    return L.lib.lc_call_packed(entry, struct.pack(fmt, *words), len(words))


@pytest.mark.parametrize("entry,fmt,words,ints", [
    (3, "QqqqQQQQQQQ", SAMPLE, SAMPLE_INTS),
    (2, "QqQqQqqqqqqQqQqqqqdQQQQ", DECODE, DECODE_INTS),
], ids=["sample", "decode"])
def test_words_beyond_an_int(entry, fmt, words, ints):
    assert call(entry, fmt, words) == 0
    for at, name in ints.items():
        for wrap in (1 << 32, -(1 << 32), 5 << 40):
            bad = list(words)
            bad[at] += wrap
            assert call(entry, fmt, bad) == INVALID, name
    # 64-bit parameters take 64 bits
    wide = list(words)
    wide[1] = 1 << 33
    assert call(entry, fmt, wide) == 0
