"""The UTF-8 grammar of the generator, without a GPU: its states against
Python's strict decoder, its masks against its states."""
from __future__ import annotations

import random

import numpy as np
import pytest

from leo_amd.generate import END, utf8_masks, utf8_table


def accepts(data: bytes):
    """The state after `data`, -1 where it is no beginning of UTF-8."""
    table, state = utf8_table(), 0
    for byte in data:
        state = int(table[state, byte])
        if state < 0:
            return -1
    return state


def decodes(data: bytes) -> bool:
    try:
        data.decode()
        return True
    except UnicodeDecodeError:
        return False


def test_sequences_of_one_and_two_bytes():
    for a in range(256):
        assert (accepts(bytes([a])) == 0) == decodes(bytes([a]))
        for b in range(256):
            assert (accepts(bytes([a, b])) == 0) == decodes(bytes([a, b]))


@pytest.mark.parametrize("length", [3, 4])
def test_longer_sequences_at_every_edge(length):
    edges = [0x00, 0x7F, 0x80, 0x8F, 0x90, 0x9F, 0xA0, 0xBF, 0xC0, 0xC1, 0xC2, 0xDF, 0xE0, 0xE1, 0xEC, 0xED, 0xEE,
             0xEF, 0xF0, 0xF1, 0xF3, 0xF4, 0xF5, 0xFF]
    rng = random.Random(length)
    for lead in range(0xC0, 0x100):
        for second in edges:
            for _ in range(40):
                data = bytes([lead, second] + [rng.choice(edges) for _ in range(length - 2)])
                assert (accepts(data) == 0) == decodes(data), data


def test_every_code_point_passes():
    for point in list(range(0, 0x3000, 7)) + list(range(0xD700, 0xE100)) + list(range(0xFF00, 0x110000, 997)):
        if not 0xD800 <= point < 0xE000:
            assert accepts(chr(point).encode()) == 0


def test_masks_hold_the_allowed_symbols():
    masks, table = utf8_masks(), utf8_table()
    assert masks.shape == (8, 9) and masks.dtype == np.int32
    for state in range(8):
        for symbol in range(288):
            bit = int(masks[state, symbol // 32]) >> (symbol % 32) & 1
            want = table[state, symbol] >= 0 if symbol < 256 else symbol == END and state == 0
            assert bool(bit) == bool(want), (state, symbol)
    # every state leaves something
    assert all(masks[state].any() for state in range(8))
