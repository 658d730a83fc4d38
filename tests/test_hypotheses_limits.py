"""Sizes of beam selection, reordered states and products that no call may take, without a GPU."""
from __future__ import annotations

import ctypes

import pytest

from leo_amd import native


def _refused(function, *args):
    lib = native.load()
    assert getattr(lib, function)(*args) == native.ERR_INVALID_ARGUMENT
    return native.last_error(lib)


@pytest.mark.parametrize("groups, beams", [((1 << 58) + 1, 64), (1 << 63, 2), ((1 << 63) + 5, 2), ((1 << 64) - 1, 64),
                                           (65_536, 1), (1024, 64), (21_846, 3)])
def test_more_hypotheses_than_the_most_are_refused(groups, beams):
    size = ctypes.c_uint64()
    assert "too many" in _refused("leo_beam_workspace_bytes", groups, beams, 4, 40_000, ctypes.byref(size))
    args = native.LeoBeams(groups=groups, beams=beams, kept=4, symbols=40_000, logits=1 << 44, logits_stride=40_000,
                           type=native.TYPE_F32, scores=1 << 20, out_symbols=1 << 21, out_parents=1 << 22,
                           out_scores=1 << 23, end=-1, workspace=1 << 40, workspace_bytes=1 << 40)
    assert "too many" in _refused("leo_beam_select", ctypes.byref(args), None)


def test_the_most_hypotheses_have_a_workspace():
    lib, size = native.load(), ctypes.c_uint64()
    for groups, beams in ((65_535, 1), (1023, 64), (21_845, 3)):
        assert lib.leo_beam_workspace_bytes(groups, beams, 4, 40_000, ctypes.byref(size)) == native.OK
        assert size.value > 0
