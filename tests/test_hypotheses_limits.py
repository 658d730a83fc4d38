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


def _array(source, target, **more):
    return native.LeoStateArray(**{**dict(source=source, target=target, outer=8, width=64, source_row=1024, source_outer=128,
                                          target_row=1024, target_outer=128), **more})


@pytest.mark.parametrize("groups, beams, kept", [(1, 1, 1), (1, 2, 1), (1, 1, 2), (2, 4, 4)])
def test_pieces_that_meet_are_refused_in_single_rows_too(groups, beams, kept):
    at, lib = 1 << 20, native.load()
    for first, second in (((1 << 30, at), (1 << 31, at + 63)),                      # targets, by one byte
                          ((1 << 30, at), (at + 64 + 127, 1 << 31)),                # a source, by one byte past the end
                          ((1 << 30, at), (1 << 31, at)), ((1 << 30, at), (at, 1 << 31))):
        entries = (native.LeoStateArray * 2)(_array(*first), _array(*second))
        args = native.LeoReorder(arrays=ctypes.addressof(entries), count=2, groups=groups, beams=beams, kept=kept, parents=256)
        assert "overlaps another array" in _refused("leo_reorder_states", ctypes.byref(args), None)
    entries = (native.LeoStateArray * 2)(_array(1 << 30, at, outer=1), _array(1 << 31, at + 63, outer=1))
    args = native.LeoReorder(arrays=ctypes.addressof(entries), count=2, groups=1, beams=1, kept=1, parents=256)
    assert "overlaps another array" in _refused("leo_reorder_states", ctypes.byref(args), None)


@pytest.mark.parametrize("outputs, inputs, rows", [((1 << 30) + 1, 64, 1), (1 << 31, 1, 16), ((1 << 28) + 1, 64, 17),
                                                   ((1 << 29) + 1, 2000, 16)])
def test_results_past_a_launch_are_refused(outputs, inputs, rows):
    lib, shape, size = native.load(), native.LeoQ8Shape(outputs=outputs, inputs=inputs), ctypes.c_uint64()
    assert lib.leo_q8_workspace_bytes(ctypes.byref(shape), rows, native.TYPE_F32, ctypes.byref(size)) == native.OK
    product = native.LeoQ8Product(shape=shape, layout=1 << 44, layout_bytes=1 << 43, rows=rows, x=1 << 20, x_stride=inputs,
                                  y=1 << 45, y_stride=outputs, x_type=native.TYPE_F32, y_type=native.TYPE_F32,
                                  workspace=1 << 40, workspace_bytes=1 << 43)
    assert "too large" in _refused("leo_q8_matmul", ctypes.byref(product), None)


@pytest.mark.parametrize("rows, y, y_type", [(2, 8192, native.TYPE_F32), (3, 8192 - 4 * 20, native.TYPE_F32),
                                             (1, 8192 + 4, native.TYPE_F32), (1, 8192 - 4 * 15, native.TYPE_F32),
                                             (1, 8192, native.TYPE_F16), (1, 8192 + 62, native.TYPE_BF16)])
def test_results_over_the_bias_are_refused(rows, y, y_type):
    good = dict(layout=1 << 20, layout_bytes=1 << 20, rows=rows, x=1 << 28, x_stride=128, bias=8192, y=y, y_stride=20,
                x_type=native.TYPE_F32, y_type=y_type, workspace=1 << 24, workspace_bytes=1 << 20)
    eight = native.LeoQ8Product(shape=native.LeoQ8Shape(outputs=16, inputs=128), **good)
    assert "overlaps the bias" in _refused("leo_q8_matmul", ctypes.byref(eight), None)
    four = native.LeoQ4Product(shape=native.LeoQ4Shape(outputs=16, inputs=128, group=32, scale_type=native.TYPE_F32), **good)
    assert "overlaps the bias" in _refused("leo_q4_matvec", ctypes.byref(four), None)
