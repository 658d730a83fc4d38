"""Refusals of the decoding operators that need no GPU: masks that are not there."""
from __future__ import annotations

import ctypes

import pytest

from leo_amd import native


def refusal(function, struct, fields):
    lib = native.load()
    assert getattr(lib, function)(ctypes.byref(struct(**fields)), None) == native.ERR_INVALID_ARGUMENT
    return native.last_error(lib)


@pytest.mark.parametrize("change", [dict(mask_rows=256), dict(mask_count=3), dict(mask_count=3, mask_rows=256)])
def test_masks_that_are_not_there_shut_nothing_silently(change):
    # a table without rows has no memory: its rows' numbers must not pass as "no masks"
    good = dict(rows=2, symbols=257, logits=256, logits_stride=257, out=4096, out_stride=257, type=native.TYPE_F32)
    assert "masks" in refusal("leo_control_logits", native.LeoLogitControl, {**good, **change})
