"""Edges of the decoding operators on the GPU: empty mask tables, quotients at the
ends of float32, temperatures that are no powers of two, operands of every
alignment, results that share memory with their operands, scales at the ends of
their type."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leo_amd import decode, native
from tests.test_gpu_decode_q4 import check, dense, make
from tests.test_gpu_decode_symbols import DEVICE, TYPES, compare, gumbel, per_row

pytestmark = pytest.mark.gpu


def refused(call):
    with pytest.raises(native.LeoError) as err:
        call()
    assert err.value.code == native.ERR_INVALID_ARGUMENT and str(err.value)


def test_an_empty_table_of_masks_is_refused(require_gpu):
    z = torch.randn(3, 100, device=DEVICE)
    empty = torch.zeros(0, 4, dtype=torch.int32, device=DEVICE)
    refused(lambda: decode.control_logits(z, masks=empty))
    refused(lambda: decode.control_logits(z, masks=empty, mask_rows=torch.zeros(3, dtype=torch.int32, device=DEVICE)))
    refused(lambda: decode.control_logits(z, masks=empty, mask_rows=torch.full((3,), -1, dtype=torch.int32, device=DEVICE)))


@pytest.mark.parametrize("rows", [1, 3, 20, 70])
def test_results_beside_their_operands(require_gpu, rows):
    # columns of one buffer, and neighbours in memory, share nothing
    codes, scales, z = make(96, 128, 32, torch.float16, True, 21)
    weight = decode.Q4Weight(codes, scales, z, inputs=128, group=32)
    w = dense(codes, scales, z, 128, 32)
    for dtype in TYPES:
        x = torch.randn(rows, 128, device=DEVICE).to(dtype)
        wide = torch.zeros(rows, 300, device=DEVICE, dtype=dtype)
        flat = torch.zeros(rows * 224, device=DEVICE, dtype=dtype)
        for a, out in ((wide[:, 40:168], wide[:, 168:264]), (wide[:, 96:224], wide[:, :96]),
                       (flat[:rows * 128].view(rows, 128), flat[rows * 128:].view(rows, 96)),
                       (flat[rows * 96:].view(rows, 128), flat[:rows * 96].view(rows, 96))):
            a.copy_(x)
            check(decode.q4_matvec(a, weight, out=out), x, w, None, dtype)
            assert torch.equal(a, x)
        refused(lambda: decode.q4_matvec(wide[:, :128], weight, out=wide[:, 100:196]))
    z = torch.randn(rows, 400, device=DEVICE)
    want = decode.control_logits(z[:, :180], presence=per_row([1.0] * rows))
    assert torch.equal(decode.control_logits(z[:, :180], out=z[:, 200:380]), want)
    assert torch.equal(decode.control_logits(z[:, 200:380], out=z[:, 20:200]), want)
    refused(lambda: decode.control_logits(z[:, :180], out=z[:, 20:200]))
    assert torch.equal(decode.control_logits(z[:, 20:200], out=z[:, 20:200]), want)
