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
