"""Edges of the reordering of states: single rows, and the largest arrays."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from leo_amd import decode
from tests.test_gpu_reorder import expected, random_parents, random_state, same

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


@pytest.mark.parametrize("groups, beams, kept", [(1, 1, 1), (1, 2, 1), (1, 1, 2), (2, 1, 1)])
def test_arrays_that_interleave_in_one_row(require_gpu, groups, beams, kept):
    """Keys and values side by side in each place of a cache, with one hypothesis before or after."""
    rng = np.random.default_rng(8)
    parents = random_parents(rng, groups, kept, beams, outside=True)
    source = random_state(rng, (groups * beams, 9, 2, 24), torch.float16)
    views = [source[:, :, 0], source[:, :, 1]]
    want = [expected(v, parents, beams) for v in views]
    target = random_state(rng, (groups * kept, 9, 2, 24), torch.float16)
    into = [target[:, :, 0], target[:, :, 1]]
    decode.reorder_states(views, parents, out=into)
    assert all(same(v, w) for v, w in zip(into, want))
    if beams == kept:
        decode.reorder_states(views, parents, out=views)
        assert all(same(v, w) for v, w in zip(views, want))


def test_more_than_2_32_threads_reorder(require_gpu):
    """2^31 - 1 pieces of two bytes, each of which may touch two columns."""
    pieces = 2 ** 31 - 1
    source = torch.randint(-2 ** 15, 2 ** 15, (1, pieces, 2), device=DEVICE, dtype=torch.int16)
    target = torch.zeros(1, pieces, 2, device=DEVICE, dtype=torch.int16)
    parents = torch.zeros(1, 1, device=DEVICE, dtype=torch.int32)
    decode.reorder_states(source[:, :, :1], parents, out=target[:, :, :1])
    for begin in range(0, pieces, 1 << 28):
        part = slice(begin, begin + (1 << 28))
        assert torch.equal(target[0, part, 0], source[0, part, 0]) and not bool(target[0, part, 1].any())
