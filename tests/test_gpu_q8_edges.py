"""Edges of the 8-bit products that random inputs do not reach."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from leo_amd import decode
from tests.test_gpu_q8 import check, make

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def largest_for(scale):
    """A float32 whose product with float(1 / 127) is `scale`."""
    inverse = np.float32(1) / np.float32(127)
    at = np.float32(np.float64(scale) / np.float64(inverse))
    for value in (at, np.nextafter(at, np.float32(np.inf)), np.nextafter(at, np.float32(0))):
        if np.float32(value * inverse) == scale:
            return value
    return None


@pytest.mark.parametrize("seed", range(4))
def test_codes_next_to_a_half_of_odd_scales(require_gpu, seed):
    """Half of a scale in [2^-126, 2^-125) with an odd last bit is no float."""
    rng = np.random.default_rng(seed)
    scale = largest = None
    while largest is None:
        scale = np.float32(2.0 ** -126 * (1 + (2 * int(rng.integers(0, 1 << 22)) + 1) * 2.0 ** -23))
        largest = largest_for(scale)
    values = []
    for n in range(-127, 127):
        border = np.float32((n + 0.5) * np.float64(scale))
        values += [border, np.nextafter(border, np.float32(np.inf)), np.nextafter(border, np.float32(-np.inf))]
    values = torch.tensor(np.array(values, dtype=np.float32), device=DEVICE).clamp(-float(largest), float(largest))
    want = torch.round(values.double() / float(scale))
    # a row for each value, beside the one that sets the scale
    rows = torch.stack([torch.full_like(values, float(largest)), values], dim=1)
    codes = torch.tensor([[0, 1], [1, 0]], device=DEVICE, dtype=torch.int8)
    got = decode.q8_matmul(rows, decode.Q8Weight(codes, torch.ones(2, device=DEVICE)))
    assert torch.equal((got[:, 0].double() / float(scale)).round(), want)
    # and all in one row, each read by its own output
    row = torch.cat([torch.tensor([float(largest)], device=DEVICE), values])[None]
    eye = torch.eye(row.shape[1], device=DEVICE).to(torch.int8)
    got = decode.q8_matmul(row, decode.Q8Weight(eye, torch.ones(row.shape[1], device=DEVICE)))
    assert torch.equal((got[0, 1:].double() / float(scale)).round(), want)


def test_more_than_2_32_threads_join(require_gpu):
    """A result of 2^32 values of two slices."""
    rows = outputs = 65_536
    inputs = 131_073
    gen = torch.Generator(DEVICE).manual_seed(1)
    codes = torch.randint(-128, 128, (outputs, inputs), generator=gen, device=DEVICE, dtype=torch.int8)
    scales = torch.rand(outputs, generator=gen, device=DEVICE) * 0.01
    one = torch.randn(1, inputs, generator=gen, device=DEVICE, dtype=torch.bfloat16)
    weight = decode.Q8Weight(codes, scales)
    some = torch.tensor([0, 1, 255, 256, 4097, 30_000, 65_279, 65_280, 65_534, 65_535], device=DEVICE)
    kept = codes[some]
    del codes
    got = decode.q8_matmul(one.expand(rows, inputs), weight)
    check(got[:1][:, some].contiguous(), one, kept, scales[some], None)
    for begin in range(0, rows, 4096):
        assert bool((got[begin:begin + 4096] == got[:1]).all())


def test_one_row_is_added_to_its_bias(require_gpu):
    """The bias may be the result itself where there is one row: y = y + x W^T."""
    for inputs, outputs in ((64, 8), (1024, 257), (100_000, 257), (9000, 2100)):
        x, codes, scales, bias = make(inputs, 1, inputs, outputs, torch.float32, torch.float32)
        weight, y = decode.Q8Weight(codes, scales), bias[None].clone()
        decode.q8_matmul(x, weight, y[0], out=y)
        check(y, x, codes, scales, bias)
        packed = decode.Q4Weight.quantize(torch.randn(outputs, inputs, device=DEVICE))
        want, y = decode.q4_matvec(x, packed, bias), bias[None].clone()
        decode.q4_matvec(x, packed, y[0], out=y)
        assert torch.equal(y, want)
