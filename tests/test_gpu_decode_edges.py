"""Edges of the decoding operators on the GPU: empty mask tables, quotients at the
ends of float32, temperatures that are no powers of two, operands of every
alignment, results that share memory with their operands, scales at the ends of
their type."""
from __future__ import annotations

import math

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("symbols", [5, 257, 20_001])
def test_rows_of_the_types_lowest_value_have_a_symbol(require_gpu, dtype, symbols):
    # finite logits that a temperature below 1 takes out of float32: the row is not one of -inf
    lowest, t = torch.finfo(dtype).min, [0.7, 1.0, 1.3, 0.0, 0.5, 0.7]
    logits = torch.full((6, symbols), lowest, device=DEVICE, dtype=dtype)
    logits[4, 0] = -math.inf
    logits[5] = -lowest
    noise = torch.zeros(6, symbols, device=DEVICE)
    noise[:, 3] = 1.0
    for extra in ({}, {"top_k": torch.full((6,), 2, dtype=torch.int32, device=DEVICE)}, {"top_p": per_row([0.5] * 6)},
                  {"min_p": per_row([0.5] * 6)}):
        got, logprob = decode.sample(logits, noise, temperature=per_row(t), **extra)
        # next to such a logit the noise is below a float32 step: all are equal, the lowest comes first
        assert got.tolist() == [0, 0, 0, 0, 1, 0]
        want = torch.full((6,), -math.log(symbols), device=DEVICE)
        want[4] = -math.log(symbols - 1)
        assert bool(((logprob - want).abs() <= 1e-5 * (1 + want.abs())).all())


def test_a_lowest_value_among_others_is_out_of_the_race(require_gpu):
    logits = torch.full((2, 300), torch.finfo(torch.float32).min, device=DEVICE)
    logits[0, 77] = -3.0
    logits[1, 44] = 3e38
    got, logprob = decode.sample(logits, torch.zeros(2, 300, device=DEVICE), temperature=per_row([0.6, 0.6]))
    assert got.tolist() == [77, 44] and logprob.tolist() == [0.0, 0.0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("symbols", [3000, 16_384, 16_385, 40_001])
def test_temperatures_that_are_no_powers_of_two(require_gpu, dtype, symbols):
    # top-k counts are whole numbers, so the symbol is exact where z is the float32 quotient: this holds the corrected
    # product with the reciprocal to a division, and the undivided bound that values are gathered by to its margin
    gen = torch.Generator(DEVICE).manual_seed(symbols)
    t = [0.7, 0.8, 1.3, 0.6, 3.1, 0.05, 17.3, 1e-3, 911.0, 0.9999999, 1.0000001, 0.333]
    rows = len(t)
    logits = (torch.randn(rows, symbols, generator=gen, device=DEVICE) * 2.5).to(dtype)
    noise = gumbel(gen, rows, symbols)
    for scale in (1.0, -3.0):      # against the order of the values: many turns before one that stays
        for k in ([1, 2, 40, 500, 7, 3, 1000, symbols, 40, 5, 60, 20], [40] * rows):
            compare(logits, noise + (scale < 0) * scale * logits.float() / per_row(t)[:, None], t, k, [1.0] * rows, [0.0] * rows)


@pytest.mark.parametrize("symbols", [3000, 40_001])
@pytest.mark.parametrize("size", [1e-20, 1e20])
def test_temperatures_with_small_and_large_logits(require_gpu, symbols, size):
    gen = torch.Generator(DEVICE).manual_seed(symbols + 1)
    logits = torch.randn(6, symbols, generator=gen, device=DEVICE) * size
    t = [0.7 * size, 1.3 * size, 0.8, 0.011 * size, 2.9 * size, 0.6]
    compare(logits, gumbel(gen, 6, symbols), t, [40, 3, 1000, 40, 500, 2], [1.0] * 6, [0.0] * 6)


@pytest.mark.parametrize("symbols", [3000, 40_001])
def test_min_p_at_temperatures_that_are_no_powers_of_two(require_gpu, symbols):
    # quarters over t: the distances to the largest are k / 4 t, and the cut lies between two of them, 2 % of it away
    gen = torch.Generator(DEVICE).manual_seed(symbols + 2)
    t = [0.7, 0.8, 1.3, 0.6]
    logits = (torch.randn(4, symbols, generator=gen, device=DEVICE) * 10).round() / 4
    floor = [math.exp(-(k + 0.5) / 4 / u) for k, u in zip([3, 9, 14, 20], t)]
    noise = gumbel(gen, 4, symbols)
    compare(logits, noise, t, [symbols] * 4, [1.0] * 4, floor)
    compare(logits, noise - 3 * logits / per_row(t)[:, None], t, [symbols, 50, symbols, 400], [1.0] * 4, floor)


@pytest.mark.parametrize("rows,inputs,outputs", [(17, 128, 64), (32, 640, 100), (32, 1000, 257), (24, 24_002, 40),
                                                 (40, 1002, 70)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_on_and_off_word_boundaries(require_gpu, rows, inputs, outputs, dtype):
    # rows at multiples of 4 bytes (even base and stride), a base off them with an even stride, and an odd stride
    for group, scale, zeros in ((32, torch.float16, True), (64, torch.bfloat16, False), (128, torch.float32, True)):
        codes, scales, z = make(outputs, inputs, group, scale, zeros, rows + inputs)
        weight = decode.Q4Weight(codes, scales, z, inputs=inputs, group=group)
        w = dense(codes, scales, z, inputs, group)
        for pad, begin in ((0, 0), (4, 1), (2, 2), (5, 0), (5, 3)):
            x = torch.randn(rows, inputs + pad, device=DEVICE).to(dtype)[:, begin:begin + inputs]
            check(decode.q4_matvec(x, weight), x, w, None, dtype)


def test_scales_that_their_type_cannot_hold_are_refused(require_gpu):
    w = torch.randn(4, 64, device=DEVICE)
    for value in (460_000.0, 1e30, math.inf, math.nan):
        large = w.clone()
        large[1, 40] = value
        refused(lambda: decode.Q4Weight.quantize(large, 32, torch.float16))
    large[1, 40] = 460_000.0
    for dtype in (torch.float32, torch.bfloat16):
        y = decode.q4_matvec(torch.eye(64, device=DEVICE), decode.Q4Weight.quantize(large, 32, dtype))
        assert bool(torch.isfinite(y).all()) and abs(y[40, 1].item() / 460_000.0 - 1) <= 2.0 ** -8


@pytest.mark.parametrize("scale", TYPES)
def test_small_weights_move_by_half_a_step_at_most(require_gpu, scale):
    # groups whose scale is a few of the smallest steps of float16: the scale in its type is the step
    for size in (1e-9, 1e-7, 2.5e-7, 6e-7, 1e-6, 3e-5, 1e-3):
        w = torch.randn(64, 96, device=DEVICE) * size
        weight = decode.Q4Weight.quantize(w, 32, scale)
        got = decode.q4_matvec(torch.eye(96, device=DEVICE), weight, out_dtype=torch.float32).t()
        largest = w.abs().view(64, 3, 32).amax(2)
        # the step is the scale as its type holds it: the largest over 7, or the next of the type's values above it
        grid = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[scale]
        step = largest / 7 * (1 + grid) + (2.0 ** -24 if scale == torch.float16 else 0.0)
        off = (got - w).abs().view(64, 3, 32)
        assert bool((off <= (step * (0.5 + 1e-5))[:, :, None]).all()), (size, (off / step[:, :, None]).max().item())


def test_results_are_tensors(require_gpu):
    weight = decode.Q4Weight.quantize(torch.randn(8, 64, device=DEVICE))
    x = torch.randn(2, 64, device=DEVICE)
    for out in (0, 1, 2, -1, True, 1 << 70):
        refused(lambda: decode.q4_matvec(x, weight, out=out))
        refused(lambda: decode.q4_matvec(x, weight, out_dtype=torch.float32, out=out))


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


def test_a_weight_is_rounded_inside_a_graph(require_gpu):
    w, x = torch.randn(40, 96, device=DEVICE), torch.randn(2, 96, device=DEVICE)
    fixed = w.clone()
    decode.q4_matvec(x, decode.Q4Weight.quantize(w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = decode.q4_matvec(x, decode.Q4Weight.quantize(fixed))
    for factor in (1.0, 3.0, -0.5):
        fixed.copy_(w * factor)
        graph.replay()
        eager = decode.q4_matvec(x, decode.Q4Weight.quantize(w * factor))
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_a_parameter_is_rounded(require_gpu):
    w = torch.nn.Parameter(torch.randn(20, 64, device=DEVICE))
    x = torch.randn(3, 64, device=DEVICE)
    for scale in TYPES:
        got = decode.q4_matvec(x, decode.Q4Weight.quantize(w, 64, scale))
        assert torch.equal(got, decode.q4_matvec(x, decode.Q4Weight.quantize(w.detach().clone(), 64, scale)))
    for scale in (torch.float64, torch.int32, torch.uint8, None):
        refused(lambda: decode.Q4Weight.quantize(w, 64, scale))


@pytest.mark.parametrize("rows", [16_000, 16_384, 16_400])
def test_slices_of_the_most_rows(require_gpu, rows):
    # up to 16,384 rows a product is split over its inputs and joined
    codes, scales, z = make(16, 1100, 32, torch.float16, True, rows)
    weight = decode.Q4Weight(codes, scales, z, inputs=1100, group=32)
    x = torch.randn(rows, 1100, device=DEVICE).to(torch.bfloat16)
    check(decode.q4_matvec(x, weight), x, dense(codes, scales, z, 1100, 32), None, torch.bfloat16)
