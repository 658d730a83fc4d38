"""8-bit products on the GPU against the formula in whole numbers and 64 bits.

The quantised rows and the sums of codes are the formula's own. A sum is rounded to float,
so is its product with the output's scale, and the last product with the bias added: 2^-24
each, two of the term and one of the result, which is no larger than the terms are together.
Then half a step of the result's type, or half of its smallest value."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from leo_amd import decode, native

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def quantized(x):
    """Codes and scales of x (float64 of values that float32 holds), as the formula says."""
    largest = x.abs().amax(dim=1)
    scale = (largest.float() * float(np.float32(1) / np.float32(127))).clamp_min(2.0 ** -126)
    good = torch.isfinite(largest)
    scale = torch.where(good, scale, torch.full_like(scale, torch.nan))
    codes = torch.where(good[:, None], torch.round(x / scale.double()[:, None]), torch.zeros_like(x))
    return codes, scale.double()


def reference(x, codes, scales, bias):
    """The result and the magnitude of its terms, in 64 bits on the GPU."""
    q, s = quantized(x.double())
    # exact: whole numbers below 2^53
    sums = q @ codes.double().t()
    terms = sums * s[:, None] * scales.double()
    return terms + (bias.double() if bias is not None else 0.0), terms.abs() + (bias.double().abs() if bias is not None else 0.0)


def check(got, x, codes, scales, bias):
    want, terms = reference(x, codes, scales, bias)
    dtype = got.dtype
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    got, rounded = got.double(), want.to(dtype).double()
    fine = torch.isfinite(rounded) & ~nan
    assert torch.equal(got[~fine & ~nan], rounded[~fine & ~nan])
    bound = want.abs() * (torch.finfo(dtype).eps / 2) + terms * (3.001 * 2.0 ** -24) + TINY[dtype] / 2
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (float(off.max()), int(off.argmax()))


def make(seed, rows, inputs, outputs, dtype, scale_dtype, spread=1.0):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    codes = torch.randint(-128, 128, (outputs, inputs), generator=gen, device=DEVICE, dtype=torch.int8)
    scales = (torch.rand(outputs, generator=gen, device=DEVICE) * 0.01 + 0.001).to(scale_dtype)
    x = (torch.randn(rows, inputs, generator=gen, device=DEVICE) * spread).to(dtype)
    bias = torch.randn(outputs, generator=gen, device=DEVICE)
    return x, codes, scales, bias


SIZES = [(1, 1, 1), (1, 15, 16), (2, 16, 17), (15, 17, 15), (16, 63, 257), (17, 64, 31), (1, 1024, 257), (31, 65, 33),
         (33, 127, 100), (64, 129, 257), (65, 257, 48), (130, 500, 257), (4, 5001, 1030), (300, 1000, 130), (257, 2049, 513),
         (8, 20_001, 257), (1, 40_000, 3), (2, 9000, 2050), (7, 4097, 2100), (16, 3000, 9700), (16, 2048, 257), (140, 300, 20), (200, 1025, 400), (512, 640, 768), (1, 8192, 2048), (48, 4097, 700)]


@pytest.mark.parametrize("rows, inputs, outputs", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes_and_types(require_gpu, rows, inputs, outputs, dtype):
    scale = {"f32": torch.float16, "f16": torch.float32, "bf16": torch.bfloat16}[dtype]
    x, codes, scales, bias = make(rows + inputs + outputs, rows, inputs, outputs, TYPES[dtype], scale)
    weight = decode.Q8Weight(codes, scales)
    check(decode.q8_matmul(x, weight, bias), x, codes, scales, bias)
    check(decode.q8_matmul(x, weight, out_dtype=torch.float32), x, codes, scales, None)
    for to in TYPES.values():
        check(decode.q8_matmul(x[:1], weight, bias, out_dtype=to), x[:1], codes, scales, bias)


@pytest.mark.parametrize("rows", [1, 3, 20, 100, 150])
@pytest.mark.parametrize("inputs, outputs", [(300, 70), (4100, 257)])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(require_gpu, rows, inputs, outputs, dtype):
    x, codes, scales, bias = make(5, rows, inputs + 3, outputs, TYPES[dtype], torch.float32)
    wide = torch.randint(-128, 128, (outputs, inputs + 5), device=DEVICE, dtype=torch.int8)
    codes = wide[:, 3:3 + inputs]
    weight = decode.Q8Weight(codes, scales)
    buffer = torch.full((rows, outputs + 9), 7.0, device=DEVICE, dtype=TYPES[dtype])
    for start in range(4):      # rows off 16-byte boundaries
        mine = x[:, start:start + inputs]
        got = decode.q8_matmul(mine, weight, bias, out=buffer[:, 2:2 + outputs])
        check(got, mine, codes, scales, bias)
        assert bool((buffer[:, :2] == 7).all()) and bool((buffer[:, 2 + outputs:] == 7).all())
    one = x[:1, :inputs].expand(rows, inputs)
    check(decode.q8_matmul(one, weight, bias), one, codes, scales, bias)
    check(decode.q8_matmul(x[0, :inputs], weight, bias)[None], x[:1, :inputs], codes, scales, bias)


@pytest.mark.parametrize("rows", [1, 5, 33])
@pytest.mark.parametrize("inputs", [131_072, 131_073, 300_001])
def test_sums_past_32_bits(require_gpu, rows, inputs):
    codes = torch.full((18, inputs), -128, device=DEVICE, dtype=torch.int8)
    codes[1:9] = 127
    codes[9::2, ::3] = -127
    x = torch.full((rows, inputs), 0.75, device=DEVICE)
    x[rows // 2:] *= -3.0
    scales = torch.full((18,), 0.5, device=DEVICE)
    check(decode.q8_matmul(x, decode.Q8Weight(codes, scales)), x, codes, scales, None)


@pytest.mark.parametrize("rows", [8, 24, 200])
@pytest.mark.parametrize("inputs", [70, 3000])
def test_rows_of_special_values(require_gpu, rows, inputs):
    x, codes, scales, bias = make(9, rows, inputs, 40, torch.float32, torch.float32)
    x[0] = 0
    x[1, inputs // 2] = torch.inf
    x[2, 3] = -torch.inf
    x[3, inputs - 1] = torch.nan
    x[4] *= 1e-40                                  # below the smallest normal float
    x[5] *= 3e37
    x[6, 1:] = 2.0 ** -149
    x[7] = torch.where(torch.arange(inputs, device=DEVICE) % 2 == 0, 127.0, 0.5)     # quotients of exactly a half
    x[7, 1::4] = -1.5
    weight = decode.Q8Weight(codes, scales)
    for to in TYPES.values():
        got = decode.q8_matmul(x, weight, bias, out_dtype=to)
        check(got, x, codes, scales, bias)
        assert bool(torch.isnan(got[1:4]).all()) and not bool(torch.isnan(got[4:]).any())
        if to is torch.float32:
            assert torch.equal(got[0], bias)


@pytest.mark.parametrize("scale", [3.0, 0.7, 1.1e-3, 2.0 ** -126])
def test_codes_next_to_a_half(require_gpu, scale):
    """The rounding of every quotient near a half, seen through weights of one code each."""
    s = np.float32(scale)
    values = [127 * s]
    for n in range(-127, 127):
        border = np.float32((n + 0.5) * np.float64(s))
        values += [border, np.nextafter(border, np.float32(np.inf)), np.nextafter(border, np.float32(-np.inf))]
    x = torch.tensor(np.array(values, dtype=np.float32), device=DEVICE)
    # a row for each value, beside the one that sets the scale
    rows = torch.stack([torch.full_like(x, float(values[0])), x], dim=1)
    codes = torch.tensor([[0, 1], [1, 0]], device=DEVICE, dtype=torch.int8)
    unit = torch.ones(2, device=DEVICE)
    got = decode.q8_matmul(rows, decode.Q8Weight(codes, unit))
    check(got, rows, codes, unit, None)
    q, units = quantized(rows.double())
    assert torch.equal((got[:, 0].double() / units).round(), q[:, 1])


@pytest.mark.parametrize("rows, inputs, outputs", [(2048, 300, 8300), (130, 131_200, 130), (700, 64, 2500), (129, 1, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_tiles(require_gpu, rows, inputs, outputs, dtype):
    x, codes, scales, bias = make(rows, rows, inputs, outputs, TYPES[dtype], torch.float32)
    buffer = torch.full((rows, outputs + 5), 7.0, device=DEVICE, dtype=TYPES[dtype])
    got = decode.q8_matmul(x, decode.Q8Weight(codes, scales), bias, out=buffer[:, 3:3 + outputs])
    check(got, x, codes, scales, bias)
    assert bool((buffer[:, :3] == 7).all()) and bool((buffer[:, 3 + outputs:] == 7).all())


def test_offsets_past_32_bits(require_gpu):
    # rows of x and of the result 2^30 values apart
    wide, out = torch.empty(3, 1 << 30, dtype=torch.bfloat16, device=DEVICE), torch.empty(3, 1 << 30, dtype=torch.float16, device=DEVICE)
    x, codes, scales, bias = make(1, 3, 1100, 300, torch.bfloat16, torch.float32)
    wide[:, 7:1107] = x
    got = decode.q8_matmul(wide[:, 7:1107], decode.Q8Weight(codes, scales), bias, out=out[:, 5:305])
    check(got, x, codes, scales, bias)
    del wide, out, got
    # weights past 4 GiB
    gen = torch.Generator(DEVICE).manual_seed(4)
    codes = torch.randint(-128, 128, (33_000, 140_000), generator=gen, device=DEVICE, dtype=torch.int8)
    scales = torch.rand(33_000, generator=gen, device=DEVICE) * 0.01
    weight = decode.Q8Weight(codes, scales)
    some = torch.tensor([0, 1, 15_339, 15_340, 16_400, 32_000, 32_990, 32_998, 32_999], device=DEVICE)
    for rows in (1, 20, 140):
        x = torch.randn(rows, 140_000, generator=gen, device=DEVICE)
        check(decode.q8_matmul(x, weight)[:, some].contiguous(), x, codes[some], scales[some], None)


@pytest.mark.parametrize("rows", [90, 1000])
@pytest.mark.parametrize("outputs", [1, 16, 17, 33, 49, 112])
def test_many_rows_of_few_outputs(require_gpu, rows, outputs):
    for inputs in (70, 5000):
        x, codes, scales, bias = make(rows + outputs, rows, inputs, outputs, torch.bfloat16, torch.float32)
        check(decode.q8_matmul(x, decode.Q8Weight(codes, scales), bias, out_dtype=torch.float32), x, codes, scales, bias)


def test_two_streams_at_once(require_gpu):
    cases = []
    for rows, inputs, outputs in ((1, 200_000, 257), (40, 9000, 900), (600, 1500, 700), (8, 70_000, 257)):
        x, codes, scales, bias = make(rows, rows, inputs, outputs, torch.bfloat16, torch.float32)
        weight = decode.Q8Weight(codes, scales)
        cases.append((x, weight, bias, decode.q8_matmul(x, weight, bias, out_dtype=torch.float32)))
    torch.cuda.synchronize()
    streams, found = [torch.cuda.Stream() for _ in range(3)], []
    for turn in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                x, weight, bias, want = cases[(turn + i) % len(cases)]
                found.append((decode.q8_matmul(x, weight, bias, out_dtype=torch.float32), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in found)


def test_results_and_workspaces_are_freed(require_gpu):
    weight = decode.Q8Weight.quantize(torch.randn(257, 70_000, device=DEVICE))
    few, many = torch.randn(5, 70_000, device=DEVICE), torch.randn(40, 70_000, device=DEVICE)
    wrong = torch.zeros(3, 5, device=DEVICE)
    before = torch.cuda.memory_allocated()
    for _ in range(10):
        decode.q8_matmul(few, weight)
        decode.q8_matmul(many, weight)
        for call in (lambda: decode.q8_matmul(wrong, weight), lambda: decode.q8_matmul(few, weight, out=wrong)):
            with pytest.raises(native.LeoError):
                call()
    assert torch.cuda.memory_allocated() == before


def test_cancelling_sums_are_exact(require_gpu):
    gen = torch.Generator(DEVICE).manual_seed(3)
    half = torch.randint(-127, 128, (64, 2048), generator=gen, device=DEVICE, dtype=torch.int8)
    codes = torch.cat([half, -half], dim=1)
    codes[:, 0] = -half[:, 0] + 1 - 2 * (half[:, 0] < 0)
    x = torch.randn(20, 2048, generator=gen, device=DEVICE).repeat(1, 2)
    unit = torch.ones(64, device=DEVICE)
    check(decode.q8_matmul(x, decode.Q8Weight(codes, unit)), x, codes, unit, None)


def test_quantize(require_gpu):
    gen = torch.Generator(DEVICE).manual_seed(8)
    weight = torch.randn(50, 333, generator=gen, device=DEVICE)
    weight[3] = 0
    weight[4] *= 1e-40
    packed = decode.Q8Weight.quantize(weight)
    # the identity reads the weight back: each entry off by half of its row's scale, and the roundings beside
    eye = torch.eye(333, device=DEVICE)
    read = decode.q8_matmul(eye, packed).t().double()
    scale = (weight.abs().amax(dim=1) / 127).double().clamp_min(2.0 ** -126)
    assert bool(((read - weight.double()).abs() <= scale[:, None] * (0.5 + 2.0 ** -15) + 2.0 ** -149).all())
    assert bool((read[3] == 0).all())
    for bad in (torch.inf, torch.nan):
        weight[0, 0] = bad
        with pytest.raises(native.LeoError):
            decode.Q8Weight.quantize(weight)


def test_results_are_the_same_each_time(require_gpu):
    for rows, inputs, outputs in ((1, 100_000, 257), (40, 9000, 500), (600, 1500, 700)):
        x, codes, scales, bias = make(1, rows, inputs, outputs, torch.bfloat16, torch.float32)
        weight = decode.Q8Weight(codes, scales)
        first = decode.q8_matmul(x, weight, bias, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(decode.q8_matmul(x, weight, bias, out_dtype=torch.float32), first)


def test_streams_and_graphs(require_gpu):
    cases = []
    for rows, inputs, outputs in ((1, 1024, 257), (6, 70_000, 257), (40, 3000, 600), (300, 1024, 512)):
        x, codes, scales, bias = make(rows, rows, inputs, outputs, torch.float32, torch.float32)
        cases.append((x, decode.Q8Weight(codes, scales), bias, codes, scales))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [decode.q8_matmul(x, w, b) for x, w, b, _, _ in cases]
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        held = []
        for graph in graphs:
            with torch.cuda.graph(graph, stream=side):
                held.append([decode.q8_matmul(x, w, b) for x, w, b, _, _ in cases])
    torch.cuda.synchronize()
    for _ in range(3):
        for x, *_ in cases:
            x.normal_()
        eager = [decode.q8_matmul(x, w, b) for x, w, b, _, _ in cases]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in held:
            for a, b, (x, _, bias, codes, scales) in zip(got, eager, cases):
                assert torch.equal(a, b)
                check(a, x, codes, scales, bias)


def test_refusals(require_gpu):
    x, codes, scales, bias = make(2, 4, 64, 8, torch.float32, torch.float32)
    weight = decode.Q8Weight(codes, scales)
    buffer = torch.zeros(8, 64, device=DEVICE)
    for call in (
        lambda: decode.q8_matmul(x[:, :63], weight),
        lambda: decode.q8_matmul(x.t(), weight),
        lambda: decode.q8_matmul(x.int(), weight),
        lambda: decode.q8_matmul(x.cpu(), weight),
        lambda: decode.q8_matmul([[1.0] * 64], weight),
        lambda: decode.q8_matmul(x, weight, bias[:7]),
        lambda: decode.q8_matmul(x, weight, bias.half()),
        lambda: decode.q8_matmul(x, weight, 1.0),
        lambda: decode.q8_matmul(x, weight, out=1),
        lambda: decode.q8_matmul(x, weight, out_dtype=torch.int8),
        lambda: decode.q8_matmul(x, weight, out=torch.zeros(4, 9, device=DEVICE)),
        lambda: decode.q8_matmul(x, weight, out_dtype=torch.float16, out=torch.zeros(4, 8, device=DEVICE)),
        lambda: decode.q8_matmul(x[0], weight, out=torch.zeros(8, device=DEVICE)),
        lambda: decode.q8_matmul(buffer, weight, out=buffer[:, :8]),
        lambda: decode.Q8Weight(codes.float(), scales),
        lambda: decode.Q8Weight(codes.cpu(), scales),
        lambda: decode.Q8Weight(codes, scales.cpu()),
        lambda: decode.Q8Weight(codes, scales[:7]),
        lambda: decode.Q8Weight(codes, scales[:, None]),
        lambda: decode.Q8Weight(codes, scales.double()),
        lambda: decode.Q8Weight(codes.t(), scales),
        lambda: decode.Q8Weight(codes[:0], scales[:0]),
        lambda: decode.Q8Weight.quantize(codes),
        lambda: decode.Q8Weight.quantize(torch.zeros(0, 4, device=DEVICE)),
    ):
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT and str(err.value)
    assert decode.q8_matmul(x[:0], weight, bias).shape == (0, 8)
