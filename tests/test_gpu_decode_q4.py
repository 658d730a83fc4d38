"""4-bit readout products (leo_q4_layout, leo_q4_matvec) against the formula in
64 bits. The bound is derived, not fitted: every product enters an fp32 sum over
at most inputs/16 + 64 additions, of relative error 2^-24 each against the sum
of magnitudes; a 32-bit x may be split in two halves that keep 22 bits of each
value and 2^-38 of a row's largest; the result is rounded once to its type."""
from __future__ import annotations

import math

import pytest
import torch

from leo_amd import decode, native

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def make(outputs, inputs, group, scale, zeros, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    codes = torch.randint(0, 256, (outputs, (inputs + 1) // 2), generator=gen, device=DEVICE, dtype=torch.uint8)
    groups = -(-inputs // group)
    scales = (torch.rand(outputs, groups, generator=gen, device=DEVICE) - 0.3).to(scale)
    z = torch.randint(0, 16, (outputs, groups), generator=gen, device=DEVICE, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def dense(codes, scales, zeros, inputs, group):
    """The matrix in 64 bits."""
    n = codes.shape[0]
    u = torch.empty(n, 2 * codes.shape[1], device=DEVICE, dtype=torch.float64)
    u[:, 0::2] = (codes & 15).double()
    u[:, 1::2] = (codes >> 4).double()
    at = torch.arange(inputs, device=DEVICE) // group
    z = zeros.double()[:, at] if zeros is not None else 8.0
    return (u[:, :inputs] - z) * scales.double()[:, at]


def check(y, x, w, bias, dtype):
    x64 = x.double()
    want = x64 @ w.t() + (bias.double() if bias is not None else 0.0)
    total = x64.abs() @ w.abs().t() + (bias.double().abs() if bias is not None else 0.0)
    inputs = w.shape[1]
    bound = 2.0 ** -24 * (inputs / 16 + 64) * total
    if x.dtype == torch.float32:
        bound = bound + 2.0 ** -22 * total + 2.0 ** -38 * x64.abs().amax(1, keepdim=True) * w.abs().sum(1)[None]
    bound = bound + HALF_ULP[dtype] * (want.abs() + bound) + SMALLEST[dtype]
    off = (y.double() - want).abs()
    assert y.dtype == dtype
    assert bool((off <= bound).all()), (off / bound).max().item()


SHAPES = [(1, 1, 1), (1, 31, 15), (2, 32, 16), (3, 33, 17), (5, 127, 33), (16, 128, 257), (17, 129, 64), (1, 1000, 257),
          (33, 257, 40), (64, 640, 100), (65, 1001, 50), (4, 4099, 257), (1, 20_000, 31), (130, 300, 20)]


@pytest.mark.parametrize("rows,inputs,outputs", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_products_match_the_formula(require_gpu, rows, inputs, outputs, group):
    for i, dtype in enumerate((torch.float32, torch.float16, torch.bfloat16)):
        scale = (torch.float16, torch.bfloat16, torch.float32)[(i + group // 64) % 3]
        for zeros in (False, True):
            codes, scales, z = make(outputs, inputs, group, scale, zeros, rows + inputs)
            weight = decode.Q4Weight(codes, scales, z, inputs=inputs, group=group)
            x = torch.randn(rows, inputs, device=DEVICE).to(dtype)
            bias = torch.randn(outputs, device=DEVICE) if zeros else None
            check(decode.q4_matvec(x, weight, bias), x, dense(codes, scales, z, inputs, group), bias, dtype)


@pytest.mark.parametrize("scale", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_every_scale_and_result_type(require_gpu, scale, out_dtype):
    codes, scales, z = make(70, 300, 64, scale, True, 1)
    weight = decode.Q4Weight(codes, scales, z, inputs=300, group=64)
    for dtype in HALF_ULP:
        x = (torch.randn(7, 300, device=DEVICE) * 0.1).to(dtype)
        check(decode.q4_matvec(x, weight, out_dtype=out_dtype), x, dense(codes, scales, z, 300, 64), None, out_dtype)


def test_long_rows_are_joined_over_many_slices(require_gpu):
    # one row against few outputs: the inputs are shared out
    codes, scales, z = make(257, 262_144 + 77, 32, torch.float16, True, 2)
    weight = decode.Q4Weight(codes, scales, z, inputs=262_144 + 77, group=32)
    w = dense(codes, scales, z, 262_144 + 77, 32)
    for rows in (1, 3, 20):
        x = torch.randn(rows, 262_144 + 77, device=DEVICE)
        first = decode.q4_matvec(x, weight)
        # a random sum's error grows with the root of its length: a thousandth of the worst case's bound
        total = x.double().abs() @ w.abs().t()
        assert bool(((first.double() - x.double() @ w.t()).abs() <= 2.0 ** -24 * 64 * total).all())
        for _ in range(3):
            assert torch.equal(decode.q4_matvec(x, weight), first)


def test_strides_and_alignment(require_gpu):
    codes, scales, z = make(45, 517, 32, torch.float16, True, 3)
    wide_codes = torch.zeros(45, codes.shape[1] + 3, device=DEVICE, dtype=torch.uint8)
    wide_codes[:, 1:-2] = codes
    wide_scales = torch.zeros(45, scales.shape[1] + 5, device=DEVICE, dtype=torch.float16)
    wide_scales[:, 3:-2] = scales
    weight = decode.Q4Weight(wide_codes[:, 1:-2], wide_scales[:, 3:-2], z, inputs=517, group=32)
    w = dense(codes, scales, z, 517, 32)
    for dtype in HALF_ULP:
        buffer = torch.randn(9, 517 + 13, device=DEVICE).to(dtype)
        for begin in (0, 1, 3):
            x = buffer[:, begin:begin + 517]
            out = torch.full((9, 45 + 11), 7.0, device=DEVICE, dtype=dtype)
            got = decode.q4_matvec(x, weight, out=out[:, 5:50])
            check(got, x, w, None, dtype)
            assert bool((out[:, :5] == 7).all()) and bool((out[:, 50:] == 7).all())
        x = buffer[2:3, :517].expand(4, 517)          # one row, four times
        check(decode.q4_matvec(x, weight), x, w, None, dtype)
        check(decode.q4_matvec(buffer[::2, :517], weight), buffer[::2, :517], w, None, dtype)
        assert torch.equal(decode.q4_matvec(buffer[1, :517], weight), decode.q4_matvec(buffer[1:2, :517], weight)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_ranges_of_x(require_gpu, dtype):
    # values over the whole exponent range of their type, rows apart
    codes, scales, z = make(40, 700, 64, torch.float32, True, 4)
    scales = scales * 1e-3
    weight = decode.Q4Weight(codes, scales, z, inputs=700, group=64)
    w = dense(codes, scales, z, 700, 64)
    exponent = torch.tensor([-126.0, -60.0, -20.0, 0.0, 20.0, 60.0, 120.0], device=DEVICE)
    x = (torch.randn(7, 700, device=DEVICE) * torch.exp2(exponent)[:, None]).to(dtype)
    check(decode.q4_matvec(x, weight), x, w, None, dtype)
    mixed = (torch.randn(3, 700, device=DEVICE) * torch.exp2(torch.randint(-12, 3, (3, 700), device=DEVICE))).to(dtype)
    check(decode.q4_matvec(mixed, weight), mixed, w, None, dtype)
    subnormal = (torch.randn(2, 700, device=DEVICE) * 2.0 ** -130).to(dtype)
    off = (decode.q4_matvec(subnormal, weight).double() - subnormal.double() @ w.t()).abs()
    # a subnormal x may count as 0
    assert bool((off <= 2.0 ** -125 * w.abs().sum(1)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_infinities_and_nan_stay_in_their_row(require_gpu, dtype):
    codes, scales, z = make(50, 260, 32, torch.float16, True, 5)
    weight = decode.Q4Weight(codes, scales, z, inputs=260, group=32)
    w = dense(codes, scales, z, 260, 32)
    x = torch.randn(6, 260, device=DEVICE).to(dtype)
    clean = decode.q4_matvec(x, weight)
    x[1, 7] = math.inf
    x[2, 259] = -math.inf
    x[3, 130] = math.nan
    got = decode.q4_matvec(x, weight)
    for row in (0, 4, 5):
        assert torch.equal(got[row], clean[row])
    assert bool(torch.isnan(got[3]).all())
    for row, k, sign in ((1, 7, 1.0), (2, 259, -1.0)):
        want = sign * math.inf * w[:, k]      # a weight of 0 times infinity is no number
        assert torch.equal(torch.isnan(got[row]), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert torch.equal(got[row][fine].double(), want[fine])


def test_a_group_of_zeros_and_the_largest_codes(require_gpu):
    # scale 0, codes at both ends
    codes = torch.zeros(16, 64, device=DEVICE, dtype=torch.uint8)
    codes[1::2] = 0xff
    scales = torch.ones(16, 4, device=DEVICE)
    scales[3] = 0.0
    x = torch.randn(2, 128, device=DEVICE)
    for zeros in (None, torch.full((16, 4), 15, device=DEVICE, dtype=torch.uint8)):
        weight = decode.Q4Weight(codes, scales, zeros, inputs=128, group=32)
        y = decode.q4_matvec(x, weight)
        check(y, x, dense(codes, scales, zeros, 128, 32), None, torch.float32)
        assert bool((y[:, 3] == 0).all())


def test_rounding_a_matrix(require_gpu):
    # a value moves by half a step of its group at most
    w = torch.randn(257, 1000, device=DEVICE) * 0.05
    for group in (32, 64, 128):
        weight = decode.Q4Weight.quantize(w, group, torch.float32)
        got = decode.q4_matvec(torch.eye(1000, device=DEVICE), weight).t()
        padded = torch.nn.functional.pad(w, (0, -1000 % group)).view(257, -1, group)
        step = (padded.abs().amax(2) / 7).repeat_interleave(group, 1)[:, :1000]
        assert bool(((got - w).abs() <= step * (0.5 + 1e-5)).all())
    assert bool((decode.q4_matvec(torch.ones(1, 40, device=DEVICE),
                                  decode.Q4Weight.quantize(torch.zeros(3, 40, device=DEVICE))) == 0).all())


def test_other_streams_and_graphs(require_gpu):
    codes, scales, z = make(257, 9000, 64, torch.float16, False, 6)
    weight = decode.Q4Weight(codes, scales, z, inputs=9000, group=64)
    x = torch.randn(2, 9000, device=DEVICE)
    want = decode.q4_matvec(x, weight)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    results = []
    with torch.cuda.stream(side):
        for _ in range(10):
            results.append(decode.q4_matvec(x, weight))
    here = [decode.q4_matvec(x, weight) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results + here)
    graph, fixed = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        y = decode.q4_matvec(fixed, weight)
    for scale in (1.0, 2.0, -1.0):
        fixed.copy_(x * scale)
        graph.replay()
        eager = decode.q4_matvec(x * scale, weight)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_no_rows(require_gpu):
    codes, scales, z = make(20, 64, 32, torch.float16, False, 7)
    weight = decode.Q4Weight(codes, scales, z, inputs=64, group=32)
    assert decode.q4_matvec(torch.empty(0, 64, device=DEVICE), weight).shape == (0, 20)


def test_refusals(require_gpu):
    codes, scales, z = make(20, 100, 32, torch.float16, True, 8)
    weight = decode.Q4Weight(codes, scales, z, inputs=100, group=32)
    x = torch.randn(2, 100, device=DEVICE)
    bad = [
        lambda: decode.Q4Weight(codes, scales, z, inputs=100, group=16),
        lambda: decode.Q4Weight(codes, scales, z, inputs=99 * 2, group=32),
        lambda: decode.Q4Weight(codes.int(), scales, z, inputs=100, group=32),
        lambda: decode.Q4Weight(codes, scales[:, :2], z, inputs=100, group=32),
        lambda: decode.Q4Weight(codes, scales, z[:5], inputs=100, group=32),
        lambda: decode.Q4Weight(codes, scales.double(), z, inputs=100, group=32),
        lambda: decode.Q4Weight(codes.t(), scales, z, inputs=40, group=32),
        lambda: decode.Q4Weight(codes.cpu(), scales, z, inputs=100, group=32),
        lambda: decode.Q4Weight.quantize(codes, 32),
        lambda: decode.q4_matvec(x[:, :99], weight),
        lambda: decode.q4_matvec(x.double(), weight),
        lambda: decode.q4_matvec(x.cpu(), weight),
        lambda: decode.q4_matvec(torch.randn(100, 2, device=DEVICE).t(), weight),
        lambda: decode.q4_matvec(x, weight, torch.zeros(19, device=DEVICE)),
        lambda: decode.q4_matvec(x, weight, torch.zeros(20, device=DEVICE, dtype=torch.float16)),
        lambda: decode.q4_matvec(x, weight, out=torch.empty(2, 19, device=DEVICE)),
        lambda: decode.q4_matvec(x, weight, out=torch.empty(1, 20, device=DEVICE).expand(2, 20)),
    ]
    for call in bad:
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT
