"""Lists past 16 bits in the control of logits, and what the operators' binding does
with results, memory and values that are no tensors."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from leo_amd import decode, native
from tests.test_gpu_decode_symbols import compare, gumbel

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


@pytest.mark.parametrize("symbols", [300, 9001, 40_000])
@pytest.mark.parametrize("entries", [65_534, 65_535, 65_536, 90_000])
def test_long_bias_lists(require_gpu, symbols, entries):
    # quarters below 2^13, so that every sum is exact; the last entry for a symbol counts
    rng = np.random.default_rng(entries + symbols)
    rows = 3
    logits = rng.integers(-400, 400, (rows, symbols)).astype(np.float32) / 4
    lengths = [entries, 5, entries]
    ids = [rng.integers(-1, symbols + 1, n).astype(np.int32) for n in lengths]
    values = [rng.integers(-400, 400, n).astype(np.float32) / 4 for n in lengths]
    history = [rng.integers(0, symbols, 40).astype(np.int32) for _ in lengths]
    want = logits.copy()
    for i in range(rows):
        count = np.bincount(history[i], minlength=symbols)
        want[i] -= np.where(count > 0, 0.5 + 0.25 * count, 0).astype(np.float32)
        for v, b in dict(zip(ids[i].tolist(), values[i].tolist())).items():
            if 0 <= v < symbols:
                want[i, v] += b

    def joined(lists):
        offsets = np.concatenate([[0], np.cumsum([len(v) for v in lists])])
        return torch.from_numpy(np.concatenate(lists)).to(DEVICE), torch.from_numpy(offsets.astype(np.int64)).to(DEVICE)

    at, offsets = joined(ids)
    got = decode.control_logits(torch.from_numpy(logits).to(DEVICE), history=joined(history),
                                presence=torch.full((rows,), 0.5, device=DEVICE),
                                frequency=torch.full((rows,), 0.25, device=DEVICE),
                                bias=(at, joined(values)[0], offsets))
    assert np.array_equal(got.cpu().numpy(), want)


def test_results_and_workspaces_are_freed(require_gpu):
    weight = decode.Q4Weight.quantize(torch.randn(257, 4096, device=DEVICE))
    x, z = torch.randn(5, 4096, device=DEVICE), torch.randn(4, 20_000, device=DEVICE)
    wrong = torch.zeros(3, 5, device=DEVICE)
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        decode.sample(decode.control_logits(z))
        decode.q4_matvec(x, weight)
        for call in (lambda: decode.q4_matvec(wrong, weight), lambda: decode.sample(z, wrong),
                     lambda: decode.control_logits(z, out=wrong)):
            with pytest.raises(native.LeoError):
                call()
    assert torch.cuda.memory_allocated() == before


def test_what_is_no_tensor_is_refused(require_gpu):
    weight = decode.Q4Weight.quantize(torch.randn(8, 64, device=DEVICE))
    x = torch.randn(2, 64, device=DEVICE)
    for call in (
        lambda: decode.q4_matvec([[1.0] * 64], weight),
        lambda: decode.q4_matvec(x, weight, 1.0),
        lambda: decode.q4_matvec(x, weight, out=[]),
        lambda: decode.q4_matvec(x, weight, out_dtype=torch.int32),
        lambda: decode.q4_matvec(x, weight, out_dtype=torch.float16, out=torch.empty(2, 8, device=DEVICE)),
        lambda: decode.control_logits(None),
        lambda: decode.control_logits(x, masks=7),
        lambda: decode.control_logits(x, bias=(None, None, torch.zeros(3, dtype=torch.int64, device=DEVICE))),
        lambda: decode.sample(None),
        lambda: decode.sample(x, temperature=1.0),
        lambda: decode.sample(x.cpu()),
    ):
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT and str(err.value)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("symbols", [16_383, 16_384, 16_385, 20_001])
def test_draws_around_the_longest_row_of_one_workgroup(require_gpu, dtype, symbols):
    # quarters and temperatures that are powers of two: every z is exact
    gen = torch.Generator(DEVICE).manual_seed(symbols)
    rows = 12
    wide = (torch.randn(rows, symbols + 1, generator=gen, device=DEVICE) * 10).round() / 4
    wide[3] = -torch.inf
    noise = gumbel(gen, rows, symbols)
    # two rows whose race the lowest value left wins each time: many turns before one that stays
    wide[4:6] = -(torch.arange(symbols + 1, device=DEVICE) % 47) / 4
    noise[4:6] = -5 * wide[4:6, 1:]
    compare(wide.to(dtype)[:, 1:], noise, [0.0, 0.5, 1.0, 1.0, 1.0, 1.0] + [1.0, 2.0] * 3,
            [40, 40, 1, 5, 3, symbols] + [symbols, 2, 40] * 2, [1.0, 0.9137, 0.5113, 1.0, 2.0, 0.9137] + [0.9137, 1.0, 0.0517] * 2,
            [0.0, 0.0317, 0.0, 0.0, 0.0, 0.0317] + [0.0, 0.0317, 0.41] * 2)
