"""Edges of the beam selection that random logits do not reach."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leo_amd import decode
from tests.test_gpu_beams import compare

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


@pytest.mark.parametrize("symbols", [900, 32_001, 131_075, 262_147, 2_000_003, 1 << 26])
@pytest.mark.parametrize("top", [0.0, 5.3, -8.7, 1000.1, 1023.9, -1013.3, -70_000.3, 3.0e6])
def test_one_large_logit_above_a_flat_tail(require_gpu, symbols, top):
    """The error of one small term is that of all, so nothing averages out. The bound is that of
    the other selections' sums: 2^-21 of the log."""
    tops, tails = [], []
    for shift in np.linspace(-0.9, 1.1, 16):      # the tail has about as much of the mass as the one
        tops.append(np.float32(top))
        tails.append(np.float32(np.float64(tops[-1]) - math.log(symbols) + shift))
    z = torch.empty(16, symbols, device=DEVICE)
    z.copy_(torch.tensor(np.array(tails), device=DEVICE)[:, None])
    place = symbols // 3
    z[:, place] = torch.tensor(np.array(tops), device=DEVICE)
    assert all(b < a for a, b in zip(tops, tails))
    below = [np.float64(b) - np.float64(a) for a, b in zip(tops, tails)]
    lse = [math.log1p((symbols - 1) * math.exp(d)) for d in below]
    # scores that take the largest logit's log probability back, so that little is left to round
    scores = torch.tensor(lse, device=DEVICE, dtype=torch.float32)[None]
    for rows in ([0], [9], [15], list(range(16))):
        got = decode.beam_select(z[rows[0]:rows[-1] + 1], scores[:, rows[0]:rows[-1] + 1].contiguous(), len(rows) + 2)
        for symbol, parent, score in zip(got.symbols[0].tolist(), got.parents[0].tolist(), got.scores[0].tolist()):
            b = rows[parent]
            want = float(scores[0, b]) + (0.0 if symbol == place else below[b]) - lse[b]
            assert abs(score - want) <= abs(want) * 2.0 ** -24 + 2.0 ** -21, (b, symbol, score - want)
        assert got.symbols[0].tolist()[:len(rows)] == [place] * len(rows)


@pytest.mark.parametrize("symbols", [900, 33_000])
def test_spans_far_apart(require_gpu, symbols):
    """What a row's parts leave is joined exactly, however far apart they lie."""
    rng = np.random.default_rng(symbols)
    for low, high in ((-30.0, 4.0), (1e5, 1.1e5), (-2e6, 12.5), (12.5, 3e6), (-3e38, 3e38), (2.0e6, 2.0e6 + 2), (1048574.0, 1048578.0),
                      (1000.0, 1048.0), (-1048.0, -1000.0), (1020.0, 1026.0), (-1026.0, -1020.0), (-2010.0, -1990.0), (-5000.0, -4990.0)):
        z = torch.from_numpy(rng.uniform(low, high, (4, symbols)).astype(np.float32)).to(DEVICE)
        z[0, ::3] = -1e9
        z[1] = z[1].sort().values
        z[2, symbols // 2:] = low
        z[3, :symbols // 2] = -torch.inf
        compare(z, torch.tensor([[-1.0, -1.5], [-2.0, -1.0]], device=DEVICE), 5)


@pytest.mark.parametrize("penalty", [1.0, 2.0, 3.0, 0.5, 1.5, -1.0])
def test_hypotheses_of_one_rank_come_in_their_order(require_gpu, penalty):
    """Scores that are whole multiples of their length's power: the quotients tie, whatever the length."""
    rng = np.random.default_rng(5)
    for turn in range(6):
        lengths = rng.permutation(np.arange(1, 65))
        if penalty in (1.0, 2.0):
            lengths += 64 * (turn % 3)
        elif penalty in (0.5, 1.5):
            lengths = lengths ** 2
        elif penalty == -1.0:
            lengths = rng.choice([n for n in range(1, 5041) if 5040 % n == 0], 64)
        scores = -5040.0 / lengths if penalty < 0 else -3.0 * np.float64(lengths) ** penalty
        assert (np.float32(scores) == scores).all() and (scores == np.round(scores)).all()
        for symbols in (70, 5000):
            z = torch.randn(64, symbols, device=DEVICE)
            got = decode.beam_select(z, torch.from_numpy(scores.astype(np.float32)).to(DEVICE)[None],
                                     finished=torch.ones(1, 64, dtype=torch.bool, device=DEVICE),
                                     lengths=torch.from_numpy(lengths.astype(np.int32)).to(DEVICE)[None],
                                     length_penalty=penalty)
            assert got.parents[0].tolist() == list(range(64))
            assert got.scores[0].tolist() == scores.tolist()
