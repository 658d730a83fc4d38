"""Beam selection on the GPU against its definition in 64 bits.

A score is the sum of a score, a logit less the largest, and the log of a sum of
exponentials, rounded to float: half a step of its value, and the error of the sum, each
of whose float terms may be off by 2^-22 of itself: 2^-21 covers it.

The order: candidates of one hypothesis share its error, so theirs is exact, and so are
ties of hypotheses with the same logits and scores. Ranks of different hypotheses may each
be off by e = 2^-21 over the length's power. The k-th largest of numbers that are off by e
at most is off by e at most, so the one found at place k has a rank within 2 e of the k-th
exact one. Hypotheses whose logits are the same in another order come that close."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leo_amd import decode, native

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def reference(logits, scores, kept, finished=None, lengths=None, penalty=0.0, end=None):
    """(symbols, parents, scores, finished, lengths) as nested lists, from the definition."""
    z = logits.detach().cpu().double().numpy()
    s = scores.cpu().double().numpy()
    groups, beams = s.shape
    done = np.zeros_like(s, dtype=bool) if finished is None else finished.cpu().numpy()
    length = np.zeros_like(s, dtype=np.int64) if lengths is None else lengths.cpu().numpy().astype(np.int64)
    z = np.where(np.isnan(z), -np.inf, z)
    out, ranks, off = [], [], [0.0] * groups
    for g in range(groups):
        found = []      # (-rank, hypothesis, place in its row's order, symbol, score)
        for b in range(beams):
            if not s[g, b] > -np.inf:
                continue

            def rank(score, n):
                return score / float(max(n, 1)) ** penalty

            step = 2.0 ** -21 / float(max(length[g, b] + (0 if done[g, b] else 1), 1)) ** penalty
            off[g] = max(off[g], step)
            if done[g, b]:
                found.append((-rank(s[g, b], length[g, b]), b, 0, -1, s[g, b]))
                continue
            row = z[g * beams + b]
            top = row.max()
            if top == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                d = np.where(row == top, 0.0, row - top)
            lse = math.log(np.exp(d).sum())
            for place, v in enumerate(np.lexsort((np.arange(row.size), -row))[:kept]):
                if row[v] > -np.inf and d[v] > -np.inf:
                    score = s[g, b] + (d[v] - lse)
                    found.append((-rank(score, length[g, b] + 1), b, place, int(v), score))
        found.sort()
        ranks.append({(f[1], f[3]): (f[2], -f[0], f[4]) for f in found})
        found = found[:kept]
        rest = kept - len(found)
        out.append(([f[3] for f in found] + [-1] * rest, [f[1] for f in found] + [0] * rest,
                    [f[4] for f in found] + [-np.inf] * rest,
                    [bool(done[g, f[1]]) or (end is not None and f[3] == end) for f in found] + [False] * rest,
                    [int(length[g, f[1]]) + (0 if done[g, f[1]] else 1) for f in found] + [int(length[g, 0])] * rest))
    return [[o[i] for o in out] for i in range(5)], ranks, off


def reorder(want, ranks, off, got):
    """The reference in the order that was found, where it lies within the bound above."""
    for g, (symbols, parents) in enumerate(zip(got.symbols.tolist(), got.parents.tolist())):
        if symbols == want[0][g] and parents == want[1][g]:
            continue
        was = [(want[1][g][k], want[0][g][k], *(w[g][k] for w in want[2:])) for k in range(len(symbols))]
        exact = [ranks[g][p, s][1] if x > -np.inf else None for p, s, x, *_ in was]
        places = {}
        for k, (p, s) in enumerate(zip(parents, symbols)):
            if exact[k] is None:
                assert (s, p) == (-1, 0)
                continue
            place, rank, score = ranks[g][p, s]
            assert place == places.get(p, 0), "out of order within one hypothesis"
            places[p] = place + 1
            assert abs(rank - exact[k]) <= 2 * off[g]
            want[2][g][k] = score
        lookup = {(w[0], w[1]): w[3:] for w in was}
        want[0][g], want[1][g] = symbols, parents
        for i in (3, 4):      # one that took a kept one's place within the bound is not among those
            want[i][g] = [lookup[p, s][i - 3] if (p, s) in lookup else None for p, s in zip(parents, symbols)]


def compare(logits, scores, kept, finished=None, lengths=None, penalty=0.0, end=None, exact=False):
    got = decode.beam_select(logits, scores, kept, finished=finished, lengths=lengths, length_penalty=penalty, end=end)
    want, ranks, off = reference(logits, scores, kept, finished, lengths, penalty, end)
    if not exact:
        reorder(want, ranks, off, got)
    assert got.symbols.tolist() == want[0]
    assert got.parents.tolist() == want[1]
    w, g = np.array(want[2]), got.scores.cpu().double().numpy()
    with np.errstate(over="ignore"):
        fine = np.isfinite(w.astype(np.float32))
    assert np.array_equal(np.isneginf(g), ~fine)
    assert (np.abs(g[fine] - w[fine]) <= np.abs(w[fine]) * 2.0 ** -24 + 2.0 ** -21).all()
    assert (got.finished is None) == (finished is None and end is None)
    def alike(found, wanted):
        return all(w is None or f == w for a, b in zip(found.tolist(), wanted) for f, w in zip(a, b))

    if got.finished is not None:
        assert got.finished.dtype is torch.bool and alike(got.finished, want[3])
    assert (got.lengths is None) == (lengths is None)
    if got.lengths is not None:
        assert got.lengths.dtype is torch.int32 and alike(got.lengths, want[4])
    return got


def make(seed, groups, beams, symbols, dtype, pad=0):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    z = torch.randn(groups * beams, symbols + pad, generator=gen, device=DEVICE) * 3
    z = torch.where(torch.rand(z.shape, generator=gen, device=DEVICE) < 0.1, torch.full_like(z, -torch.inf), z)
    scores = -10 - 3 * torch.rand(groups, beams, generator=gen, device=DEVICE)
    return z.to(dtype)[:, pad:], scores, gen


SIZES = [(1, 1, 1, 1), (1, 1, 5, 3), (2, 3, 4, 2), (1, 4, 257, 4), (3, 4, 257, 8), (2, 8, 1000, 8), (1, 16, 257, 32), (2, 5, 4099, 5),
         (1, 64, 257, 64), (2, 64, 50, 64), (1, 3, 32_001, 6), (1, 8, 70_003, 16), (1, 1, 262_147, 64), (4, 2, 16_385, 1),
         (1, 2, 131_075, 33), (70, 2, 300, 2)]


@pytest.mark.parametrize("groups, beams, symbols, kept", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes_and_types(require_gpu, groups, beams, symbols, kept, dtype):
    z, scores, gen = make(symbols + kept, groups, beams, symbols, TYPES[dtype])
    compare(z, scores, kept)
    finished = torch.rand(groups, beams, generator=gen, device=DEVICE) < 0.3
    lengths = torch.randint(0, 300, (groups, beams), generator=gen, device=DEVICE, dtype=torch.int32)
    compare(z, scores, kept, finished, lengths, 0.7, symbols - 1)
    compare(z, scores, kept, None, lengths, -0.3, 0)
    first = torch.full_like(scores, -torch.inf)
    first[:, 0] = 0.0
    compare(z, first, kept, end=int(z[0].argmax()))


@pytest.mark.parametrize("symbols", [257, 5003, 40_001])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_off_word_boundaries(require_gpu, symbols, dtype):
    for pad in (1, 2, 3, 5):
        z, scores, _ = make(pad, 2, 3, symbols, TYPES[dtype], pad)
        compare(z, scores, 6)


@pytest.mark.parametrize("symbols", [64, 257, 3000, 33_000])
@pytest.mark.parametrize("beams, kept", [(1, 7), (4, 4), (5, 64)])
def test_ties_go_to_the_lowest(require_gpu, symbols, beams, kept):
    groups = 2
    scores = torch.full((groups, beams), -3.0, device=DEVICE)
    z = torch.zeros(groups * beams, symbols, device=DEVICE)
    compare(z, scores, kept, exact=True)                            # everything ties
    z = (torch.arange(symbols, device=DEVICE) % 5).float().repeat(groups * beams, 1)
    compare(z, scores, kept, exact=True)
    compare(-z.flip(1), scores, kept, exact=True)
    z[:] = -torch.inf
    z[:, -1] = 1.0
    compare(z, scores, kept, exact=True)                            # one symbol a row
    z[:, 0] = -0.0
    z[:, symbols // 2] = 0.0
    z[:, -1] = -torch.inf
    compare(z, scores, kept, exact=True)                            # zeros of either sign are equal


@pytest.mark.parametrize("symbols", [130, 2049, 20_000])
@pytest.mark.parametrize("kept", [1, 4, 16, 64])
def test_order_of_rows(require_gpu, symbols, kept):
    """Rows in rising and falling order, and with their largest side by side in every place."""
    rising = torch.linspace(-20, 20, symbols, device=DEVICE)
    rows = [rising, rising.flip(0)]
    for at in (0, 1, 63, 64, symbols // 2, symbols - 65, symbols - 64, symbols - 1):
        row = torch.randn(symbols, device=DEVICE, generator=torch.Generator(DEVICE).manual_seed(at))
        row[max(0, at):at + kept] = 30 + rising[:kept][:max(0, symbols - at)]
        rows.append(row)
    z = torch.stack(rows)
    scores = torch.full((len(rows), 1), -1.0, device=DEVICE)
    for dtype in (torch.float32, torch.bfloat16):
        compare(z.to(dtype), scores, kept)
    compare(z, scores.view(2, -1), kept)


@pytest.mark.parametrize("beams, symbols, kept", [(8, 131_075, 64), (3, 100_000, 40), (64, 9000, 64), (16, 2000, 17)])
def test_more_than_the_pool_holds(require_gpu, beams, symbols, kept):
    """Rows in falling order, whose first lists hold all; ties; one hypothesis of many."""
    gen = torch.Generator(DEVICE).manual_seed(symbols)
    z = torch.randn(beams, symbols, generator=gen, device=DEVICE).sort(dim=1, descending=True).values
    scores = -5 - torch.rand(1, beams, generator=gen, device=DEVICE)
    compare(z, scores, kept)
    compare(z.bfloat16(), scores, kept)
    compare(torch.zeros_like(z), torch.full_like(scores, -1.0), kept, exact=True)
    for alive in (0, beams - 1):
        one = torch.full_like(scores, -torch.inf)
        one[0, alive] = -2.0
        compare(z, one, kept, exact=True)
        compare(z, one, kept, torch.arange(beams, device=DEVICE)[None] == alive, exact=True)


@pytest.mark.parametrize("symbols", [40, 300, 17_000])
def test_special_values(require_gpu, symbols):
    z, scores, _ = make(3, 10, 2, symbols, torch.float32)
    z[0] = -torch.inf                       # a row without a way
    z[2] = z[3] = -torch.inf                # a group without one
    z[4, 5] = torch.nan
    z[5] = torch.nan
    z[6, [3, 7, 11]] = torch.inf            # share all probability
    z[7, 9] = torch.inf
    z[8] = torch.finfo(torch.float32).min   # the type's lowest value
    z[9] = torch.finfo(torch.float32).min
    z[9, 4] = torch.finfo(torch.float32).max
    scores[5] = -torch.inf
    scores[6, 0] = torch.nan
    scores[7] = -1e30
    scores[8] = 0.0
    z[18, 1:] = -torch.inf                  # a probability of 1
    for kept in (1, 2, 5, 64):
        compare(z, scores, kept)
        finished = torch.zeros(10, 2, dtype=torch.bool, device=DEVICE)
        finished[1] = True                  # their logits hold nothing, and are not read
        finished[5] = True
        finished[7, 1] = True
        compare(z, scores, kept, finished, torch.full((10, 2), 7, device=DEVICE, dtype=torch.int32), 1.0, 2)


@pytest.mark.parametrize("dtype, bits, quiet, signalling", [(torch.float32, torch.int32, 0x7fc00000, 0x7f800001),
                                                            (torch.bfloat16, torch.int16, 0x7fc0, 0x7f81),
                                                            (torch.float16, torch.int16, 0x7e00, 0x7c01)])
@pytest.mark.parametrize("symbols", [100, 5000])
def test_every_nan_is_no_way_on(require_gpu, dtype, bits, quiet, signalling, symbols):
    z, scores, _ = make(11, 1, 3, symbols, dtype)
    z = z.contiguous()
    raw = z.view(bits)
    raw[0, ::3] = quiet
    raw[1, ::2] = signalling
    raw[2, 1::5] = signalling
    raw[2, 2::5] = quiet - (1 << 15) if bits is torch.int16 else quiet - (1 << 31)      # with the sign set
    compare(z, scores, 8)


@pytest.mark.parametrize("beams, symbols, kept", [(1, 5_000_003, 7), (2, 8_400_000, 64)])
def test_very_long_rows(require_gpu, beams, symbols, kept):
    gen = torch.Generator(DEVICE).manual_seed(symbols)
    z = torch.randn(beams, symbols, generator=gen, device=DEVICE).clamp_(max=5)
    at = torch.randint(0, symbols, (beams, kept), generator=gen, device=DEVICE)
    top = 20 - 0.125 * torch.arange(beams * kept, device=DEVICE).view(kept, beams).t()      # hypotheses in turn
    z.scatter_(1, at, top)
    assert all(len(set(row)) == kept for row in at.tolist())
    lse = torch.logsumexp(z.double(), dim=1)
    scores = lse.float()[None]      # ranks are the logits, as far as floats go
    got = decode.beam_select(z, scores, kept)
    ranks = (z.double().gather(1, at) - lse[:, None] + scores.double().t()).t().reshape(-1)
    assert got.parents[0].tolist() == [k % beams for k in range(kept)]
    assert got.symbols[0].tolist() == at.t().reshape(-1)[:kept].tolist()
    assert float((got.scores[0].double() - ranks[:kept]).abs().max()) <= 25 * 2.0 ** -24 + 2.0 ** -21


def test_offsets_past_32_bits(require_gpu):
    wide = torch.empty(5, 1 << 30, dtype=torch.bfloat16, device=DEVICE)
    z, scores, _ = make(12, 1, 5, 3000, torch.bfloat16)
    wide[:, 3:3003] = z
    compare(wide[:, 3:3003], scores, 9)
    wide[:, 3:260] = z[:, :257]
    compare(wide[:, 3:260], scores, 9)


def test_lengths(require_gpu):
    z, scores, _ = make(4, 3, 4, 100, torch.float32)
    lengths = torch.tensor([[0, 1, 2, 3], [-5, 2**31 - 2, 0, 10], [2**31 - 2, 1, 1, 1]], device=DEVICE, dtype=torch.int32)
    finished = torch.tensor([[False, True, False, True], [True, False, True, False], [False] * 4], device=DEVICE)
    for penalty in (0.0, 1.0, 2.5, -1.0, 30.0):
        compare(z, scores, 6, finished, lengths, penalty, 7)
    compare(z, scores, 6, torch.ones_like(finished), lengths, 0.5)


def test_results_are_the_same_each_time(require_gpu):
    z, scores, _ = make(6, 2, 8, 90_001, torch.bfloat16)
    first = decode.beam_select(z, scores, 16)
    for _ in range(5):
        again = decode.beam_select(z, scores, 16)
        assert all(torch.equal(a, b) for a, b in zip(first[:3], again[:3]))


def test_streams_and_graphs(require_gpu):
    cases = [make(7, 2, 4, 257, torch.float32)[:2], make(8, 1, 8, 50_001, torch.bfloat16)[:2]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    with torch.cuda.stream(side):
        for graph in graphs:
            with torch.cuda.graph(graph, stream=side):
                held.append([decode.beam_select(z, s, 8, end=1) for z, s in cases])
    torch.cuda.synchronize()
    for _ in range(3):
        for z, s in cases:
            z.normal_()
            s.uniform_(-9, -7)
        eager = [decode.beam_select(z, s, 8, end=1) for z, s in cases]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in held:
            for a, b, (z, s) in zip(got, eager, cases):
                assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))
        compare(*cases[0], 8, end=1)


def test_two_streams_at_once(require_gpu):
    cases = [make(7, 2, 4, 257, torch.float32)[:2], make(8, 1, 8, 50_001, torch.bfloat16)[:2], make(9, 3, 2, 9000, torch.float16)[:2]]
    want = [decode.beam_select(z, s, 8) for z, s in cases]
    torch.cuda.synchronize()
    streams, found = [torch.cuda.Stream() for _ in range(3)], []
    for turn in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                which = (turn + i) % 3
                found.append((decode.beam_select(*cases[which], 8), want[which]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for a, b in found for x, y in zip(a[:3], b[:3]))


def test_results_and_workspaces_are_freed(require_gpu):
    z, scores, _ = make(6, 2, 8, 20_001, torch.bfloat16)
    parents = torch.zeros(2, 8, dtype=torch.int32, device=DEVICE)
    before = torch.cuda.memory_allocated()
    for _ in range(10):
        found = decode.beam_select(z, scores, 16, end=1)
        decode.reorder_states([z, scores.view(16, 1)], found.parents)
        del found
        for call in (lambda: decode.beam_select(z, scores[:1]), lambda: decode.reorder_states([z, scores], parents),
                     lambda: decode.reorder_states([z], parents, out=[scores])):
            with pytest.raises(native.LeoError):
                call()
    assert torch.cuda.memory_allocated() == before


def test_refusals(require_gpu):
    z, scores, _ = make(9, 2, 3, 50, torch.float32)
    flags, lengths = torch.zeros(2, 3, dtype=torch.bool, device=DEVICE), torch.ones(2, 3, dtype=torch.int32, device=DEVICE)
    for call in (
        lambda: decode.beam_select(z[:5], scores),
        lambda: decode.beam_select(z.t(), scores),
        lambda: decode.beam_select(z.cpu(), scores),
        lambda: decode.beam_select(z.double(), scores),
        lambda: decode.beam_select(z[:, :0], scores),
        lambda: decode.beam_select(z, scores.cpu()),
        lambda: decode.beam_select(z, scores.half()),
        lambda: decode.beam_select(z, scores.view(6)),
        lambda: decode.beam_select(z, scores.t()),
        lambda: decode.beam_select(z, scores, 0),
        lambda: decode.beam_select(z, scores, 65),
        lambda: decode.beam_select(z, scores, -1),
        lambda: decode.beam_select(torch.zeros(65, 50, device=DEVICE), torch.zeros(1, 65, device=DEVICE)),
        lambda: decode.beam_select(z, scores, finished=lengths),
        lambda: decode.beam_select(z, scores, finished=flags[:1]),
        lambda: decode.beam_select(z, scores, lengths=lengths.long()),
        lambda: decode.beam_select(z, scores, lengths=lengths[:, :2]),
        lambda: decode.beam_select(z, scores, length_penalty=1.0),
        lambda: decode.beam_select(z, scores, lengths=lengths, length_penalty=float("nan")),
        lambda: decode.beam_select(z, scores, end=50),
        lambda: decode.beam_select(z, scores, end=-1),
        lambda: decode.beam_select(None, scores),
        lambda: decode.beam_select(z, None),
    ):
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT and str(err.value)
    empty = decode.beam_select(z[:0], scores[:0], 4)
    assert empty.symbols.shape == (0, 4)
