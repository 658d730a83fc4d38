"""Control of logits and the draw (leo_control_logits, leo_sample) against plain
statements of their definitions."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leo_amd import decode, native

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def ragged(lists, dtype):
    offsets = np.zeros(len(lists) + 1, dtype=np.int64)
    offsets[1:] = np.cumsum([len(v) for v in lists])
    flat = np.array([e for v in lists for e in v], dtype=dtype)
    return torch.from_numpy(flat).to(DEVICE), torch.from_numpy(offsets).to(DEVICE)


def per_row(values):
    return torch.tensor(values, dtype=torch.float32, device=DEVICE)


def controlled(z, history, r, p, f, bias, masks, mask_rows):
    """(logits, magnitudes) in 64 bits, by the definition, one row after the other."""
    z = z.copy()
    size = np.abs(z)
    rows, symbols = z.shape
    for i in range(rows):
        for v in set(history[i]):
            if 0 <= v < symbols:
                c = history[i].count(v)
                z[i, v] = z[i, v] / r[i] if z[i, v] > 0 else z[i, v] * r[i]
                z[i, v] -= p[i] + f[i] * c
                size[i, v] = size[i, v] * max(r[i], 1 / r[i]) + abs(p[i]) + abs(f[i]) * c
        for v, b in dict(bias[i]).items():
            if 0 <= v < symbols:
                z[i, v] += b
                size[i, v] += abs(b)
        if masks is not None and mask_rows[i] != -1:
            for v in range(symbols):
                word = int(masks[mask_rows[i]][v // 32]) & 0xffffffff if 0 <= mask_rows[i] < len(masks) else 0
                if not word >> (v % 32) & 1:
                    z[i, v] = -math.inf
    return z, size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("symbols", [1, 31, 32, 33, 257, 4095, 4097, 9001])
def test_control_matches_the_definition(require_gpu, dtype, symbols):
    rng = np.random.default_rng(symbols)
    rows = 6
    wide = torch.from_numpy(rng.normal(0, 4, (rows, symbols + 5)).astype(np.float32)).to(DEVICE).to(dtype)
    logits = wide[:, 2:2 + symbols]
    lengths = [0, 1, 2, 300, 1000, 50]
    history = [rng.integers(-1, symbols + 2, n).tolist() for n in lengths]
    history[4] = [int(v) for v in (rng.random(1000) ** 5 * symbols)]
    bias = [[(int(rng.integers(-1, symbols + 1)), float(np.float32(rng.normal()))) for _ in range(n)]
            for n in (3, 0, 1, 64, 64, 2)]
    r, p, f = ([float(np.float32(v)) for v in rng.uniform(0.5, 1.5, rows)] for _ in range(3))
    words = (symbols + 31) // 32
    masks = rng.integers(-2 ** 31, 2 ** 31, (4, words)).astype(np.int32)
    masks[3] = 0
    mask_rows = [0, -1, 3, 2, 7, -2]          # one allows nothing; the last two are no masks' numbers
    ids, offsets = ragged([[v for v, _ in row] for row in bias], np.int32)
    values = torch.tensor([b for row in bias for _, b in row], dtype=torch.float32, device=DEVICE)
    call = dict(history=ragged(history, np.int32), repetition=per_row(r), presence=per_row(p), frequency=per_row(f),
                bias=(ids, values, offsets), masks=torch.from_numpy(masks).to(DEVICE),
                mask_rows=torch.tensor(mask_rows, dtype=torch.int32, device=DEVICE))
    got = decode.control_logits(logits, **call)
    want, size = controlled(logits.double().cpu().numpy(), history, r, p, f, bias, masks, mask_rows)
    out = got.double().cpu().numpy()
    assert got.dtype == dtype and got.shape == logits.shape
    assert np.array_equal(np.isneginf(out), np.isneginf(want))
    fine = np.isfinite(want)
    # six roundings in 32 bits at most, then one to the type
    bound = 6 * 2.0 ** -24 * size + HALF_ULP[dtype] * (np.abs(want) + size * 2.0 ** -21) + 2.0 ** -24
    assert bool((np.abs(out - want)[fine] <= bound[fine]).all())
    # what no list and no mask touches keeps its bits
    bare = decode.control_logits(logits)
    assert torch.equal(bare, logits)
    again = wide.clone()
    into = again[:, 2:2 + symbols]
    assert decode.control_logits(into, **call, out=into) is into
    assert torch.equal(into, got) and torch.equal(again[:, :2], wide[:, :2])
    assert torch.equal(again[:, 2 + symbols:], wide[:, 2 + symbols:])


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_places_may_hold_anything(require_gpu, dtype):
    symbols = 300
    lowest = torch.finfo(dtype).min
    row = [math.nan, math.inf, -math.inf, lowest, -lowest, 0.0]
    logits = torch.tensor([row * 50] * 3, device=DEVICE, dtype=dtype)
    masks = torch.zeros(3, 10, dtype=torch.int32, device=DEVICE)
    masks[1, :] = 0x20            # of the first 32 symbols, the sixth alone
    masks[2, :] = -1
    got = decode.control_logits(logits, masks=masks)
    assert bool(torch.isneginf(got[0]).all())
    allowed = torch.arange(symbols, device=DEVICE) % 32 == 5
    assert torch.equal(got[1][allowed], logits[1][allowed]) and bool(torch.isneginf(got[1][~allowed]).all())
    assert torch.equal(torch.nan_to_num(got[2], nan=5.0), torch.nan_to_num(logits[2], nan=5.0))
    assert torch.equal(torch.isnan(got[2]), torch.isnan(logits[2]))
    one = decode.control_logits(logits, masks=masks[1:2])      # one mask for every row
    assert torch.equal(one[0], got[1]) and torch.equal(one[2], got[1])
    # values at the type's ends under penalties and biases
    history = ragged([[3, 4, 1, 2]] * 3, np.int32)
    got = decode.control_logits(logits[:, :6], history=history, repetition=per_row([2.0] * 3)).float()
    assert got[0, 1] == math.inf and got[0, 2] == -math.inf and got[0, 3] == -math.inf
    assert got[0, 4] == -lowest / 2 and math.isnan(got[0, 0])


def test_long_histories_and_many_rows(require_gpu):
    # counts past 16 bits, every row its own list; the last row's offsets end at the list's end
    symbols, rows = 5000, 70
    logits = torch.randn(rows, symbols, device=DEVICE)
    lists = [[7] * (70_000 if i == 3 else i) + [i] * 2 for i in range(rows)]
    got = decode.control_logits(logits, history=ragged(lists, np.int32), frequency=per_row([0.5] * rows))
    want = logits.clone()
    for i in range(rows):
        counts = {7: lists[i].count(7), i: lists[i].count(i)}
        for v, c in counts.items():
            if c:
                want[i, v] = logits[i, v] - 0.5 * c
    assert torch.equal(got, want)


def test_offsets_outside_the_list_are_held_inside(require_gpu):
    logits = torch.zeros(2, 64, device=DEVICE)
    history = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEVICE)
    offsets = torch.tensor([-5, 2, 1 << 40], dtype=torch.int64, device=DEVICE)
    got = decode.control_logits(logits, history=(history, offsets), presence=per_row([1.0, 1.0]))
    assert got.nonzero().tolist() == [[0, 1], [0, 2], [1, 3]]


# --- the draw ---------------------------------------------------------------------------------------------------------

def drawn(z, noise, t, k, p, floor):
    """One row's symbol and logprob by the definition; z float32."""
    z = np.where(np.isnan(z), np.float32(-np.inf), z)
    if np.isneginf(z).all():
        return -1, -math.inf
    if t > 0:
        z = (z / np.float32(t)).astype(np.float32)
    w = np.where(z == z.max(), 1.0, np.exp(z.astype(np.float64) - float(z.max())))
    if t > 0:
        larger = np.array([(z > v).sum() for v in z]) if z.size < 3000 else None
        if larger is None:
            order = np.sort(z)
            larger = z.size - np.searchsorted(order, z, side="right")
        levels, inverse = np.unique(z, return_inverse=True)
        level_mass = np.bincount(inverse, weights=w)
        mass = (level_mass.sum() - np.cumsum(level_mass))[inverse]
        stays = (larger < max(k, 1)) & ((mass < p * w.sum()) | (p >= 1)) & (w >= floor)
        stays |= z == z.max()
        race = np.where(stays & ~np.isneginf(z), z + noise, -np.inf)
        at = int(np.argmax(race))
    else:
        at = int(np.argmax(z))
    return at, (0.0 if z[at] == z.max() else float(z[at]) - float(z.max())) - math.log(w.sum())


def compare(logits, noise, t, k, p, floor):
    rows = logits.shape[0]
    got, logprob = decode.sample(logits, noise, temperature=per_row(t), top_k=torch.tensor(k, dtype=torch.int32, device=DEVICE),
                                 top_p=per_row(p), min_p=per_row(floor))
    z, g = logits.float().cpu().numpy(), noise.cpu().numpy()
    for i in range(rows):
        at, lp = drawn(z[i], g[i], t[i], k[i], p[i], floor[i])
        assert got[i].item() == at, (i, got[i].item(), at, t[i], k[i], p[i], floor[i])
        # the sum of up to 2^19 terms in a tree of 32-bit additions, then one log: well under 1e-5
        assert logprob[i].item() == lp if math.isinf(lp) else abs(logprob[i].item() - lp) <= 1e-5 * (1 + abs(lp))


def gumbel(gen, rows, symbols):
    return -torch.log(torch.empty(rows, symbols, device=DEVICE).exponential_(generator=gen).clamp_min(1e-30))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("symbols", [1, 2, 63, 64, 65, 257, 1023, 1025, 8193, 40_001])
def test_draws_match_the_definition(require_gpu, dtype, symbols):
    gen = torch.Generator(DEVICE).manual_seed(symbols)
    rows = 24
    # values on a grid of quarters and temperatures that are powers of two: every z is exact, ties are many, and the
    # masses' steps are far wider than a sum's error
    wide = (torch.randn(rows, symbols + 3, generator=gen, device=DEVICE) * 10).round() / 4
    wide = torch.where(torch.rand(rows, symbols + 3, generator=gen, device=DEVICE) < 0.1, torch.full_like(wide, -math.inf), wide)
    wide[5] = -math.inf
    if symbols > 2:
        wide[6, 3] = math.nan
        wide[7, 2:] = 1.5          # all equal
    logits = wide.to(dtype)[:, 1:1 + symbols]
    noise = gumbel(gen, rows, symbols + 1)[:, 1:]
    rng = np.random.default_rng(symbols)
    t = rng.choice([0.0, 0.5, 1.0, 2.0], rows).tolist()
    k = rng.choice([1, 2, 5, 40, symbols, 2 ** 31 - 1], rows).tolist()
    p = rng.choice([1.0, 0.9137, 0.5113, 0.0517, 2.0], rows).tolist()
    floor = rng.choice([0.0, 0.0, 0.0317, 0.41], rows).tolist()
    compare(logits, noise, t, k, p, floor)


def test_noise_that_picks_the_rarest_first(require_gpu):
    # each race is won by the lowest value left: many passes before one that stays
    symbols = 3000
    logits = torch.linspace(-60, 0, symbols, device=DEVICE)[None].repeat(4, 1)
    noise = torch.linspace(100, 0, symbols, device=DEVICE)[None].repeat(4, 1) * 4
    compare(logits, noise, [1.0] * 4, [1, 3, symbols, symbols], [1.0, 1.0, 0.5, 1.0], [0.0, 0.0, 0.0, 0.9])


def test_noise_that_is_no_number_or_infinite(require_gpu):
    logits = torch.randn(3, 500, device=DEVICE)
    noise = torch.full((3, 500), math.nan, device=DEVICE)
    noise[1] = -math.inf
    noise[2] = math.inf
    got, _ = decode.sample(logits, noise, top_k=torch.full((3,), 7, dtype=torch.int32, device=DEVICE))
    for i in range(3):
        kept = torch.topk(logits[i], 7).indices
        assert got[i].item() == kept.min().item()      # equals: the lowest


def test_greedy_rows_ties_and_infinities(require_gpu):
    logits = torch.zeros(5, 9000, device=DEVICE)
    logits[0, [700, 8000]] = 3.0
    logits[1, 8999] = math.inf
    logits[2] = -math.inf
    logits[2, 44] = -5.0
    logits[3] = math.nan
    logits[4, [10, 20]] = math.inf
    for noise in (None, torch.zeros(5, 9000, device=DEVICE)):
        t = None if noise is None else per_row([0.0] * 5)
        got, logprob = decode.sample(logits, noise, temperature=t)
        assert got.tolist() == [700, 8999, 44, -1, 10]
        want = [-math.log(2 + 8998 * math.exp(-3.0)), 0.0, 0.0, -math.inf, -math.log(2)]
        for a, b in zip(logprob.tolist(), want):
            assert a == b or abs(a - b) <= 1e-5 * (1 + abs(b))


def test_parameters_out_of_their_range_keep_the_largest(require_gpu):
    logits = torch.randn(4, 700, device=DEVICE)
    noise = gumbel(torch.Generator(DEVICE).manual_seed(3), 4, 700)
    best = logits.argmax(1).tolist()
    zero = torch.zeros(4, dtype=torch.int32, device=DEVICE)
    assert decode.sample(logits, noise, top_k=zero)[0].tolist() == best
    assert decode.sample(logits, noise, top_k=zero - 9)[0].tolist() == best
    for value in (0.0, -1.0, math.nan):
        assert decode.sample(logits, noise, top_p=per_row([value] * 4))[0].tolist() == best
    assert decode.sample(logits, noise, min_p=per_row([1.5] * 4))[0].tolist() == best
    for value in (-1.0, math.nan):
        assert decode.sample(logits, noise, temperature=per_row([value] * 4))[0].tolist() == best


def test_draws_follow_the_distribution(require_gpu):
    # 40,000 draws of 6 symbols, top-k 4: each frequency within five standard deviations
    n = 40_000
    logits = torch.tensor([2.0, 1.0, 0.5, 0.0, -0.5, -3.0], device=DEVICE)
    noise = gumbel(torch.Generator(DEVICE).manual_seed(9), n, 6)
    got, _ = decode.sample(logits[None].expand(n, 6), noise, top_k=torch.full((n,), 4, dtype=torch.int32, device=DEVICE))
    share = torch.bincount(got, minlength=6).double().cpu() / n
    want = torch.softmax(logits[:4].double().cpu(), 0)
    assert share[4:].sum() == 0
    assert bool(((share[:4] - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all())


def test_draw_in_a_graph_and_on_another_stream(require_gpu):
    gen = torch.Generator(DEVICE).manual_seed(5)
    logits, noise = torch.randn(3, 70_000, device=DEVICE), gumbel(gen, 3, 70_000)
    kept = dict(top_p=per_row([0.9] * 3))
    torch.cuda.synchronize()
    side, results = torch.cuda.Stream(), []
    with torch.cuda.stream(side):
        for _ in range(5):
            results.append(decode.sample(logits, noise, **kept))
    here = [decode.sample(logits, noise, **kept) for _ in range(5)]
    torch.cuda.synchronize()
    for r in results + here[1:]:
        assert torch.equal(r[0], here[0][0]) and torch.equal(r[1], here[0][1])
    graph, fixed = torch.cuda.CUDAGraph(), logits.clone()
    with torch.cuda.graph(graph):
        controlled_logits = decode.control_logits(fixed)
        inside = decode.sample(controlled_logits, noise, **kept)
    for step in range(3):
        fixed.copy_(logits.roll(step * 1000, dims=1))
        graph.replay()
        eager = decode.sample(logits.roll(step * 1000, dims=1), noise, **kept)
        torch.cuda.synchronize()
        assert torch.equal(inside[0], eager[0]) and torch.equal(inside[1], eager[1])


def test_nothing_to_do(require_gpu):
    assert decode.sample(torch.empty(0, 50, device=DEVICE))[0].shape == (0,)
    assert decode.control_logits(torch.empty(0, 50, device=DEVICE)).shape == (0, 50)
    assert decode.control_logits(torch.empty(3, 0, device=DEVICE)).shape == (3, 0)


def test_refusals(require_gpu):
    z = torch.randn(3, 100, device=DEVICE)
    i32 = dict(dtype=torch.int32, device=DEVICE)
    offsets = torch.zeros(4, dtype=torch.int64, device=DEVICE)
    none = torch.zeros(0, **i32)
    bad = [
        lambda: decode.control_logits(z.double()),
        lambda: decode.control_logits(z.cpu()),
        lambda: decode.control_logits(z.t()),
        lambda: decode.control_logits(z[0]),
        lambda: decode.control_logits(z, out=z.half()),
        lambda: decode.control_logits(z, out=z[:2]),
        lambda: decode.control_logits(z, out=z[:1].expand(3, 100)),
        lambda: decode.control_logits(z, history=(none.long(), offsets)),
        lambda: decode.control_logits(z, history=(none, offsets[:3])),
        lambda: decode.control_logits(z, history=(none, offsets.int())),
        lambda: decode.control_logits(z, repetition=per_row([1.0, 1.0])),
        lambda: decode.control_logits(z, bias=(none, per_row([1.0]), offsets)),
        lambda: decode.control_logits(z, masks=torch.zeros(3, 3, **i32)),
        lambda: decode.control_logits(z, masks=torch.zeros(2, 4, **i32)),
        lambda: decode.control_logits(z, masks=torch.zeros(3, 4, device=DEVICE)),
        lambda: decode.control_logits(z, mask_rows=torch.zeros(3, **i32)),
        lambda: decode.control_logits(z, masks=torch.zeros(3, 4, **i32), mask_rows=torch.zeros(2, **i32)),
        lambda: decode.sample(z[:, :0]),
        lambda: decode.sample(z.double()),
        lambda: decode.sample(z, z[:, :50]),
        lambda: decode.sample(z, z.half()),
        lambda: decode.sample(z, z.cpu()),
        lambda: decode.sample(z, z, temperature=per_row([1.0])),
        lambda: decode.sample(z, z, top_k=per_row([1.0] * 3)),
        lambda: decode.sample(z, z, top_p=torch.ones(3)),
    ]
    for call in bad:
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT
