"""Reordered states on the GPU against indexing on the CPU, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from leo_amd import decode, native

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def expected(state, parents, beams):
    """On the CPU: rows by their parents, zeros where there is none."""
    state, parents = state.cpu(), parents.cpu()
    groups, kept = parents.shape
    out = torch.zeros((groups * kept, *state.shape[1:]), dtype=state.dtype)
    for g in range(groups):
        for k in range(kept):
            p = int(parents[g, k])
            if 0 <= p < beams:
                out[g * kept + k] = state[g * beams + p]
    return out


def same(a, b):
    a, b = a.detach().cpu().contiguous(), b.contiguous()
    return a.shape == b.shape and a.dtype == b.dtype and a.view(torch.uint8).equal(b.view(torch.uint8))


def random_state(rng, shape, dtype):
    if dtype is torch.bool:
        return torch.from_numpy(rng.integers(0, 2, shape).astype(bool)).to(DEVICE)
    count = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    raw = torch.from_numpy(rng.integers(0, 256, max(count, 1), dtype=np.uint8))[:count]      # any bits, NaN among them
    return raw.view(dtype).view(shape).to(DEVICE)


def random_parents(rng, groups, kept, beams, outside=False):
    low, high = (-2, beams + 2) if outside else (0, beams)
    return torch.from_numpy(rng.integers(low, high, (groups, kept)).astype(np.int32)).to(DEVICE)


DTYPES = [torch.float32, torch.bfloat16, torch.int8, torch.int64, torch.bool, torch.float64, torch.complex64]


@pytest.mark.parametrize("groups, beams, kept", [(1, 1, 1), (1, 4, 4), (3, 2, 5), (2, 8, 3), (5, 3, 6), (1, 64, 64), (2, 17, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_many_widths(require_gpu, groups, beams, kept, dtype):
    rng = np.random.default_rng(groups * 100 + beams + kept)
    states = [random_state(rng, (groups * beams, *shape), dtype)
              for shape in ((), (1,), (3,), (15,), (16,), (17,), (5, 33), (1000,), (4099,), (3, 1, 700))]
    parents = random_parents(rng, groups, kept, beams, outside=True)
    for state, got in zip(states, decode.reorder_states(states, parents)):
        assert same(got, expected(state, parents, beams))
    got = decode.reorder_states(states[6], parents)
    assert isinstance(got, torch.Tensor) and same(got, expected(states[6], parents, beams))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float32])
@pytest.mark.parametrize("groups, beams", [(1, 4), (3, 6), (2, 16), (1, 33), (2, 64)])
def test_in_place(require_gpu, groups, beams, dtype):
    rng = np.random.default_rng(beams)
    states = [random_state(rng, (groups * beams, *shape), dtype) for shape in ((), (7,), (4, 129), (2, 3000))]
    for parents in (random_parents(rng, groups, beams, beams), random_parents(rng, groups, beams, beams, outside=True),
                    torch.arange(beams - 1, -1, -1, device=DEVICE, dtype=torch.int32).repeat(groups, 1),
                    torch.arange(beams, device=DEVICE, dtype=torch.int32).roll(1).repeat(groups, 1),
                    torch.arange(beams, device=DEVICE, dtype=torch.int32).repeat(groups, 1)):
        want = [expected(s, parents, beams) for s in states]
        got = decode.reorder_states(states, parents, out=states)
        for a, s, w in zip(got, states, want):
            assert a.data_ptr() == s.data_ptr() and same(s, w)


def test_filled_parts_of_caches(require_gpu):
    rng = np.random.default_rng(4)
    groups, beams, kept = 2, 3, 3
    rows, heads, capacity, width = groups * beams, 5, 40, 33
    for dtype in (torch.bfloat16, torch.int8):
        for length in (0, 1, 2, 17, 39, 40):
            whole = random_state(rng, (rows, heads, capacity, width), dtype)
            state, parents = whole[:, :, :length], random_parents(rng, groups, kept, beams)
            want = expected(state, parents, beams)
            assert same(decode.reorder_states(state, parents), want)
            # into another cache, and in place: what is not filled stays
            other = random_state(rng, (rows, heads, capacity + 3, width), dtype)
            keep = other.clone()
            decode.reorder_states([state], parents, out=[other[:, :, :length]])
            assert same(other[:, :, :length], want) and same(other[:, :, length:], keep[:, :, length:].cpu())
            keep = whole.clone()
            decode.reorder_states([state], parents, out=[state])
            assert same(whole[:, :, :length], want) and same(whole[:, :, length:], keep[:, :, length:].cpu())


def test_layouts(require_gpu):
    rng = np.random.default_rng(5)
    groups, beams = 2, 4
    parents = random_parents(rng, groups, beams, beams)
    rows = groups * beams
    # keys and values side by side, layer by layer, in one buffer; all views in place at once
    buffer = random_state(rng, (rows, 3, 2, 5, 24), torch.float16)
    views = [buffer[:, l, i] for l in range(3) for i in range(2)]
    want = [expected(v, parents, beams) for v in views]
    decode.reorder_states(views, parents, out=views)
    assert all(same(v, w) for v, w in zip(views, want))
    # the same inside each head
    buffer = random_state(rng, (rows, 5, 2, 24), torch.int8)
    views = [buffer[:, :, 0], buffer[:, :, 1]]
    want = [expected(v, parents, beams) for v in views]
    decode.reorder_states(views, parents, out=views)
    assert all(same(v, w) for v, w in zip(views, want))
    # from one half of a buffer into the other
    buffer = random_state(rng, (rows, 2, 50), torch.float32)
    want = expected(buffer[:, 0], parents, beams)
    decode.reorder_states(buffer[:, 0], parents, out=buffer[:, 1])
    assert same(buffer[:, 1], want)
    # rows inside layers, every second value, one row for all
    layers = random_state(rng, (3, rows, 100), torch.bfloat16)
    for state in (layers.transpose(0, 1), layers[0][:, ::2], layers[0][:1].expand(rows, 100), layers[1][:, 3:70]):
        assert same(decode.reorder_states(state, parents), expected(state, parents, beams))
    state = layers.transpose(0, 1)
    want = expected(state, parents, beams)
    decode.reorder_states(state, parents, out=state)
    assert same(state, want)


def test_many_arrays(require_gpu):
    rng = np.random.default_rng(6)
    states = [random_state(rng, (6, 1 + i % 37), torch.int16) for i in range(150)]
    parents = random_parents(rng, 2, 3, 3)
    for state, got in zip(states, decode.reorder_states(states, parents)):
        assert same(got, expected(state, parents, 3))
    want = [expected(s, parents, 3) for s in states]
    fresh = [torch.empty_like(s) for s in states[::2]]
    out = [fresh[i // 2] if i % 2 == 0 else s for i, s in enumerate(states)]      # some in place
    decode.reorder_states(states, parents, out=out)
    assert all(same(o, w) for o, w in zip(out, want))
    assert decode.reorder_states([], parents) == []


def test_offsets_past_32_bits(require_gpu):
    # rows 3 GiB apart, their pieces 1 GiB apart
    whole = torch.zeros(4, 3, 1 << 30, dtype=torch.int8, device=DEVICE)
    state = whole[:, :, (1 << 30) - 5000:]
    state.copy_(torch.randint(-128, 128, (4, 3, 5000), dtype=torch.int8, device=DEVICE))
    parents = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device=DEVICE)
    want = expected(state, parents, 2)
    assert same(decode.reorder_states(state, parents), want)
    decode.reorder_states(state, parents, out=state)
    assert same(state, want)


def test_empty_shapes(require_gpu):
    parents = torch.zeros(0, 3, dtype=torch.int32, device=DEVICE)
    assert decode.reorder_states(torch.zeros(0, 7, device=DEVICE), parents).shape == (0, 7)
    parents = torch.zeros(2, 3, dtype=torch.int32, device=DEVICE)
    assert decode.reorder_states(torch.zeros(4, 0, 5, device=DEVICE), parents).shape == (6, 0, 5)


def test_streams_and_graphs(require_gpu):
    rng = np.random.default_rng(7)
    states = [random_state(rng, (8, 3, 500), torch.int32), random_state(rng, (8, 9), torch.int8)]
    parents = random_parents(rng, 2, 4, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            fresh = decode.reorder_states(states, parents)
            decode.reorder_states(states, parents, out=states)
    torch.cuda.synchronize()
    for turn in range(4):
        parents.copy_(random_parents(rng, 2, 4, 4))
        for s in states:
            s.copy_(random_state(rng, tuple(s.shape), s.dtype))
        want = [expected(s, parents, 4) for s in states]
        again = decode.reorder_states(states, parents)
        graph.replay()
        torch.cuda.synchronize()
        for a, f, s, w in zip(again, fresh, states, want):
            assert same(a, w) and same(f, w) and same(s, w), turn


def test_refusals(require_gpu):
    state, parents = torch.zeros(8, 16, device=DEVICE), torch.zeros(2, 4, dtype=torch.int32, device=DEVICE)
    wide = torch.zeros(8, 40, device=DEVICE)
    for call in (
        lambda: decode.reorder_states(state, parents.long()),
        lambda: decode.reorder_states(state, parents[0]),
        lambda: decode.reorder_states(state, parents.t()),
        lambda: decode.reorder_states(state, parents.cpu()),
        lambda: decode.reorder_states(state.cpu(), parents),
        lambda: decode.reorder_states([state, 3], parents),
        lambda: decode.reorder_states(state, None),
        lambda: decode.reorder_states(state[:7], parents),
        lambda: decode.reorder_states([state, state[:6]], parents),
        lambda: decode.reorder_states(state[0, 0], parents),
        lambda: decode.reorder_states(torch.zeros(2 * 65, 4, device=DEVICE), parents),
        lambda: decode.reorder_states(state, torch.zeros(2, 65, dtype=torch.int32, device=DEVICE)),
        lambda: decode.reorder_states(state, torch.zeros(2, 0, dtype=torch.int32, device=DEVICE)),
        lambda: decode.reorder_states(state, parents, out=torch.zeros(8, 15, device=DEVICE)),
        lambda: decode.reorder_states(state, parents, out=torch.zeros(8, 16, device=DEVICE, dtype=torch.float16)),
        lambda: decode.reorder_states([state], parents, out=[]),
        lambda: decode.reorder_states(state, parents[:, :3].contiguous(), out=state),
        lambda: decode.reorder_states(wide[:, :16], parents, out=wide[:, 8:24]),
        lambda: decode.reorder_states([wide[:, :16], wide[:, 20:36]], parents, out=[wide[:, 20:36], wide[:, :16]]),
        lambda: decode.reorder_states([state, state], parents, out=[state, state]),
        lambda: decode.reorder_states(state, parents, out=torch.zeros(1, 16, device=DEVICE).expand(8, 16)),
        lambda: decode.reorder_states(torch.zeros(8, 3, 4, 5, 6, device=DEVICE)[:, ::2, ::2, ::2], parents),
        lambda: decode.reorder_states(torch.zeros(8, 4, device=DEVICE, dtype=torch.complex64).conj(), parents),
    ):
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT and str(err.value)
