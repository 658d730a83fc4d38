"""Performance cases of the operators that take Leo from activations to the next
symbol: the readout's matrix-vector product with 4-bit weights and group scales,
the control of its logits (penalties, biases, grammar masks) and the draw.

A case names its operator ("op") and sizes. `run` computes it with elementary
torch operations in 32 bits, or, where `own` is true, through leo_amd.decode.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MOST_WEIGHTS = 257 << 20      # the largest readout here: 1,048,576 neurons
MOST_LOGITS = 128 * 131_075


def listed():
    return [
        # the readout of a 1,024-neuron model for one story: latency alone
        _matvec("readout 1k, one row", 1, 1024, 257, 32, "f32", "f16", False, 0.02),
        # eight stories answered together by a 131,072-neuron model
        _matvec("readout 131k, 8 rows", 8, 131_072, 257, 64, "bf16", "bf16", True, 0.05),
        # one story of a 1,048,576-neuron model: a long, flat weight matrix
        _matvec("readout 1M, one row", 1, 1_048_576, 257, 128, "f32", "f32", False, 0.02),
        # a dense square projection for one row, the usual shape of single-symbol serving
        _matvec("dense 8192, one row", 1, 8192, 8192, 128, "bf16", "f16", False, 1.0),
        # a full batch against odd sizes: rows that end inside a group and inside a tile
        _matvec("dense odd, 64 rows", 64, 5001, 11_007, 32, "f16", "f16", True, 1.0),
        # one story's byte logits with a UTF-8 mask and penalties: latency alone
        _control("bytes, one row", 1, 257, "f32", 256, 8, True, 0),
        # a small server's batch over a word-piece vocabulary
        _control("32k symbols, 16 rows", 16, 32_001, "bf16", 1000, 100, True, 0),
        # a full batch over a large vocabulary with long histories, rows of a padded buffer
        _control("131k symbols, 128 rows", 128, 131_075, "f32", 8192, 300, True, 61),
        # one story's next byte: latency alone
        _sample("bytes, one draw", 1, 257, "f32", 40, 0.95, 0.0, 0),
        # a small server's batch, 16-bit logits with many ties
        _sample("32k symbols, 16 draws", 16, 32_001, "bf16", 50, 0.9, 0.0, 0),
        # few long rows: the row has to be shared among workgroups
        _sample("262k symbols, 2 draws", 2, 262_147, "f32", 0, 0.95, 0.02, 0),
        # a full batch over a large vocabulary
        _sample("131k symbols, 128 draws", 128, 131_075, "f32", 200, 0.9, 0.01, 61),
    ]


def _matvec(name, rows, inputs, outputs, group, dtype, scale, zeros, activity):
    return {"name": name, "op": "matvec", "rows": rows, "inputs": inputs, "outputs": outputs, "group": group,
            "dtype": dtype, "scale": scale, "zeros": zeros, "activity": activity}


def _control(name, rows, symbols, dtype, history, biases, masked, pad):
    return {"name": name, "op": "control", "rows": rows, "symbols": symbols, "dtype": dtype, "history": history,
            "biases": biases, "masked": masked, "pad": pad}


def _sample(name, rows, symbols, dtype, top_k, top_p, min_p, pad):
    return {"name": name, "op": "sample", "rows": rows, "symbols": symbols, "dtype": dtype, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "pad": pad}


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["matvec", "control", "sample"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "matvec":
        outputs = 257 if rng.random() < 0.4 else _log_int(rng, 31, 16_384)
        rows = _log_int(rng, 1, 64)
        # rows beyond 16 multiply the products, wide rows of x their bytes
        most = min(MOST_WEIGHTS // (outputs * (1 + rows // 8)), (1 << 21) // rows, 1 << 20)
        inputs = _log_int(rng, min(200, most), most)
        case = _matvec("", rows, inputs, outputs, rng.choice([32, 64, 128]), dtype, rng.choice(["f16", "bf16", "f32"]),
                       rng.random() < 0.5, rng.choice([0.02, 1.0]))
    else:
        rows = _log_int(rng, 1, 128)
        symbols = 257 if rng.random() < 0.25 else _log_int(rng, 200, min(262_147, MOST_LOGITS // rows))
        pad = rng.choice([0, 0, 7, 64])
        if op == "control":
            case = _control("", rows, symbols, dtype, _log_int(rng, 1, 8192), rng.choice([0, 5, 250]),
                            rng.random() < 0.7, pad)
        else:
            case = _sample("", rows, symbols, dtype, rng.choice([0, 1, 20, 500]), rng.choice([1.0, 0.95, 0.5]),
                           rng.choice([0.0, 0.05]), pad)
    del case["name"]
    return case


# --- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    state = {"case": case}
    {"matvec": _prepare_matvec, "control": _prepare_control, "sample": _prepare_sample}[case["op"]](case, gen, state)
    return state


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _uniform(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEVICE)


def _integers(gen, low, high, *shape, dtype=torch.int64):
    return torch.randint(low, high, shape, generator=gen, device=DEVICE, dtype=dtype)


def _padded(values, pad, dtype):
    """`values` as rows of a buffer that is `pad` elements wider."""
    rows, width = values.shape
    buffer = torch.full((rows, width + pad), 7.0, device=DEVICE, dtype=dtype)
    buffer[:, :width] = values.to(dtype)
    return buffer[:, :width]


def _prepare_matvec(case, gen, state):
    m, k, n, g = case["rows"], case["inputs"], case["outputs"], case["group"]
    groups = -(-k // g)
    # two inputs a byte, the even one in the low half; the halves of normal weights cluster about 8
    low, high = (((_normal(gen, n, -(-k // 2)) * 3.0).round() + 8).clamp(0, 15).to(torch.uint8) for _ in range(2))
    state["codes"] = low | (high << 4)
    state["scales"] = (0.004 + 0.02 * _uniform(gen, n, groups)).to(TYPES[case["scale"]])
    state["zeros"] = _integers(gen, 5, 12, n, groups, dtype=torch.uint8) if case["zeros"] else None
    x = _normal(gen, m, k)
    if case["activity"] < 1:      # Leo's activations: few, and none below zero
        x = torch.where(_uniform(gen, m, k) < case["activity"], x.abs(), torch.zeros_like(x))
    state["x"] = x.to(TYPES[case["dtype"]])
    state["bias"] = _normal(gen, n) * 0.5
    if own:
        from leo_amd import decode

        # a serving program lays its weights out once
        state["weight"] = decode.Q4Weight(state["codes"], state["scales"], state["zeros"], inputs=k, group=g)


def _ragged(gen, rows, most):
    """Offsets of `rows` lists of up to `most` entries, every eighth list empty where there are several."""
    lengths = _integers(gen, max(1, most // 2), most + 1, rows) if most else torch.zeros(rows, device=DEVICE, dtype=torch.int64)
    if rows > 1:
        lengths[3::8] = 0
    offsets = torch.zeros(rows + 1, device=DEVICE, dtype=torch.int64)
    torch.cumsum(lengths, 0, out=offsets[1:])
    return offsets, int(offsets[-1])


def _prepare_control(case, gen, state):
    b, v = case["rows"], case["symbols"]
    logits = _normal(gen, b, v) * 3.0
    offsets, total = _ragged(gen, b, case["history"])
    # frequent symbols come often; one in a hundred stands outside the vocabulary (a begin mark)
    symbols = (v * _uniform(gen, total) ** 4).to(torch.int32).clamp(max=v - 1)
    symbols = torch.where(_uniform(gen, total) < 0.01, torch.full_like(symbols, v + 1), symbols)
    state["history"] = (symbols, offsets)
    state["repetition"] = 1.0 + 0.3 * _uniform(gen, b)
    state["presence"] = 0.5 * _uniform(gen, b)
    state["frequency"] = 0.2 * _uniform(gen, b)
    state["bias"] = state["masks"] = state["mask_rows"] = None
    if case["biases"]:
        offsets, total = _ragged(gen, b, case["biases"])
        state["bias"] = (_integers(gen, 0, v, total, dtype=torch.int32), _normal(gen, total) * 2.0, offsets)
    if case["masked"]:
        # a grammar of 32 states; the last allows nothing
        words = -(-v // 32)
        masks = _integers(gen, -(1 << 31), 1 << 31, 32, words).to(torch.int32)
        masks[31] = 0
        state["masks"] = masks
        state["mask_rows"] = (_integers(gen, -1, 31, b)).to(torch.int32)
        state["mask_rows"][b // 2] = 31 if b > 4 else 0
        # what a grammar excludes may hold anything
        at = torch.arange(v, device=DEVICE)
        shut = ((masks[0, at // 32] >> (at % 32)) & 1) == 0
        shut = shut & (state["mask_rows"] == 0)[:, None] & (at % 5 == 0)
        logits = torch.where(shut & (at % 2 == 0), torch.full_like(logits, math.nan), logits)
        logits = torch.where(shut & (at % 2 == 1), torch.full_like(logits, math.inf), logits)
    state["logits"] = _padded(logits, case["pad"], TYPES[case["dtype"]])


def _prepare_sample(case, gen, state):
    b, v = case["rows"], case["symbols"]
    logits = _normal(gen, b, v) * 2.5
    logits = torch.where(_uniform(gen, b, v) < 0.1, torch.full_like(logits, -math.inf), logits)
    if b > 4:
        logits[b // 2] = -math.inf      # a row that its grammar left empty
    state["logits"] = _padded(logits, case["pad"], TYPES[case["dtype"]])
    state["noise"] = -torch.log(torch.empty(b, v, device=DEVICE).exponential_(generator=gen).clamp_min(1e-30))
    state["temperature"] = 0.6 + 0.8 * _uniform(gen, b)
    state["temperature"][5::8] = 0.0     # greedy rows among the others
    state["top_k"] = torch.full((b,), case["top_k"] or v, device=DEVICE, dtype=torch.int32)
    state["top_p"] = torch.full((b,), case["top_p"], device=DEVICE)
    state["min_p"] = torch.full((b,), case["min_p"], device=DEVICE)


# --- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        from leo_amd import decode

        if op == "matvec":
            return decode.q4_matvec(state["x"], state["weight"], state["bias"])
        if op == "control":
            return decode.control_logits(state["logits"], history=state["history"], repetition=state["repetition"],
                                         presence=state["presence"], frequency=state["frequency"],
                                         bias=state["bias"], masks=state["masks"], mask_rows=state["mask_rows"])
        return decode.sample(state["logits"], state["noise"], temperature=state["temperature"],
                             top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    return {"matvec": _plain_matvec, "control": _plain_control, "sample": _plain_sample}[op](state)


def _plain_matvec(state):
    case, codes = state["case"], state["codes"]
    k, g = case["inputs"], case["group"]
    weight = torch.stack((codes & 15, codes >> 4), dim=2).view(codes.shape[0], -1)[:, :k].float()
    if state["zeros"] is None:
        weight = weight - 8.0
    else:
        weight = weight - state["zeros"].float().repeat_interleave(g, dim=1)[:, :k]
    weight = weight * state["scales"].float().repeat_interleave(g, dim=1)[:, :k]
    return (state["x"].float() @ weight.t() + state["bias"]).to(state["x"].dtype)


def _row_of(offsets, total):
    """The row that each of `total` list entries belongs to."""
    return torch.searchsorted(offsets, torch.arange(total, device=offsets.device), right=True) - 1


def _plain_control(state):
    logits = state["logits"]
    b, v = logits.shape
    z = logits.float()
    symbols, offsets = state["history"]
    inside = (symbols >= 0) & (symbols < v)
    place = _row_of(offsets, symbols.numel()) * v + torch.where(inside, symbols, torch.zeros_like(symbols))
    count = torch.zeros(b * v, device=z.device).index_add_(0, place, inside.float()).view(b, v)
    repetition, presence, frequency = (state[w][:, None] for w in ("repetition", "presence", "frequency"))
    seen = torch.where(z > 0, z / repetition, z * repetition) - (presence + frequency * count)
    z = torch.where(count > 0, seen, z)
    if state["bias"] is not None:
        ids, values, offsets = state["bias"]
        place = _row_of(offsets, ids.numel()) * v + ids
        last = torch.full((b * v,), -1, device=z.device, dtype=torch.int64)
        last = last.scatter_reduce(0, place, torch.arange(ids.numel(), device=z.device), "amax").view(b, v)
        if ids.numel():
            z = torch.where(last >= 0, z + values[last.clamp(min=0)], z)
    if state["masks"] is not None:
        at = torch.arange(v, device=z.device)
        rows = state["mask_rows"]
        words = state["masks"][rows.clamp(min=0).long()][:, at // 32]
        allowed = ((words >> (at % 32).int()) & 1).bool() | (rows < 0)[:, None]
        z = torch.where(allowed, z, torch.full_like(z, -math.inf))
    return z.to(logits.dtype)


def _plain_sample(state):
    z = state["logits"].float()
    b, v = z.shape
    greedy = (state["temperature"] == 0)[:, None]
    z = z / torch.where(greedy, torch.ones_like(state["temperature"])[:, None], state["temperature"][:, None])
    top = z.amax(dim=1, keepdim=True)
    ordered = z.sort(dim=1, descending=True).values
    mass = torch.where(ordered == top, torch.ones_like(z), (ordered - top).exp())
    mass = torch.where(torch.isneginf(ordered), torch.zeros_like(z), mass)
    upto = mass.cumsum(dim=1)
    whole = upto[:, -1:]
    # the number of strictly larger symbols, and their mass
    above = torch.searchsorted(-ordered, -ordered)
    before = torch.where(above > 0, upto.gather(1, (above - 1).clamp(min=0)), torch.zeros_like(z))
    stays = (above < state["top_k"][:, None]) & (before < state["top_p"][:, None] * whole)
    stays = stays & (mass >= state["min_p"][:, None])
    bar = torch.where(stays, ordered, torch.full_like(z, math.inf)).amin(dim=1, keepdim=True)
    race = torch.where(z >= bar, z + state["noise"], torch.full_like(z, -math.inf))
    race = torch.where(greedy, z, race)
    best = race.amax(dim=1, keepdim=True)
    at = torch.arange(v, device=z.device)
    symbol = torch.where(race == best, at, torch.full_like(at, v)).amin(dim=1, keepdim=True)
    empty = torch.isneginf(top)
    logprob = z.gather(1, symbol) - top - whole.log()
    symbol = torch.where(empty, torch.full_like(symbol, -1), symbol).to(torch.int32)
    logprob = torch.where(empty, torch.full_like(logprob, -math.inf), logprob)
    return symbol.view(b), logprob.view(b)


# --- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    b = case["rows"]
    e = BYTES[case["dtype"]]
    if case["op"] == "matvec":
        n, k = case["outputs"], case["inputs"]
        groups = n * -(-k // case["group"])
        weights = n * k / 2 + groups * (BYTES[case["scale"]] + (0.5 if case["zeros"] else 0))
        return {"bytes": weights + b * k * e + b * n * e + 4 * n, "flops": 2.0 * b * n * k}
    v = case["symbols"]
    if case["op"] == "control":
        lists = b * 0.7 * (4 * case["history"] + 8 * case["biases"])
        masks = min(b, 32) * v / 8 if case["masked"] else 0
        return {"bytes": 2.0 * b * v * e + lists + masks + 44 * b, "flops": 6.0 * b * v}
    return {"bytes": b * v * (e + 4.0) + 24 * b, "flops": 8.0 * b * v}


# --- the definition in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"matvec": _exact_matvec, "control": _exact_control, "sample": _exact_sample}[case["op"]](case, state)


def _exact_matvec(case, state):
    # y = b + sum over groups of s (sum x u - z sum x), a run of groups at a time
    n, k, g = case["outputs"], case["inputs"], case["group"]
    x = state["x"].double()
    y = state["bias"].double().expand(x.shape[0], n).clone()
    step = max(g, (1 << 24) // n // g * g)
    for begin in range(0, k, step):
        end = min(k, begin + step)
        width = -(-(end - begin) // g) * g
        part = torch.zeros(x.shape[0], width, device=DEVICE, dtype=torch.float64)
        part[:, :end - begin] = x[:, begin:end]
        u = torch.zeros(n, width, device=DEVICE, dtype=torch.float64)
        packed = state["codes"][:, begin // 2:(end + 1) // 2]
        u[:, 0:2 * packed.shape[1]:2] = (packed % 16).double()
        u[:, 1:2 * packed.shape[1]:2] = (packed // 16).double()
        scale = state["scales"][:, begin // g:-(-end // g)].double()
        zero = state["zeros"][:, begin // g:-(-end // g)].double() if case["zeros"] else 8.0
        w = ((u.view(n, -1, g) - (zero[:, :, None] if case["zeros"] else zero)) * scale[:, :, None]).view(n, width)
        y += part @ w.t()
    return y


def _exact_control(case, state):
    z = state["logits"].double().cpu().numpy().copy()
    b, v = z.shape
    symbols, offsets = (t.cpu().numpy() for t in state["history"])
    bias = [t.cpu().numpy() for t in state["bias"]] if state["bias"] is not None else None
    r, p, f = (state[w].double().cpu().numpy() for w in ("repetition", "presence", "frequency"))
    for i in range(b):
        mine = symbols[offsets[i]:offsets[i + 1]]
        ids, counts = np.unique(mine[(mine >= 0) & (mine < v)], return_counts=True)
        old = z[i, ids]
        z[i, ids] = np.where(old > 0, old / r[i], old * r[i]) - p[i] - f[i] * counts
        if bias is not None:
            last = dict(zip(bias[0][bias[2][i]:bias[2][i + 1]].tolist(), bias[1][bias[2][i]:bias[2][i + 1]].tolist()))
            z[i, list(last)] += np.array(list(last.values()), dtype=np.float64)
        if state["masks"] is not None and int(state["mask_rows"][i]) >= 0:
            words = state["masks"][int(state["mask_rows"][i])].cpu().numpy().view(np.uint8)
            allowed = np.unpackbits(words, bitorder="little", count=v).astype(bool)
            z[i, ~allowed] = -np.inf
    return z


def _exact_sample(case, state):
    # row by row: the prefix of the sorted row that stays, the race among it, and the winner's share of the whole row;
    # the symbol itself is a whole number and has no value here
    logits, noise = state["logits"].double(), state["noise"].double()
    t, k, p, floor = (state[w].double().tolist() for w in ("temperature", "top_k", "top_p", "min_p"))
    found = torch.full((case["rows"],), -math.inf, device=DEVICE, dtype=torch.float64)
    for i in range(case["rows"]):
        z = logits[i] / (t[i] or 1.0)
        if torch.isneginf(z).all():
            continue
        share = torch.softmax(z, dim=0)
        if t[i] == 0:
            found[i] = share.max().log()
            continue
        values, counts = torch.unique(share, return_counts=True)      # ascending
        values, counts = values.flip(0), counts.flip(0)
        larger = counts.cumsum(0) - counts
        mass = (values * counts).cumsum(0) - values * counts
        stays = (larger < k[i]) & (mass < p[i]) & (values >= floor[i] * values[0])
        bar = values[stays].min()
        winner = torch.where(share >= bar, z + noise[i], torch.full_like(z, -math.inf)).argmax()
        found[i] = share[winner].log()
    return None, found
