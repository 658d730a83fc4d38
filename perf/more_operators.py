"""Performance cases of the operators that answer with several hypotheses at once:
products with 8-bit weights and 8-bit activations (a scale for each output and each
row), beam search's selection over beams and symbols, and the reordering of the
beams' states by their parents.

A case names its operator ("op") and sizes. `run` computes it with elementary
torch operations, or, where `own` is true, through leo_amd.decode.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i8": 1}
MOST_WEIGHTS = 257 << 20              # the largest readout here: 1,048,576 neurons
MOST_PRODUCTS = 2048 * 8192 * 8192
MOST_LOGITS = 256 * 131_075
MOST_STATE = 540 << 20                # bytes written by a reordering


def listed():
    return [
        # the readout of a 1,024-neuron model for one story: latency alone
        _product("8-bit readout 1k, one row", 1, 1024, 257, "f32", "f32", 0.02),
        # eight hypotheses of a 131,072-neuron model read out together
        _product("8-bit readout 131k, 8 rows", 8, 131_072, 257, "bf16", "f32", 0.05),
        # one story of a 1,048,576-neuron model: a long, flat weight matrix, sums past 32 bits
        _product("8-bit readout 1M, one row", 1, 1_048_576, 257, "f32", "f16", 0.02),
        # a full batch against odd sizes: rows that end inside a block and inside a tile
        _product("8-bit dense odd, 64 rows", 64, 5001, 11_007, "f16", "bf16", 1.0),
        # all rows of a long text at once: the products themselves are what counts
        _product("8-bit dense 8192, 2048 rows", 2048, 8192, 8192, "bf16", "f32", 1.0),
        # one story's next bytes: latency alone
        _beams("bytes, 4 beams", 1, 4, 4, 257, "f32", True, 0),
        # a small server's searches over a word-piece vocabulary, 16-bit logits with many ties
        _beams("32k symbols, 16 x 4 beams", 16, 4, 4, 32_001, "bf16", True, 0),
        # one search over a large vocabulary, keeping twice its beams: few long rows
        _beams("262k symbols, 8 beams to 16", 1, 8, 16, 262_147, "f32", False, 0),
        # a full batch of searches over a large vocabulary, rows of a padded buffer
        _beams("131k symbols, 32 x 8 beams", 32, 8, 8, 131_075, "f32", True, 61),
        # four hypotheses of a 1,024-neuron model, four arrays each: latency alone
        _states("4 small arrays, 4 beams", 1, 4, 4, 4, 1, 1, 1, 1024, "f32"),
        # eight hypotheses' neuron state over 1,048,576 neurons, eight planes
        _states("8 planes of 1M neurons, 8 beams", 1, 8, 8, 8, 1, 1, 1, 1_048_576, "f32"),
        # 8-bit caches with odd rows, two hypotheses of each three kept twice
        _states("odd 8-bit caches, 20 x 3 beams to 4", 20, 3, 4, 6, 5, 700, 1001, 99, "i8"),
    ]


def _product(name, rows, inputs, outputs, dtype, scale, activity):
    return {"name": name, "op": "product", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "scale": scale, "activity": activity}


def _beams(name, groups, beams, kept, symbols, dtype, ends, pad):
    return {"name": name, "op": "beams", "groups": groups, "beams": beams, "kept": kept, "symbols": symbols,
            "dtype": dtype, "ends": ends, "pad": pad}


def _states(name, groups, beams, kept, arrays, heads, length, capacity, width, dtype):
    return {"name": name, "op": "states", "groups": groups, "beams": beams, "kept": kept, "arrays": arrays,
            "heads": heads, "length": length, "capacity": capacity, "width": width, "dtype": dtype}


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))))


def draw(rng):
    op = rng.choice(["product", "beams", "states"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "product":
        outputs = 257 if rng.random() < 0.4 else _log_int(rng, 31, 16_384)
        rows = _log_int(rng, 1, 4096)
        most = min(MOST_WEIGHTS // outputs, MOST_PRODUCTS // (rows * outputs), (1 << 24) // rows)
        case = _product("", rows, _log_int(rng, min(200, most), most), outputs, dtype,
                        rng.choice(["f32", "f16", "bf16"]), rng.choice([0.02, 1.0]))
    else:
        groups, beams = _log_int(rng, 1, 32), _log_int(rng, 1, 16)
        kept = rng.choice([beams, beams, 2 * beams, _log_int(rng, 1, 32)])
        if op == "beams":
            symbols = 257 if rng.random() < 0.25 else _log_int(rng, 200, min(262_147, MOST_LOGITS // (groups * beams)))
            case = _beams("", groups, beams, kept, symbols, dtype, rng.random() < 0.6, rng.choice([0, 0, 7, 64]))
        else:
            arrays, heads = _log_int(rng, 1, 16), rng.choice([1, 1, 4, 7])
            dtype = rng.choice(["f32", "bf16", "i32", "i8"])
            width = _log_int(rng, 1, 256) if heads > 1 else _log_int(rng, 1, 65_536)
            row = MOST_STATE // (max(beams, kept) * groups * arrays * heads * width * BYTES[dtype])
            length = _log_int(rng, 1, max(1, min(row, 2048)))
            case = _states("", groups, beams, kept, arrays, heads, length, length + rng.choice([0, 1, length // 2]),
                           width, dtype)
    del case["name"]
    return case


# --- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    state = {"case": case}
    {"product": _prepare_product, "beams": _prepare_beams, "states": _prepare_states}[case["op"]](case, gen, state)
    return state


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _uniform(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEVICE)


def _integers(gen, low, high, *shape, dtype=torch.int64):
    return torch.randint(low, high, shape, generator=gen, device=DEVICE, dtype=dtype)


def _prepare_product(case, gen, state):
    m, k, n = case["rows"], case["inputs"], case["outputs"]
    # normal weights, the largest of a row at 127
    state["codes"] = (_normal(gen, n, k) * 30.0).round_().clamp_(-127, 127).to(torch.int8)
    state["scales"] = (0.0005 + 0.002 * _uniform(gen, n)).to(TYPES[case["scale"]])
    x = _normal(gen, m, k)
    if case["activity"] < 1:      # Leo's activations: few, and none below zero
        x = torch.where(_uniform(gen, m, k) < case["activity"], x.abs(), torch.zeros_like(x))
    state["x"] = x.to(TYPES[case["dtype"]])
    state["bias"] = _normal(gen, n) * 0.5
    if own:
        from leo_amd import decode

        # a serving program lays its weights out once
        state["weight"] = decode.Q8Weight(state["codes"], state["scales"])


def _prepare_beams(case, gen, state):
    g, b, v = case["groups"], case["beams"], case["symbols"]
    logits = _normal(gen, g * b, v) * 2.5
    # what a grammar has taken out
    logits = torch.where(_uniform(gen, g * b, v) < 0.1, torch.full_like(logits, -math.inf), logits)
    buffer = torch.full((g * b, v + case["pad"]), 7.0, device=DEVICE, dtype=TYPES[case["dtype"]])
    buffer[:, :v] = logits.to(buffer.dtype)
    state["logits"] = buffer[:, :v]
    # sums of log probabilities that lie close together
    scores = -20.0 - 4.0 * _uniform(gen, g, b)
    scores[3::8, 1:] = -math.inf      # searches that have just begun
    state["scores"] = scores
    state["finished"] = state["lengths"] = state["end"] = None
    state["penalty"] = 0.0
    if case["ends"]:
        state["finished"] = _uniform(gen, g, b) < 0.2
        state["finished"][:, 0] = False
        state["lengths"] = _integers(gen, 1, 200, g, b, dtype=torch.int32)
        state["end"] = v - 1
        state["penalty"] = 0.6
        if g > 4:
            scores[g // 2] = -math.inf      # a search that its grammar left without a way


def _prepare_states(case, gen, state):
    rows = case["groups"] * case["beams"]
    shape = (rows, case["heads"], case["capacity"], case["width"])
    if case["dtype"] in ("i32", "i8"):
        whole = [_integers(gen, -128, 128, *shape, dtype=TYPES[case["dtype"]]) for _ in range(case["arrays"])]
    else:
        whole = [_normal(gen, *shape).to(TYPES[case["dtype"]]) for _ in range(case["arrays"])]
    state["states"] = [t[:, :, :case["length"]] for t in whole]      # what has been filled so far
    state["parents"] = _integers(gen, 0, case["beams"], case["groups"], case["kept"], dtype=torch.int32)


# --- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        from leo_amd import decode

        if op == "product":
            return decode.q8_matmul(state["x"], state["weight"], state["bias"])
        if op == "beams":
            found = decode.beam_select(state["logits"], state["scores"], state["case"]["kept"], finished=state["finished"],
                                       lengths=state["lengths"], length_penalty=state["penalty"], end=state["end"])
            return [t for t in found if t is not None]
        return decode.reorder_states(state["states"], state["parents"])
    return {"product": _plain_product, "beams": _plain_beams, "states": _plain_states}[op](state)


def _plain_product(state):
    x = state["x"].float()
    scale = (x.abs().amax(dim=1, keepdim=True) / 127.0).clamp_min(2.0 ** -126)
    # 64 bits: quotients next to a half
    codes = (x.double() / scale.double()).round().float()
    sums = codes @ state["codes"].float().t()
    return (sums * scale * state["scales"].float() + state["bias"]).to(state["x"].dtype)


def _plain_beams(state):
    # 64 bits throughout: the order of candidates next to each other
    case = state["case"]
    g, b, v, k = case["groups"], case["beams"], case["symbols"], case["kept"]
    z = state["logits"].double()
    top = z.amax(dim=1, keepdim=True)
    top = torch.where(torch.isneginf(top), torch.zeros_like(top), top)
    score = state["scores"].double().view(g * b, 1) + (z - top - (z - top).exp().sum(dim=1, keepdim=True).log())
    score = torch.where(torch.isneginf(z), z, score)
    rank = score
    if case["ends"]:
        done = state["finished"].view(g * b, 1)
        still = torch.full_like(score, -math.inf)
        still[:, 0] = state["scores"].double().view(g * b)
        score = torch.where(done, still, score)
        length = state["lengths"].view(g * b, 1) + (~done).int()
        rank = score / length.double() ** state["penalty"]
    rank, at = rank.view(g, b * v).sort(dim=1, descending=True, stable=True)
    rank, at = rank[:, :k], at[:, :k]
    kept = score.view(g, b * v).gather(1, at)
    empty = torch.isneginf(kept)
    parents = torch.where(empty, torch.zeros_like(at), at // v)
    symbols = torch.where(empty, torch.full_like(at, -1), at % v)
    found = [kept.float()]
    if case["ends"]:
        was = state["finished"].gather(1, parents) & ~empty
        symbols = torch.where(was, torch.full_like(at, -1), symbols)
        length = state["lengths"].gather(1, parents) + (~was & ~empty).int()
        found += [was | (symbols == state["end"]), length]
    return [symbols.int(), parents.int()] + found


def _plain_states(state):
    parents = state["parents"].long()
    first = torch.arange(parents.shape[0], device=parents.device) * state["case"]["beams"]
    rows = (parents + first[:, None]).view(-1)
    return [t.index_select(0, rows) for t in state["states"]]


# --- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "product":
        m, k, n, e = case["rows"], case["inputs"], case["outputs"], BYTES[case["dtype"]]
        return {"bytes": n * k + n * (BYTES[case["scale"]] + 4.0) + (m * k + m * n) * e, "flops": 2.0 * m * n * k}
    g, b, k = case["groups"], case["beams"], case["kept"]
    if case["op"] == "beams":
        v = case["symbols"]
        live = 1 - 0.2 * (b - 1) / b if case["ends"] else 1.0      # finished beams' logits need no reading
        return {"bytes": live * g * b * v * BYTES[case["dtype"]] + 9.0 * g * b + 17.0 * g * k, "flops": 4.0 * live * g * b * v}
    row = case["arrays"] * case["heads"] * case["length"] * case["width"] * BYTES[case["dtype"]]
    read = b * (1 - (1 - 1 / b) ** k)      # rows that are a parent at all
    return {"bytes": float(g * (read + k) * row + 4 * g * k), "flops": 0.0}


# --- the definition in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "states":
        return None      # copies
    return {"product": _exact_product, "beams": _exact_beams}[case["op"]](case, state)


def _exact_product(case, state):
    # whole sums of codes, a run of inputs at a time
    n, k = case["outputs"], case["inputs"]
    x = state["x"].double()
    largest = x.abs().max(dim=1).values
    unit = torch.clamp((largest.float() / 127).double(), min=2.0 ** -126)
    y = torch.zeros(x.shape[0], n, device=DEVICE, dtype=torch.float64)
    step = max(64, (1 << 26) // n)
    for begin in range(0, k, step):
        part = torch.round(x[:, begin:begin + step] / unit[:, None])
        y += part @ state["codes"][:, begin:begin + step].double().t()
    return y * unit[:, None] * state["scales"].double() + state["bias"].double()


def _exact_beams(case, state):
    # group by group: each beam's best symbols, then the best among those
    g, b, k = case["groups"], case["beams"], case["kept"]
    scores, logits = state["scores"].double(), state["logits"]
    kept = torch.full((g, k), -math.inf, device=DEVICE, dtype=torch.float64)
    for i in range(g):
        found, ranks = [], []
        for j in range(b):
            s = scores[i, j]
            if torch.isneginf(s):
                continue
            if case["ends"] and bool(state["finished"][i, j]):
                mine, length = s.view(1), int(state["lengths"][i, j])
            else:
                z = logits[i * b + j].double()
                mine = torch.log_softmax(z, dim=0).topk(min(k, z.numel())).values + s
                length = int(state["lengths"][i, j]) + 1 if case["ends"] else 1
            found.append(mine)
            ranks.append(mine / float(length) ** state["penalty"])
        if found:
            found, ranks = torch.cat(found), torch.cat(ranks)
            best = ranks.argsort(descending=True, stable=True)[:k]
            kept[i, :best.numel()] = found[best]
    return [None, None, kept] + ([None, None] if case["ends"] else [])
