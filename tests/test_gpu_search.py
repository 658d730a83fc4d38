"""The generator's search end to end: the readout of all hypotheses, the control of their
logits, the selection and the reordering of what they carry, against a search on the host
over the same logits; and the 8-bit readout."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leo_amd import decode, native
from leo_amd.generate import END, Generator, main
from leo_amd.model import BEGIN_DOCUMENT, Model
from leo_amd.runtime import HipRuntime
from tests.helpers import small_redundant_config, story

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def trained():
    runtime = HipRuntime(Model.synthetic(small_redundant_config(), weight_sigma=0.05), max_lanes=1)
    for i in range(4):
        runtime.train_batch([story(i, 300)], native.TRAINING, replay=False)
    yield runtime
    runtime.close()


def logits_after(generator, text):
    r = generator.runtime
    r.begin_document()
    r.advance_frozen_batch([(s, None) for s in [BEGIN_DOCUMENT, *text][:-1]])
    r.step([BEGIN_DOCUMENT, *text][-1], None, native.FROZEN)
    return generator.logits()[0].double().cpu().numpy()


def search_on_the_host(generator, prompt, count, beams, penalty=0.0, repetition=1.0, presence=0.0, frequency=0.0,
                       history=64, allow_end=True):
    """[(bytes, score)], in 64 bits from the generator's logits of one hypothesis at a time."""
    kept = [(0.0, b"", 0, 0, False)]      # score, bytes, state of UTF-8, length, finished
    for byte in prompt:
        kept = [(0.0, b"", int(generator._next[kept[0][2], byte]), 0, False)]
    for _ in range(count):
        found = []
        for place, (score, text, state, length, done) in enumerate(kept):
            if done:
                found.append((-score / max(length, 1) ** penalty, place, 0, (score, text, state, length, True)))
                continue
            z = logits_after(generator, prompt + text)
            recent = list((prompt + text)[max(0, len(prompt + text) - history):])
            for v in set(recent):
                z[v] = z[v] / repetition if z[v] > 0 else z[v] * repetition
                z[v] -= presence + frequency * recent.count(v)
            z[:256][generator._next[state] < 0] = -np.inf
            if state != 0 or not allow_end:
                z[END] = -np.inf
            logp = z - z.max() - math.log(np.exp(z - z.max()).sum())
            for order, v in enumerate(np.argsort(-z, kind="stable")[:beams]):
                if z[v] > -np.inf:
                    s = score + logp[v]
                    more = (s, text, state, length + 1, True) if v == END else \
                        (s, text + bytes([v]), int(generator._next[state, v]), length + 1, False)
                    found.append((-s / (length + 1) ** penalty, place, order, more))
        found.sort(key=lambda f: f[:3])
        kept = [f[3] for f in found[:beams]]
        if all(k[4] for k in kept):
            break
    return [(text, score) for score, text, *_ in kept]


@pytest.mark.parametrize("readout", ["device", "q4", "q8"])
@pytest.mark.parametrize("beams, options", [
    (1, {}), (4, {}), (5, dict(penalty=0.7)), (3, dict(repetition=1.3, presence=0.2, frequency=0.1, history=5)),
    (4, dict(allow_end=False, history=0)),
])
def test_search_finds_what_the_host_finds(require_gpu, trained, readout, beams, options):
    generator = Generator(trained, readout=readout)
    prompt = "once upon café ".encode()[:-2]      # ends inside a character
    want = search_on_the_host(generator, prompt, 12, beams, **options)
    generator.prompt(prompt)
    renamed = {"length_penalty" if k == "penalty" else k: v for k, v in options.items()}
    got = generator.search(12, beams=beams, **renamed)
    assert [t for t, _ in got] == [t for t, _ in want]
    # 12 sums of float32 logits' log probabilities, each rounded: 2^-24 of a logit or a score, 2^-21 of the selection's sum
    assert max(abs(a - b) for (_, a), (_, b) in zip(got, want)) < 12 * (2.0 ** -21 + 2.0 ** -23 * 64)


def test_more_beams_find_no_worse(require_gpu, trained):
    generator = Generator(trained, readout="q8")
    best = []
    for beams in (1, 8):
        generator.prompt(b"the ")
        found = generator.search(10, beams=beams, allow_end=False)
        assert len(found) == beams and len(set(t for t, _ in found)) == beams
        assert all(len(t) == 10 for t, _ in found)
        assert [s for _, s in found] == sorted((s for _, s in found), reverse=True)
        best.append(found[0][1])
    assert best[1] >= best[0] - 1e-5


def test_one_beam_is_the_greedy_text(require_gpu, trained):
    for readout in ("q4", "q8", "device"):
        generator = Generator(trained, readout=readout)
        generator.prompt(b"once")
        text, logprobs = generator.write(15, temperature=0.0, allow_end=False, repetition=1.2)
        generator.prompt(b"once")
        (again, score), = generator.search(15, beams=1, allow_end=False, repetition=1.2)
        assert again == text and abs(score - sum(logprobs)) < 1e-4


def test_the_end_and_biases(require_gpu, trained):
    generator = Generator(trained, readout="q8")
    generator.prompt(b"a")
    found = generator.search(30, beams=3, bias={END: 1e4})
    assert found[0][0] == b"" and found[0][1] == pytest.approx(0.0, abs=1e-6)
    generator.prompt(b"a")
    found = generator.search(5, beams=2, bias={ord("z"): 1e4})
    assert found[0][0] == b"zzzzz"
    generator.prompt(b"a")
    assert generator.search(0) == [(b"", 0.0)]


def test_the_prompts_document_has_ended(require_gpu, trained):
    generator = Generator(trained)
    generator.prompt(b"the ")
    generator.search(2, beams=2)
    for call in (lambda: generator.search(2), lambda: generator.write(2)):
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT and "document" in str(err.value)
    generator.prompt(b"the ")
    for beams in (0, 65, -1):
        with pytest.raises(native.LeoError):
            generator.search(2, beams=beams)


def test_the_parameters_stay_as_they_are(require_gpu, trained):
    before = trained.model()
    generator = Generator(trained, readout="q8")
    generator.prompt(b"the ")
    generator.search(5, beams=3)
    after = trained.model()
    assert np.array_equal(before.out_weight, after.out_weight) and np.array_equal(before.rec_weight, after.rec_weight)
    assert before.parameter_revision == after.parameter_revision


def test_eight_bit_readout_is_within_half_a_step_of_the_weights(require_gpu, trained):
    generator = Generator(trained, readout="q8")
    generator.prompt(b"once upon a time")
    got = generator.logits()[0].double().cpu().numpy()
    model = trained.model()
    ids, values = trained._read_active()
    assert ids.size > 0
    rows = model.out_weight.reshape(257, -1).astype(np.float64)[:, ids]
    values = values.astype(np.float64)
    want = model.bias.astype(np.float64) + rows @ values
    # a weight is off by half of its row's step, an activation by half of the largest over 127, and their roundings
    step = np.abs(model.out_weight.reshape(257, -1)).max(1) / 127 * 0.5001
    off = np.abs(values).max() / 127 * 0.5001
    bound = (step[:, None] * (np.abs(values) + off)).sum(1) + np.abs(rows).sum(1) * off + 1e-5
    assert (np.abs(got - want) <= bound).all()


def test_a_readout_follows_the_model(require_gpu):
    with HipRuntime(Model.synthetic(small_redundant_config(), weight_sigma=0.05), max_lanes=1) as runtime:
        generator = Generator(runtime, readout="q8")
        generator.prompt(b"once")
        before = generator.logits().clone()
        runtime.train_batch([story(1, 300)], native.TRAINING, replay=False)
        generator.prompt(b"once")
        fresh = Generator(runtime, readout="q8")
        assert torch.equal(generator.logits(), fresh.logits()) and not torch.equal(generator.logits(), before)


def test_operators_together_on_several_searches(require_gpu):
    """A readout, the control, the selection and the states of six searches at once, step by step,
    captured into a graph and replayed, against the same calls made one search at a time."""
    gen = torch.Generator("cuda").manual_seed(2)
    groups, beams, neurons, symbols = 6, 4, 700, 257
    weight = decode.Q8Weight.quantize(torch.randn(symbols, neurons, generator=gen, device="cuda") * 0.1)
    active = torch.randn(groups * beams, neurons, generator=gen, device="cuda").relu()
    state = torch.randn(groups * beams, neurons, generator=gen, device="cuda")
    scores = torch.randn(groups, beams, generator=gen, device="cuda") - 5
    masks = torch.randint(-2 ** 31, 2 ** 31, (3, 9), generator=gen, device="cuda").to(torch.int32)
    rows = torch.randint(-1, 3, (groups * beams,), generator=gen, device="cuda", dtype=torch.int32)
    lengths = torch.ones(groups, beams, device="cuda", dtype=torch.int32)
    finished = torch.zeros(groups, beams, device="cuda", dtype=torch.bool)

    def step(part):
        some = slice(part.start * beams, part.stop * beams)
        logits = decode.control_logits(decode.q8_matmul(active[some], weight), masks=masks, mask_rows=rows[some].contiguous())
        found = decode.beam_select(logits, scores[part], finished=finished[part], lengths=lengths[part], length_penalty=0.6,
                                   end=256)
        return found, decode.reorder_states([active[some], state[some]], found.parents)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(slice(0, groups))
        with torch.cuda.graph(graph, stream=side):
            held, carried = step(slice(0, groups))
    torch.cuda.synchronize()
    for _ in range(4):
        single = [step(slice(g, g + 1)) for g in range(groups)]
        graph.replay()
        torch.cuda.synchronize()
        for i in range(5):
            assert torch.equal(held[i], torch.cat([f[i] for f, _ in single]))
        for i in range(2):
            assert torch.equal(carried[i], torch.cat([s[i] for _, s in single]))
        active.copy_(carried[0] + 0.1 * carried[1].abs())
        state.copy_(carried[1].flip(1))
        scores.copy_(held.scores)
        finished.copy_(held.finished)
        lengths.copy_(held.lengths)


def test_command(require_gpu, capsys):
    assert main(["--stories", "2", "--bytes", "12", "--prompt", "the ", "--beams", "3", "--readout", "q8",
                 "--length-penalty", "0.5"]) == 0
    out, err = capsys.readouterr()
    assert out.startswith("the ") and "bits a byte" in err
