"""What a generator keeps and what it must not: a mirror's marks, the model's weights
after training, documents that have ended, whole UTF-8."""
from __future__ import annotations

import codecs

import pytest
import torch

from leo_amd import native
from leo_amd.generate import END, Generator
from leo_amd.model import Model
from leo_amd.runtime import HipRuntime
from tests.helpers import assert_models_equal, small_redundant_config, story

pytestmark = pytest.mark.gpu


@pytest.fixture
def runtime():
    with HipRuntime(Model.synthetic(small_redundant_config(), weight_sigma=0.05), max_lanes=2) as r:
        r.train_batch([story(0, 200)], native.TRAINING, replay=False)
        yield r


@pytest.mark.parametrize("tracked", [False, True])
def test_a_mirror_still_gets_its_changes(require_gpu, runtime, tracked):
    mirror = runtime.model()
    if tracked:
        runtime.enable_parameter_tracking()
    runtime.train_batch([story(1, 200), story(2, 200)], native.TRAINING, replay=True)
    if tracked:
        runtime.enable_parameter_tracking()
    Generator(runtime)
    runtime.synchronize_model(mirror)
    assert_models_equal(mirror, runtime.model())


def no_document(call):
    with pytest.raises(native.LeoError) as err:
        call()
    assert err.value.code == native.ERR_INVALID_ARGUMENT and "document" in str(err.value)


def learn_by_batch(r):
    r.train_batch([story(1, 300)], native.TRAINING, replay=False)


def learn_by_lanes(r):
    r.train_batch([story(1, 300), story(2, 300)], native.TRAINING, replay=True)


def learn_by_steps(r):
    r.begin_document()
    for a, b in zip(b"once upon a tim", b"nce upon a time"):
        r.step(a, b, native.TRAINING)


def take_another_model(r):
    r.set_model(Model.synthetic(r.config, weight_sigma=0.2))


@pytest.mark.parametrize("change", [learn_by_batch, learn_by_lanes, learn_by_steps, take_another_model])
def test_answers_come_from_the_current_model(require_gpu, runtime, change):
    generator = Generator(runtime)
    generator.prompt(b"once upon ")
    generator.write(5, temperature=0.0, allow_end=False)
    change(runtime)
    answers = []
    for g in (generator, Generator(runtime)):
        g.prompt(b"once upon ")
        logits = g.logits().clone()
        answers.append((logits, *g.write(20, temperature=0.0, allow_end=False)))
    assert torch.equal(answers[0][0], answers[1][0])
    assert answers[0][1:] == answers[1][1:]


def test_weights_are_kept_while_the_model_stays(require_gpu, runtime):
    generator = Generator(runtime)
    kept = generator.weight
    generator.prompt(b"once upon ")
    generator.write(5)
    runtime.evaluate([story(3, 50)])
    generator.prompt(b"the ")
    generator.write(5)
    assert generator.weight is kept


@pytest.mark.parametrize("readout", ["q4", "device"])
def test_writing_needs_an_open_document(require_gpu, runtime, readout):
    generator = Generator(runtime, readout=readout)
    no_document(lambda: generator.write(3))
    generator.prompt(b"a")
    assert generator.write(5, bias={END: 1e4}) == (b"", [])
    no_document(lambda: generator.write(5))
    generator.prompt(b"a")
    assert len(generator.write(5, allow_end=False)[0]) == 5
    assert len(generator.write(5, allow_end=False)[0]) == 5      # it is still open
    for ends in (runtime.finish_document, runtime.begin_document, runtime.reset_transient_state, lambda: learn_by_batch(runtime),
                 lambda: runtime.evaluate([story(3, 50)]), lambda: Generator(runtime).prompt(b"b")):
        generator.prompt(b"a")
        ends()
        no_document(lambda: generator.write(5))


@pytest.mark.parametrize("readout", ["q4", "device"])
def test_every_prefix_is_utf8(require_gpu, runtime, readout):
    for seed in range(6):
        generator = Generator(runtime, readout=readout, seed=seed)
        start = "café ".encode()[:-2]                            # ends inside a character
        generator.prompt(start)
        text, _ = generator.write(60, temperature=2.0, top_k=257, top_p=1.0, allow_end=False)
        decoder = codecs.getincrementaldecoder("utf-8")("strict")
        decoder.decode(start + text, final=False)                # raises at the first byte that cannot stand there
        assert (generator._state == 0) == (decoder.getstate()[0] == b"")
