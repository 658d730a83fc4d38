"""The generator end to end: a trained model's active neurons through the 4-bit
readout, the control of its logits and the draw."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from leo_amd import native
from leo_amd.generate import END, Generator, main
from leo_amd.model import Model
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


def test_four_bit_readout_is_within_half_a_step_of_the_weights(require_gpu, trained):
    generator = Generator(trained, group=32)
    generator.prompt(b"once upon a time")
    got = generator.logits()[0].double().cpu().numpy()
    model = trained.model()
    ids, values = trained._read_active()
    assert ids.size > 0
    rows = model.out_weight.reshape(257, -1).astype(np.float64)
    want = model.bias.astype(np.float64) + rows[:, ids] @ values.astype(np.float64)
    # a group's step is its largest magnitude over 7, held in half precision; rounding moves a weight by half of it
    step = np.abs(np.pad(rows, ((0, 0), (0, -rows.shape[1] % 32))).reshape(257, -1, 32)).max(2) / 7
    bound = (step[:, ids // 32] * np.abs(values)).sum(1) * (0.5 + 2.0 ** -8) + 1e-4
    assert (np.abs(got - want) <= bound).all()


def test_device_readout_is_the_runtimes(require_gpu, trained):
    generator = Generator(trained, readout="device")
    generator.prompt(b"the cat")
    assert np.array_equal(generator.logits()[0].cpu().numpy(), trained.read_state("logits"))


@pytest.mark.parametrize("readout", ["q4", "device"])
def test_what_is_written_is_utf8_and_repeats_with_its_seed(require_gpu, trained, readout):
    texts = []
    for seed in (1, 1, 2):
        generator = Generator(trained, readout=readout, seed=seed)
        generator.prompt("café ".encode()[:-2])      # ends inside a character
        text, logprobs = generator.write(60, temperature=2.0, top_k=257, top_p=1.0, allow_end=False)
        assert len(text) == len(logprobs) == 60 and all(p <= 0 for p in logprobs)
        whole = "café ".encode()[:-2] + text
        whole.decode(errors="strict" if generator._state == 0 else "ignore")
        assert 0x80 <= text[0] <= 0xBF
        texts.append(text)
    assert texts[0] == texts[1] != texts[2]


def test_greedy_bytes_are_the_largest_allowed_logits(require_gpu, trained):
    generator = Generator(trained)
    generator.prompt(b"once")
    text, _ = generator.write(20, temperature=0.0, allow_end=False)
    again = Generator(trained)
    again.prompt(b"once")
    state = 0
    for byte in text:
        logits = again.logits()[0]
        allowed = torch.tensor(again._next[state] >= 0, device=logits.device)
        assert int(torch.where(allowed, logits[:256], float("-inf")).argmax()) == byte
        state = int(again._next[state, byte])
        trained.step(byte, None, native.FROZEN)


def test_penalties_biases_and_the_end(require_gpu, trained):
    generator = Generator(trained)
    generator.prompt(b"a")
    text, _ = generator.write(30, bias={ord("z"): 1e4})
    assert text == b"z" * 30
    generator.prompt(b"a")
    text, _ = generator.write(30, bias={ord("z"): 50.0, ord("y"): 49.0}, frequency=10.0, temperature=0.0, top_k=1)
    assert set(text[:2]) == set(b"zy")
    generator.prompt(b"a")
    assert generator.write(30, bias={END: 1e4}) == (b"", [])


def test_the_parameters_stay_as_they_are(require_gpu, trained):
    before = trained.model()
    generator = Generator(trained)
    generator.prompt(b"the ")
    generator.write(10)
    after = trained.model()
    assert np.array_equal(before.out_weight, after.out_weight) and np.array_equal(before.rec_weight, after.rec_weight)
    assert before.parameter_revision == after.parameter_revision


def test_refusals(require_gpu, trained):
    for call in (lambda: Generator(trained, readout="f32"), lambda: Generator(trained, group=17),
                 lambda: Generator(trained).prompt(b"\xff")):
        with pytest.raises(native.LeoError) as err:
            call()
        assert err.value.code == native.ERR_INVALID_ARGUMENT


def test_command(require_gpu, capsys):
    assert main(["--stories", "2", "--bytes", "24", "--prompt", "the "]) == 0
    out, err = capsys.readouterr()
    assert out.startswith("the ") and "bits a byte" in err
