"""Text from a trained model: a prompt, then one drawn byte after the other.

    python -m leo_amd.generate --checkpoint model.psc --prompt "once upon" --bytes 200

Each byte is one frozen step of the runtime and three operators of
`leo_amd.decode` on its active neurons: the readout with 4-bit weights, the
control of its 257 logits (penalties for repeated bytes, biases, and the bytes
that UTF-8 allows next) and the draw. The loop is that of the reference's
generation (crates/leo-cli/src/main.rs:834-1009), with its UTF-8 state
(crates/leo-core/src/utf8.rs:4-87) as a grammar mask.

The 4-bit readout answers from the neurons alone, without the context's share. Its
weights are an eighth of the output weights' size, beside those, which the runtime
keeps. readout="device" takes the runtime's own logits, which every step leaves and
which are quicker to have: 58 us a byte against 180 at 1,024 neurons, 60 against 132
at 1,048,576, where the product of all weights alone takes 39 us and the active
neurons come by way of the host.
"""
from __future__ import annotations

import argparse
import sys
from typing import Dict, List, Optional, Sequence, Tuple

from . import decode  # torch before the first call into libleo_hip.so

import numpy as np
import torch

from . import native
from .model import BEGIN_DOCUMENT, OUTPUT_CLASSES, Model
from .runtime import HipRuntime

END = 256      # the output class that ends a document

# States of UTF-8: the bytes that may come next, and where they lead. Overlong
# forms, surrogates and code points beyond 10FFFF have no way through.
_LEADS = [(0x00, 0x7F, 0), (0xC2, 0xDF, 1), (0xE0, 0xE0, 4), (0xE1, 0xEC, 2), (0xED, 0xED, 5), (0xEE, 0xEF, 2),
          (0xF0, 0xF0, 6), (0xF1, 0xF3, 3), (0xF4, 0xF4, 7)]
_STATES = [_LEADS, [(0x80, 0xBF, 0)], [(0x80, 0xBF, 1)], [(0x80, 0xBF, 2)], [(0xA0, 0xBF, 1)], [(0x80, 0x9F, 1)],
           [(0x90, 0xBF, 2)], [(0x80, 0x8F, 2)]]


def utf8_table() -> np.ndarray:
    """next[state, byte]: the state after a byte, -1 where UTF-8 does not allow it."""
    table = np.full((len(_STATES), 256), -1, dtype=np.int64)
    for state, ranges in enumerate(_STATES):
        for low, high, to in ranges:
            table[state, low:high + 1] = to
    return table


def utf8_masks() -> np.ndarray:
    """The masks of `decode.control_logits`, one a state; a document may end in state 0 only."""
    allowed = np.zeros((len(_STATES), 288), dtype=bool)
    allowed[:, :256] = utf8_table() >= 0
    allowed[0, END] = True
    return np.packbits(allowed, axis=1, bitorder="little").view(np.int32)


class Generator:
    """Writes with a runtime's current model. The runtime's document state is this
    object's while it writes; its parameters stay as they are (frozen steps)."""

    def __init__(self, runtime: HipRuntime, *, group: int = 32, readout: str = "q4", seed: int = 0):
        if readout not in ("q4", "device"):
            raise native.LeoError(native.ERR_INVALID_ARGUMENT, f"readout must be q4 or device, not {readout}")
        self.runtime = runtime
        self.device = torch.device("cuda", runtime.device)
        self.neurons = runtime.config.model.neuron_count
        self.readout = readout
        self.group = group
        self.weight: Optional[decode.Q4Weight] = None
        self.bias: Optional[torch.Tensor] = None
        self._version = -1      # of the parameters that weight and bias were made from
        if readout == "q4":
            self._take_weights()
        self._active = torch.zeros(1, self.neurons, device=self.device)
        self._noise = torch.Generator(self.device).manual_seed(seed)
        self._next = utf8_table()
        self._masks = torch.from_numpy(utf8_masks()).to(self.device)
        self._state = 0
        self._written: List[int] = []
        self._document: Optional[int] = None      # the runtime's count while the prompt's document is open

    def _take_weights(self) -> None:
        version = self.runtime.parameter_version
        if version != self._version:
            rows, bias = self.runtime._read_readout()
            self.weight = decode.Q4Weight.quantize(torch.from_numpy(rows).to(self.device), self.group)
            self.bias = torch.from_numpy(bias).to(self.device)
            self._version = version

    def logits(self) -> torch.Tensor:
        """[1, 257]: the readout of the last step, with the model's weights as they are now."""
        if self.readout == "device":
            return torch.from_numpy(self.runtime.read_state("logits")).to(self.device)[None]
        self._take_weights()
        ids, values = self.runtime._read_active()
        self._active.zero_()
        self._active[0, torch.from_numpy(ids).to(self.device)] = torch.from_numpy(values).to(self.device)
        return decode.q4_matvec(self._active, self.weight, self.bias)

    def prompt(self, text: bytes) -> None:
        """Begins a document and reads `text`, which has to be UTF-8 as far as it goes."""
        state = 0
        for i, byte in enumerate(text):
            state = int(self._next[state, byte])
            if state < 0:
                raise native.LeoError(native.ERR_INVALID_ARGUMENT, f"byte {i} of the prompt is not UTF-8")
        self.runtime.begin_document()
        symbols = [BEGIN_DOCUMENT, *text]
        self.runtime.advance_frozen_batch([(s, None) for s in symbols[:-1]])
        self.runtime.step(symbols[-1], None, native.FROZEN)
        self._state = state
        self._written = list(text)
        self._document = self.runtime.documents

    def write(self, count: int, *, temperature: float = 0.8, top_k: int = 40, top_p: float = 0.95, min_p: float = 0.0,
              repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0, history: int = 64,
              bias: Optional[Dict[int, float]] = None, allow_end: bool = True) -> Tuple[bytes, List[float]]:
        """Up to `count` bytes after the prompt, and their logprobs; fewer where the
        model ends the document. Needs the document that `prompt` began, ended neither
        by the model nor by another use of the runtime. The penalties look at the last
        `history` bytes, the prompt's among them; `bias` adds to single bytes' logits
        (256: the end). A top_k below 1 keeps the largest alone, as 1 does."""
        if self._document != self.runtime.documents:
            raise native.LeoError(native.ERR_INVALID_ARGUMENT, "no document is open: begin one with prompt()")

        def one(value, dtype=torch.float32):
            return torch.tensor([value], dtype=dtype, device=self.device)

        per_row = {"temperature": one(temperature), "top_k": one(top_k, torch.int32), "top_p": one(top_p),
                   "min_p": one(min_p)}
        penalties = {"repetition": one(repetition), "presence": one(presence), "frequency": one(frequency)}
        biases = dict(bias or {})
        if not allow_end:
            biases[END] = float("-inf")
        listed = (torch.tensor(list(biases), dtype=torch.int32, device=self.device),
                  torch.tensor(list(biases.values()), dtype=torch.float32, device=self.device),
                  torch.tensor([0, len(biases)], device=self.device)) if biases else None
        written, logprobs = [], []
        for _ in range(count):
            recent = self._written[max(0, len(self._written) - history):]
            logits = decode.control_logits(
                self.logits(), history=(torch.tensor(recent, dtype=torch.int32, device=self.device),
                                        torch.tensor([0, len(recent)], device=self.device)),
                bias=listed, masks=self._masks, mask_rows=one(self._state, torch.int32), **penalties)
            noise = -torch.log(torch.empty(1, OUTPUT_CLASSES, device=self.device)
                               .exponential_(generator=self._noise).clamp_min(1e-30))
            drawn, logprob = decode.sample(logits, noise, **per_row)
            symbol = int(drawn)
            if symbol < 0:
                raise native.LeoError(native.ERR_NUMERICAL, "no byte is left to draw")
            if symbol == END:
                self.runtime.finish_document()
                break
            written.append(symbol)
            logprobs.append(float(logprob))
            self._written.append(symbol)
            self._state = int(self._next[self._state, symbol])
            self.runtime.step(symbol, None, native.FROZEN)
        return bytes(written), logprobs


def _trained(neurons: int, stories: int) -> HipRuntime:
    """A small model that has seen some synthetic stories."""
    from .workload import WORKLOADS, story_list, synthetic_stories, workload_config

    w = WORKLOADS["A"]
    config = workload_config(w)
    config.model.neuron_count, config.model.block_count = neurons, neurons // config.model.neurons_per_block
    config.model.max_active_global = config.model.block_count * config.model.max_active_per_block
    runtime = HipRuntime(Model.synthetic(config, topology=w.topology, weight_sigma=0.05), max_lanes=1)
    for story in story_list(*synthetic_stories(w, stories)):
        runtime.train_batch([story], native.TRAINING, replay=False)
    return runtime


def main(argv: Optional[Sequence[str]] = None) -> int:
    parser = argparse.ArgumentParser(prog="python -m leo_amd.generate", description="Writes text with a trained model.")
    parser.add_argument("--checkpoint", help="a PSCLS100 checkpoint; without one a small model is trained first")
    parser.add_argument("--neurons", type=int, default=1024, help="of the small model")
    parser.add_argument("--stories", type=int, default=16, help="synthetic stories it is trained on")
    parser.add_argument("--prompt", default="the ")
    parser.add_argument("--bytes", type=int, default=160)
    parser.add_argument("--readout", choices=("q4", "device"), default="q4")
    parser.add_argument("--group", type=int, default=32, choices=(32, 64, 128))
    parser.add_argument("--seed", type=int, default=0)
    for name, default in (("temperature", 0.8), ("top-p", 0.95), ("min-p", 0.0), ("repetition", 1.1), ("presence", 0.0),
                          ("frequency", 0.0)):
        parser.add_argument("--" + name, type=float, default=default)
    parser.add_argument("--top-k", type=int, default=40, help="bytes to draw from; below 2 the likeliest alone, 257 for all")
    parser.add_argument("--history", type=int, default=64)
    args = parser.parse_args(argv)
    if args.checkpoint:
        from .formats import load_model

        runtime = HipRuntime(load_model(args.checkpoint), max_lanes=1)
    else:
        runtime = _trained(args.neurons, args.stories)
    with runtime:
        generator = Generator(runtime, group=args.group, readout=args.readout, seed=args.seed)
        generator.prompt(args.prompt.encode())
        text, logprobs = generator.write(
            args.bytes, temperature=args.temperature, top_k=args.top_k, top_p=args.top_p, min_p=args.min_p,
            repetition=args.repetition, presence=args.presence, frequency=args.frequency, history=args.history)
    print(args.prompt + text.decode(errors="replace"))
    if logprobs:
        print(f"{len(logprobs)} bytes, {-sum(logprobs) / len(logprobs) / np.log(2):.3f} bits a byte under its own "
              "distribution", file=sys.stderr)
    return 0


if __name__ == "__main__":
    sys.exit(main())
