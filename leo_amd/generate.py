"""Text from a trained model: a prompt, then one drawn byte after the other.

    python -m leo_amd.generate --checkpoint model.psc --prompt "once upon" --bytes 200

Each byte is one frozen step of the runtime and three operators of
`leo_amd.decode` on its active neurons: the readout with 4-bit weights (or 8-bit
ones), the control of its 257 logits (penalties for repeated bytes, biases, and the
bytes that UTF-8 allows next) and the draw. With `--beams` a search over several
hypotheses takes the draw's place. The loop is that of the reference's
generation (crates/leo-cli/src/main.rs:834-1009), with its UTF-8 state
(crates/leo-core/src/utf8.rs:4-87) as a grammar mask.

The 4-bit readout answers from the neurons alone, without the context's share. Its
weights are an eighth of the output weights' size, beside those, which the runtime
keeps. readout="device" takes the runtime's own logits, which every step leaves and
which are quicker to have: 58 us a byte against 180 at 1,024 neurons, 60 against 132
at 1,048,576, where the product of all weights alone takes 39 us and the active
neurons come by way of the host. The 8-bit readout's weights are a quarter of the output
weights' size, and its bytes take as long as the 4-bit one's.

A search of 4 hypotheses takes 3.4 to 4.9 ms a byte in texts of 100 bytes: the runtime has one
document, so each step writes every hypothesis from its beginning.
"""
from __future__ import annotations

import argparse
import sys
from typing import Dict, List, Optional, Sequence, Tuple, Union

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
        if readout not in ("q4", "q8", "device"):
            raise native.LeoError(native.ERR_INVALID_ARGUMENT, f"readout must be q4, q8 or device, not {readout}")
        self.runtime = runtime
        self.device = torch.device("cuda", runtime.device)
        self.neurons = runtime.config.model.neuron_count
        self.readout = readout
        self.group = group
        self.weight: Union[None, decode.Q4Weight, decode.Q8Weight] = None
        self.bias: Optional[torch.Tensor] = None
        self._version = -1      # of the parameters that weight and bias were made from
        if readout != "device":
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
            weight = torch.from_numpy(rows).to(self.device)
            self.weight = decode.Q8Weight.quantize(weight) if self.readout == "q8" else decode.Q4Weight.quantize(weight, self.group)
            self.bias = torch.from_numpy(bias).to(self.device)
            self._version = version

    def logits(self) -> torch.Tensor:
        """[1, 257]: the readout of the last step, with the model's weights as they are now."""
        if self.readout == "device":
            return torch.from_numpy(self.runtime.read_state("logits")).to(self.device)[None]
        self._active.zero_()
        self._take_active(self._active[0])
        return self._read_out(self._active)

    def _take_active(self, row: torch.Tensor) -> None:
        """The last step's activations into a row of zeros."""
        ids, values = self.runtime._read_active()
        row[torch.from_numpy(ids).to(self.device)] = torch.from_numpy(values).to(self.device)

    def _read_out(self, active: torch.Tensor) -> torch.Tensor:
        self._take_weights()
        product = decode.q8_matmul if self.readout == "q8" else decode.q4_matvec
        return product(active, self.weight, self.bias)

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

    def _need_document(self) -> None:
        if self._document != self.runtime.documents:
            raise native.LeoError(native.ERR_INVALID_ARGUMENT, "no document is open: begin one with prompt()")

    def _biases(self, bias: Optional[Dict[int, float]], allow_end: bool, rows: int):
        """The biases of `decode.control_logits` for `rows` rows."""
        biases = dict(bias or {})
        if not allow_end:
            biases[END] = float("-inf")
        if not biases:
            return None
        return (torch.tensor(list(biases) * rows, dtype=torch.int32, device=self.device),
                torch.tensor(list(biases.values()) * rows, dtype=torch.float32, device=self.device),
                torch.arange(rows + 1, device=self.device) * len(biases))

    def write(self, count: int, *, temperature: float = 0.8, top_k: int = 40, top_p: float = 0.95, min_p: float = 0.0,
              repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0, history: int = 64,
              bias: Optional[Dict[int, float]] = None, allow_end: bool = True) -> Tuple[bytes, List[float]]:
        """Up to `count` bytes after the prompt, and their logprobs; fewer where the
        model ends the document. Needs the document that `prompt` began, ended neither
        by the model nor by another use of the runtime. The penalties look at the last
        `history` bytes, the prompt's among them; `bias` adds to single bytes' logits
        (256: the end). A top_k below 1 keeps the largest alone, as 1 does."""
        self._need_document()

        def one(value, dtype=torch.float32):
            return torch.tensor([value], dtype=dtype, device=self.device)

        per_row = {"temperature": one(temperature), "top_k": one(top_k, torch.int32), "top_p": one(top_p),
                   "min_p": one(min_p)}
        penalties = {"repetition": one(repetition), "presence": one(presence), "frequency": one(frequency)}
        listed = self._biases(bias, allow_end, 1)
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

    def search(self, count: int, *, beams: int = 4, length_penalty: float = 0.0, repetition: float = 1.0,
               presence: float = 0.0, frequency: float = 0.0, history: int = 64, bias: Optional[Dict[int, float]] = None,
               allow_end: bool = True) -> List[Tuple[bytes, float]]:
        """The likeliest texts of up to `count` bytes after the document's bytes so far,
        the best first, with the sums of their bytes' log probabilities (and the end's,
        where they end): beam search by score / length^length_penalty, at most `beams` of
        them (64 at most). Penalties and biases are those of `write`, whose probabilities
        they change.

        The runtime has one document at a time, so each step writes every hypothesis
        from its beginning, with frozen steps, and the readout, the control and the
        selection take all of them at once. The prompt's document has ended
        afterwards."""
        self._need_document()
        if not 1 <= beams <= 64:
            raise native.LeoError(native.ERR_INVALID_ARGUMENT, f"beams must be 1 to 64, not {beams}")
        if count < 1:
            self._document = None
            return [(b"", 0.0)]
        prefix = self._written
        # what each hypothesis has on the GPU: its bytes, with those before it, and its state of UTF-8
        text = torch.zeros(1, len(prefix) + count, dtype=torch.int32, device=self.device)
        text[0, :len(prefix)] = torch.tensor(prefix, dtype=torch.int32, device=self.device)
        states = torch.full((1,), self._state, dtype=torch.int32, device=self.device)
        following = torch.from_numpy(self._next.astype(np.int32)).to(self.device)
        scores, lengths = torch.zeros(1, 1, device=self.device), torch.zeros(1, 1, dtype=torch.int32, device=self.device)
        finished = torch.zeros(1, 1, dtype=torch.bool, device=self.device)
        written: List[List[int]] = [[]]
        done, alive = [False], [True]
        logits = self.logits()
        for at in range(len(prefix), len(prefix) + count):
            rows = len(written)
            if at > len(prefix):
                logits = self._logits_of(prefix, written, [a and not d for a, d in zip(alive, done)])

            def each(value, rows=rows):
                return torch.full((rows,), value, device=self.device)

            recent = text[:, max(0, at - history):at].reshape(-1) if history > 0 else text[:, :0].reshape(-1)
            logits = decode.control_logits(
                logits, history=(recent, torch.arange(rows + 1, device=self.device) * (recent.numel() // rows)),
                repetition=each(repetition), presence=each(presence), frequency=each(frequency),
                bias=self._biases(bias, allow_end, rows), masks=self._masks, mask_rows=states)
            found = decode.beam_select(logits, scores, beams, finished=finished, lengths=lengths,
                                       length_penalty=length_penalty, end=END)
            scores, finished, lengths = found.scores, found.finished, found.lengths
            if rows == beams:
                decode.reorder_states([text, states], found.parents, out=[text, states])
            else:
                text, states = decode.reorder_states([text, states], found.parents)
            grows = (found.symbols[0] >= 0) & (found.symbols[0] < END)
            byte = torch.where(grows, found.symbols[0], torch.zeros_like(found.symbols[0]))
            text[:, at] = byte
            states = torch.where(grows, following[states.long(), byte.long()], states)
            symbols, parents = found.symbols[0].tolist(), found.parents[0].tolist()
            done, alive = finished[0].tolist(), [s > -np.inf for s in scores[0].tolist()]
            written = [written[p] + ([s] if 0 <= s < END else []) for s, p in zip(symbols, parents)]
            if all(d or not a for d, a in zip(done, alive)):
                break
        self._document = None
        if not any(alive):
            raise native.LeoError(native.ERR_NUMERICAL, "no byte is left to take")
        return [(bytes(w), s) for w, s, a in zip(written, scores[0].tolist(), alive) if a]

    def _logits_of(self, prefix: List[int], written: List[List[int]], wanted: List[bool]) -> torch.Tensor:
        """[hypotheses, 257]: the readouts after each of the wanted hypotheses; the others' rows hold anything."""
        active = torch.zeros(len(written), OUTPUT_CLASSES if self.readout == "device" else self.neurons, device=self.device)
        for row, hypothesis, wants in zip(active, written, wanted):
            if not wants:
                continue
            self.runtime.begin_document()
            symbols = [BEGIN_DOCUMENT, *prefix, *hypothesis]
            self.runtime.advance_frozen_batch([(s, None) for s in symbols[:-1]])
            self.runtime.step(symbols[-1], None, native.FROZEN)
            if self.readout == "device":
                row.copy_(torch.from_numpy(self.runtime.read_state("logits")))
            else:
                self._take_active(row)
        return active if self.readout == "device" else self._read_out(active)


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
    parser.add_argument("--readout", choices=("q4", "q8", "device"), default="q4")
    parser.add_argument("--group", type=int, default=32, choices=(32, 64, 128))
    parser.add_argument("--seed", type=int, default=0)
    for name, default in (("temperature", 0.8), ("top-p", 0.95), ("min-p", 0.0), ("repetition", 1.1), ("presence", 0.0),
                          ("frequency", 0.0)):
        parser.add_argument("--" + name, type=float, default=default)
    parser.add_argument("--top-k", type=int, default=40, help="bytes to draw from; below 2 the likeliest alone, 257 for all")
    parser.add_argument("--history", type=int, default=64)
    parser.add_argument("--beams", type=int, default=0, help="hypotheses of a search, which takes the draw's place; 0 draws")
    parser.add_argument("--length-penalty", type=float, default=0.0, help="of the search")
    args = parser.parse_args(argv)
    if args.checkpoint:
        from .formats import load_model

        runtime = HipRuntime(load_model(args.checkpoint), max_lanes=1)
    else:
        runtime = _trained(args.neurons, args.stories)
    with runtime:
        generator = Generator(runtime, group=args.group, readout=args.readout, seed=args.seed)
        generator.prompt(args.prompt.encode())
        penalties = dict(repetition=args.repetition, presence=args.presence, frequency=args.frequency, history=args.history)
        if args.beams:
            text, score = generator.search(args.bytes, beams=args.beams, length_penalty=args.length_penalty, **penalties)[0]
            logprobs = [score / max(1, len(text))] * len(text)
        else:
            text, logprobs = generator.write(args.bytes, temperature=args.temperature, top_k=args.top_k, top_p=args.top_p,
                                             min_p=args.min_p, **penalties)
    print(args.prompt + text.decode(errors="replace"))
    if logprobs:
        print(f"{len(logprobs)} bytes, {-sum(logprobs) / len(logprobs) / np.log(2):.3f} bits a byte under its own "
              "distribution", file=sys.stderr)
    return 0


if __name__ == "__main__":
    sys.exit(main())
