"""The operators that take a model from activations to its next symbol, on torch
tensors: 4-bit readout products, control of logits, and the draw.

    Q4Weight, q4_matvec   y = b + x W^T with 4-bit codes and group scales
    control_logits        penalties for repeated symbols, biases, grammar masks
    sample                temperature, top-k, top-p, min-p and the draw

Each call goes through the C-ABI of include/leo_decode.h into libleo_hip.so and
enqueues its work on the current stream of its tensors' device. Failed checks
raise ``LeoError`` with ``native.ERR_INVALID_ARGUMENT``. There is no CPU
fallback. Calls may be captured into a graph.

The step runtime does not use torch; this module does, and torch brings a HIP
runtime of its own. One process must have one: import torch (or this module)
before the first call into libleo_hip.so.
"""
from __future__ import annotations

import ctypes
import sys
from typing import Dict, Optional, Tuple

from . import native

if "torch" not in sys.modules and native._lib is not None:
    raise ImportError("import torch (or leo_amd.decode) before the first HipRuntime: libleo_hip.so is already bound "
                      "to another HIP runtime than torch's")

import torch  # noqa: E402

_TYPES = {torch.float32: native.TYPE_F32, torch.float16: native.TYPE_F16, torch.bfloat16: native.TYPE_BF16}


def _refuse(message: str) -> None:
    raise native.LeoError(native.ERR_INVALID_ARGUMENT, message)


def _matrix(name: str, t: torch.Tensor, dtypes, device: Optional[torch.device] = None) -> None:
    """`t` is a 2-D device tensor of one of `dtypes` whose last axis is dense."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{name} must be a tensor on the GPU")
    if device is not None and t.device != device:
        _refuse(f"{name} is on {t.device}, not on {device}")
    if t.dtype not in dtypes:
        _refuse(f"{name} has type {t.dtype}")
    if t.dim() != 2:
        _refuse(f"{name} must have two axes, not {t.dim()}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        _refuse(f"{name}'s last axis must be dense")


def _vector(name: str, t: Optional[torch.Tensor], dtype: torch.dtype, device: torch.device,
            count: Optional[int] = None) -> Optional[int]:
    """The address of a dense 1-D tensor (None for none)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.device != device:
        _refuse(f"{name} must be a tensor on {device}")
    if t.dtype != dtype:
        _refuse(f"{name} must have type {dtype}, not {t.dtype}")
    if t.dim() != 1 or not t.is_contiguous():
        _refuse(f"{name} must be a dense vector")
    if count is not None and t.shape[0] != count:
        _refuse(f"{name} has {t.shape[0]} entries, not {count}")
    return t.data_ptr()


def _call(function: str, args: ctypes.Structure, device: torch.device, need: int = 0) -> None:
    lib = native.load()
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(function, args, device, need)
    stream = torch.cuda.current_stream(device).cuda_stream
    if need:      # the caching allocator's: free again in the stream's order
        space = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = space.data_ptr(), need
    native.check(lib, getattr(lib, function)(ctypes.byref(args), stream))


class Q4Weight:
    """A 4-bit weight matrix [outputs, inputs], laid out once for `q4_matvec`:

        w[n, k] = scales[n, k // group] * (code[n, k] - zeros[n, k // group])

    codes   uint8 [outputs, ceil(inputs / 2)], input 2j in the low half of byte j
    scales  float32, float16 or bfloat16 [outputs, ceil(inputs / group)]
    zeros   uint8 0..15 of the scales' shape; None: 8 everywhere
    group   32, 64 or 128 inputs; the last group of a row may be short

    The layout is the object's own; the arguments are not kept.
    """

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
                 inputs: int, group: int):
        _matrix("codes", codes, (torch.uint8,))
        self.device = codes.device
        _matrix("scales", scales, _TYPES, self.device)
        if zeros is not None:
            _matrix("zeros", zeros, (torch.uint8,), self.device)
        if group not in (32, 64, 128):
            _refuse(f"group must be 32, 64 or 128, not {group}")
        outputs, groups = codes.shape[0], -(-inputs // group)
        if inputs < 1 or outputs < 1 or codes.shape[1] != (inputs + 1) // 2:
            _refuse(f"codes of {inputs} inputs have {(inputs + 1) // 2} bytes a row, not {codes.shape[1]}")
        for name, t in (("scales", scales), ("zeros", zeros)):
            if t is not None and tuple(t.shape) != (outputs, groups):
                _refuse(f"{name} must be {(outputs, groups)}, not {tuple(t.shape)}")
        self.outputs, self.inputs, self.group = outputs, inputs, group
        self.shape = native.LeoQ4Shape(outputs=outputs, inputs=inputs, group=group, scale_type=_TYPES[scales.dtype],
                                       has_zeros=zeros is not None)
        lib, size = native.load(), ctypes.c_uint64()
        native.check(lib, lib.leo_q4_layout_bytes(ctypes.byref(self.shape), ctypes.byref(size)))
        self.layout = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        source = native.LeoQ4Source(
            shape=self.shape, codes=codes.data_ptr(), codes_stride=codes.stride(0), scales=scales.data_ptr(),
            scales_stride=scales.stride(0), zeros=None if zeros is None else zeros.data_ptr(),
            zeros_stride=0 if zeros is None else zeros.stride(0), layout=self.layout.data_ptr(),
            layout_bytes=size.value)
        _call("leo_q4_layout", source, self.device)
        self._workspace_bytes: Dict[Tuple[int, int], int] = {}

    def workspace_bytes(self, rows: int, x_type: int) -> int:
        """Bytes of workspace that a product with `rows` rows of x needs."""
        found = self._workspace_bytes.get((rows, x_type))
        if found is None:
            lib, size = native.load(), ctypes.c_uint64()
            native.check(lib, lib.leo_q4_workspace_bytes(ctypes.byref(self.shape), rows, x_type, ctypes.byref(size)))
            found = self._workspace_bytes[rows, x_type] = size.value
        return found

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 32, scale_dtype: torch.dtype = torch.float16) -> "Q4Weight":
        """A floating matrix [outputs, inputs] rounded to codes about 8: a group's
        scale is its largest magnitude over 7 (0 for a group of zeros)."""
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not weight.is_floating_point():
            _refuse("weight must be a floating matrix")
        if group not in (32, 64, 128):
            _refuse(f"group must be 32, 64 or 128, not {group}")
        outputs, inputs = weight.shape
        padded = torch.nn.functional.pad(weight.float(), (0, -inputs % group)).view(outputs, -1, group)
        scales = (padded.abs().amax(dim=2) / 7.0).to(scale_dtype)
        divide = torch.where(scales == 0, torch.ones_like(scales), scales).float()
        codes = ((padded / divide[:, :, None]).round().clamp(-8, 7) + 8).to(torch.uint8)
        codes = codes.view(outputs, -1)[:, :inputs + inputs % 2].contiguous()
        return cls(codes[:, 0::2] | (codes[:, 1::2] << 4), scales, inputs=inputs, group=group)


def q4_matvec(x: torch.Tensor, weight: Q4Weight, bias: Optional[torch.Tensor] = None, *,
              out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bias + x W^T for x [rows, inputs] (or [inputs]) of float32, float16 or
    bfloat16: sums in 32 bits, rounded once to `out_dtype` (x's type by default).
    bias: float32 [outputs]."""
    if isinstance(x, torch.Tensor) and x.dim() == 1:
        if out is not None:
            _refuse("out needs x with two axes")
        return q4_matvec(x[None], weight, bias, out_dtype=out_dtype)[0]
    _matrix("x", x, _TYPES, weight.device)
    rows = x.shape[0]
    if x.shape[1] != weight.inputs:
        _refuse(f"x has {x.shape[1]} inputs, the weight {weight.inputs}")
    if out is None:
        out = torch.empty((rows, weight.outputs), dtype=out_dtype or x.dtype, device=x.device)
    _matrix("out", out, _TYPES, weight.device)
    if out.shape[0] != rows or out.shape[1] != weight.outputs or (out_dtype is not None and out.dtype != out_dtype):
        _refuse(f"out must be {(rows, weight.outputs)} of {out_dtype or out.dtype}")
    args = native.LeoQ4Product(
        shape=weight.shape, layout=weight.layout.data_ptr(), layout_bytes=weight.layout.numel(), rows=rows,
        x=x.data_ptr(), x_stride=x.stride(0), bias=_vector("bias", bias, torch.float32, weight.device, weight.outputs),
        y=out.data_ptr(), y_stride=out.stride(0), x_type=_TYPES[x.dtype], y_type=_TYPES[out.dtype])
    _call("leo_q4_matvec", args, weight.device, weight.workspace_bytes(rows, args.x_type))
    return out


def control_logits(logits: torch.Tensor, *, history: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                   repetition: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None,
                   bias: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                   masks: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [rows, symbols] after, in this order and for a symbol that stands c
    times in its row's history: z / repetition (z * repetition where z <= 0) and
    - (presence + frequency * c) where c > 0; + bias; -inf where the mask's bit is 0.

    history    (symbols int32, offsets int64 [rows + 1]); entries outside the vocabulary are ignored
    repetition, presence, frequency   float32 [rows]; without them 1, 0 and 0
    bias       (ids int32, values float32, offsets int64 [rows + 1]); a row's last entry for a symbol counts
    masks      int32 [n, ceil(symbols / 32)], symbol v at bit v % 32 of word v // 32
    mask_rows  int32 [rows]: each row's mask, -1 for none, any other number outside 0..n-1 allows nothing;
               without it n is 1 or the number of rows
    out        may be `logits`
    """
    _matrix("logits", logits, _TYPES)
    device = logits.device
    rows, symbols = logits.shape
    if out is None:
        out = torch.empty((rows, symbols), dtype=logits.dtype, device=device)
    else:
        _matrix("out", out, (logits.dtype,), device)
        if out.shape != logits.shape:
            _refuse(f"out must be {(rows, symbols)}")
    args = native.LeoLogitControl(rows=rows, symbols=symbols, logits=logits.data_ptr(),
                                  logits_stride=logits.stride(0), out=out.data_ptr(), out_stride=out.stride(0),
                                  type=_TYPES[logits.dtype])
    if history is not None:
        args.history = _vector("history", history[0], torch.int32, device)
        args.history_offsets = _vector("history offsets", history[1], torch.int64, device, rows + 1)
        args.history_count = history[0].shape[0]
    args.repetition = _vector("repetition", repetition, torch.float32, device, rows)
    args.presence = _vector("presence", presence, torch.float32, device, rows)
    args.frequency = _vector("frequency", frequency, torch.float32, device, rows)
    if bias is not None:
        args.bias_ids = _vector("bias ids", bias[0], torch.int32, device)
        args.bias_count = bias[0].shape[0]
        args.bias_values = _vector("bias values", bias[1], torch.float32, device, args.bias_count)
        args.bias_offsets = _vector("bias offsets", bias[2], torch.int64, device, rows + 1)
    if masks is not None:
        _matrix("masks", masks, (torch.int32,), device)
        if masks.shape[1] != (symbols + 31) // 32:
            _refuse(f"masks of {symbols} symbols have {(symbols + 31) // 32} words, not {masks.shape[1]}")
        args.masks, args.masks_stride, args.mask_count = masks.data_ptr(), masks.stride(0), masks.shape[0]
    elif mask_rows is not None:
        _refuse("mask_rows without masks")
    args.mask_rows = _vector("mask_rows", mask_rows, torch.int32, device, rows)
    _call("leo_control_logits", args, device)
    return out


def sample(logits: torch.Tensor, noise: Optional[torch.Tensor] = None, *, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(symbols int32 [rows], logprobs float32 [rows]) drawn from logits [rows, symbols].

    With z = logits / temperature and w = exp(z - max z), a symbol stays if fewer
    than top_k symbols have a larger z, those have less than top_p of the mass
    (top_p >= 1: any), and w >= min_p; the largest always stays. The one that
    stays with the largest z + noise is drawn, the lowest of equals. noise
    float32 [rows, symbols] holds Gumbel noise, -log of an exponential draw;
    without it, or at a temperature of 0, the largest logit is taken. logprobs are
    z - log sum exp z over the whole row. A NaN logit counts as -inf; a row of
    -inf alone gives -1 and -inf. temperature, top_p, min_p float32 [rows] and
    top_k int32 [rows]; without them 1, 1, 0 and all.
    """
    _matrix("logits", logits, _TYPES)
    device = logits.device
    rows, symbols = logits.shape
    if symbols < 1:
        _refuse("no symbols to draw from")
    if noise is not None:
        _matrix("noise", noise, (torch.float32,), device)
        if noise.shape != logits.shape:
            _refuse(f"noise must be {(rows, symbols)}, not {tuple(noise.shape)}")
    drawn = torch.empty(rows, dtype=torch.int32, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    args = native.LeoSample(
        rows=rows, symbols=symbols, logits=logits.data_ptr(), logits_stride=logits.stride(0),
        type=_TYPES[logits.dtype], noise=None if noise is None else noise.data_ptr(),
        noise_stride=0 if noise is None else noise.stride(0),
        temperature=_vector("temperature", temperature, torch.float32, device, rows),
        top_k=_vector("top_k", top_k, torch.int32, device, rows),
        top_p=_vector("top_p", top_p, torch.float32, device, rows),
        min_p=_vector("min_p", min_p, torch.float32, device, rows),
        out_symbols=drawn.data_ptr(), out_logprobs=logprobs.data_ptr())
    _call("leo_sample", args, device, _sample_workspace(rows, symbols))
    return drawn, logprobs


_sample_spaces: Dict[Tuple[int, int], int] = {}


def _sample_workspace(rows: int, symbols: int) -> int:
    found = _sample_spaces.get((rows, symbols))
    if found is None:
        lib, size = native.load(), ctypes.c_uint64()
        native.check(lib, lib.leo_sample_workspace_bytes(rows, symbols, ctypes.byref(size)))
        found = _sample_spaces[rows, symbols] = size.value
    return found
