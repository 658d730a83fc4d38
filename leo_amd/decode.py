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
before the first call into libleo_hip.so; any other order raises ``ImportError``.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import pathlib
import sys
from typing import Optional, Tuple

from . import native

_ORDER = ("import torch (or leo_amd.decode) before the first HipRuntime: libleo_hip.so is already bound to another HIP "
          "runtime than torch's")
if "torch" not in sys.modules and native._lib is not None:
    raise ImportError(_ORDER)

import torch  # noqa: E402

_TYPES = {torch.float32: native.TYPE_F32, torch.float16: native.TYPE_F16, torch.bfloat16: native.TYPE_BF16}


def _refuse(message: str) -> None:
    raise native.LeoError(native.ERR_INVALID_ARGUMENT, message)


def _device(name: str, t: torch.Tensor) -> int:
    """The number of the GPU that `t` is on."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{name} must be a tensor on the GPU")
    return t.get_device()


def _matrix(name: str, t: torch.Tensor, dtypes, index: int) -> Tuple[int, int, int]:
    """(rows, width, row stride) of a 2-D tensor of one of `dtypes` on GPU `index` whose last axis is dense."""
    if isinstance(t, torch.Tensor) and t.get_device() == index and t.dtype in dtypes and t.dim() == 2:
        rows, width = t.shape
        stride, last = t.stride()
        if last == 1 or width <= 1:
            return rows, width, stride
        _refuse(f"{name}'s last axis must be dense")
    if _device(name, t) != index:
        _refuse(f"{name} is on GPU {t.get_device()}, not on {index}")
    _refuse(f"{name} has type {t.dtype}" if t.dtype not in dtypes else f"{name} must have two axes, not {t.dim()}")


def _public_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# torch's own accessor of the same number, without the Stream object that costs more than a small launch's checks
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _check_runtime(lib: ctypes.CDLL) -> None:
    """Refuses a library that calls another HIP runtime than torch: torch may have
    come after the library, and then each is bound to its own."""
    hip = pathlib.Path(torch.__file__).with_name("lib") / "libtorch_hip.so"
    if hip.exists():
        ours, theirs = (ctypes.cast(l.hipLaunchKernel, ctypes.c_void_p).value for l in (lib, ctypes.CDLL(str(hip))))
        if ours != theirs:
            raise ImportError(_ORDER)


def _load_binding():
    path = native.LIB_PATH.with_name("leo_decode_binding.so")
    if not path.exists():
        raise ImportError(f"{path} is missing: build it with `python -m leo_amd.build` (no fallback exists)")
    _check_runtime(native.load())
    loader = importlib.machinery.ExtensionFileLoader("leo_decode_binding", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader(loader.name, loader))
    loader.exec_module(module)
    module.setup(native.LeoError, _stream_of)
    return module


_binding = _load_binding()   # the products', the control's and the draw's checks, results and calls


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
        self.index = _device("codes", codes)
        self.device = codes.device
        outputs, width, codes_stride = _matrix("codes", codes, (torch.uint8,), self.index)
        if group not in (32, 64, 128):
            _refuse(f"group must be 32, 64 or 128, not {group}")
        if inputs < 1 or outputs < 1 or width != (inputs + 1) // 2:
            _refuse(f"codes of {inputs} inputs have {(inputs + 1) // 2} bytes a row, not {width}")
        strides = []
        for name, t, dtypes in (("scales", scales, _TYPES), ("zeros", zeros, (torch.uint8,))):
            if t is None and name == "zeros":
                strides.append(0)
                continue
            *shape, stride = _matrix(name, t, dtypes, self.index)
            if shape != [outputs, -(-inputs // group)]:
                _refuse(f"{name} must be {(outputs, -(-inputs // group))}, not {tuple(shape)}")
            strides.append(stride)
        self.outputs, self.inputs, self.group = outputs, inputs, group
        self.shape = native.LeoQ4Shape(outputs=outputs, inputs=inputs, group=group, scale_type=_TYPES[scales.dtype],
                                       has_zeros=zeros is not None)
        lib, size = native.load(), ctypes.c_uint64()
        native.check(lib, lib.leo_q4_layout_bytes(ctypes.byref(self.shape), ctypes.byref(size)))
        self.layout = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        source = native.LeoQ4Source(
            shape=self.shape, codes=codes.data_ptr(), codes_stride=codes_stride, scales=scales.data_ptr(),
            scales_stride=strides[0], zeros=None if zeros is None else zeros.data_ptr(), zeros_stride=strides[1],
            layout=self.layout.data_ptr(), layout_bytes=size.value)
        with torch.cuda.device(self.index):
            native.check(lib, lib.leo_q4_layout(ctypes.byref(source), _stream_of(self.index)))
        self._shape = bytes(self.shape)

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 32, scale_dtype: torch.dtype = torch.float16) -> "Q4Weight":
        """A floating matrix [outputs, inputs] rounded to codes about 8: a group's
        scale is its largest magnitude over 7 (0 for a group of zeros). Refuses a
        weight with a scale that `scale_dtype` does not hold; the check waits for the
        GPU and is left out while a graph is captured."""
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not weight.is_floating_point():
            _refuse("weight must be a floating matrix")
        _device("weight", weight)
        if group not in (32, 64, 128):
            _refuse(f"group must be 32, 64 or 128, not {group}")
        if scale_dtype not in _TYPES:
            _refuse(f"scales have type float32, float16 or bfloat16, not {scale_dtype}")
        outputs, inputs = weight.shape
        padded = torch.nn.functional.pad(weight.detach().float(), (0, -inputs % group)).view(outputs, -1, group)
        largest = padded.abs().amax(dim=2)
        scales = (largest / 7.0).to(scale_dtype)
        # among the type's smallest values, where rounding may have left too little, its next one
        bits = scales.view(torch.int32 if scale_dtype is torch.float32 else torch.int16)
        scales = (bits + (largest > 7.5 * scales.float())).view(scale_dtype)
        if not torch.cuda.is_current_stream_capturing() and not bool(scales.isfinite().all()):
            _refuse(f"a group's largest magnitude over 7 is no finite {scale_dtype}")
        divide = torch.where(scales == 0, torch.ones_like(scales), scales).float()
        codes = ((padded / divide[:, :, None]).round().clamp(-8, 7) + 8).to(torch.uint8)
        codes = codes.view(outputs, -1)[:, :inputs + inputs % 2].contiguous()
        return cls(codes[:, 0::2] | (codes[:, 1::2] << 4), scales, inputs=inputs, group=group)


def q4_matvec(x: torch.Tensor, weight: Q4Weight, bias: Optional[torch.Tensor] = None, *,
              out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bias + x W^T for x [rows, inputs] (or [inputs]) of float32, float16 or
    bfloat16: sums in 32 bits, rounded once to `out_dtype` (x's type by default). A
    float32 x enters with 22 bits of each value, and to 2^-39 of the largest of its
    row's 128 neighbouring inputs, to which a bfloat16 x is held too; scales have to
    stay below 2^100. bias: float32 [outputs]. `out` and x share no memory."""
    if isinstance(x, torch.Tensor) and x.dim() == 1:
        if out is not None:
            _refuse("out needs x with two axes")
        return q4_matvec(x[None], weight, bias, out_dtype=out_dtype)[0]
    if out is None:
        out = -1 if out_dtype is None else _TYPES.get(out_dtype, len(_TYPES))
    elif not isinstance(out, torch.Tensor):      # a number would pass for a type
        _refuse("out must be a tensor on the GPU")
    elif out_dtype is not None and out.dtype is not out_dtype:
        _refuse(f"out must have type {out_dtype}")
    return _binding.q4_matvec(x, weight.layout, weight._shape, bias, out)


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
    masks      int32 [n, ceil(symbols / 32)] with n >= 1, symbol v at bit v % 32 of word v // 32
    mask_rows  int32 [rows]: each row's mask, -1 for none, any other number outside 0..n-1 allows nothing;
               without it n is 1 or the number of rows
    out        may be `logits`, but share no memory with them otherwise
    """
    entries, offsets = (None, None) if history is None else history
    ids, values, bias_offsets = (None, None, None) if bias is None else bias
    return _binding.control_logits(logits, entries, offsets, repetition, presence, frequency, ids, values, bias_offsets,
                                   masks, mask_rows, out)


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
    return _binding.sample(logits, noise, temperature, top_k, top_p, min_p)
