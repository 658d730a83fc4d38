"""The decoding operators' C-ABI without a GPU: exports, argument structs and
refusals that come before any device work."""
from __future__ import annotations

import ctypes
import re
import subprocess
import sys

import pytest

from leo_amd import native
from tests.test_abi import ROOT, _declared_functions

STRUCTS = ("LeoQ4Shape", "LeoQ4Source", "LeoQ4Product", "LeoLogitControl", "LeoSample")


def test_every_declared_function_is_exported_and_bound():
    lib = ctypes.CDLL(str(native.LIB_PATH))
    declared = _declared_functions("leo_decode.h")
    assert declared == set(native.DECODE_SIGNATURES)
    assert all(hasattr(lib, name) for name in declared)


def test_struct_layouts_match_the_header(tmp_path):
    fields = {name: [f for f, _ in getattr(native, name)._fields_] for name in STRUCTS}
    lines = [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n in STRUCTS for f in fields[n]]
    lines += [f'printf("{n} %zu\\n", sizeof({n}));' for n in STRUCTS]
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "leo_decode.h"\nint main(void) {\n'
                      + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(source), "-o", str(tmp_path / "layout")], check=True)
    said = dict(line.split() for line in
                subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for n in STRUCTS:
        struct = getattr(native, n)
        assert int(said[n]) == ctypes.sizeof(struct)
        for f in fields[n]:
            assert int(said[f"{n}.{f}"]) == getattr(struct, f).offset, (n, f)
    header = (ROOT / "include" / "leo_decode.h").read_text()
    for i, name in enumerate(("LEO_TYPE_F32", "LEO_TYPE_F16", "LEO_TYPE_BF16")):
        assert re.search(rf"{name} = {i}\b", header)
    assert (native.TYPE_F32, native.TYPE_F16, native.TYPE_BF16) == (0, 1, 2)


def _refused(function, *args):
    lib = native.load()
    assert getattr(lib, function)(*args) == native.ERR_INVALID_ARGUMENT
    return native.last_error(lib)


def test_null_arguments_are_refused():
    for name in ("leo_q4_layout", "leo_q4_matvec", "leo_control_logits", "leo_sample"):
        assert "null" in _refused(name, None, None)
    size = ctypes.c_uint64()
    _refused("leo_q4_layout_bytes", None, ctypes.byref(size))
    _refused("leo_q4_workspace_bytes", None, 1, native.TYPE_F32, ctypes.byref(size))
    _refused("leo_sample_workspace_bytes", 1, 1, None)


@pytest.mark.parametrize("change", [dict(group=0), dict(group=48), dict(group=256), dict(scale_type=3),
                                    dict(scale_type=-1), dict(outputs=0), dict(inputs=0), dict(inputs=2 ** 40)])
def test_bad_shapes_are_refused(change):
    good = dict(outputs=257, inputs=1024, group=32, scale_type=native.TYPE_F16, has_zeros=0)
    size = ctypes.c_uint64()
    lib = native.load()
    assert lib.leo_q4_layout_bytes(ctypes.byref(native.LeoQ4Shape(**good)), ctypes.byref(size)) == native.OK
    # 17 tiles of 8 blocks: codes, then a 16-bit scale for each of a block's four groups and 16 outputs
    assert size.value == 17 * 8 * (1024 + 16 * 4 * 2)
    _refused("leo_q4_layout_bytes", ctypes.byref(native.LeoQ4Shape(**{**good, **change})), ctypes.byref(size))


def test_bad_products_are_refused():
    shape = native.LeoQ4Shape(outputs=16, inputs=128, group=128, scale_type=native.TYPE_F32, has_zeros=0)
    good = dict(shape=shape, layout=256, layout_bytes=1 << 20, rows=1, x=256, x_stride=128, y=256, y_stride=16,
                x_type=native.TYPE_F32, y_type=native.TYPE_F32)
    for change in (dict(layout=None), dict(x=None), dict(y=None), dict(layout=128), dict(layout_bytes=1024),
                   dict(x_type=9), dict(y_type=-1), dict(x_stride=-1), dict(rows=2, y_stride=15), dict(rows=1 << 40)):
        _refused("leo_q4_matvec", ctypes.byref(native.LeoQ4Product(**{**good, **change})), None)
    source = dict(shape=shape, codes=256, codes_stride=64, scales=256, scales_stride=1, layout=256, layout_bytes=1 << 20)
    for change in (dict(codes=None), dict(scales=None), dict(layout=None), dict(layout=8), dict(layout_bytes=1024),
                   dict(codes_stride=63), dict(scales_stride=0), dict(zeros=256, zeros_stride=1)):
        _refused("leo_q4_layout", ctypes.byref(native.LeoQ4Source(**{**source, **change})), None)


def test_bad_controls_and_draws_are_refused():
    good = dict(rows=2, symbols=257, logits=256, logits_stride=257, out=256, out_stride=257, type=native.TYPE_F32)
    for change in (dict(logits=None), dict(out=None), dict(type=5), dict(logits_stride=-257), dict(out_stride=256),
                   dict(rows=1 << 33), dict(symbols=1 << 40), dict(history_offsets=256, history_count=1),
                   dict(bias_offsets=256, bias_count=1, bias_ids=256), dict(masks=256), dict(masks=256, mask_count=3),
                   dict(masks=256, mask_count=2, masks_stride=-1)):
        _refused("leo_control_logits", ctypes.byref(native.LeoLogitControl(**{**good, **change})), None)
    good = dict(rows=2, symbols=257, logits=256, logits_stride=257, type=native.TYPE_F32, out_symbols=256,
                out_logprobs=256)
    for change in (dict(logits=None), dict(out_symbols=None), dict(out_logprobs=None), dict(type=5), dict(symbols=0),
                   dict(symbols=1 << 40), dict(rows=1 << 33), dict(logits_stride=-1),
                   dict(noise=256, noise_stride=-1)):
        _refused("leo_sample", ctypes.byref(native.LeoSample(**{**good, **change})), None)


def test_torch_has_to_come_first():
    # one process, one HIP runtime: torch's
    code = ("from leo_amd import native\nnative.load()\ntry:\n    import leo_amd.decode\n"
            "except ImportError as e:\n    assert 'before the first HipRuntime' in str(e)\nelse:\n    raise SystemExit(1)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(ROOT))
    subprocess.run([sys.executable, "-c", "import leo_amd.decode\nfrom leo_amd import native\nnative.load()\n"],
                   check=True, cwd=str(ROOT))
