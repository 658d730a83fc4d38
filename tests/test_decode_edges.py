"""Refusals of the decoding operators that need no GPU: masks that are not there, a
second HIP runtime in the process, results over their operands."""
from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest

from leo_amd import native
from tests.test_abi import ROOT


def refusal(function, struct, fields):
    lib = native.load()
    assert getattr(lib, function)(ctypes.byref(struct(**fields)), None) == native.ERR_INVALID_ARGUMENT
    return native.last_error(lib)


@pytest.mark.parametrize("change", [dict(mask_rows=256), dict(mask_count=3), dict(mask_count=3, mask_rows=256)])
def test_masks_that_are_not_there_shut_nothing_silently(change):
    # a table without rows has no memory: its rows' numbers must not pass as "no masks"
    good = dict(rows=2, symbols=257, logits=256, logits_stride=257, out=4096, out_stride=257, type=native.TYPE_F32)
    assert "masks" in refusal("leo_control_logits", native.LeoLogitControl, {**good, **change})


@pytest.mark.parametrize("first", ["native.load()", "ctypes.CDLL(str(native.LIB_PATH))"])
def test_a_torch_that_came_later_is_refused(first):
    # the library is bound to one HIP runtime, torch has brought another
    code = (f"import ctypes\nfrom leo_amd import native\n{first}\nimport torch\ntry:\n    import leo_amd.decode\n"
            "except ImportError as e:\n    assert 'before the first HipRuntime' in str(e)\nelse:\n    raise SystemExit(1)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(ROOT))


def test_torch_before_the_library_is_one_runtime():
    code = ("import torch\nfrom leo_amd import native\nnative.load()\nimport leo_amd.decode, leo_amd.generate\n"
            "assert len({l.split()[-1] for l in open('/proc/self/maps') if 'libamdhip64' in l}) == 1\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(ROOT))


MATRIX = dict(rows=4, x_stride=128, y_stride=128)


@pytest.mark.parametrize("x,y,change", [
    (1 << 20, 1 << 20, {}), (1 << 20, (1 << 20) + 4, {}), ((1 << 20) + 4 * 127, 1 << 20, {}),
    (1 << 20, (1 << 20) + 4 * 128 * 4 - 4, {}), (1 << 20, (1 << 20) + 4 * 100, dict(x_stride=300, y_stride=300)),
    (1 << 20, (1 << 20) + 4 * 250, dict(x_stride=300, y_stride=300)), (1 << 20, (1 << 20) + 4 * 64, dict(x_stride=0)),
    (1 << 20, (1 << 20) + 4 * 130, dict(x_stride=257, y_stride=200))])
def test_results_over_their_operand_are_refused(x, y, change):
    # other workgroups read x while the first results are stored
    shape = native.LeoQ4Shape(outputs=128, inputs=128, group=128, scale_type=native.TYPE_F32, has_zeros=0)
    assert "overlaps x" in refusal("leo_q4_matvec", native.LeoQ4Product, dict(
        shape=shape, layout=1 << 30, layout_bytes=1 << 20, x=x, y=y, x_type=native.TYPE_F32, y_type=native.TYPE_F32,
        workspace=1 << 31, workspace_bytes=1 << 30, **{**MATRIX, **change}))


@pytest.mark.parametrize("out,change", [
    (4, {}), (-4, {}), (4 * 256, {}), (4 * 257 * 3, {}), (0, dict(out_stride=300)), (0, dict(logits_stride=0)),
    (4 * 200, dict(logits_stride=400, out_stride=400))])
def test_controlled_logits_beside_the_logits_are_refused(out, change):
    # in place is exactly in place
    assert "overlaps the logits" in refusal("leo_control_logits", native.LeoLogitControl, {**dict(
        rows=4, symbols=257, logits=1 << 20, logits_stride=257, out=(1 << 20) + out, out_stride=257,
        type=native.TYPE_F32), **change})


def test_a_weight_off_the_gpu_is_refused():
    code = ("import torch\nfrom leo_amd import decode, native\ntry:\n    decode.Q4Weight.quantize(torch.ones(4, 64))\n"
            "except native.LeoError as e:\n    assert e.code == native.ERR_INVALID_ARGUMENT and 'on the GPU' in str(e)\n"
            "else:\n    raise SystemExit(1)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(ROOT))
