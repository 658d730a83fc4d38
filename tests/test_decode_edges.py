"""Refusals of the decoding operators that need no GPU: masks that are not there, a
second HIP runtime in the process."""
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
