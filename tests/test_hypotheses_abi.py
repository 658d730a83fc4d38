"""The C-ABI of 8-bit products, beam selection and reordered states without a GPU:
argument structs, and refusals that come before any device work."""
from __future__ import annotations

import ctypes
import subprocess

import pytest

from leo_amd import native
from tests.test_abi import ROOT

STRUCTS = ("LeoQ8Shape", "LeoQ8Source", "LeoQ8Product", "LeoBeams", "LeoStateArray", "LeoReorder")


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


def _refused(function, *args):
    lib = native.load()
    assert getattr(lib, function)(*args) == native.ERR_INVALID_ARGUMENT
    return native.last_error(lib)


def test_null_arguments_are_refused():
    for name in ("leo_q8_layout", "leo_q8_matmul", "leo_beam_select", "leo_reorder_states"):
        assert "null" in _refused(name, None, None)
    size = ctypes.c_uint64()
    _refused("leo_q8_layout_bytes", None, ctypes.byref(size))
    _refused("leo_q8_workspace_bytes", None, 1, native.TYPE_F32, ctypes.byref(size))
    _refused("leo_beam_workspace_bytes", 1, 1, 1, 1, None)


def test_bad_products_are_refused():
    shape = native.LeoQ8Shape(outputs=16, inputs=128)
    size, lib = ctypes.c_uint64(), native.load()
    assert lib.leo_q8_layout_bytes(ctypes.byref(shape), ctypes.byref(size)) == native.OK
    assert size.value == 2 * 1024 + 256      # two blocks of one tile, and its scales
    for change in (dict(outputs=0), dict(inputs=0), dict(outputs=2 ** 40), dict(inputs=2 ** 40)):
        _refused("leo_q8_layout_bytes", ctypes.byref(native.LeoQ8Shape(**{**dict(outputs=16, inputs=128), **change})),
                 ctypes.byref(size))
    _refused("leo_q8_workspace_bytes", ctypes.byref(shape), 1 << 40, native.TYPE_F32, ctypes.byref(size))
    _refused("leo_q8_workspace_bytes", ctypes.byref(shape), 1, 7, ctypes.byref(size))
    good = dict(shape=shape, layout=256, layout_bytes=1 << 20, rows=1, x=256, x_stride=128, y=4096, y_stride=16,
                x_type=native.TYPE_F32, y_type=native.TYPE_F32, workspace=1 << 20, workspace_bytes=1 << 30)
    for change in (dict(layout=None), dict(x=None), dict(y=None), dict(layout=128), dict(layout_bytes=1024),
                   dict(x_type=9), dict(y_type=-1), dict(x_stride=-1), dict(rows=2, y_stride=15), dict(rows=1 << 40),
                   dict(y=512)):
        _refused("leo_q8_matmul", ctypes.byref(native.LeoQ8Product(**{**good, **change})), None)
    # a product that needs a workspace
    wide = {**good, "shape": native.LeoQ8Shape(outputs=257, inputs=1 << 20), "layout_bytes": 1 << 40, "x_stride": 1 << 20,
            "rows": 8, "y": 1 << 30, "y_stride": 257}
    for change in (dict(workspace=None), dict(workspace=(1 << 20) + 8), dict(workspace_bytes=16)):
        assert "workspace" in _refused("leo_q8_matmul", ctypes.byref(native.LeoQ8Product(**{**wide, **change})), None)
    source = dict(shape=shape, codes=256, codes_stride=128, scales=256, scale_type=0, layout=256, layout_bytes=1 << 20)
    for change in (dict(codes=None), dict(scales=None), dict(layout=None), dict(layout=8), dict(layout_bytes=1024),
                   dict(codes_stride=127), dict(scale_type=3), dict(scale_type=-1)):
        _refused("leo_q8_layout", ctypes.byref(native.LeoQ8Source(**{**source, **change})), None)


def test_bad_selections_are_refused():
    good = dict(groups=2, beams=3, kept=3, symbols=40_000, logits=1 << 24, logits_stride=40_000, type=native.TYPE_F32,
                scores=256, out_symbols=512, out_parents=768, out_scores=1024, end=-1, workspace=1 << 20,
                workspace_bytes=1 << 20)
    for change in (dict(beams=0), dict(beams=65), dict(kept=0), dict(kept=65), dict(symbols=0), dict(symbols=(1 << 26) + 1),
                   dict(groups=1 << 20), dict(type=4), dict(logits=None), dict(scores=None), dict(out_symbols=None),
                   dict(out_parents=None), dict(out_scores=None), dict(logits_stride=-1), dict(length_penalty=0.5),
                   dict(lengths=2048, length_penalty=float("nan")), dict(lengths=2048, length_penalty=float("inf")),
                   dict(out_lengths=256), dict(end=40_000), dict(end=-2), dict(workspace=None), dict(workspace_bytes=8),
                   dict(workspace=(1 << 20) + 128)):
        _refused("leo_beam_select", ctypes.byref(native.LeoBeams(**{**good, **change})), None)
    for change in (dict(out_scores=256), dict(out_scores=256 + 20), dict(out_parents=512), dict(out_symbols=(1 << 24) + 8),
                   dict(finished=1024 + 23), dict(lengths=2048, out_lengths=2048), dict(out_finished=256 - 5),
                   dict(out_symbols=(1 << 24) + 4 * (5 * 40_000 + 39_999))):
        assert "overlap" in _refused("leo_beam_select", ctypes.byref(native.LeoBeams(**{**good, **change})), None)
    size = ctypes.c_uint64()
    for sizes in ((1, 65, 1, 5), (1, 1, 65, 5), (1 << 17, 1, 1, 5), (1, 1, 1, 0)):
        _refused("leo_beam_workspace_bytes", *sizes, ctypes.byref(size))


def _reorder(listed, **more):
    entries = (native.LeoStateArray * max(1, len(listed)))(*[native.LeoStateArray(**a) for a in listed])
    args = {**dict(arrays=ctypes.addressof(entries), count=len(listed), groups=2, beams=4, kept=4, parents=256), **more}
    return native.LeoReorder(**args), entries


def _array(source, target, width=64, outer=1, row=64, piece=64, **more):
    return {**dict(source=source, target=target, outer=outer, width=width, source_row=row, source_outer=piece,
                   target_row=row, target_outer=piece), **more}


def test_bad_reorderings_are_refused():
    one = _array(1 << 20, 1 << 21)
    for more in (dict(beams=0), dict(beams=65), dict(kept=0), dict(kept=65), dict(groups=1 << 17), dict(parents=None),
                 dict(arrays=None), dict(count=1 << 20)):
        args, _ = _reorder([one], **more)
        _refused("leo_reorder_states", ctypes.byref(args), None)
    for change in (dict(source=None), dict(target=None), dict(source_row=-1), dict(target_outer=-64), dict(width=1 << 50),
                   dict(outer=1 << 40), dict(target_row=63), dict(outer=2, target_outer=63), dict(outer=2, target_row=64),
                   dict(target_row=1 << 50)):
        args, _ = _reorder([{**one, **change}])
        _refused("leo_reorder_states", ctypes.byref(args), None)
    # an array that is its own target: the same strides, and as many kept
    args, _ = _reorder([_array(1 << 20, 1 << 20, target_row=128)])
    assert "own target" in _refused("leo_reorder_states", ctypes.byref(args), None)
    args, _ = _reorder([_array(1 << 20, 1 << 20)], kept=3)
    assert "own target" in _refused("leo_reorder_states", ctypes.byref(args), None)


def _meets(arrays, **more):
    args, _ = _reorder(arrays, **more)
    return "overlaps another array" in _refused("leo_reorder_states", ctypes.byref(args), None)


def test_targets_that_overlap_are_refused():
    at = 1 << 20
    assert _meets([_array(at, at + 32)])                                      # by half a row
    assert _meets([_array(at, at + 8 * 64 - 1)])                              # by one byte at the end
    assert _meets([_array(at, 1 << 21), _array(1 << 22, at)])                 # another array's source
    assert _meets([_array(at, 1 << 21), _array(1 << 22, (1 << 21) + 64)])     # another target
    assert _meets([_array(at, at), _array(at, 1 << 21)])                      # a source that is reordered in place
    # columns of one buffer, one byte too wide, in rows and in pieces of rows
    assert _meets([_array(at, at, row=128, width=65), _array(at + 64, at + 64, row=128, width=64)])
    assert _meets([_array(at, at, row=1024, outer=8, piece=128, width=65),
                   _array(at + 64, at + 64, row=1024, outer=8, piece=128, width=64)])
    # what wraps round the common divisor
    assert _meets([_array(at + 100, at + 100, row=128, width=40), _array(at + 128, at + 128, row=128, width=40)])


def test_targets_over_the_parents_are_refused():
    args, _ = _reorder([_array(1 << 20, 256 + 31)])
    assert "parents" in _refused("leo_reorder_states", ctypes.byref(args), None)


def test_nothing_to_reorder_is_no_error():
    lib = native.load()
    for args, _ in (_reorder([]), _reorder([_array(1 << 20, 1 << 21)], groups=0), _reorder([_array(1 << 20, 1 << 21, width=0)])):
        assert lib.leo_reorder_states(ctypes.byref(args), None) == native.OK
    beams = native.LeoBeams(groups=0, beams=1, kept=1, symbols=1)
    assert lib.leo_beam_select(ctypes.byref(beams), None) == native.OK
    product = native.LeoQ8Product(shape=native.LeoQ8Shape(outputs=1, inputs=1), rows=0)
    assert lib.leo_q8_matmul(ctypes.byref(product), None) == native.OK
