"""Refusals of the beam search calls that need no GPU: the C ABI checks every argument before it looks
at a device, so addresses that are never read do for buffers."""
import ctypes

import pytest
import torch  # noqa: F401  before the library: a process has one HIP runtime, and torch brings its own

import radx_amd
from radx_amd import capi

BASE = 0x7f0000000000


def refused(code, text):
    assert code == 1, code  # hipErrorInvalidValue
    got = capi.lib.radx_hip_error_string().decode()
    assert text in got, got


def select_args(**change):
    a = dict(logits=BASE, row_stride=1000, cum=BASE + (1 << 30), allowed=None, allowed_stride=0, finished=None, scores=BASE + (2 << 30),
             parents=BASE + (3 << 30), tokens=BASE + (4 << 30), out_finished=None, batch=2, beams=4, vocab=1000, k=8, dtype=1, normalize=1,
             end_token=0)
    a.update(change)
    return capi.BEAM_SELECT_ARGS.pack(*(value or 0 for value in a.values()))


@pytest.mark.parametrize("change,text", [
    (dict(beams=0), "beams"), (dict(beams=65), "beams"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1), "vocab"),
    (dict(batch=1 << 20, beams=8), "batch x beams"), (dict(k=0), "k must"), (dict(k=129), "k must"), (dict(batch=(1 << 20) + 1), "batch"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
    (dict(logits=None), "NULL"), (dict(cum=None), "NULL"), (dict(scores=None), "NULL"), (dict(parents=None), "NULL"), (dict(tokens=None), "NULL"),
    (dict(row_stride=999), "row_stride"), (dict(row_stride=1 << 41), "stride out of range"), (dict(row_stride=(1 << 36) + 1), "stride out of range"),
    (dict(allowed=BASE + (5 << 30), allowed_stride=31), "allowed_stride"),
    (dict(finished=BASE + (5 << 30)), "go together"), (dict(out_finished=BASE + (5 << 30)), "go together"),
    (dict(finished=BASE + (5 << 30), out_finished=BASE + (6 << 30), end_token=-1), "end_token"),
    (dict(finished=BASE + (5 << 30), out_finished=BASE + (6 << 30), end_token=1000), "end_token"),
    (dict(logits=BASE + 1), "aligned"), (dict(cum=BASE + (1 << 30) + 2), "aligned"), (dict(tokens=BASE + (4 << 30) + 2), "aligned"),
    (dict(scores=BASE + (1 << 30)), "an output overlaps an input"), (dict(tokens=BASE + 15996), "an output overlaps an input"),
    (dict(tokens=BASE + (3 << 30) + 60), "two outputs overlap"),
    (dict(finished=BASE + (5 << 30), out_finished=BASE + (5 << 30), end_token=0), "an output overlaps an input"),
    (dict(), "handle is NULL"), (dict(row_stride=0), "handle is NULL"), (dict(allowed=BASE + (5 << 30), allowed_stride=0), "handle is NULL"),
])
def test_select_refuses(change, text):
    refused(capi.lib.radx_hip_beam_select(None, select_args(**change), None), text)


def test_an_empty_batch_is_no_error():
    assert capi.lib.radx_hip_beam_select(None, select_args(batch=0), None) == 0
    assert capi.lib.radx_hip_beam_reorder(None, 0, None, None, 0, 4, 4, 4, None) == 0
    assert capi.lib.radx_hip_beam_backtrace(None, None, None, 0, 2, 4, None, 0, None) == 0
    assert capi.lib.radx_hip_beam_destroy(None) == 0


def test_create_refuses_limits():
    h = ctypes.c_void_p(None)
    for limits, text in (((0, 4, 100, 8), "batch"), ((1, 65, 100, 8), "beams"), ((1, 4, 0, 8), "vocab"), ((1, 4, 100, 129), "k must")):
        refused(capi.lib.radx_hip_beam_create(0, *limits, ctypes.byref(h)), text)
        assert capi.lib.radx_hip_beam_scratch_bytes(*limits) == 0
    refused(capi.lib.radx_hip_beam_create(0, 1, 1, 1, 1, None), "out is NULL")
    assert 0 < capi.lib.radx_hip_beam_scratch_bytes(1, 1, 1, 1) < capi.lib.radx_hip_beam_scratch_bytes(64, 8, 131072, 16) < 1 << 24


def state(**change):
    s = dict(src=BASE, dst=BASE, src_row=4096, dst_row=4096, src_outer=(0, 0), dst_outer=(0, 0), unit_bytes=64, units=64, outer=(1, 1))
    s.update(change)
    flat = []
    for value in s.values():
        flat += value if isinstance(value, tuple) else [value or 0]
    return capi.BEAM_STATE.pack(*flat)


def reorder(states, batch=2, src=4, dst=4, k=4, parents=BASE + (1 << 30)):
    return capi.lib.radx_hip_beam_reorder(b"".join(states), len(states), parents, None, batch, src, dst, k, None)


def test_struct_formats_are_the_headers(tmp_path):
    """The packed formats are the C structs, field by field."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = ["logits", "row_stride", "cum", "allowed", "allowed_stride", "finished", "scores", "parents", "tokens", "out_finished", "batch",
              "beams", "vocab", "k", "dtype", "normalize", "end_token"]
    state_fields = ["src", "dst", "src_row", "dst_row", "src_outer", "dst_outer", "unit_bytes", "units", "outer"]
    lines = ["offsetof(radx_hip_beam_select_args, %s)" % f for f in fields] + ["sizeof(radx_hip_beam_select_args)"]
    lines += ["offsetof(radx_hip_beam_state, %s)" % f for f in state_fields] + ["sizeof(radx_hip_beam_state)"]
    src = tmp_path / "o.c"
    src.write_text('#include <stdio.h>\n#include "radx_hip.h"\nint main(void) {' + "".join('printf("%%zu\\n", %s);' % e for e in lines) + "return 0; }\n")
    subprocess.run(["gcc", "-I" + os.path.join(root, "include"), "-o", str(tmp_path / "o"), str(src)], check=True, timeout=60)
    got = [int(v) for v in subprocess.run([str(tmp_path / "o")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [8 * i for i in range(10)] + [80 + 4 * i for i in range(7)] + [capi.BEAM_SELECT_ARGS.size] + \
        [0, 8, 16, 24, 32, 48, 64, 72, 80] + [capi.BEAM_STATE.size]


@pytest.mark.parametrize("change,text", [
    (dict(src=None), "NULL"), (dict(dst=None), "NULL"), (dict(src_row=8192), "two layouts"), (dict(dst_row=4095, src_row=4095), "rows overlap"),
    (dict(dst=BASE + 4096), "source and destination overlap"), (dict(dst=BASE + 8 * 4096 - 1), "source and destination overlap"),
    (dict(units=1 << 41), "too long"), (dict(units=1 << 30, src_row=1 << 37, dst_row=1 << 37), "too long for one call"), (dict(unit_bytes=1 << 30, units=1 << 30), "too long"), (dict(src_row=1 << 41, dst_row=1 << 41), "out of range"),
    (dict(outer=(1 << 13, 1 << 12)), "pieces"), (dict(outer=(2, 1), src_outer=(100, 0), dst_outer=(100, 0)), "pieces overlap"),
    (dict(outer=(2, 1), src_outer=(4096, 0), dst_outer=(4096, 0)), "rows and pieces overlap"),
    (dict(outer=(2, 1), src_outer=(6144, 0), dst_outer=(6144, 0)), "rows and pieces overlap"),
    (dict(outer=(3, 2), src_outer=(4096, 8192), dst_outer=(4096, 8192), src_row=1 << 16, dst_row=1 << 16), "rows and pieces overlap"),
    (dict(outer=(2, 1), src_outer=(1 << 41, 0), dst_outer=(1 << 41, 0)), "out of range"),
    (dict(outer=(2, 1), src_outer=(8192, 0), dst_outer=(4096, 0)), "two layouts"),
])
def test_reorder_refuses_states(change, text):
    refused(reorder([state(**change)]), text)


def test_reorder_refuses_calls():
    refused(reorder([state()], k=0), "k must")
    refused(reorder([state()], k=65, dst=65), "k must")
    refused(reorder([state()], k=5), "exceeds the rows")
    refused(reorder([state()], src=0), "beams")
    refused(reorder([state()], batch=65536), "batch")
    refused(reorder([state()], batch=1 << 10, src=1 << 15, dst=1 << 15), "2^24 rows")
    refused(reorder([state()], parents=None), "NULL")
    refused(reorder([state()], parents=BASE + 2), "aligned")
    refused(reorder([state(), state()]), "written twice")
    refused(reorder([state(dst=BASE + (1 << 28)), state(src=BASE + (1 << 28), dst=BASE + (1 << 29))]), "written twice, or read and written")
    refused(reorder([state()], src=5), "two layouts")
    assert reorder([state(units=0, src=None, dst=None)], batch=0) == 0


def test_backtrace_refuses():
    def call(tokens=BASE, parents=BASE + (1 << 30), steps=None, total=10, batch=2, k=4, out=BASE + (2 << 30), stride=10):
        return capi.lib.radx_hip_beam_backtrace(tokens, parents, steps, total, batch, k, out, stride, None)
    refused(call(k=0), "k must")
    refused(call(k=129), "k must")
    refused(call(batch=65536), "batch")
    refused(call(total=1 << 24), "total_steps")
    refused(call(tokens=None), "NULL")
    refused(call(parents=None), "NULL")
    refused(call(out=None), "NULL")
    refused(call(stride=9), "out_stride")
    refused(call(stride=(1 << 36) + 1), "out_stride")
    refused(call(tokens=BASE + 1), "aligned")
    refused(call(out=BASE + 316), "out overlaps")
    refused(call(steps=BASE + (2 << 30)), "out overlaps")


def test_the_c_plus_plus_layer_compiles():
    """harness/beam_test.cpp drives include/radx/radx_beam.hpp; tests/test_gpu_beam.py runs it."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    made = subprocess.run(["make", "-C", root, "-W", "harness/beam_test.cpp", "harness/beam_test"], capture_output=True, text=True, timeout=600)
    assert made.returncode == 0, made.stdout + made.stderr
    assert "warning" not in made.stderr, made.stderr


def test_host_tensors_are_refused():
    import torch
    with pytest.raises(ValueError, match="device tensor"):
        radx_amd.beam_reorder(torch.zeros(4, 8), torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="device tensor"):
        radx_amd.beam_backtrace(torch.zeros(3, 1, 4, dtype=torch.int32), torch.zeros(3, 1, 4, dtype=torch.int32))


@pytest.mark.parametrize("shape,order,row_dim,length_dim,want", [
    # [rows, heads, positions, width]: a piece for each head, a position is 16 elements
    ((8, 3, 5, 16), (0, 1, 2, 3), 0, 2, (480, (3, 160), 32, 5)),
    # [rows, positions, heads, width]: one piece
    ((8, 5, 3, 16), (0, 1, 2, 3), 0, 1, (480, (1, 0), 96, 5)),
    ((8, 5, 3, 16), (0, 1, 2, 3), 0, None, (480, (1, 0), 480, 1)),
    # [layers, rows, positions, width]: the layers are pieces
    ((4, 8, 5, 16), (0, 1, 2, 3), 1, 2, (160, (4, 1280), 32, 5)),
])
def test_rows_are_cut_into_pieces(shape, order, row_dim, length_dim, want):
    import torch
    from radx_amd.beam import _pieces
    t = torch.zeros(shape, dtype=torch.bfloat16).permute(order)
    src_row, dst_row, src_outer, dst_outer, outer, unit, units = _pieces(t.shape, t.stride(), t.stride(), 2, row_dim, length_dim)
    assert src_row == dst_row == want[0] and src_outer == dst_outer
    assert (outer[1], src_outer[1]) == want[1] and outer[0] == 1
    assert (unit, units) == want[2:]


def test_scattered_rows_are_refused():
    import torch
    from radx_amd.beam import _pieces
    t = torch.zeros(8, 3, 4, 5, 16)[:, :2, :3, :4, :15]
    with pytest.raises(ValueError, match="scattered"):
        _pieces(t.shape, t.stride(), t.stride(), 4, 0, None)
    t = torch.zeros(8, 3, 5, 16)[:, :, :, :15]
    with pytest.raises(ValueError, match="contiguous"):
        _pieces(t.shape, t.stride(), t.stride(), 4, 0, 2)
