"""Positions with several axes, positions of their own for appended tokens, and
tokens read back, without a GPU: plans, argument structs, and what every call
refuses before any device work."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from kunlunxin_fft_amd import (PagedCache, RotaryAxes, RotaryScaling, append_paged_cache, execute_rotary_plan, native,
                               plan_rotary, read_paged_cache)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I32 = dict(dtype=torch.int32)


def test_blocks_on_a_shared_ladder():
    plan = plan_rotary(16, axes=RotaryAxes((2, 3, 3)))
    assert plan.axis_of == (0, 0, 1, 1, 1, 2, 2, 2) and plan.axes == 3
    assert plan.frequencies == plan_rotary(16).frequencies
    assert plan is plan_rotary(16, axes=RotaryAxes((2, 3, 3))) and plan is not plan_rotary(16)


def test_cycle_leaves_out_axes_that_are_done():
    plan = plan_rotary(16, axes=RotaryAxes((2, 5, 1), order="cycle", ladder="own"))
    assert plan.axis_of == (0, 1, 2, 0, 1, 1, 1, 1)
    places = (0, 0, 0, 1, 1, 2, 3, 4)
    want = [10000.0 ** (-i / (2, 5, 1)[a]) for a, i in zip(plan.axis_of, places)]
    assert plan.frequencies == pytest.approx(want, rel=1e-14)


def test_a_ladder_of_its_own_is_that_of_a_head_of_its_own():
    plan = plan_rotary(64, base=100.0, axes=RotaryAxes((16, 16), ladder="own"))
    assert plan.frequencies == plan_rotary(32, base=100.0).frequencies * 2


@pytest.mark.parametrize("kind", ["linear", "base", "parts"])
def test_scalings_go_by_each_pair(kind):
    scaling = RotaryScaling(kind, 4.0, 4096 if kind == "parts" else 0)
    shared = plan_rotary(64, scaling=scaling, axes=RotaryAxes((8, 12, 12), "cycle"))
    assert shared.frequencies == plan_rotary(64, scaling=scaling).frequencies
    own = plan_rotary(64, scaling=scaling, axes=RotaryAxes((16, 16), ladder="own"))
    assert own.frequencies == plan_rotary(32, scaling=scaling).frequencies * 2


def test_without_axes_positions_are_numbers():
    assert plan_rotary(64).axes == 0 and plan_rotary(64).axis_of == ()
    assert plan_rotary(64, axes=RotaryAxes((32,))).axes == 1


@pytest.mark.parametrize("axes,error", [
    ((8, 24), TypeError), (RotaryAxes((8, 23)), ValueError), (RotaryAxes(()), ValueError), (RotaryAxes((0, 32)), ValueError),
    (RotaryAxes((33, -1)), ValueError), (RotaryAxes((8, 8, 8, 4, 4)), ValueError),
    (RotaryAxes((8, 24), order="rows"), ValueError), (RotaryAxes((8, 24), ladder="each"), ValueError),
], ids=str)
def test_plan_refuses(axes, error):
    with pytest.raises(error):
        plan_rotary(64, axes=axes)


@pytest.mark.parametrize("pairs", [(8.0, 24.0), (True, 31), [8, 24], 32, "ab"], ids=str)
def test_axes_are_a_tuple_of_ints(pairs):
    plan_rotary(64, axes=RotaryAxes((8, 24)))
    plan_rotary(64, axes=RotaryAxes((1, 31)))
    with pytest.raises(TypeError, match="tuple of ints"):  # and never the plan of equal numbers
        plan_rotary(64, axes=RotaryAxes(pairs))


def test_base_scaling_needs_two_pairs_of_an_axis():
    with pytest.raises(ValueError, match="two pairs"):
        plan_rotary(64, scaling=RotaryScaling("base", 4.0), axes=RotaryAxes((1, 31), ladder="own"))
    plan_rotary(64, scaling=RotaryScaling("base", 4.0), axes=RotaryAxes((1, 31)))


@pytest.mark.parametrize("shape", [(3,), (2, 3), (3, 4), (3, 1, 3), (1, 3, 3)], ids=str)
def test_rotary_refuses_positions_of_other_shapes(shape):
    plan = plan_rotary(64, axes=RotaryAxes((8, 12, 12)))
    with pytest.raises(ValueError, match=r"\(3, 3\).*3 axes"):
        execute_rotary_plan(plan, torch.zeros(3, 2, 64), torch.zeros(shape, **I32))


def test_rotary_refuses_batches_of_other_shapes():
    plan = plan_rotary(64, axes=RotaryAxes((8, 24)))
    for shape in ((2, 4, 3), (2, 3, 2), (5,), (4, 5)):
        with pytest.raises(ValueError, match="positions"):
            execute_rotary_plan(plan, torch.zeros(4, 5, 2, 64), torch.zeros(shape, **I32))


AXES = plan_rotary(64, axes=RotaryAxes((8, 24)))


@pytest.mark.parametrize("kw,error,text", [
    (dict(rotary=AXES), ValueError, "2 axes"), (dict(positions=torch.zeros(3, **I32)), ValueError, "give rotary"),
    (dict(rotary=AXES, positions=torch.zeros(3, **I32)), ValueError, "shape"),
    (dict(rotary=AXES, positions=torch.zeros(2, 4, **I32)), ValueError, "shape"),
    (dict(rotary=AXES, positions=torch.zeros(2, 3)), TypeError, "int32 or int64"),
    (dict(rotary=AXES, positions=[1, 2, 3]), TypeError, "Tensor"),
    (dict(rotary=plan_rotary(64), positions=torch.zeros(2, 3, **I32)), ValueError, "shape"),
    (dict(rotary=AXES, positions=torch.zeros(2, 3, device="meta", **I32)), ValueError, "like the cache"),
], ids=str)
def test_append_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        append_paged_cache(PagedCache.empty(4, 2, 64, 16, device="cpu"), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64),
                           torch.zeros(3, 2, **I32), torch.zeros(3, **I32), **kw)


def _read(**change):
    kw = dict(cache=PagedCache.empty(4, 2, 64, 16, device="cpu"), page_table=torch.zeros(3, 2, **I32),
              starts=torch.zeros(3, **I32), tokens=6)
    return read_paged_cache(**{**kw, **change})


@pytest.mark.parametrize("change,error", [
    (dict(cache=None), TypeError), (dict(page_table=torch.zeros(3, 2)), TypeError), (dict(page_table=torch.zeros(3, 0, **I32)), ValueError),
    (dict(starts=torch.zeros(2, **I32)), ValueError), (dict(starts=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(tokens=6.0), TypeError), (dict(tokens=True), TypeError), (dict(tokens=torch.tensor(6)), TypeError), (dict(tokens=-1), ValueError),
    (dict(tokens=1 << 31), ValueError), (dict(tokens=7), ValueError), (dict(offsets=torch.zeros(3, **I32)), ValueError),
    (dict(offsets=torch.zeros(4)), TypeError), (dict(dtype=torch.float64), TypeError), (dict(dtype="bf16"), TypeError),
], ids=str)
def test_read_refuses(change, error):
    with pytest.raises(error):
        _read(**change)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the refusal of a machine without a GPU")
def test_no_gpu_is_an_error():
    with pytest.raises(RuntimeError, match="GPU"):
        _read()


def header_layout(tmp_path, name):
    """(size, [(field, offset, values)]) of a struct of the C header, by a C compiler."""
    src = open(os.path.join(ROOT, "include", "mfft.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct \{([^{}]*)\} " + name + ";", src).group(1), flags=re.S)
    fields = []
    for decl in body.split(";"):
        for f in re.sub(r"^\s*(const\s+)?\w+\s*", "", decl.strip()).split(",") if decl.strip() else ():
            m = re.match(r"[*\s]*(\w+)(?:\[(\d+)\])?", f.strip())
            fields.append((m.group(1), int(m.group(2) or 1)))
    c = '#include <stdio.h>\n#include <stddef.h>\n#include "mfft.h"\nint main(void) {\n' + f'printf("%zu\\n", sizeof({name}));\n'
    c += "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f, _ in fields)
    (tmp_path / "s.c").write_text(c + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    size, *at = map(int, subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split())
    return size, [(f, o, n) for (f, n), o in zip(fields, at)]


def check_layout(tmp_path, name, st):
    size, fields = header_layout(tmp_path, name)
    assert st.size == size
    total, at = sum(n for _, _, n in fields), 0
    for f, offset, n in fields:
        values = [0] * total
        values[at] = 1
        assert st.pack(*values).index(1) == offset, f
        at += n
    assert len(st.unpack(bytes(size))) == total


def test_read_struct_matches_the_header(tmp_path):
    check_layout(tmp_path, "mfft_read_args", native.READ_ARGS)


def test_c_entries_refuse_before_device_work():
    """The C entries' own checks (made-up addresses, never touched)."""
    lib = native.load()
    p = 1 << 20
    cache = native.CACHE_ARGS.pack(p, p + (1 << 18), p, p, 4, 2, 64, 16)
    good = [p << 10, p << 11, 128, 64, 128, 64, p, p, 0, 2, 6, 2, 3, native.F16]
    for i, value, rc, text in ((13, 7, native.ERR_TYPE, b"type"), (10, 7, native.ERR_VALUE, b"as many"), (10, -1, native.ERR_VALUE, b"tokens"),
                               (12, 0, native.ERR_VALUE, b"sequences"), (11, 0, native.ERR_VALUE, b"column"), (6, 0, native.ERR_VALUE, b"NULL"),
                               (7, 0, native.ERR_VALUE, b"NULL"), (8, p + 1, native.ERR_VALUE, b"offsets"), (2, -1, native.ERR_VALUE, b"stride"),
                               (2, 132, native.ERR_VALUE, b"aligned"), (0, (p << 10) + 8, native.ERR_VALUE, b"aligned"), (1, 0, native.ERR_VALUE, b"NULL"),
                               (2, 64, native.ERR_VALUE, b"overlap"), (1, p << 10, native.ERR_VALUE, b"overlap"), (0, p + 64, native.ERR_VALUE, b"overlap")):
        v = list(good)
        v[i] = value
        assert lib.mfft_cache_read(cache, native.READ_ARGS.pack(*v), None) == rc, (i, value)
        assert text in lib.mfft_last_error(), (i, value, lib.mfft_last_error())
    assert lib.mfft_cache_read(None, None, None) == native.ERR_VALUE
    assert lib.mfft_cache_read(cache, None, None) == native.ERR_VALUE
    assert lib.mfft_rotary_execute_axes(None, None, 0, None) == native.ERR_VALUE
    assert lib.mfft_cache_append_at(cache, None, None, p, 0, 1, 0, None) == native.ERR_VALUE


def test_create_axes_refuses():
    lib = native.load()
    h = ctypes.c_void_p()
    f = (ctypes.c_double * 2)(1.0, 0.5)

    def axis(*v):
        return (ctypes.c_int32 * len(v))(*v)

    for args, text in (((f, axis(0, 2), 2, 2, 1024, 1.0, 0), b"axis_of"), ((f, axis(-1, 0), 2, 2, 1024, 1.0, 0), b"axis_of"),
                       ((f, None, 2, 2, 1024, 1.0, 0), b"axis_of"), ((f, axis(0, 0), 2, 0, 1024, 1.0, 0), b"axes"),
                       ((f, axis(0, 0), 2, 5, 1024, 1.0, 0), b"axes"), ((f, axis(0, 0), 0, 1, 1024, 1.0, 0), b"pairs")):
        assert lib.mfft_rotary_create_axes(ctypes.byref(h), *args) == native.ERR_VALUE and not h.value
        assert text in lib.mfft_last_error()
