"""The language-model operators without a GPU: rotary plans, the argument
structs' layout, and what every call refuses before any device work."""
import os
import re
import subprocess

import pytest
import torch

from kunlunxin_fft_amd import (PagedCache, RotaryScaling, append_paged_cache, attend_paged_cache, execute_rotary_plan,
                               native, plan_rotary)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plans_are_memoised_and_host_only():
    a = plan_rotary(128, base=500000.0)
    assert a is plan_rotary(128, base=500000.0) and a is not plan_rotary(128)
    assert a.rot_dim == 128 and len(a.frequencies) == 64 and a.frequencies[0] == 1.0


@pytest.mark.parametrize("args,kw,error", [
    ((127,), {}, ValueError), ((0,), {}, ValueError), ((128.0,), {}, TypeError), ((128,), {"rot_dim": 3}, ValueError),
    ((128,), {"rot_dim": 130}, ValueError), ((1024,), {}, ValueError), ((128,), {"layout": "pairs"}, ValueError),
    ((128,), {"base": 0.0}, ValueError), ((128,), {"base": float("inf")}, ValueError), ((128,), {"base": "e"}, TypeError),
    ((128,), {"max_positions": 0}, ValueError), ((128,), {"max_positions": (1 << 24) + 1}, ValueError),
    ((128,), {"scaling": 4.0}, TypeError), ((128,), {"scaling": RotaryScaling("cubic", 2.0)}, ValueError),
    ((128,), {"scaling": RotaryScaling("linear", 0.0)}, ValueError),
    ((128,), {"scaling": RotaryScaling("parts", 4.0)}, ValueError),
    ((128,), {"scaling": RotaryScaling("parts", 4.0, 4096, 32.0, 1.0)}, ValueError),
    ((2,), {"scaling": RotaryScaling("base", 4.0)}, ValueError),
])
def test_plan_rotary_refuses(args, kw, error):
    with pytest.raises(error):
        plan_rotary(*args, **kw)


def test_argument_structs_match_the_header(tmp_path):
    """Sizes and offsets of the packed structs against a C compiler's."""
    src = open(os.path.join(ROOT, "include", "mfft.h")).read()
    fields = {}
    for body, name in re.findall(r"typedef struct \{([^{}]*)\} (mfft_(?:rotary_args|cache|append_args|attend_args));", src, re.S):
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields[name] = [re.sub(r"\[.*", "", f.strip().lstrip("*")) for decl in body.split(";") if decl.strip()
                        for f in re.sub(r"^\s*(const\s+)?\w+\s*", "", decl.strip()).split(",")]
    assert set(fields) == {"mfft_rotary_args", "mfft_cache", "mfft_append_args", "mfft_attend_args"}
    c = '#include <stdio.h>\n#include <stddef.h>\n#include "mfft.h"\nint main(void) {\n'
    for name, fs in fields.items():
        c += f'printf("{name} %zu", sizeof({name}));\n'
        c += "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fs) + 'printf("\\n");\n'
    (tmp_path / "s.c").write_text(c + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = dict((line.split()[0], [int(x) for x in line.split()[1:]])
               for line in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.splitlines())
    arrays = {"in_strides": 3, "out_strides": 3, "position_strides": 2}
    for name, st in (("mfft_rotary_args", native.ROTARY_ARGS), ("mfft_cache", native.CACHE_ARGS),
                     ("mfft_append_args", native.APPEND_ARGS), ("mfft_attend_args", native.ATTEND_ARGS)):
        assert got[name][0] == st.size, name
        # the byte at which each field's first value lands
        n = {f: (arrays.get(f, 2) if name == "mfft_rotary_args" else 2) if f.endswith("strides") else 1
             for f in fields[name]}
        total = sum(n.values())
        at = 0
        for f, off in zip(fields[name], got[name][1:]):
            values = [0] * total
            values[at] = 1
            packed = st.pack(*values)
            first = next(i for i, v in enumerate(packed) if v)
            # 1.0f has its first nonzero byte third
            assert first == off + (2 if f == "scale" else 0), (name, f)
            at += n[f]


def _cache(pages=4, heads=2, size=16, dim=64):
    return PagedCache.empty(pages, heads, dim, size, device="cpu")


def _codes(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


@pytest.mark.parametrize("change,error", [
    (dict(k=torch.zeros(4, 2, 16, 64)), TypeError), (dict(k="k"), TypeError),
    (dict(k=_codes(4, 2, 16)), ValueError), (dict(k=_codes(4, 2, 24, 64)), ValueError),
    (dict(k=_codes(4, 2, 16, 80)), ValueError), (dict(v=_codes(4, 2, 16, 64)), ValueError),
    (dict(v=_codes(4, 2, 1, 16, 64).transpose(3, 4)), ValueError), (dict(k_scale=torch.zeros(4)), ValueError),
    (dict(v_scale=torch.zeros(4, 2, dtype=torch.float64)), TypeError), (dict(k=_codes(0, 2, 16, 64)), ValueError),
])
def test_cache_refuses(change, error):
    c = _cache()
    with pytest.raises(error):
        PagedCache(**{**dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale), **change})


def test_empty_refuses_page_sizes():
    for size in (0, 8, 17, 1040, 16.0):
        with pytest.raises(ValueError):
            PagedCache.empty(1, 1, 64, size, device="cpu")


I32 = dict(dtype=torch.int32)


def _append(**change):
    kw = dict(cache=_cache(), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), page_table=torch.zeros(3, 2, **I32),
              starts=torch.zeros(3, **I32))
    kw.update(change)
    return append_paged_cache(**kw)


@pytest.mark.parametrize("change,error", [
    (dict(cache=1), TypeError), (dict(k=[1]), TypeError), (dict(k=torch.zeros(3, 2, 64, dtype=torch.float64)), TypeError),
    (dict(v=torch.zeros(3, 2, 64).bfloat16()), TypeError), (dict(k=torch.zeros(3, 1, 64)), ValueError),
    (dict(k=torch.zeros(3, 2, 32)), ValueError), (dict(v=torch.zeros(2, 2, 64)), ValueError),
    (dict(k=torch.zeros(3, 2, 128)[..., ::2]), ValueError), (dict(page_table=torch.zeros(3, 2)), TypeError),
    (dict(page_table=torch.zeros(3, **I32)), ValueError), (dict(page_table=torch.zeros(3, 0, **I32)), ValueError),
    (dict(starts=torch.zeros(2, **I32)), ValueError), (dict(starts=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(offsets=torch.zeros(3, **I32)), ValueError), (dict(offsets=torch.zeros(4)), TypeError),
    (dict(k=torch.zeros(4, 2, 64), v=torch.zeros(4, 2, 64)), ValueError), (dict(q=torch.zeros(2, 2, 64)), ValueError),
    (dict(q=torch.zeros(3, 2, 64).half()), TypeError), (dict(rotary=3), TypeError), (dict(rotary=plan_rotary(128)), ValueError),
])
def test_append_refuses(change, error):
    with pytest.raises(error):
        _append(**change)


def _attend(**change):
    kw = dict(cache=_cache(), q=torch.zeros(3, 4, 64).half(), page_table=torch.zeros(3, 2, **I32),
              lengths=torch.zeros(3, **I32))
    kw.update(change)
    return attend_paged_cache(**kw)


@pytest.mark.parametrize("change,error", [
    (dict(cache=None), TypeError), (dict(q=torch.zeros(3, 4, 64)), TypeError), (dict(q=torch.zeros(3, 3, 64).half()), ValueError),
    (dict(q=torch.zeros(3, 0, 64).half()), ValueError), (dict(q=torch.zeros(3, 4, 96).half()), ValueError),
    (dict(q=torch.zeros(4, 4, 64).half()), ValueError), (dict(lengths=torch.zeros(4, **I32)), ValueError),
    (dict(window=0), ValueError), (dict(window=True), ValueError), (dict(window=2.5), ValueError),
    (dict(max_length=-1), ValueError), (dict(offsets=torch.zeros(3, **I32)), ValueError),
])
def test_attend_refuses(change, error):
    with pytest.raises(error):
        _attend(**change)


@pytest.mark.parametrize("change,error", [
    (dict(plan=1), TypeError), (dict(x=[1]), TypeError), (dict(x=torch.zeros(3, 2, 64, dtype=torch.float64)), TypeError),
    (dict(positions=torch.zeros(3)), TypeError), (dict(x=torch.zeros(3, 64)), ValueError),
    (dict(x=torch.zeros(3, 2, 32)), ValueError), (dict(positions=torch.zeros(2, **I32)), ValueError),
    (dict(x=torch.zeros(3, 2, 128)[..., ::2]), ValueError), (dict(out=torch.zeros(3, 2, 32)), ValueError),
    (dict(out=torch.zeros(3, 2, 64).half()), TypeError),
    (dict(x=torch.zeros(3, 2, 64, requires_grad=True), out=torch.zeros(3, 2, 64)), ValueError),
])
def test_rotary_refuses(change, error):
    kw = dict(plan=plan_rotary(64), x=torch.zeros(3, 2, 64), positions=torch.zeros(3, **I32))
    kw.update(change)
    with pytest.raises(error):
        execute_rotary_plan(**kw)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the refusal of a machine without a GPU")
def test_no_gpu_is_an_error():
    with pytest.raises(RuntimeError, match="GPU"):
        _append()
    with pytest.raises(RuntimeError, match="GPU"):
        _attend()
    with pytest.raises(RuntimeError, match="GPU"):
        execute_rotary_plan(plan_rotary(64), torch.zeros(3, 2, 64), torch.zeros(3, **I32))


def _c(fmt, *values):
    return fmt.pack(*values)


def test_c_entries_refuse_before_device_work():
    """The C entries' own checks (made-up addresses, never touched)."""
    lib = native.load()
    p = 1 << 20
    cache = native.CACHE_ARGS.pack(p, p, p, p, 4, 2, 64, 16)
    att = [p, p << 10, 0, 128, 64, 128, 64, p, p, 0, 2, 3, 2, 3, 2, native.F16, 0.125, 1, 0, 0, 0, 0]

    def attend(**at):
        v = list(att)
        for i, x in at.items():
            v[int(i[1:])] = x
        return lib.mfft_cache_attend(cache, native.ATTEND_ARGS.pack(*v), None)

    assert lib.mfft_cache_attend(None, None, None) == native.ERR_VALUE
    for change, rc, text in ((dict(i15=native.F32), native.ERR_TYPE, b"type"), (dict(i16=float("nan")), native.ERR_VALUE, b"scale"),
                             (dict(i16=-1.0), native.ERR_VALUE, b"scale"), (dict(i14=3), native.ERR_VALUE, b"multiple"),
                             (dict(i11=4), native.ERR_VALUE, b"as many"), (dict(i13=0), native.ERR_VALUE, b"sequences"),
                             (dict(i12=0), native.ERR_VALUE, b"column"), (dict(i7=0), native.ERR_VALUE, b"NULL"),
                             (dict(i0=p + 2), native.ERR_VALUE, b"aligned"), (dict(i3=100), native.ERR_VALUE, b"aligned"),
                             (dict(i5=0), native.ERR_VALUE, b"overlap"), (dict(i1=p), native.ERR_VALUE, b"overlap"),
                             (dict(i3=-8), native.ERR_VALUE, b"stride"), (dict(i18=-1), native.ERR_VALUE, b"window"),
                             (dict(i19=-1), native.ERR_VALUE, b"max_length")):
        assert attend(**change) == rc, change
        assert text in lib.mfft_last_error(), (change, lib.mfft_last_error())
    for bad, text in (((p, p, p, p, 4, 2, 72, 16), b"head_dim"), ((p, p, p, p, 4, 2, 64, 20), b"page_size"),
                      ((p, p, p, p, 0, 2, 64, 16), b"pages"), ((p, p, p, p, 4, 0, 64, 16), b"kv_heads"),
                      ((p + 8, p, p, p, 4, 2, 64, 16), b"aligned"), ((0, p, p, p, 4, 2, 64, 16), b"NULL")):
        assert lib.mfft_cache_attend(native.CACHE_ARGS.pack(*bad), native.ATTEND_ARGS.pack(*att), None) in (
            native.ERR_VALUE, native.ERR_UNSUPPORTED)
        assert text in lib.mfft_last_error()
    assert lib.mfft_rotary_execute(None, None, None) == native.ERR_VALUE
    assert lib.mfft_rotary_destroy(None) == 0
    assert lib.mfft_cache_append(cache, None, None, None) == native.ERR_VALUE


def test_rotary_create_refuses():
    import ctypes

    lib = native.load()
    h = ctypes.c_void_p()
    f = (ctypes.c_double * 4)(1.0, 0.5, float("nan"), 0.1)
    for args, text in (((f, 0, 1024, 1.0, 0), b"pairs"), ((f, 257, 1024, 1.0, 0), b"pairs"), ((f, 2, 0, 1.0, 0), b"max_positions"),
                       ((f, 2, 1024, float("inf"), 0), b"amplitude"), ((f, 2, 1024, 1.0, 2), b"layout"),
                       ((f, 4, 1024, 1.0, 0), b"frequency"), ((None, 2, 1024, 1.0, 0), b"NULL")):
        assert lib.mfft_rotary_create(ctypes.byref(h), *args) == native.ERR_VALUE and not h.value
        assert text in lib.mfft_last_error()
