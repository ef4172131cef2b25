"""CPU tests of the host side of the grouped and 8-bit calls: what the binding hands to the C entry points, what it refuses
before it hands anything over, and what the C entry points refuse without a context.  No GPU: the library is replaced by a
recorder, and the context's "device" is the one torch reports for CPU tensors."""
import os
import sys

import pytest
import torch

import maize_b200
from maize_b200 import _ffi, build

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


class Recorder:
    """Takes any entry point's place and keeps the arguments of the last call."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return _ffi.OK
        return entry


@pytest.fixture
def ctx():
    sys.modules["maize_b200.gemm"]._types()
    c = maize_b200.Context.__new__(maize_b200.Context)
    c._lib = c._calls = Recorder()
    c._h, c._ctx, c.device = None, None, -1
    given = maize_b200.Context._result
    c._result = lambda out, shape, dtype, stream: (torch.empty(shape, dtype=dtype) if out is None
                                                   else given(c, out, shape, dtype, stream))
    return c


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def offs(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_grouped_arguments(ctx):
    a, b, o = t(10, 32)[:, :16], t(3, 24, 40)[:, :, :16], offs(0, 4, 4, 9)
    out = ctx.grouped_gemm(a, b, o, stream=7)
    name, args = ctx._lib.calls[-1]
    assert name == "maize_grouped_gemm_bf16" and out.shape == (10, 24) and out.dtype == BF16
    assert args == (None, a.data_ptr(), 32, b.data_ptr(), 40, 24 * 40, out.data_ptr(), 24, o.data_ptr(), 3, 10, 24, 16, 7)
    b = t(3, 16, 24)
    out = ctx.grouped_gemm_kn(a, b, o, out=t(10, 30)[:, :24], stream=7)
    name, args = ctx._lib.calls[-1]
    assert name == "maize_grouped_gemm_bf16_kn"
    assert args == (None, a.data_ptr(), 32, b.data_ptr(), 24, 16 * 24, out.data_ptr(), 30, o.data_ptr(), 3, 10, 24, 16, 7)
    dc = t(10, 24)
    out = ctx.grouped_gemm_wgrad(a, dc, o, stream=7)
    name, args = ctx._lib.calls[-1]
    assert name == "maize_grouped_gemm_bf16_wgrad" and out.shape == (3, 24, 16)
    assert args == (None, a.data_ptr(), 32, dc.data_ptr(), 24, out.data_ptr(), 16, 24 * 16, o.data_ptr(), 3, 10, 24, 16, 7)


def test_strides_of_single_rows_do_not_matter(ctx):
    """torch may report any stride for a dimension of one."""
    a = torch.as_strided(t(64), (1, 13), (3, 1))
    b = torch.as_strided(t(128), (1, 13, 8), (1, 8, 1))
    ctx.grouped_gemm_kn(a, b, offs(0, 1), stream=7)
    args = ctx._lib.calls[-1][1]
    assert args[2] == 16 and args[4] == 8  # pitches that the loads can take
    a, s = torch.as_strided(t(64, dtype=F8), (1, 32), (1, 1)), torch.as_strided(t(8, dtype=torch.float32), (1, 1), (5, 1))
    ctx.gemm_e4m3(a, s, a, s, stream=7)
    args = ctx._lib.calls[-1][1]
    assert args[2] == 32 and args[4] == 1 and args[6] == 32 and args[8] == 1


def test_e4m3_arguments(ctx):
    x = t(5, 300)
    q, s = ctx.quantize_e4m3(x, stream=7)
    assert q.shape == (5, 300) and q.dtype == F8 and s.shape == (5, 3) and s.dtype == torch.float32
    assert ctx._lib.calls[-1] == ("maize_quantize_e4m3", (None, x.data_ptr(), 300, 5, 300, 1, q.data_ptr(), 300, s.data_ptr(), 3, 7))
    q, s = ctx.quantize_e4m3(t(300, 129), 128, stream=7)
    assert s.shape == (3, 2)
    a, b, sa, sb = t(5, 272, dtype=F8), t(200, 272, dtype=F8), t(5, 3, dtype=torch.float32), t(2, 3, dtype=torch.float32)
    c = ctx.gemm_e4m3(a, sa, b, sb, stream=7)
    assert ctx._lib.calls[-1] == ("maize_gemm_e4m3", (None, a.data_ptr(), 272, sa.data_ptr(), 3, b.data_ptr(), 272, sb.data_ptr(), 3,
                                                      c.data_ptr(), 200, 5, 200, 272, 7))


def test_refused_before_the_library_is_called(ctx):
    a, b, o, f32 = t(10, 16), t(2, 24, 16), offs(0, 4, 10), torch.float32
    qa, sa, qb, sb = t(10, 256, dtype=F8), t(10, 2, dtype=f32), t(200, 256, dtype=F8), t(2, 2, dtype=f32)
    bad = [
        lambda: ctx.grouped_gemm(a, t(2, 24, 8), o), lambda: ctx.grouped_gemm(a, t(3, 24, 16), o),
        lambda: ctx.grouped_gemm(a, b, o.long()), lambda: ctx.grouped_gemm(a.float(), b, o),
        lambda: ctx.grouped_gemm(a, t(24, 16), o), lambda: ctx.grouped_gemm(t(16, 10).T, b, o),
        lambda: ctx.grouped_gemm(a, b, o, out=t(10, 23)), lambda: ctx.grouped_gemm(a, b, o, out=t(10, 24, dtype=f32)),
        lambda: ctx.grouped_gemm(a, b, torch.stack([o, o], 1)[:, 0]), lambda: ctx.grouped_gemm(a, b, o[None]),
        lambda: ctx.grouped_gemm_kn(a, b, o),
        lambda: ctx.grouped_gemm_wgrad(a, t(9, 24), o), lambda: ctx.grouped_gemm_wgrad(a, t(10, 24), o[:0]),
        lambda: ctx.grouped_gemm_wgrad(a, t(10, 24), o, out=t(2, 16, 24)), lambda: ctx.grouped_gemm_wgrad(a, t(10, 24), o[None]),
        lambda: ctx.quantize_e4m3(a, 64), lambda: ctx.quantize_e4m3(a.float()), lambda: ctx.quantize_e4m3(t(16, 10).T),
        lambda: ctx.quantize_e4m3(a, out=t(10, 16)), lambda: ctx.quantize_e4m3(a, scales=t(10, 2, dtype=f32)),
        lambda: ctx.gemm_e4m3(qa, sa, qb[:, :128], sb), lambda: ctx.gemm_e4m3(qa, sa[:9], qb, sb),
        lambda: ctx.gemm_e4m3(qa, sa, qb, sb[:1]), lambda: ctx.gemm_e4m3(qa.view(torch.uint8), sa, qb, sb),
        lambda: ctx.gemm_e4m3(qa, sa.double(), qb, sb), lambda: ctx.gemm_e4m3(qa, sa, qb, sb, out=t(10, 199)),
    ]
    for call in bad:
        with pytest.raises(maize_b200.MaizeError) as e:
            call()
        assert e.value.status == _ffi.INVALID_ARG
    assert ctx._lib.calls == []


def test_sizes_beyond_the_entry_points_range_are_refused(ctx):
    """The C entry points take 32-bit sizes: 2^32 + 10 rows may not arrive there as ten."""
    many = (1 << 32) + 10
    f32 = torch.float32

    def tall(cols, dtype=BF16):
        return t(1, cols, dtype=dtype).expand(many, cols)

    o = offs(0, 10)
    calls = [
        lambda: ctx.grouped_gemm(tall(16), t(1, 24, 16), o, out=tall(24), stream=7),
        lambda: ctx.grouped_gemm(t(10, 16), t(1, 1, 16).expand(1, many, 16), o, out=t(10, 1).expand(10, many), stream=7),
        lambda: ctx.grouped_gemm_kn(tall(16), t(1, 16, 24), o, out=tall(24), stream=7),
        lambda: ctx.grouped_gemm_wgrad(tall(16), tall(24), o, out=t(1, 24, 16), stream=7),
        lambda: ctx.quantize_e4m3(tall(16), out=tall(16, F8), scales=tall(1, f32), stream=7),
        lambda: ctx.gemm_e4m3(tall(16, F8), tall(1, f32), t(24, 16, dtype=F8), t(1, 1, dtype=f32), out=tall(24), stream=7),
        lambda: ctx.gemm_e4m3(t(10, 16, dtype=F8), t(10, 1, dtype=f32), tall(16, F8),
                              t(1, 1, dtype=f32).expand(-(-many // 128), 1), out=t(10, 1).expand(10, many), stream=7),
    ]
    for call in calls:
        with pytest.raises(maize_b200.MaizeError) as e:
            call()
        assert e.value.status == _ffi.UNSUPPORTED
    assert ctx._lib.calls == []


def test_results_are_allocated_on_the_contexts_device(ctx, monkeypatch):
    """The short way to a new tensor gives one of the current device: it is taken only where that is the context's."""
    gemm = sys.modules["maize_b200.gemm"]
    asked = []
    monkeypatch.setattr(gemm, "_empty", lambda shape, strides, dtype: asked.append((shape, strides, dtype)))
    monkeypatch.setattr(gemm, "_current_device", lambda: 1)
    monkeypatch.setattr(gemm, "_devices", (torch.device("cpu"), torch.device("cpu")))
    result = maize_b200.Context._result
    ctx.device = 0
    assert result(ctx, None, (3, 5), BF16, None).shape == (3, 5) and asked == []
    ctx.device = 1
    result(ctx, None, (3, 5), F8, None)
    result(ctx, None, (2, 3, 5), BF16, None)
    assert asked == [((3, 5), (5, 1), F8), ((2, 3, 5), (15, 5, 1), BF16)]
    for shape in ((0, 5), (3, 0), (2, 0, 5)):
        out = result(ctx, None, shape, BF16, None)
        assert out.shape == shape and out.is_contiguous()
    assert len(asked) == 2
    monkeypatch.setattr(gemm, "_empty", None)
    assert result(ctx, None, (3, 5), BF16, None).shape == (3, 5)


@pytest.mark.parametrize("fault", ["signature", "shape", "strides", "dtype", "none"])
def test_an_undocumented_allocation_is_tried_before_it_is_used(ctx, monkeypatch, fault):
    """A torch that keeps the name of the short way to a new tensor but not what it does: results come by torch.empty."""
    gemm = sys.modules["maize_b200.gemm"]
    asked = []

    def other(shape, strides, dtype):
        asked.append(shape)
        if fault == "signature":
            raise TypeError("takes 2 positional arguments but 3 were given")
        shape, strides = ((5, 3), (3, 1)) if fault == "shape" else (shape, (1, shape[0]) if fault == "strides" else strides)
        return torch.empty_strided(shape, strides, dtype=torch.float32 if fault == "dtype" else dtype)

    monkeypatch.setattr(gemm, "_empty", gemm._on_trial(other))
    monkeypatch.setattr(gemm, "_current_device", lambda: -1)  # as CPU tensors have it
    monkeypatch.setattr(gemm, "_devices", (torch.device("cpu"),))
    for _ in range(3):
        out = maize_b200.Context._result(ctx, None, (3, 5), BF16, None)
        assert out.shape == (3, 5) and out.is_contiguous() and out.dtype is BF16
    assert len(asked) == (3 if fault == "none" else 1) and gemm._empty is (other if fault == "none" else None)


def test_module_functions_refuse_cpu_tensors():
    a = t(4, 16)
    for call in (lambda: maize_b200.grouped_gemm(a, t(1, 8, 16), offs(0, 4)), lambda: maize_b200.quantize_e4m3(a),
                 lambda: maize_b200.grouped_gemm_wgrad(a, a, offs(0, 4)),
                 lambda: maize_b200.gemm_e4m3(a.to(F8), t(4, 1), a.to(F8), t(1, 1))):
        with pytest.raises(maize_b200.MaizeError) as e:
            call()
        assert e.value.status == _ffi.INVALID_ARG


def test_null_context_is_rejected():
    lib = _ffi.load()
    assert lib.maize_grouped_gemm_bf16(None, None, 8, None, 8, 64, None, 8, None, 1, 1, 8, 8, None) == _ffi.INVALID_ARG
    assert lib.maize_grouped_gemm_bf16_kn(None, None, 8, None, 8, 64, None, 8, None, 1, 1, 8, 8, None) == _ffi.INVALID_ARG
    assert lib.maize_grouped_gemm_bf16_wgrad(None, None, 8, None, 8, None, 8, 64, None, 1, 1, 8, 8, None) == _ffi.INVALID_ARG
    assert lib.maize_quantize_e4m3(None, None, 8, 1, 8, 1, None, 8, None, 1, None) == _ffi.INVALID_ARG
    assert lib.maize_gemm_e4m3(None, None, 16, None, 1, None, 16, None, 1, None, 8, 1, 8, 16, None) == _ffi.INVALID_ARG


def test_compiled_calls_agree_with_ctypes():
    """The compiled callables have the entry points' names and give their status codes."""
    lib, calls = _ffi.load(), _ffi.load_calls()
    if calls is lib:
        pytest.skip("built without a C compiler or Python's headers")
    for name in ("maize_grouped_gemm_bf16", "maize_grouped_gemm_bf16_kn", "maize_grouped_gemm_bf16_wgrad", "maize_quantize_e4m3",
                 "maize_gemm_e4m3"):
        count = len(_ffi.SYMBOLS[name][1])
        assert getattr(calls, name)(*[None] * count) == getattr(lib, name)(*[None] + [0] * (count - 1)) == _ffi.INVALID_ARG
        with pytest.raises(TypeError):
            getattr(calls, name)(*[0] * (count - 1))
        with pytest.raises(TypeError):
            getattr(calls, name)(*["0"] * count)


def test_no_read_only_loads_beside_the_kernel_before():
    """A kernel launched with programmatic stream serialization runs while the one before it still writes: none of these may
    read by the read-only path.  The two files that do hold kernels launched in plain stream order."""
    import re
    found = {f.name: len(re.findall(r"\b__ldg\(|ld\.global[.\w:]*\.nc\b", f.read_text())) for f in sorted(build.CSRC.glob("*.cu*"))}
    # the pitch-aligning copy, and the pushes of the multi-GPU path
    assert {name: n for name, n in found.items() if n} == {"gemm_common.cuh": 1, "mc_bcast.cuh": 1}


def compiler(tmp_path, monkeypatch, script):
    """Puts a C compiler of its own in front, and the callables where it may write them."""
    cc = tmp_path / "cc"
    cc.write_text("#!/bin/sh\n" + script)
    cc.chmod(0o755)
    monkeypatch.setattr(build, "CALLS_OUT", tmp_path / "calls.so")
    monkeypatch.setattr(build, "_calls_compiler", lambda: str(cc))
    monkeypatch.setattr(build, "is_stale", lambda: False)
    monkeypatch.setattr(build, "find_nvcc", lambda: pytest.fail("the library is not stale"))
    return build.CALLS_OUT


WRITES_ITS_OUTPUT = 'while [ "$1" != -o ]; do shift; done; echo x > "$2"\n'


def test_a_failing_c_compiler_does_not_stop_the_build(tmp_path, monkeypatch, capsys):
    out = compiler(tmp_path, monkeypatch, "echo no such symbol >&2; exit 1\n")
    out.write_text("of an earlier build")
    os.utime(out, (1, 1))
    assert build.build() == build.OUT
    assert not out.exists()  # what the old callables were built for is gone
    err = capsys.readouterr().err
    assert "no such symbol" in err and "ctypes" in err


def test_missing_and_old_callables_are_built(tmp_path, monkeypatch):
    out = compiler(tmp_path, monkeypatch, WRITES_ITS_OUTPUT)
    assert build.calls_are_stale()
    build.build()
    assert out.exists() and not build.calls_are_stale()
    os.utime(out, (1, 1))
    assert build.calls_are_stale()
    monkeypatch.setattr(build, "_calls_compiler", lambda: None)
    assert not build.calls_are_stale()  # nothing can be built here: the library alone is up to date


def test_callables_that_do_not_load_leave_ctypes(tmp_path, monkeypatch):
    lib = _ffi.load()
    monkeypatch.setattr(_ffi, "LIB_PATH", tmp_path / "libmaize_gemm.so")
    monkeypatch.setattr(_ffi, "_calls", None)
    (tmp_path / build.CALLS_OUT.name).write_text("not a module")
    assert _ffi.load_calls() is lib
