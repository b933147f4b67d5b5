"""The W8A8 operators' refusals: no call below reaches a device."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from dynamicscaler_amd import _lib, ops
from dynamicscaler_amd._lib import DS_EPI_GEGLU, DS_EPI_SILU, DsError

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, F32, I8 = torch.float16, torch.float32, torch.int8


def product(**kw):
    c = dict(A=torch.zeros((4, 32), dtype=I8), W=torch.zeros((64, 32), dtype=I8), a_scale=torch.ones(4), w_scale=torch.ones(64))
    c.update(kw)
    return c


@pytest.mark.parametrize("change,says", [
    (dict(A=torch.zeros((4, 32))), "gemm_i8\\(A\\).*float32"),
    (dict(A=torch.zeros((4, 32, 1), dtype=I8)), "\\[rows, columns\\]"),
    (dict(W=torch.zeros((64, 31), dtype=I8)), "gemm_i8\\(W\\).*expected 64 x 32"),
    (dict(A=torch.zeros((32, 4), dtype=I8).t()), "contiguous"),
    (dict(A=torch.zeros((1, 32), dtype=I8).expand(4, 32)), "overlap"),
    (dict(a_scale=torch.ones(5)), "a_scale.*4 values"),
    (dict(a_scale=torch.ones(4, dtype=F16)), "a_scale"),
    (dict(a_scale=torch.ones(8)[::2]), "a_scale"),
    (dict(w_scale=torch.ones(1)), "w_scale.*64 values"),
    (dict(w_scale=torch.ones((64, 1))), "w_scale"),
    (dict(bias=torch.ones(63)), "bias"),
    (dict(residual=torch.zeros((4, 63), dtype=F16)), "residual.*expected 4 x 64"),
    (dict(residual=torch.zeros((4, 64), dtype=torch.float64)), "residual"),
    (dict(out=torch.zeros((4, 64), dtype=I8)), "out"),
    (dict(out=torch.zeros((1, 64), dtype=F16).expand(4, 64)), "overlap"),
    (dict(out=torch.zeros((4, 64), dtype=F16), epilogue=DS_EPI_GEGLU), "out.*expected 4 x 32"),
    (dict(out_dtype=torch.bfloat16), "out_dtype"),
    (dict(epilogue=4), "epilogue 4"),
    (dict(epilogue=8 | DS_EPI_SILU), "epilogue"),
    (dict(epilogue=-1), "epilogue"),
    (dict(), "no CPU fallback"),
    (dict(A=[[1]]), "not a tensor"),
])
def test_product_refuses(change, says):
    with pytest.raises(DsError, match=says):
        ops.gemm_i8(**product(**change))


@pytest.mark.parametrize("change,says", [(dict(A=[[1]]), "not a tensor"), (dict(W=None), "not a tensor"), (dict(A=torch.zeros((4, 32, 1), dtype=I8)), "\\[rows, columns\\]"),
                                         (dict(W=torch.zeros(32, dtype=I8)), "\\[rows, columns\\]"), (dict(A=torch.zeros((), dtype=I8)), "\\[rows, columns\\]"),
                                         (dict(W=torch.zeros((64, 31), dtype=I8)), "expected 64 x 32"), (dict(), "no CPU fallback")])
def test_product_refuses_the_same_under_a_timing_hook(change, says):
    ops.set_timing_hook(lambda name, flops, launch, info: launch())
    try:
        with pytest.raises(DsError, match=says):
            ops.gemm_i8(**product(**change))
    finally:
        ops.set_timing_hook(None)


X = torch.zeros((4, 32), dtype=F16)


@pytest.mark.parametrize("call,says", [
    (lambda: ops.rmsnorm(X.to(torch.bfloat16), torch.ones(32)), "x"),
    (lambda: ops.rmsnorm(X, torch.ones(31)), "gamma.*32 values"),
    (lambda: ops.rmsnorm(X, torch.ones(32, dtype=F16)), "gamma"),
    (lambda: ops.rmsnorm(X, torch.ones(32), residual=torch.zeros((3, 32))), "residual.*expected 4 x 32"),
    (lambda: ops.rmsnorm(X, torch.ones(32), residual=X, sum_out=torch.zeros((4, 32))), "sum_out.*float32"),
    (lambda: ops.rmsnorm(X, torch.ones(32), sum_out=X), "without a residual"),
    (lambda: ops.rmsnorm(X, torch.ones(32), out=torch.zeros((4, 32), dtype=I8)), "out"),
    (lambda: ops.rmsnorm(X, torch.ones(32), out_dtype=I8), "out_dtype"),
    (lambda: ops.rmsnorm(X[:, :0], torch.ones(0)), "without values"),
    (lambda: ops.rmsnorm_i8(X, torch.ones(32), out=X), "out"),
    (lambda: ops.rmsnorm_i8(X, torch.ones(32), scale=torch.ones(3)), "scale.*4 values"),
    (lambda: ops.rmsnorm_i8(X, torch.ones(32)), "no CPU fallback"),
    (lambda: ops.quantize_rows_i8(X.to(I8)), "x"),
    (lambda: ops.quantize_rows_i8(X[:, :0]), "without values"),
    (lambda: ops.quantize_rows_i8(X, out=torch.zeros((4, 33), dtype=I8)), "expected 4 x 32"),
    (lambda: ops.quantize_rows_i8(X, scale=torch.ones((4, 1))), "scale"),
    (lambda: ops.quantize_rows_i8(X.t()[:, :2]), "contiguous"),
    (lambda: ops.quantize_rows_i8(X), "no CPU fallback"),
    (lambda: ops.dequantize_rows_i8(X, torch.ones(4)), "q"),
    (lambda: ops.dequantize_rows_i8(X.to(I8), torch.ones(5)), "scale"),
    (lambda: ops.dequantize_rows_i8(X.to(I8), torch.ones(4), dtype=I8), "dtype"),
    (lambda: ops.dequantize_rows_i8(X.to(I8), torch.ones(4), out=X[:3]), "expected 4 x 32"),
    (lambda: ops.dequantize_rows_i8(X.to(I8), torch.ones(4)), "no CPU fallback"),
])
def test_rows_refuse(call, says):
    with pytest.raises(DsError, match=says):
        call()


def refused(rc, says):
    assert rc == -1 and re.search(says, _lib.load().ds_last_error().decode()), _lib.load().ds_last_error()


P = 1 << 20      # stands for an aligned device address; a refused call does not follow it


@pytest.mark.parametrize("fields,args,says", [
    (dict(K=131072, lda=131072, ldw=131072), {}, "131071"),
    (dict(M=-1), {}, "negative"),
    (dict(epilogue=16), {}, "epilogue"),
    (dict(epilogue=DS_EPI_GEGLU | DS_EPI_SILU), {}, "exclude"),
    (dict(epilogue=DS_EPI_GEGLU, N=96, ldc=96), {}, "N % 64"),
    (dict(epilogue=DS_EPI_GEGLU, ldr=64), dict(residual=P), "no residual"),
    (dict(lda=31), {}, "row stride"),
    (dict(ldw=0), {}, "row stride"),
    (dict(ldc=63), {}, "row stride"),
    (dict(ldr=63), dict(residual=P), "row stride"),
    ({}, dict(A=0), "NULL"),
    ({}, dict(w_scale=0), "NULL"),
    ({}, dict(out=0), "NULL"),
    ({}, dict(out=P + 1), "aligned"),
    (dict(ldr=64, epilogue=8), dict(residual=P + 2), "aligned"),
    ({}, dict(bias=P + 2), "aligned"),
])
def test_product_c_entry_refuses(fields, args, says):
    d = _lib.GemmI8Desc()
    for k, v in dict(dict(M=4, N=64, K=32, lda=32, ldw=32, ldc=64, ldr=0, epilogue=0), **fields).items():
        setattr(d, k, v)
    a = dict(dict(A=P, W=P, a_scale=P, w_scale=P, bias=0, residual=0, out=P), **args)
    refused(_lib.load().ds_gemm_i8(a["A"], a["W"], a["a_scale"], a["w_scale"], a["bias"], a["residual"], a["out"], C.byref(d), 0, 0, 0), says)


def test_product_c_entry_refuses_no_desc_and_accepts_nothing_to_do():
    lib = _lib.load()
    refused(lib.ds_gemm_i8(P, P, P, P, 0, 0, P, None, 0, 0, 0), "desc")
    d = _lib.GemmI8Desc(M=0, N=64, K=32, lda=32, ldw=32, ldc=64)
    assert lib.ds_gemm_i8(P, P, P, P, 0, 0, P, C.byref(d), 0, 0, 0) == 0


def test_product_workspace():
    """Rows of whole 16s need none; odd ones room for both operands' rows rounded up to 16; a short or crooked one is refused."""
    lib = _lib.load()
    d = _lib.GemmI8Desc(M=2057, N=997, K=1280, lda=1280, ldw=1280, ldc=997)
    assert lib.ds_gemm_i8_workspace_bytes(P, P, C.byref(d)) == 0
    assert lib.ds_gemm_i8_workspace_bytes(P + 16, P, C.byref(d)) == 0
    assert lib.ds_gemm_i8_workspace_bytes(P + 4, P, C.byref(d)) == 2057 * 1280
    assert lib.ds_gemm_i8_workspace_bytes(P, P + 1, C.byref(d)) == 997 * 1280
    d.K = d.lda = d.ldw = 1273
    need = lib.ds_gemm_i8_workspace_bytes(P, P, C.byref(d))
    assert need == (2057 + 997) * 1280
    refused(lib.ds_gemm_i8(P, P, P, P, 0, 0, P, C.byref(d), P, need - 1, 0), "workspace")
    refused(lib.ds_gemm_i8(P, P, P, P, 0, 0, P, C.byref(d), P + 8, need, 0), "workspace")
    d.M = 64                                     # few rows are read as they lie
    assert lib.ds_gemm_i8_workspace_bytes(P, P, C.byref(d)) == 0
    assert lib.ds_gemm_i8_workspace_bytes(P, P, None) == 0


@pytest.mark.parametrize("fields", [dict(K=131072, lda=131073, ldw=131073), dict(epilogue=16), dict(epilogue=DS_EPI_GEGLU, N=997), dict(epilogue=DS_EPI_GEGLU | DS_EPI_SILU, N=1024),
                                    dict(M=-5), dict(N=-5), dict(K=-5)])
def test_product_that_is_refused_needs_no_workspace(fields):
    d = _lib.GemmI8Desc(**dict(dict(M=2057, N=997, K=1273, lda=1273, ldw=1273, ldc=997), **fields))
    assert _lib.load().ds_gemm_i8_workspace_bytes(P, P, C.byref(d)) == 0


NORM = dict(x=P, xt=0, ldx=32, r=P, rt=0, ldr=32, g=P, s=P, lds=32, y=P, yt=2, ldy=32, scale=P, rows=4, C=32, eps=1e-6)


@pytest.mark.parametrize("change,says", [
    (dict(C=0), "C 0"), (dict(rows=-1), "rows -1"), (dict(xt=2), "type 2"), (dict(rt=3), "type"), (dict(yt=5), "result type"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(x=0), "NULL"), (dict(g=0), "NULL"),
    (dict(scale=0), "NULL"), (dict(r=0), "without a residual"), (dict(ldx=31), "row stride"), (dict(lds=31), "row stride"),
    (dict(ldr=0), "row stride"), (dict(ldy=31), "row stride"), (dict(x=P + 1), "aligned"), (dict(r=P + 2, rt=1), "aligned"), (dict(g=P + 2), "aligned")])
def test_norm_c_entry_refuses(change, says):
    c = dict(NORM, **change)
    d = _lib.RmsnormDesc(c["ldx"], c["ldr"], c["lds"], c["ldy"], c["rows"], c["C"], c["xt"], c["rt"], c["yt"], c["eps"])
    refused(_lib.load().ds_rmsnorm_rows(c["x"], c["r"], c["g"], c["s"], c["y"], c["scale"], C.byref(d), 0), says)


def test_norm_c_entry_refuses_no_desc():
    refused(_lib.load().ds_rmsnorm_rows(P, 0, P, 0, P, P, None, 0), "desc")


@pytest.mark.parametrize("args,says", [((P, 2, 32, P, 32, P, 4, 32), "type"), ((P, 0, 31, P, 32, P, 4, 32), "row stride"), ((P, 0, 32, 0, 32, P, 4, 32), "NULL"),
                                       ((P, 0, 32, P, 32, P + 2, 4, 32), "aligned"), ((P, 0, 32, P, 32, P, 4, 0), "C 0")])
def test_quantize_c_entry_refuses(args, says):
    refused(_lib.load().ds_quantize_rows_i8(*args, 0), says)


@pytest.mark.parametrize("args,says", [((P, 32, P, P, 2, 32, 4, 32), "type"), ((P, 31, P, P, 0, 32, 4, 32), "row stride"), ((P, 32, 0, P, 0, 32, 4, 32), "NULL"),
                                       ((P, 32, P, P + 2, 1, 32, 4, 32), "aligned")])
def test_dequantize_c_entry_refuses(args, says):
    refused(_lib.load().ds_dequantize_rows_i8(*args, 0), says)


@pytest.mark.parametrize("name,cls", [("ds_gemm_i8_desc", _lib.GemmI8Desc), ("ds_rmsnorm_desc", _lib.RmsnormDesc)])
def test_desc_layout_matches_the_header(name, cls):
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "dynscaler_hip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, flags=re.S).group(1)
    fields = [(n.strip(), t) for t, names in re.findall(r"(int32_t|int64_t|float) ([^;]+);", body) for n in names.split(",")]
    assert [(n, {C.c_int64: "int64_t", C.c_int32: "int32_t", C.c_float: "float"}[t]) for n, t in cls._fields_] == fields


@pytest.mark.parametrize("source", ["gemm_i8.hip", "rows_i8.hip"])
def test_sources_compile_without_warnings(source):
    """Among them -Walign-mismatch: loads and stores at any element are declared so, whatever the hardware accepts."""
    from dynamicscaler_amd import build
    if not os.path.exists(build.HIPCC):
        pytest.skip("needs hipcc")
    r = subprocess.run([build.HIPCC] + build.FLAGS + build.SOURCE_FLAGS[source] + ["-Werror", "-Wno-unused-command-line-argument", "--cuda-device-only", "-fsyntax-only",
                                                                                   "-x", "hip", os.path.join(build.CSRC, source)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


class Compiler:
    """Stands for subprocess.run in the build: counts the calls, compiles nothing."""
    def __init__(self):
        self.calls = 0

    def __call__(self, cmd, **kw):
        self.calls += 1
        return subprocess.CompletedProcess(cmd, 0, "", "")


def test_the_front_end_is_built_anew_where_that_is_asked_for_or_torch_has_changed(monkeypatch, tmp_path):
    from dynamicscaler_amd import build
    run = Compiler()
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build, "_newer", lambda sources, target: False)
    counts = []
    for force, version in ((False, None), (False, None), (True, None), (False, "99.0"), (False, "99.0")):
        if version:
            monkeypatch.setattr(torch, "__version__", version)
        assert build.build_torch(force=force, verbose=False)
        counts.append(run.calls)
    assert counts == [1, 1, 2, 3, 3]


@pytest.mark.parametrize("missing", ["torch", "g++", "headers"])
def test_a_build_without_torch_leaves_out_the_front_end_alone(monkeypatch, missing, capsys):
    import sys
    import torch.utils.cpp_extension as ext
    from dynamicscaler_amd import build
    run = Compiler()
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "_newer", lambda sources, target: False)
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif missing == "g++":
        monkeypatch.setattr(build.shutil, "which", lambda name: None)
    else:
        monkeypatch.setattr(ext, "include_paths", lambda: [])
    assert build.build(verbose=False) == build.LIB and run.calls == 0
    assert "_w8a8.so not built" in capsys.readouterr().err
