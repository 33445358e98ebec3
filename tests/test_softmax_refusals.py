"""CPU tests of what the softmax operators refuse at the C interface (als_sample_rows, als_distill_rows,
als_distill_topk_f32): every call here is turned away before anything is launched, so no GPU is needed and the addresses
are never read.  Also the option struct and the workspace sizes."""
import ctypes
import os
import re

import pytest

from recommender_amd import _lib
from recommender_amd._lib import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                        # an address: aligned, never read


CODE = {n: int(v) for n, v in re.findall(r"#define ALS_ERR_(\w+) (\d)", open(os.path.join(ROOT, "include", "als_hip.h")).read())}


def refused(rc, code, word):
    assert rc == CODE[code], (rc, lib.als_last_error_string())
    assert word in lib.als_last_error_string().decode(), lib.als_last_error_string()


def sample(**over):
    o = _lib.SampleOpts(1.0, 0, 1.0, 0.0, None, None, None, None)
    a = dict(scores=P, dtype=0, lds=100, n=4, M=100, ex_ptr=None, ex_col=None, ex_rows=None, opts=ctypes.byref(o), u=P, f64=0,
             draws=1, idx=P, logp=P, ws=None, bytes=0, stream=None)
    assert not set(over) - set(a)
    a.update(over)
    return lib.als_sample_rows(*a.values())


@pytest.mark.parametrize("over, code, word", [
    (dict(scores=None), "INVALID_ARG", "null"), (dict(opts=None), "INVALID_ARG", "null"), (dict(u=None), "INVALID_ARG", "null"),
    (dict(idx=None), "INVALID_ARG", "null"), (dict(logp=None), "INVALID_ARG", "null"),
    (dict(n=0), "INVALID_ARG", "sizes"), (dict(n=-1), "INVALID_ARG", "sizes"), (dict(M=0), "INVALID_ARG", "sizes"),
    (dict(lds=99), "INVALID_ARG", "sizes"), (dict(draws=0), "INVALID_ARG", "sizes"), (dict(draws=(1 << 16) + 1), "INVALID_ARG", "sizes"),
    (dict(n=1 << 31), "INVALID_ARG", "sizes"),
    # a thread's next index behind the row would pass 32 bits
    (dict(M=(1 << 31) - 1, lds=1 << 31), "INVALID_ARG", "sizes"), (dict(M=(1 << 31) - 65535, lds=1 << 31), "INVALID_ARG", "sizes"),
    (dict(dtype=3), "UNSUPPORTED", "dtype"), (dict(dtype=-1), "UNSUPPORTED", "dtype"),
    (dict(scores=P + 2), "INVALID_ARG", "aligned"), (dict(dtype=1, scores=P + 1), "INVALID_ARG", "aligned"),
    (dict(ex_ptr=P), "INVALID_ARG", "both"), (dict(ex_col=P), "INVALID_ARG", "both"),
    (dict(M=1 << 20, lds=1 << 20), "WORKSPACE", "workspace"),
    (dict(M=1 << 20, lds=1 << 20, ws=P, bytes=64), "WORKSPACE", "workspace"),
    (dict(M=1 << 20, lds=1 << 20, ws=P + 8, bytes=1 << 40), "WORKSPACE", "workspace")])
def test_sample_rows_refuses(over, code, word):
    refused(sample(**over), code, word)


def rows(**over):
    a = dict(scores=P, dtype=0, lds=100, n=4, M=100, idx=P, val=P, ldt=10, k=10, T=1.0, weight=None, loss=P, grad=P, ldg=100, ws=None,
             bytes=0, stream=None)
    assert not set(over) - set(a)
    a.update(over)
    return lib.als_distill_rows(*a.values())


@pytest.mark.parametrize("over, code, word", [
    (dict(scores=None), "INVALID_ARG", "null"), (dict(idx=None), "INVALID_ARG", "null"), (dict(val=None), "INVALID_ARG", "null"),
    (dict(loss=None), "INVALID_ARG", "null"), (dict(grad=None), "INVALID_ARG", "null"),
    (dict(n=0), "INVALID_ARG", "sizes"), (dict(M=0), "INVALID_ARG", "sizes"), (dict(lds=99), "INVALID_ARG", "sizes"),
    (dict(ldg=99), "INVALID_ARG", "sizes"), (dict(ldt=9), "INVALID_ARG", "sizes"), (dict(n=1 << 31), "INVALID_ARG", "sizes"),
    (dict(M=(1 << 31) - 1, lds=1 << 31, ldg=1 << 31), "INVALID_ARG", "sizes"),
    (dict(k=0), "UNSUPPORTED", "k="), (dict(k=1025, ldt=1025), "UNSUPPORTED", "k="),
    (dict(dtype=3), "UNSUPPORTED", "dtype"), (dict(grad=P + 2), "INVALID_ARG", "aligned"),
    (dict(dtype=2, scores=P + 1), "INVALID_ARG", "aligned"),
    (dict(T=0.0), "INVALID_ARG", "temperature"), (dict(T=-1.0), "INVALID_ARG", "temperature"),
    (dict(T=float("nan")), "INVALID_ARG", "temperature"), (dict(T=float("inf")), "INVALID_ARG", "temperature"),
    (dict(M=1 << 20, lds=1 << 20, ldg=1 << 20), "WORKSPACE", "workspace"),
    (dict(M=1 << 20, lds=1 << 20, ldg=1 << 20, ws=P + 4, bytes=1 << 40), "WORKSPACE", "workspace")])
def test_distill_rows_refuses(over, code, word):
    refused(rows(**over), code, word)


def topk(**over):
    a = dict(X=P, x_rows=50, ldx=20, users=P, n=40, Y=P, ldy=20, M=100, f=20, idx=P, val=P, ldt=10, k=10, T=1.0, weight=None, loss=P,
             dX=P, dY=P, ws=P, bytes=1 << 40, stream=None)
    assert not set(over) - set(a)
    a.update(over)
    return lib.als_distill_topk_f32(*a.values())


@pytest.mark.parametrize("over, code, word", [
    (dict(X=None), "INVALID_ARG", "null"), (dict(Y=None), "INVALID_ARG", "null"), (dict(idx=None), "INVALID_ARG", "null"),
    (dict(val=None), "INVALID_ARG", "null"), (dict(loss=None), "INVALID_ARG", "null"), (dict(dX=None), "INVALID_ARG", "null"),
    (dict(dY=None), "INVALID_ARG", "null"),
    (dict(n=0), "INVALID_ARG", "sizes"), (dict(M=0), "INVALID_ARG", "sizes"), (dict(f=0), "INVALID_ARG", "sizes"),
    (dict(k=0), "INVALID_ARG", "sizes"), (dict(x_rows=0), "INVALID_ARG", "sizes"), (dict(users=None, n=51), "INVALID_ARG", "sizes"),
    (dict(ldx=19), "INVALID_ARG", "sizes"), (dict(ldy=19), "INVALID_ARG", "sizes"), (dict(ldt=9), "INVALID_ARG", "sizes"),
    (dict(M=(1 << 27) + 1), "INVALID_ARG", "sizes"), (dict(n=(1 << 27) + 1), "INVALID_ARG", "sizes"),
    (dict(f=_lib.MAX_FACTORS + 1, ldx=512, ldy=512), "UNSUPPORTED", "f="), (dict(k=1025, ldt=1025), "UNSUPPORTED", "k="),
    (dict(T=0.0), "INVALID_ARG", "temperature"), (dict(T=float("nan")), "INVALID_ARG", "temperature"),
    (dict(T=1e7), "INVALID_ARG", "temperature"), (dict(T=1e-7), "INVALID_ARG", "temperature"),
    (dict(ws=None), "WORKSPACE", "workspace"), (dict(bytes=1000), "WORKSPACE", "workspace"), (dict(ws=P + 8), "WORKSPACE", "workspace")])
def test_distill_topk_refuses(over, code, word):
    refused(topk(**over), code, word)


def test_workspace_sizes():
    """0 for calls that need none and for sizes that are refused; a call's own size is enough, a byte less is not."""
    assert lib.als_sample_rows_workspace_bytes(0, 4096, 59047) == 0
    assert lib.als_sample_rows_workspace_bytes(0, 1, 1 << 20) > 0
    assert lib.als_sample_rows_workspace_bytes(0, 1, (1 << 31) - 1) == 0 and lib.als_sample_rows_workspace_bytes(5, 1, 1 << 20) == 0
    assert lib.als_distill_rows_workspace_bytes(0, 8, 9724, 100) == 0
    assert lib.als_distill_rows_workspace_bytes(0, 8, 1 << 20, 100) > 0
    assert lib.als_distill_rows_workspace_bytes(0, 8, 1 << 20, 1025) == 0
    need = lib.als_distill_topk_workspace_bytes(40, 100, 20, 10)
    assert need > 0
    refused(topk(bytes=need - 1), "WORKSPACE", "%d < %d" % (need - 1, need))
    assert lib.als_distill_topk_workspace_bytes(40, 100, _lib.MAX_FACTORS + 1, 10) == 0
    # no 32-bit size anywhere: half a million users of a catalogue of a million
    assert lib.als_distill_topk_workspace_bytes(500_000, 1_000_000, 128, 200) > 1 << 32


def test_sampling_options_are_the_same_in_header_and_binding():
    hdr = open(os.path.join(ROOT, "include", "als_hip.h")).read()
    body = re.search(r"typedef struct \{([^}]*)\} als_sample_opts_t;", hdr).group(1)
    fields = []
    for decl in body.split(";"):
        decl = " ".join(decl.split())
        if decl:
            name = re.search(r"(\w+)$", decl).group(1)
            ctype = decl[: -len(name)].strip()
            fields.append((name, ctypes.c_void_p if "*" in ctype else {"int32_t": ctypes.c_int32, "float": ctypes.c_float}[ctype]))
    assert fields == list(_lib.SampleOpts._fields_)
    types = dict(re.findall(r"#define ALS_DTYPE_(\w+) (\d)", hdr))
    torch = pytest.importorskip("torch")
    assert {torch.float32: int(types["F32"]), torch.float16: int(types["F16"]), torch.bfloat16: int(types["BF16"])} == _lib.DTYPES
