"""The C ABI of include/ccv1d_layer.h without a GPU: the library exports what the header declares, its workspace
sizes, and the refusal of invalid requests before any HIP call is made."""

import ctypes as C
import os
import re

import pytest

import torch  # noqa: F401  (the library binds to torch's HIP runtime)
from causal_conv1d_triton import _ffi

_HDR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ccv1d_layer.h")
_TYPES = {"int": C.c_int, "float": C.c_float, "int64_t": C.c_int64, "size_t": C.c_size_t}
F32, F16, BF16, F64 = 0, 1, 2, 3


def _header():
    with open(_HDR) as f:
        return re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)


def _struct(name):
    body = re.search(r"struct " + name + r" \{(.*?)\};", _header(), flags=re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        head = re.match(r"(?:const )?(\w+)", decl)
        for var in decl[head.end():].split(","):
            var = var.strip()
            fields.append((var.lstrip("* "), C.c_void_p if var.startswith("*") else _TYPES[head.group(1)]))
    return type(name, (C.Structure,), {"_fields_": fields})


Delta, Update, Norm = (_struct("ccv1d_" + n) for n in ("delta_args", "delta_update_args", "norm_args"))


@pytest.fixture(scope="module")
def lib():
    lib = _ffi.load()
    for n in ("ccv1d_delta_saved_floats", "ccv1d_delta_workspace_bytes", "ccv1d_norm_workspace_bytes"):
        getattr(lib, n).restype = C.c_size_t
    return lib


def test_library_exports_every_declared_symbol(lib):
    names = set(re.findall(r"^(?:int|size_t)\s+(ccv1d_\w+)\(", _header(), flags=re.M))
    assert names == {"ccv1d_delta_saved_floats", "ccv1d_delta_workspace_bytes", "ccv1d_delta_fwd", "ccv1d_delta_bwd",
                     "ccv1d_delta_update", "ccv1d_norm_workspace_bytes", "ccv1d_norm_fwd", "ccv1d_norm_bwd"}
    for n in names:
        assert hasattr(lib, n), n


def _refused(lib, fn, args, code, msg):
    assert fn(C.byref(args)) == code
    assert msg in lib.ccv1d_last_error().decode()


def delta(**kw):
    d = dict(q=4096, k=4096, v=4096, dtype=BF16, log_decay=4096, beta=4096, log_decay_dtype=F32, beta_dtype=BF16,
             scale=1.0, batch=2, seqlen=70, key_heads=2, heads=4, key_dim=64, value_dim=64, out=4096, saved=4096,
             dout=4096, dq=4096, dk=4096, dv=4096, dlog_decay=4096, dbeta=4096, workspace=4096,
             workspace_bytes=1 << 40)
    return Delta(**{**d, **kw})


BAD_DELTA = [
    (dict(batch=-1), 1, "negative size"),
    (dict(seqlen=-1), 1, "negative size"),
    (dict(dtype=F64), 1, "dtypes"),
    (dict(log_decay_dtype=F64), 1, "dtypes"),
    (dict(beta_dtype=9), 1, "dtypes"),
    (dict(key_heads=0), 1, "multiple of key_heads"),
    (dict(heads=0), 1, "multiple of key_heads"),
    (dict(heads=3), 1, "multiple of key_heads"),
    (dict(key_dim=0), 1, "key_dim"),
    (dict(key_dim=257), 1, "key_dim"),
    (dict(value_dim=0), 1, "value_dim"),
    (dict(value_dim=1 << 21), 2, "too large"),
    (dict(seqlen=1 << 31), 2, "too large"),
    (dict(batch=1 << 31), 2, "too large"),
    (dict(batch=1 << 20, seqlen=1 << 20), 2, "too large"),
    (dict(k=0), 1, "null"),
    (dict(beta=0), 1, "null"),
    (dict(log_decay=0), 1, "null"),
    (dict(workspace=0), 3, "workspace"),
    (dict(workspace_bytes=100), 3, "workspace"),
]


@pytest.mark.parametrize("kw,code,msg", BAD_DELTA + [(dict(out=0), 1, "out is null")])
def test_delta_fwd_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_delta_fwd, delta(**kw), code, msg)


@pytest.mark.parametrize("kw,code,msg", BAD_DELTA + [
    (dict(dout=0), 1, "null"), (dict(dq=0), 1, "null"), (dict(dv=0), 1, "null"), (dict(dlog_decay=0), 1, "null"),
    (dict(dbeta=0), 1, "null"), (dict(saved=0), 1, "saved is null")])
def test_delta_bwd_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_delta_bwd, delta(**kw), code, msg)


def test_delta_sizes(lib):
    saved, ws = lib.ccv1d_delta_saved_floats, lib.ccv1d_delta_workspace_bytes
    # a state of (64, 128 or 256) by value_dim up to a multiple of 32 and 64 corrections, a chunk and head
    assert saved(C.byref(delta())) == 2 * 4 * 2 * (64 + 64) * 64
    assert saved(C.byref(delta(key_dim=65, value_dim=33))) == 2 * 4 * 2 * (128 + 64) * 64
    assert saved(C.byref(delta(seqlen=0))) == saved(C.byref(delta(batch=0))) == saved(C.byref(delta(heads=3))) == 0
    keys, heads = 2 * 2 * 2, 2 * 4 * 2  # chunks of key heads and of heads
    tri = 6 * 64 * 16
    rows = 8 * 64 * 4
    assert ws(C.byref(delta()), 0) == keys * 3 * 64 * 64 * 2 + heads * (tri * (3 + 2) + rows)
    assert ws(C.byref(delta(dtype=F32)), 0) == keys * 3 * 64 * 64 * 6 + heads * (tri * (3 + 3) + rows)
    back = keys * 4 * 64 * 64 * 2 + heads * (tri * 6 + rows + (64 + 64) * 64 * 4)
    assert ws(C.byref(delta()), 1) == back
    assert ws(C.byref(delta(seqlen=0)), 1) == 0


def update(**kw):
    d = dict(q=4096, k=4096, v=4096, dtype=BF16, log_decay=4096, beta=4096, log_decay_dtype=F32, beta_dtype=BF16,
             scale=1.0, state=4096, out=4096, rows=4, slots=4, key_heads=1, heads=2, key_dim=64, value_dim=64)
    return Update(**{**d, **kw})


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "negative size"), (dict(slots=-1, rows=0), 1, "negative size"), (dict(dtype=F64), 1, "dtypes"),
    (dict(heads=3, key_heads=2), 1, "multiple of key_heads"), (dict(key_dim=300), 1, "key_dim"),
    (dict(value_dim=0), 1, "value_dim"), (dict(rows=5), 1, "more rows than slots"), (dict(state=0), 1, "null"),
    (dict(q=0), 1, "null"), (dict(out=0), 1, "null"), (dict(rows=1 << 31, slots=1 << 31), 2, "too large"),
    (dict(rows=1 << 22, slots=1 << 22, value_dim=1 << 20), 2, "too large")])
def test_delta_update_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_delta_update, update(**kw), code, msg)


def norm(**kw):
    d = dict(x=4096, dtype=BF16, residual_dtype=BF16, post_weight=4096, pre_weight=4096, gate=4096, scale=1.0, eps=1e-6,
             activation=1, outer=3, inner=2, dim=64, r=4096, y=4096, dr=4096, dy=4096, dx=4096, dgate=4096,
             dpost_weight=4096, dpre_weight=4096, workspace=4096, workspace_bytes=1 << 30)
    return Norm(**{**d, **kw})


BAD_NORM = [
    (dict(outer=-1), 1, "negative size"),
    (dict(dim=0), 1, "dim must be"),
    (dict(dim=8193), 1, "dim must be"),
    (dict(dtype=F64), 1, "dtype"),
    (dict(residual_dtype=F16), 1, "residual_dtype"),
    (dict(residual_dtype=F32), 1, "without residual"),
    (dict(post_weight=0, pre_weight=0), 1, "post_weight and pre_weight"),
    (dict(post_dtype=F64), 1, "weights' dtypes"),
    (dict(scale_weight=4096, scale_dtype=5), 1, "weights' dtypes"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(eps=float("nan")), 1, "eps"),
    (dict(activation=3), 1, "activation"),
    (dict(outer=1 << 31), 2, "too many rows"),
    (dict(outer=1 << 20, inner=1 << 20), 2, "too many rows"),
    (dict(x=0), 1, "null"),
]


@pytest.mark.parametrize("kw,code,msg", BAD_NORM + [
    (dict(y=0), 1, "y goes with pre_weight"), (dict(pre_weight=0), 1, "y goes with pre_weight"),
    (dict(pre_weight=0, y=0, r=0), 1, "r is null")])
def test_norm_fwd_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_norm_fwd, norm(**kw), code, msg)


@pytest.mark.parametrize("kw,code,msg", BAD_NORM + [
    (dict(dpost_weight=0), 1, "gradients go with"), (dict(dscale_weight=4096), 1, "gradients go with"),
    (dict(pre_weight=0, dpre_weight=0), 1, "dy goes with"), (dict(dgate=0), 1, "dgate goes with"),
    (dict(dresidual=4096), 1, "dresidual goes with"), (dict(workspace=0), 3, "workspace"),
    (dict(workspace_bytes=8), 3, "workspace"), (dict(dx=0), 1, "null")])
def test_norm_bwd_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_norm_bwd, norm(**kw), code, msg)


def test_norm_workspace(lib):
    ws = lib.ccv1d_norm_workspace_bytes
    assert ws(C.byref(norm())) == 1 * 3 * 64 * 4  # six rows at once in one workgroup
    assert ws(C.byref(norm(outer=100, dim=300))) == 50 * 3 * 300 * 4  # four at once
    assert ws(C.byref(norm(outer=1 << 20, dim=4096))) == 1024 * 3 * 4096 * 4
    assert ws(C.byref(norm(outer=0))) == 0 and ws(C.byref(norm(dim=0))) == 0


def test_nothing_to_do(lib):
    """Empty calls touch nothing: no pointer is needed."""
    assert lib.ccv1d_delta_fwd(C.byref(Delta(dtype=BF16, batch=0, seqlen=5, key_heads=1, heads=1, key_dim=8,
                                             value_dim=8))) == 0
    assert lib.ccv1d_delta_update(C.byref(Update(dtype=BF16, key_heads=1, heads=1, key_dim=8, value_dim=8))) == 0
    assert lib.ccv1d_norm_fwd(C.byref(Norm(dtype=BF16, residual_dtype=BF16, post_weight=4096, dim=8))) == 0


def test_null_arguments(lib):
    for fn in (lib.ccv1d_delta_fwd, lib.ccv1d_delta_bwd, lib.ccv1d_delta_update, lib.ccv1d_norm_fwd,
               lib.ccv1d_norm_bwd):
        assert fn(None) == 1 and "null" in lib.ccv1d_last_error().decode()
    assert lib.ccv1d_delta_saved_floats(None) == lib.ccv1d_delta_workspace_bytes(None, 0) == 0
    assert lib.ccv1d_norm_workspace_bytes(None) == 0
