"""The C ABI of include/ccv1d_ops.h without a GPU: the library exports what the header declares, its
workspace sizes, and the refusal of invalid requests before any HIP call is made."""

import ctypes as C
import os
import re

import pytest

import torch  # noqa: F401  (the library binds to torch's HIP runtime)
from causal_conv1d_triton import _ffi

_HDR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                    "ccv1d_ops.h")
_TYPES = {"int": C.c_int, "float": C.c_float, "int64_t": C.c_int64, "size_t": C.c_size_t}
F32, F16, BF16, F64 = 0, 1, 2, 3


def _header():
    with open(_HDR) as f:
        return re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)


def _struct(name):
    """A ctypes structure from the header's declaration."""
    body = re.search(r"struct " + name + r" \{(.*?)\};", _header(), flags=re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        base = re.match(r"(?:const )?(\w+)", decl).group(1)
        rest = decl[re.match(r"(?:const )?\w+", decl).end():]
        for var in rest.split(","):
            var = var.strip()
            ptr = var.startswith("*")
            fields.append((var.lstrip("* "), C.c_void_p if ptr else _TYPES[base]))
    return type(name, (C.Structure,), {"_fields_": fields})


Rec, Update, Plan, Write, Attn = (_struct("ccv1d_" + n) for n in (
    "rec_args", "rec_update_args", "paged_plan_args", "paged_write_args", "paged_attn_args"))


@pytest.fixture(scope="module")
def lib():
    lib = _ffi.load()
    lib.ccv1d_rec_workspace_bytes.restype = C.c_size_t
    lib.ccv1d_rec_workspace_bytes.argtypes = [C.c_int64, C.c_int64, C.c_int64, C.c_int]
    lib.ccv1d_paged_attn_workspace_bytes.restype = C.c_size_t
    return lib


def test_library_exports_every_declared_symbol(lib):
    names = set(re.findall(r"^(?:int|size_t)\s+(ccv1d_\w+)\(", _header(), flags=re.M))
    assert names == {"ccv1d_rec_workspace_bytes", "ccv1d_rec_fwd", "ccv1d_rec_bwd",
                     "ccv1d_rec_update", "ccv1d_paged_plan", "ccv1d_paged_write",
                     "ccv1d_paged_attn_workspace_bytes", "ccv1d_paged_attn"}
    for n in names:
        assert hasattr(lib, n), n


def _refused(lib, fn, args, code, msg):
    assert fn(C.byref(args)) == code
    assert msg in lib.ccv1d_last_error().decode()


def rec(**kw):
    d = dict(x=4096, gate=4096, x_stride_t=8, gate_stride_t=8, dtype=BF16, decay_scale=8.0, batch=2,
             seqlen=40, dim=8, out=4096, saved=4096, dout=4096, dout_stride_t=8, dx=4096, dgate=4096,
             workspace=4096, workspace_bytes=1 << 40)
    return Rec(**{**d, **kw})


@pytest.mark.parametrize("kw,code,msg", [
    (dict(batch=-1), 1, "negative size"),
    (dict(dim=-1), 1, "negative size"),
    (dict(dtype=F64), 1, "dtype"),
    (dict(dtype=7), 1, "dtype"),
    (dict(x=0), 1, "null"),
    (dict(gate=0), 1, "null"),
    (dict(out=0), 1, "null"),
    (dict(seqlen=1 << 31), 2, "too large"),
    (dict(batch=1 << 31), 2, "too large"),
    (dict(batch=1 << 20, dim=1 << 20), 2, "too large"),
    (dict(seqlen=1000, workspace=0), 3, "workspace"),
    (dict(seqlen=1000, workspace_bytes=100), 3, "workspace"),
    (dict(decay_scale=-1.0), 1, "decay_scale"),
    (dict(decay_scale=float("nan")), 1, "decay_scale"),
])
def test_rec_fwd_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_rec_fwd, rec(**kw), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dout=0), 1, "null"),
    (dict(dx=0), 1, "null"),
    (dict(dgate=0), 1, "null"),
    (dict(saved=0), 1, "saved"),
    (dict(input_gate=4096), 1, "dinput_gate"),
    (dict(dinput_gate=4096), 1, "dinput_gate"),
    (dict(decay=4096), 1, "ddecay"),
    (dict(ddecay=4096), 1, "ddecay"),
    (dict(workspace=0), 3, "workspace"),
])
def test_rec_bwd_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_rec_bwd, rec(**kw), code, msg)


def test_null_arguments(lib):
    for fn in (lib.ccv1d_rec_fwd, lib.ccv1d_rec_bwd, lib.ccv1d_rec_update, lib.ccv1d_paged_plan,
               lib.ccv1d_paged_write, lib.ccv1d_paged_attn):
        assert fn(None) == 1 and "null" in lib.ccv1d_last_error().decode()
    assert lib.ccv1d_paged_attn_workspace_bytes(None) == 0


def test_rec_workspace(lib):
    ws = lib.ccv1d_rec_workspace_bytes
    assert ws(0, 10, 8, 0) == ws(1, 0, 8, 1) == ws(1, 10, 0, 1) == 0
    assert ws(3, 128, 70, 0) == 0  # one chunk: nothing to hand on
    # beyond one chunk: a word per channel and chunk, one per channel and group, and half a word, rounded
    # up, per 64 channels of a batch row
    assert ws(2, 129, 70, 0) == 8 * (2 * 70 * (2 + 1) + 2)
    assert ws(1, 128 * 17, 5, 0) == 8 * (5 * (17 + 2) + 1)
    # the backward's chunks are half as long, with a sum per channel and chunk
    assert ws(3, 64, 70, 1) == 4 * 3 * 70
    assert ws(2, 65, 70, 1) == 8 * (2 * 70 * (2 + 1) + 2) + 4 * 2 * 70 * 2


def update(**kw):
    d = dict(x=4096, gate=4096, dtype=BF16, decay_scale=8.0, state=4096, state_stride=8, out=4096,
             rows=4, slots=4, dim=8)
    return Update(**{**d, **kw})


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "negative size"),
    (dict(dtype=F64), 1, "dtype"),
    (dict(rows=5), 1, "more rows than slots"),
    (dict(state=0), 1, "null"),
    (dict(gate=0), 1, "null"),
    (dict(out=0), 1, "null"),
    (dict(rows=1 << 31, slots=1 << 31), 2, "too large"),
    (dict(decay_scale=-2.0), 1, "decay_scale"),
])
def test_rec_update_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_rec_update, update(**kw), code, msg)


def plan(**kw):
    d = dict(cached_lens=4096, new_lens=4096, block_tables=4096, block_table_stride=4, free_pages=4096,
             num_free=4096, requests=3, max_pages=4, num_free_pages=9, page_size=16, max_tokens=10,
             seq_lens=4096, query_start=4096, positions=4096, request_ids=4096, slot_mapping=4096,
             num_free_out=4096)
    return Plan(**{**d, **kw})


@pytest.mark.parametrize("kw,code,msg", [
    (dict(requests=-1), 1, "negative size"),
    (dict(page_size=0), 1, "page_size"),
    (dict(max_pages=1 << 30), 2, "too large"),
    (dict(page_size=1 << 31, max_pages=0), 2, "too large"),
    (dict(max_tokens=1 << 31), 2, "too large"),
    (dict(num_free=0), 1, "null"),
    (dict(num_free_out=0), 1, "null"),
    (dict(cached_lens=0), 1, "null"),
    (dict(block_tables=0), 1, "null"),
    (dict(free_pages=0), 1, "null"),
    (dict(slot_mapping=0), 1, "null"),
])
def test_paged_plan_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_paged_plan, plan(**kw), code, msg)


def write(**kw):
    d = dict(k=4096, v=4096, k_cache=4096, v_cache=4096, dtype=BF16, slot_mapping=4096, tokens=5,
             kv_heads=2, head_dim=8, num_pages=3, page_size=4)
    return Write(**{**d, **kw})


@pytest.mark.parametrize("kw,code,msg", [
    (dict(tokens=-1), 1, "negative size"),
    (dict(dtype=9), 1, "dtype"),
    (dict(page_size=0), 1, "page_size"),
    (dict(tokens=1 << 31), 2, "too large"),
    (dict(kv_heads=1 << 20, head_dim=1 << 20), 2, "too large"),
    (dict(num_pages=1 << 40, page_size=1 << 40), 1, "too large"),
    (dict(k=0), 1, "null"),
    (dict(v_cache=0), 1, "null"),
    (dict(slot_mapping=0), 1, "null"),
])
def test_paged_write_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_paged_write, write(**kw), code, msg)


def attn(**kw):
    d = dict(q=4096, k_cache=4096, v_cache=4096, dtype=BF16, block_tables=4096, block_table_stride=8,
             seq_lens=4096, out=4096, scale=0.1, rows=3, requests=3, q_heads=8, kv_heads=2, head_dim=64,
             num_pages=30, page_size=16, max_pages=8, workspace=4096, workspace_bytes=1 << 40)
    return Attn(**{**d, **kw})


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "negative size"),
    (dict(window=-1), 1, "negative size"),
    (dict(dtype=F64), 1, "dtype"),
    (dict(head_dim=60), 1, "head_dim"),
    (dict(head_dim=0), 1, "head_dim"),
    (dict(head_dim=264), 1, "head_dim"),
    (dict(q_heads=7), 1, "q_heads"),
    (dict(kv_heads=0), 1, "q_heads"),
    (dict(page_size=0), 1, "page_size"),
    (dict(max_pages=1 << 30), 2, "max_pages"),
    (dict(rows=1 << 30, requests=1 << 30), 2, "too large"),
    (dict(rows=4), 1, "more rows than requests"),
    (dict(q=0), 1, "null"),
    (dict(k_cache=0), 1, "null"),
    (dict(block_tables=0), 1, "null"),
    (dict(max_pages=100, workspace=0), 3, "workspace"),
    (dict(max_pages=100, workspace_bytes=10), 3, "workspace"),
])
def test_paged_attn_refuses(lib, kw, code, msg):
    _refused(lib, lib.ccv1d_paged_attn, attn(**kw), code, msg)


def test_paged_attn_workspace(lib):
    ws = lambda **kw: lib.ccv1d_paged_attn_workspace_bytes(C.byref(attn(**kw)))  # noqa: E731
    assert ws() == 0  # 128 positions: one span
    assert ws(rows=0) == 0
    assert ws(head_dim=60) == 0  # refused
    # spans of 128 to 1024 positions, 256 at most; head_dim sums, a maximum and a sum each
    assert ws(max_pages=100) == 3 * 8 * 13 * (64 + 2) * 4
    assert ws(rows=2000, requests=2000, max_pages=512) == 2000 * 8 * 8 * (64 + 2) * 4
    assert ws(max_pages=1 << 20) <= 3 * 8 * 256 * (64 + 2) * 4
    assert ws(max_pages=1 << 20, max_seq_len=128) == 0
    assert ws(max_pages=1 << 20, window=97) == 0


def test_paged_attn_windows_past_every_length(lib):
    """A window that no length reaches is none, up to the largest that the argument holds: the launch is
    sized for the table, and the sums of its spans have a place."""
    for kw in (dict(max_pages=1000), dict(rows=64, requests=64, q_heads=32, head_dim=128, max_pages=512),
               dict(max_pages=1000, max_seq_len=9000)):
        none = lib.ccv1d_paged_attn_workspace_bytes(C.byref(attn(**kw)))
        assert none > 0
        for window in (kw["max_pages"] * 16, 2 ** 31 - 32, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 32, 2 ** 63 - 31,
                       2 ** 63 - 1):
            a = attn(**kw, window=window)
            assert lib.ccv1d_paged_attn_workspace_bytes(C.byref(a)) == none, window
        a = attn(**kw, window=2 ** 63 - 1, workspace=0, workspace_bytes=0)
        _refused(lib, lib.ccv1d_paged_attn, a, 3, "workspace")


@pytest.mark.parametrize("rows,q_heads,kv_heads,head_dim,positions", [
    (2048, 32, 8, 128, 131072), (8192, 32, 8, 128, 131072), (8192, 32, 8, 128, 262144),
    (16384, 32, 8, 128, 131072), (1000, 64, 64, 256, 1 << 20), (100000, 8, 8, 8, 1 << 20),
    (8388607, 1, 1, 8, 1 << 20), (131071, 64, 1, 64, 1 << 30)])
def test_paged_attn_many_rows_of_a_long_table(lib, rows, q_heads, kv_heads, head_dim, positions):
    """Where the rows alone fill the card, the table's capacity does not size the workspace, and no launch
    has 2^32 threads (256 a workgroup; the join: 64 for four spans, at most 1024)."""
    a = attn(rows=rows, requests=rows, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
             max_pages=positions // 16, num_pages=positions)
    need = lib.ccv1d_paged_attn_workspace_bytes(C.byref(a))
    assert need <= 512 << 20
    each = rows * q_heads * (head_dim + 2) * 4
    assert need % each == 0
    splits = max(1, need // each)
    tiles = -(-(q_heads // kv_heads) // 16)
    assert rows * splits * kv_heads * tiles * 256 < 2 ** 32
    assert splits == 1 or rows * q_heads * min(1024, 64 * -(-splits // 4)) < 2 ** 32


@pytest.mark.parametrize("fn,args", [
    # 512 threads for 64 channels (16 bits: 128, but for a single one) and 128 rows, backward 64 rows
    ("rec_fwd", dict(batch=1, dim=1, seqlen=(1 << 30) + 1)),
    ("rec_fwd", dict(batch=1 << 23, dim=1)),
    ("rec_fwd", dict(batch=1 << 22, dim=130, seqlen=1)),
    ("rec_fwd", dict(batch=1 << 22, dim=65, seqlen=1, dtype=F32)),
    # one chunk of 1024 threads
    ("rec_fwd", dict(batch=1 << 22, dim=128, seqlen=200)),
    ("rec_bwd", dict(batch=1, dim=1, seqlen=(1 << 29) + 1)),
    ("rec_bwd", dict(batch=1 << 23, dim=1)),
    # 1024 threads for 32 channels of the decay's sum
    ("rec_bwd", dict(batch=1, dim=1 << 27, seqlen=1, decay=4096, ddecay=4096)),
])
def test_recurrence_of_2_32_threads_is_refused(lib, fn, args):
    _refused(lib, getattr(lib, "ccv1d_" + fn), rec(**args), 2, "too large for one launch")


def test_other_launches_of_2_32_threads_are_refused(lib):
    # 64 threads for 256 channels of a row
    n = 1 << 26
    _refused(lib, lib.ccv1d_rec_update, update(rows=n, slots=n), 2, "too large for one launch")
    _refused(lib, lib.ccv1d_rec_update, update(rows=n // 2, slots=n // 2, dim=257), 2, "too large for one")
    # 256 threads for one token, or for as many as have 512 pieces between them
    _refused(lib, lib.ccv1d_paged_write, write(tokens=1 << 24, kv_heads=16, head_dim=128), 2, "too large for one")
    _refused(lib, lib.ccv1d_paged_write, write(tokens=(1 << 31) - 1, kv_heads=2, head_dim=8, dtype=F32), 2,
             "too large for one")


def test_empty_requests_are_no_ops(lib):
    assert lib.ccv1d_rec_fwd(C.byref(rec(batch=0))) == 0
    assert lib.ccv1d_rec_fwd(C.byref(rec(dim=0))) == 0
    assert lib.ccv1d_rec_bwd(C.byref(rec(dim=0))) == 0
    assert lib.ccv1d_rec_update(C.byref(update(rows=0))) == 0
    assert lib.ccv1d_paged_write(C.byref(write(tokens=0))) == 0
    assert lib.ccv1d_paged_attn(C.byref(attn(rows=0))) == 0
    assert lib.ccv1d_last_error().decode() == ""
