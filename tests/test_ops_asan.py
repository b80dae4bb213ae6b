"""The host code of the C ABI of include/ccv1d_ops.h under AddressSanitizer, without a GPU: the tests of
test_ops_abi.py against _build/libccv1d_asan.so (`make -C causal-conv1d-triton_amd asan`), in a child
process that preloads clang's ASan runtime, as tests/test_asan_host.py does for ccv1d.h."""

import os
import subprocess
import sys

import pytest

from test_asan_host import _LIB, _PKG, _ROOT, _asan_runtime


def test_ops_abi_checks_under_asan():
    runtime = _asan_runtime()
    if runtime is None:
        pytest.skip("clang's shared ASan runtime is not installed")
    if not os.path.exists(_LIB):
        pytest.skip("host ASan build missing: run `make -C causal-conv1d-triton_amd asan`")
    code = (
        "import sys\n"
        f"sys.path[:0] = [{_PKG!r}, {os.path.join(_ROOT, 'tests')!r}]\n"
        "import causal_conv1d_triton._ffi as F\n"
        f"F._LIB_PATH = {_LIB!r}\n"
        "import pytest\n"
        f"sys.exit(pytest.main([{os.path.join(_ROOT, 'tests', 'test_ops_abi.py')!r}, '-q',"
        " '-p', 'no:cacheprovider']))\n"
    )
    env = dict(os.environ, LD_PRELOAD=runtime,
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:halt_on_error=1")
    r = subprocess.run([sys.executable, "-c", code], cwd=_ROOT, env=env, capture_output=True,
                       text=True, timeout=600)
    out = r.stdout + r.stderr
    assert "AddressSanitizer" not in out, out[-4000:]
    assert r.returncode == 0, out[-4000:]
    assert " passed" in out and " failed" not in out, out[-2000:]
