"""A C++ exception below a tensor call becomes a Python exception, and the interpreter goes on."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

# The library's functions are stood in for by one of the C++ runtime that throws std::bad_alloc, in a process of its own.
PROGRAM = """
import ctypes, threading
import torch
from megcc_b200 import _lib, ops
x = torch.ones((2, 64), device="cuda")
b = torch.ones((8, 64), dtype=torch.int8, device="cuda")
s = torch.ones(8, device="cuda")
w1, w2 = torch.ones((4, 64, 64), dtype=torch.int8, device="cuda"), torch.ones((4, 64, 32), dtype=torch.int8, device="cuda")
s1, s2, logits = torch.ones((4, 64), device="cuda"), torch.ones((4, 64), device="cuda"), torch.zeros((2, 4), device="cuda")
calls = _lib.tensor_calls()
throws = ctypes.cast(getattr(ctypes.CDLL("libstdc++.so.6"), "_ZSt17__throw_bad_allocv"), ctypes.c_void_p).value
size = ctypes.cast(_lib.lib().mb200_linear_s8_workspace_bytes, ctypes.c_void_p).value
msize = ctypes.cast(_lib.lib().mb200_matmul_s8_scaled_workspace_bytes, ctypes.c_void_p).value
esize = ctypes.cast(_lib.lib().mb200_moe_s8_workspace_bytes, ctypes.c_void_p).value
calls.bind(_lib.check, torch.OutOfMemoryError, throws, msize, throws, size, throws, esize, throws)
def each():
    for call in (lambda: ops.quantize_rows_s8(x), lambda: ops.linear_s8(x, b, s),
                 lambda: ops.matmul_s8_scaled(b, b, s, s), lambda: ops.moe_s8(x, logits, w1, s1, w2, s2, 2)):
        try:
            call()
        except RuntimeError as e:
            assert "bad_alloc" in str(e), e
            done.append(1)
done = []
each()
threads = [threading.Thread(target=each) for _ in range(3)]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert len(done) == 16, done
print("went on")
"""


def test_exceptions_below_a_call():
    r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["went", "on"], r.stderr[-2000:]
