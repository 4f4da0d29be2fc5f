"""A kernel of a serving call whose launch fails is the call's last: the ones behind it read what it would have written (on
the CPU, against a stand-in for the runtime's launches)."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

LIBRARY = Path(__file__).resolve().parents[1] / "risaattention_b200" / "librisa_b200.so"

STAND_IN = r"""
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
static int launches, last;
static char word[64];
int cudaGetSymbolAddress(void** address, const void* symbol) { *address = word; return 0; }
int cudaFuncSetAttribute(const void* f, int attribute, int value) { return 0; }
int cudaFuncGetAttributes(void* attributes, const void* f) {
  memset(attributes, 0, 32);
  ((int*)attributes)[7] = 80;  /* numRegs */
  return 0;
}
int cudaLaunchKernelExC(const void* config, const void* f, void** arguments) {
  if (launches++ == atoi(getenv("FAILING_LAUNCH"))) return last = 701;  /* too many resources */
  return 0;
}
int cudaGetLastError(void) { int e = last; last = 0; return e; }
int launch_count(void) { return launches; }
"""

CALLS = r"""
import ctypes as c, sys
import os
stand_in = c.CDLL(os.environ["LD_PRELOAD"])
lib = c.CDLL(sys.argv[1])
lib.risa_b200_last_error.restype = c.c_char_p
lib.risa_b200_paged_attention_scratch_size.restype = lib.risa_b200_key_weights_scratch_size.restype = c.c_size_t
class Cache(c.Structure):
    _fields_ = [(n, c.c_void_p) for n in ("keys", "values", "key_scales", "value_scales")] + [(n, c.c_int) for n in ("pages", "kv_heads", "page_size", "head_dim", "dtype_code")]
class Step(c.Structure):
    _fields_ = [(n, c.c_void_p) for n in ("page_table", "lengths", "query_offsets")] + [(n, c.c_int) for n in ("batch", "table_width", "tokens")]
A = 4096  # aligned addresses that nothing reads
cache, tokens = Cache(A, A, A, A, 8, 2, 16, 128, 4), int(sys.argv[3])
step, strides = Step(A, A, A, 1, 8, tokens), (c.c_int64 * 2)(512, 128)
p = lambda x: c.c_void_p(x)
scratch = 1 << 30
if sys.argv[2] == "attention":
    status = lib.risa_b200_paged_attention(c.byref(cache), c.byref(step), p(A), strides, 4, 2, p(A), strides, p(A), c.c_float(0.1), 1, 0, 3, p(A), c.c_size_t(scratch), p(0))
elif sys.argv[2] == "weights":
    status = lib.risa_b200_key_weights(c.byref(cache), c.byref(step), p(A), strides, 4, 2, p(A), c.c_float(0.1), 1, 0, p(0), p(A), p(A), c.c_size_t(scratch), p(0))
else:
    status = lib.risa_b200_cache_evict(c.byref(cache), c.byref(step), p(A), p(2 * A), 4, 32, 4, p(A), p(A), p(A), p(0))
print(status, stand_in.launch_count(), lib.risa_b200_last_error().decode())
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    if shutil.which("gcc") is None:
        pytest.skip("needs a C compiler")
    folder = tmp_path_factory.mktemp("stand_in")
    (folder / "launches.c").write_text(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", str(folder / "launches.c"), "-o", str(folder / "launches.so")], check=True)
    return folder / "launches.so"


@pytest.mark.parametrize("call,tokens,launches", [("attention", 1, 2), ("attention", 64, 4), ("weights", 1, 1), ("weights", 64, 3), ("evict", 1, 2)])
def test_nothing_is_launched_behind_a_launch_that_failed(stand_in, call, tokens, launches):
    for failing in range(launches + 1):
        env = {**os.environ, "LD_PRELOAD": str(stand_in), "FAILING_LAUNCH": str(failing)}
        run = subprocess.run([sys.executable, "-c", CALLS, str(LIBRARY), call, str(tokens)], env=env, capture_output=True, text=True, timeout=60)
        assert run.returncode == 0, run.stderr
        status, count, *_ = run.stdout.split()
        assert int(count) == min(failing + 1, launches)
        assert (int(status) == 0) == (failing == launches), run.stdout
