"""As in test_serving_launches_cpu: a launch that fails is its call's last, for a cache in 4 bits and for calls that move pages."""
import os
import subprocess
import sys

import pytest
from test_serving_launches_cpu import LIBRARY, stand_in  # noqa: F401

CALLS = r"""
import ctypes as c, sys
import os
stand_in = c.CDLL(os.environ["LD_PRELOAD"])
lib = c.CDLL(sys.argv[1])
lib.risa_b200_last_error.restype = c.c_char_p
class Cache(c.Structure):
    _fields_ = [(n, c.c_void_p) for n in ("keys", "values", "key_scales", "value_scales")] + [(n, c.c_int) for n in ("pages", "kv_heads", "page_size", "head_dim", "dtype_code")]
class Step(c.Structure):
    _fields_ = [(n, c.c_void_p) for n in ("page_table", "lengths", "query_offsets")] + [(n, c.c_int) for n in ("batch", "table_width", "tokens")]
A = 4096  # aligned addresses that nothing reads
call, tokens = sys.argv[2], 1 if sys.argv[2] == "step" else 64
cache, other = Cache(A, A, A, A, 8, 2, 128, 128, 5), Cache(2 * A, 2 * A, 2 * A, 2 * A, 8, 2, 128, 128, 5)
step, strides, p, much = Step(A, A, A, 1, 8, tokens), (c.c_int64 * 2)(512, 128), lambda x: c.c_void_p(x), c.c_size_t(1 << 30)
if call in ("step", "chunk"):
    status = lib.risa_b200_paged_attention_sinks(c.byref(cache), c.byref(step), p(A), strides, 4, 2, p(A), strides, p(A), c.c_float(0.1), 1, 9, 3, 3, p(A), much, p(0))
elif call == "weights":
    status = lib.risa_b200_key_weights_sinks(c.byref(cache), c.byref(step), p(A), strides, 4, 2, p(A), c.c_float(0.1), 1, 9, 3, p(0), p(A), p(A), much, p(0))
elif call == "read":
    status = lib.risa_b200_cache_read(c.byref(cache), c.byref(step), p(A), strides, p(A), strides, 2, p(0))
elif call == "fork":
    status = lib.risa_b200_fork_sequences(c.byref(cache), p(A), c.byref(step), p(A), 3, p(A), p(A), p(0))
elif call.startswith("resize"):
    status = lib.risa_b200_resize_sequences(c.byref(cache), p(A), p(A), 8, p(A), p(A), int(call[6:]), p(A), p(A), much, p(0))
else:
    status = lib.risa_b200_cache_compact(c.byref(cache), p(A), c.byref(step), c.byref(other), p(A), p(A), p(A), p(A), much, p(0))
print(status, stand_in.launch_count(), lib.risa_b200_last_error().decode())
"""


@pytest.mark.parametrize("call,launches", [("step", 2), ("chunk", 4), ("weights", 3), ("read", 1), ("fork", 1), ("resize100", 1), ("resize1000", 2), ("compact", 2)])
def test_nothing_is_launched_behind_a_launch_that_failed(stand_in, call, launches):  # noqa: F811
    for failing in range(launches + 1):
        env = {**os.environ, "LD_PRELOAD": str(stand_in), "FAILING_LAUNCH": str(failing)}
        run = subprocess.run([sys.executable, "-c", CALLS, str(LIBRARY), call], env=env, capture_output=True, text=True, timeout=60)
        assert run.returncode == 0, run.stderr
        status, count, *_ = run.stdout.split()
        assert int(count) == min(failing + 1, launches), run.stdout
        assert (int(status) == 0) == (failing == launches), run.stdout


REFUSED = CALLS[:CALLS.index("call, tokens")] + r"""
cache, strides, p, much = Cache(A, A, A, A, 8, 2, 128, 128, 5), (c.c_int64 * 2)(512, 128), lambda x: c.c_void_p(x), c.c_size_t(1 << 30)
step = Step(A, A, A, 1, 8, 64)
class Rotary(c.Structure):
    _fields_ = [("turns", c.c_void_p), ("rotary_dim", c.c_int), ("magnitude", c.c_float), ("interleaved", c.c_int)]
class Axes(c.Structure):
    _fields_ = [("axes", c.c_void_p), ("count", c.c_int), ("position_stride", c.c_int64)]
def attend(k, scale, window, sinks):
    return lib.risa_b200_paged_attention_sinks(c.byref(k), c.byref(step), p(A), strides, 4, 2, p(A), strides, p(A), c.c_float(scale), 1, window, sinks, 3, p(A), much, p(0))
def said(status, word):
    assert status != 0 and word in lib.risa_b200_last_error(), (status, lib.risa_b200_last_error())
said(attend(cache, 0.1, 0, 3), b"window")
said(attend(cache, 0.1, 9, -1), b"first keys")
said(attend(cache, 1e36, 9, 1), b"scale")          # in units of log 2 and of 2^-8 it is not finite
said(attend(Cache(A, A, None, None, 8, 2, 128, 128, 5), 0.1, 0, 0), b"scales")
said(attend(Cache(A, A, A + 4, A, 8, 2, 128, 128, 5), 0.1, 0, 0), b"aligned")
said(attend(Cache(A, A, A, A, 8, 65536, 128, 128, 5), 0.1, 0, 0), b"65535 heads")
three, rotary = (c.c_int64 * 3)(512, 128, 128), Rotary(A, 128, 1.0, 0)
for axes in (Axes(A, 0, 1), Axes(A, 9, 1), Axes(None, 2, 1)):
    said(lib.risa_b200_rotate_axes(p(A), p(A), 2, 1, 2, 3, 128, three, three, p(A), 0, c.c_int64(0), c.c_int64(1), c.byref(rotary), c.byref(axes), 0, p(0)), b"axes")
    said(lib.risa_b200_cache_append_axes(c.byref(cache), c.byref(step), p(A), strides, p(A), strides, p(A), strides, p(A), strides, 4, 2, c.byref(rotary), c.byref(axes), p(A), 0, p(0)), b"axes")
said(lib.risa_b200_cache_read(c.byref(cache), c.byref(step), p(A), strides, p(A), strides, 0, p(0)), b"float16 or bfloat16")
said(lib.risa_b200_cache_read(c.byref(cache), c.byref(step), p(A + 8), strides, p(A), strides, 2, p(0)), b"16-byte")
said(lib.risa_b200_fork_sequences(c.byref(cache), p(A), c.byref(step), p(A), 0, p(A), p(A), p(0)), b"children")
said(lib.risa_b200_resize_sequences(c.byref(cache), p(A), p(A), 8, p(A), p(A), 1, p(A), p(A), c.c_size_t(8), p(0)), b"scratch")
said(lib.risa_b200_resize_sequences(c.byref(cache), p(A), p(A), 1 << 25, p(A), p(A), 1, p(A), p(A), much, p(0)), b"2^31 - 8192")
compact = lambda other: lib.risa_b200_cache_compact(c.byref(cache), p(A), c.byref(step), c.byref(other), p(A), p(A), p(A), p(A), much, p(0))
said(compact(cache), b"another pool")
said(compact(Cache(2 * A, 2 * A, A, A, 8, 2, 64, 128, 5)), b"same kind")
assert stand_in.launch_count() == 0
"""


def test_c_entries_refuse(stand_in):  # noqa: F811
    run = subprocess.run([sys.executable, "-c", REFUSED, str(LIBRARY)], env={**os.environ, "LD_PRELOAD": str(stand_in), "FAILING_LAUNCH": "-1"},
                         capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stderr
