"""The first launch of a kernel with a raised LDS limit, by two threads at once and behind a failure.

The library's calls into the runtime go to a stand-in that is loaded before it, so this needs no GPU and launches
nothing."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = r"""
#include <stdatomic.h>
#include <time.h>
static atomic_int entered, set, launched, early;
int fail_first;
int attributes(void) { return entered; }
int launches(void) { return launched; }
int early_launches(void) { return early; }
int hipGetDevice(int *device) { *device = 0; return 0; }
int hipGetLastError(void) { return 0; }
int hipDeviceGetAttribute(int *value, int attribute, int device) { *value = 256; return 0; }
int hipFuncSetAttribute(const void *kernel, int attribute, int value) {
  if (atomic_fetch_add(&entered, 1) == 0) {
    if (fail_first) return 2;
    /* the first caller is slow: up to half a second, or until somebody launches */
    for (int i = 0; i < 500 && !launched; ++i) {
      struct timespec ms = {0, 1000000};
      nanosleep(&ms, 0);
    }
  }
  set = 1;
  return 0;
}
typedef struct { unsigned x, y, z; } three;
int __hipPushCallConfiguration(three grid, three block, unsigned long lds, void *stream) { return 0; }
int __hipPopCallConfiguration(three *grid, three *block, unsigned long *lds, void **stream) {
  *grid = *block = (three){1, 1, 1};
  *lds = 0;
  *stream = 0;
  return 0;
}
int hipLaunchKernel(const void *kernel, three grid, three block, void **args, unsigned long lds, void *stream) {
  if (!set) atomic_fetch_add(&early, 1);
  atomic_fetch_add(&launched, 1);
  return 0;
}
"""

CALLS = r"""
import ctypes as C, importlib.util, sys, threading
root, stand_in, what = sys.argv[1:4]
shim = C.CDLL(stand_in, mode=C.RTLD_GLOBAL)
spec = importlib.util.spec_from_file_location("vitk", root + "/visiontransformer_amd/vitk.py")
vitk = importlib.util.module_from_spec(spec)
spec.loader.exec_module(vitk)
d = C.CDLL(root + "/visiontransformer_amd/lib/libvitk.so")
d.vitk_last_error.restype = C.c_char_p

def newton_schulz():
    a = vitk.NewtonSchulzArgs(rows=16, cols=16, batch=1, steps=1, x=4096, ld_x=16, out=8192, ld_out=16, a=1.5, b=-0.5)
    return d.vitk_newton_schulz_f32(C.byref(a), None)

def attention_backward():
    p = C.c_void_p
    return d.vitk_sdpa_bwd(p(4096), p(8192), p(12288), C.c_int64(64), p(16384), p(20480), C.c_int64(64), p(24576), 2, 1, 64, 64,
                           C.c_float(0.125), 0, p(28672), p(32768), p(36864), C.c_int64(64), p(40960), C.c_size_t(1 << 20), None)

call = {"newton_schulz": newton_schulz, "attention": attention_backward}[what.split("/")[0]]
if what.endswith("failure"):
    C.c_int.in_dll(shim, "fail_first").value = 1
    assert call() != 0 and "LDS" in d.vitk_last_error().decode(), d.vitk_last_error()
    assert shim.launches() == 0
    assert call() == 0 and shim.attributes() == 2 and shim.launches() > 0
else:
    threads = [threading.Thread(target=call) for _ in range(2)]
    threads[0].start()
    while shim.attributes() == 0 and threads[0].is_alive():  # until it is inside the runtime
        pass
    threads[1].start()
    [t.join() for t in threads]
    assert shim.launches() >= 2
before = shim.attributes()
assert call() == 0 and shim.attributes() == before  # known by now
print("early", shim.early_launches())
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    folder = tmp_path_factory.mktemp("stand_in")
    (folder / "runtime.c").write_text(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", str(folder / "libruntime.so"), str(folder / "runtime.c")], check=True)
    return str(folder / "libruntime.so")


@pytest.mark.parametrize("what", ["newton_schulz/threads", "newton_schulz/failure", "attention/threads", "attention/failure"])
def test_no_launch_before_its_lds_limit_is_raised(stand_in, what):
    r = subprocess.run([sys.executable, "-c", CALLS, ROOT, stand_in, what], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split() == ["early", "0"], r.stdout
