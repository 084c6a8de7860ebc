"""A call on one device leaves the thread's current device as it was.

No GPU: the library is loaded behind a small stand-in for the HIP calls that
choose devices and launch, which counts two devices and keeps on which one each
launch was made.  Pointers stand for device memory and are never followed.
"""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = r"""
#include <stddef.h>
static int current = 0, launches = 0, elsewhere = 0, fails = 0;
typedef struct { unsigned x, y, z; } grid_t;
int hipGetDeviceCount(int* n) { *n = 2; return 0; }
int hipGetDevice(int* d) { *d = current; return 0; }
int hipSetDevice(int d) { current = d; return 0; }
int hipDeviceGetAttribute(int* v, int a, int d) { *v = 256; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
int hipGetLastError(void) { return fails; }
int hipPeekAtLastError(void) { return fails; }
int hipDeviceSynchronize(void) { return 0; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void* f, int b, size_t s) { *n = 2; return 0; }
int hipModuleOccupancyMaxActiveBlocksPerMultiprocessor(int* n, void* f, int b, size_t s) { *n = 2; return 0; }
int __hipPushCallConfiguration(grid_t g, grid_t b, size_t lds, void* stream) { return 0; }
int __hipPopCallConfiguration(grid_t* g, grid_t* b, size_t* lds, void** stream) { return 0; }
int hipLaunchKernel(const void* f, grid_t g, grid_t b, void** args, size_t lds, void* stream) {
    ++launches;
    elsewhere += current != 1;
    return 0;
}
void stand_in_set(int device, int error) { current = device; launches = elsewhere = 0; fails = error; }
int stand_in_current(void) { return current; }
int stand_in_launches(void) { return launches; }
int stand_in_elsewhere(void) { return elsewhere; }
"""

CALLS = r"""
import ctypes, sys
stand = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
from tropical_gemm import _native as nat
lib = nat.load()
P, W = 4096, 1 << 26
CALLS = {
    "tg_i8_quantize": (1, P, 8, P, P, 4, 8, None),
    "tg_i8_gemm": (1, P, 16, P, P, 16, P, None, P, 4, 8, 16, P, W, None),
    "tg_f8_quantize": (1, P, 8, 1, P, P, 4, 8, None),
    "tg_f8_dequantize": (1, P, 8, P, 1, 4, 1, P, 4, 8, None),
    "tg_f8_gemm": (1, P, 256, P, 1, 300, P, 256, P, 1, 3, None, P, 300, 300, 256, P, W, None),
    "tg_f8_backward_a": (1, P, 8, P, 16, P, 1, 1, P, 4, 8, 16, P, W, None),
    "tg_f8_backward_b": (0, P, 8, P, 16, P, 1, 4, P, 4, 8, 16, P, W, None),
    "tg_dropout": (1, P, 8, P, 8, 0.5, 1, None, 0, P, 4, 8, None),
    "tg_layer_norm": (1, 1, P, 8, P, 8, P, P, 1e-5, 0.5, 1, None, 0, P, P, P, P, 4, 8, None),
    "tg_layer_norm_backward": (1, 1, P, 8, P, 8, P, P, P, P, 8, 0.5, 1, None, 0, P, P, P, P, 4, 8, P, W, None),
    "tg_transpose": (0, P, 2 * P, 1, 64, 64, None),
    "tg_gemm_ws": (0, 0, 0, P, P, P, None, 64, 64, 64, P, W, None),
    "tg_backward_a": (0, 0, P, P, P, 16, 16, 16, None),
}
NO_LAUNCH = {"tg_synchronize": ()}
for name, rest in {**CALLS, **NO_LAUNCH}.items():
    for current in (0, 1):
        for error in (0, 1):  # a launch that fails
            stand.stand_in_set(current, error)
            rc = getattr(lib, name)(1, *rest)
            made = stand.stand_in_launches()
            assert (rc == 0) == (error == 0 or name in NO_LAUNCH), (name, rc, nat.last_error())
            assert (made > 0) == (name in CALLS) and stand.stand_in_elsewhere() == 0, (name, made)
            assert stand.stand_in_current() == current, (name, current, stand.stand_in_current())
    stand.stand_in_set(1, 0)
    assert getattr(lib, name)(2, *rest) != 0 and stand.stand_in_current() == 1  # no such device
print("kept", len(CALLS))
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    path = tmp_path_factory.mktemp("stand_in")
    (path / "hip.c").write_text(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-o", str(path / "hip.so"), str(path / "hip.c")], check=True)
    return path / "hip.so"


def test_calls_keep_the_current_device(stand_in):
    run = subprocess.run([sys.executable, "-c", CALLS, str(stand_in), os.path.join(ROOT, "tropical-gemm_amd")],
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().startswith("kept"), (run.stdout[-300:], run.stderr[-800:])
