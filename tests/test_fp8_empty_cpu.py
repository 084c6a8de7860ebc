"""Products and gradients of nothing: the size functions, which the calls ask
too, answer for every size and type with a zero in it, each in a process of its
own, as an arithmetic fault on the host ends one."""
import os
import subprocess
import sys

import pytest

from tropical_gemm import _native as nat

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SIZES = """
import sys
sys.path.insert(0, {path!r})
from tropical_gemm import _native as nat
lib = nat.load()
kind, P = {kind}, 4096
for m in (0, 1, 3, 64, 65, 100, 300, 5000):
    for n in (0, 1, 5, 8, 5000):
        for k in (0, 8, 128, 1000):
            if m and n and k:
                continue
            for at in (0, 1):
                need = lib.tg_f8_gemm_workspace_size(kind, P + at, k, P, k, m, n, k)
                assert need == 0, ("product", m, n, k, need)
            for size in (lib.tg_f8_backward_a_workspace_size, lib.tg_f8_backward_b_workspace_size):
                need = size(kind, P, n, m, n, k)
                assert need == 0, ("gradient", m, n, k, need)
            lib.tg_f8_gemm_plan(kind, P, k, P, k, m, n, k)
            for want_a in (0, 1):
                lib.tg_f8_backward_plan(kind, want_a, P, n, m, n, k)
print("answered")
"""


@pytest.mark.parametrize("kind", sorted(nat.FLOAT))
def test_sizes_with_a_zero(kind):
    code = SIZES.format(path=os.path.join(ROOT, "tropical-gemm_amd"), kind=nat.FLOAT[kind])
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "answered", (run.returncode, run.stderr[-500:])
