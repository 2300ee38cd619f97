"""A batch whose work list does not fit the host's memory is an error of the call, not the end of the process."""

import os
import subprocess
import sys

CHILD = """
import ctypes, resource
from turbopolar_b200 import _lib
lib = _lib.lib()
plan, lens = _lib.PromptPlan(), (ctypes.c_int64 * 1)(1 << 29)
resource.setrlimit(resource.RLIMIT_AS, (3 << 30, 3 << 30))
# 128 query heads on one KV head: 2 tokens to an item, 2^28 items of 32 bytes.
try:
    _lib.check(lib.tp_prompt_plan_make(lens, lens, 1, 128, 1, plan, None, 0))
except RuntimeError as e:
    print(e)
lens[0] = 1000
_lib.check(lib.tp_prompt_plan_make(lens, lens, 1, 128, 1, plan, None, 0))
print(plan.q_tokens)
"""


def test_too_many_items():
    from turbopolar_b200 import build
    build.build()
    run = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert run.returncode == 0, run.stderr[-500:]
    assert "out of host memory" in run.stdout and run.stdout.endswith("1000\n")
