"""What importing the package brings with it."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


def test_the_interpreter_needs_no_torch():
    """A star import included; the serving operators are imported by name, and say what is missing."""
    r = _run("import sys; sys.modules['torch'] = None\n"
             "from ktir_cpu_b200 import *\n"
             "KTIRInterpreter, KTIRParser, HardwareConfig\n"
             "import ktir_cpu_b200 as K\n"
             "assert 'kv_append' in dir(K)\n"
             "try:\n    K.kv_append\nexcept ImportError:\n    print('no torch')")
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == "no torch"


def test_the_serving_operators_are_found_by_name():
    r = _run("from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention, rotary_table")
    assert r.returncode == 0, r.stderr
