"""CPU test of importing the package where torch is not there."""

import os
import subprocess
import sys

import decode_opt_b200 as dg

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_star_import_needs_no_torch():
    """The package's names for the GEMM need the C library alone; the attention
    operators', found on first use, need torch."""
    code = ("import sys; sys.modules['torch'] = None\n"
            "from decode_opt_b200 import *\n"
            "import decode_opt_b200 as dg\n"
            "print(default_config(1, 7168, 16384) is not None, 'paged_attention' in dir(dg))\n"
            "try: dg.paged_attention\n"
            "except ImportError: print('needs torch')")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert out.stdout.split("\n")[:2] == ["True True", "needs torch"], out.stderr
    out = subprocess.run([sys.executable, "-c", "from decode_opt_b200 import *; print(paged_attention.__name__)"],
                         capture_output=True, text=True, cwd=ROOT)
    assert out.stdout.split() == ["paged_attention"], out.stderr
    assert dg.paged_attention.__module__ == "decode_opt_b200.attention" and "rotary" in dir(dg)
