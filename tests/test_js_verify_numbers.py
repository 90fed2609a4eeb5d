"""The JavaScript host takes counts as they are or not at all."""
import os
import subprocess

from .test_js_host import NODE, ROOT, ensure_addon, needs_node


@needs_node
def test_counts_are_whole_numbers():
    ensure_addon()
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "verify_numbers_cpu.js")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "js verify number checks ok" in r.stdout, r.stdout + r.stderr
