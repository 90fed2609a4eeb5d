"""Waits and barriers written as assembly have to tell the compiler that memory is what they order: without the clobber it
may move a plain LDS store past the wait that publishes it, or a read past the wait before its place is filled again."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zero-tvm_amd", "csrc")


def functions(name):
    """name -> body of the one-statement device functions of a header"""
    text = open(os.path.join(CSRC, name)).read()
    return dict(re.findall(r"__device__ __forceinline__ void (\w+)\([^)]*\) \{(.*?)\n?\}", text, re.S))


def test_waits_and_barriers_clobber_memory():
    bodies = functions("mma.h")
    for name in ("wait_vm", "wait_lgkm", "wg_barrier", "dma16", "dma4"):
        assert re.search(r'asm volatile\(.*"memory"', bodies[name], re.S), name
