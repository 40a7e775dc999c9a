"""A forked child collects nothing that its parent left in reference cycles."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import gc, os
from graphsage_amd import _lib
_lib.load()

class Held:
    def __del__(self):
        if os.getpid() != parent:
            os._exit(7)

parent = os.getpid()
gc.disable()
held = Held()
held.me = held
del held
child = os.fork()
if child == 0:
    gc.collect()
    os._exit(0)
assert os.waitstatus_to_exitcode(os.waitpid(child, 0)[1]) == 0, "collected in the child"
assert gc.collect() > 0
"""


def test_parents_cycles_are_not_collected_in_a_forked_child():
    subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, check=True, timeout=120)
