"""What the native binding remembers of the streams' scratch, while the Python function that
it asks for more changes it (another thread's request or `forget` in the meantime).  Host
bookkeeping, no GPU needed; in a process of its own, since a fault there is one of memory."""
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parents[1] / "simsd-release_b200"

CHILD = """
import gc, sys
sys.path.insert(0, sys.argv[1])
import torch
from kernels import _binding as native

made = []
inside = None


def stream_scratch(index, stream, nbytes, zeroed):
    global inside
    if inside is not None:
        act, inside = inside, None
        act()
    made.append((4096 * (len(made) + 1), nbytes, object()))
    return made[-1]


def held():
    # references beyond the list's, the loop's and getrefcount's own
    return [sys.getrefcount(t) - 3 for t in made]


native.bind({}, lambda index: 0, stream_scratch)
assert native.scratch(0, 7, 100) == (4096, 100)
assert native.scratch(0, 7, 100) == (4096, 100) and native.scratch(0, 7, 50) == (4096, 100)
base = held()
assert len(base) == 1
one = base[0]                       # what one reference of the binding counts as

for round in range(200):
    n = len(made)
    if sys.argv[2] == "forget":
        inside = native.forget
        size = 200 + round
        assert native.scratch(0, 7, size) == (4096 * (n + 1), size)
        live = [n]
    elif sys.argv[2] == "grow":     # another thread asks for more of the same stream meanwhile
        size = 1000 * (round + 1)
        inside = lambda: native.scratch(0, 7, size + 500)
        # whichever of the two is kept, it is one that was made and is large enough
        at, nbytes = native.scratch(0, 7, size)
        assert nbytes >= size and (at, nbytes) in [t[:2] for t in made[n:]]
        live = [i for i, t in enumerate(made) if t[:2] == native.scratch(0, 7, 1)]
        assert len(live) == 1 and live[0] >= n
    else:                           # other streams are remembered meanwhile
        inside = lambda: [native.scratch(0, 100 + round * 8 + k, 10) for k in range(8)]
        size = 200 + round
        native.scratch(0, 7, size)
        live = None
    junk = [bytearray(80) for _ in range(50)]          # freed memory is used again
    if live is not None:
        refs = held()
        assert [i for i, r in enumerate(refs) if r == one] == live and all(r in (one, one - 1) for r in refs), refs
native.forget()
assert all(r == one - 1 for r in held())
del made[:]
gc.collect()
print("fine")
"""


def run(kind):
    r = subprocess.run([sys.executable, "-c", CHILD, str(PKG), kind], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", (r.returncode, r.stdout, r.stderr[-2000:])


def test_forget_while_more_is_asked_for():
    run("forget")


def test_another_request_while_more_is_asked_for():
    run("grow")


def test_other_streams_while_more_is_asked_for():
    run("others")
