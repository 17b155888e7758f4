"""Windows of the peer transport over the life of a process (csrc/peer_rules.hpp): used again once every rank has let go, and not before.  In a
process of its own, whose windows are this test's only.  Nothing is exchanged, so nothing waits."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import json, struct, sys
sys.path.insert(0, %r)
import numpy as np
import nmfx

def context(rank):
    c = nmfx.Context(np.float32, 256, 150, 4)
    c.comm_init_p2p(rank, 2)
    return c, c.comm_p2p_export()

def window(handle):
    return struct.unpack_from("<Q", handle, 16)[0]

def pair():
    (a, ha), (b, hb) = context(0), context(1)
    a.comm_p2p_attach([ha, hb])
    b.comm_p2p_attach([ha, hb])
    return a, b, window(ha), window(hb)

out = {"rounds": []}
for _ in range(4):                                # both leave: both windows serve the next pair
    a, b, wa, wb = pair()
    a.close(), b.close()
    out["rounds"].append([wa, wb])
a, b, wa, wb = pair()
a.close()                                         # b may still store into wa
c, hc = context(0)
out["while_held"] = [wa, window(hc)]
b.close()                                         # now both are free; c's window is in use
d, hd = context(0)
e, he = context(1)
out["afterwards"] = [wa, wb, window(hd), window(he)]
c.close()                                         # nobody attached to c's window, but its handle went out
f, hf = context(0)
out["never_attached"] = [window(hc), window(hf)]
a, b, wa, wb = pair()
a.comm_p2p_attach(None)                           # let go, and map again
a.comm_p2p_attach([h for h in (a.comm_p2p_export(), b.comm_p2p_export())])
b.close()
g, hg = context(0)
out["mapped_again"] = [wb, window(hg)]
print(json.dumps(out))
"""


def test_windows_are_used_again_once_every_rank_has_let_go(built):
    r = subprocess.run([sys.executable, "-c", PROGRAM % os.path.join(ROOT, "nmf.jl_amd")], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    out = json.loads(r.stdout.splitlines()[-1])
    assert all(sorted(w) == sorted(out["rounds"][0]) for w in out["rounds"]) and len(set(out["rounds"][0])) == 2
    assert out["while_held"][0] != out["while_held"][1]
    assert sorted(out["afterwards"][:2]) == sorted(out["afterwards"][2:])
    assert out["never_attached"][0] != out["never_attached"][1]
    assert out["mapped_again"][0] != out["mapped_again"][1]
