"""The 4-bit kernels' place among programmatic launches: each lets its successor start only behind its own
wait. A flagged attention call (``SOLORT_DECODE_STABLE_PREFIX``) reads keys before its wait, and is right
only if what its predecessor's predecessors wrote is complete by then; the order is a race on the GPU, so
here it is read from the sources."""

from __future__ import annotations

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "solort_b200", "csrc")


def test_dependents_start_behind_the_wait():
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "int4*"))):
        with open(path) as f:
            found += re.findall(r'"(griddepcontrol[^"]*)"', f.read())
    # one statement for all of them, so that no kernel can have it the other way round
    assert found == [r"griddepcontrol.wait;\ngriddepcontrol.launch_dependents;"]


def test_every_kernel_waits():
    for name in ("int4_rows.cu", "int4_decode.cu"):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        bodies = re.split(r"__global__ void", text)[1:]
        assert len(bodies) == {"int4_rows.cu": 3, "int4_decode.cu": 2}[name]
        for body in bodies:
            assert "pdl_wait();" in body.split("\n}\n")[0]
