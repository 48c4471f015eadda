"""A warp's ring of copies in the kernel of single tokens (tur_b200/csrc/attend_plan.h): where a wait runs out, the copies still on their way
are exactly those that the warp then waits for, so that none can land in shared memory that is someone else's by then. On the CPU: the wait
that runs out is the simulation's."""
import ctypes
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = '#include "attend_plan.h"\nextern "C" int requested(int own, int taken, int stages) { return turq::ring_requested(own, taken, stages); }\n'


@pytest.fixture(scope="module")
def requested():
    with tempfile.TemporaryDirectory() as d:
        src, so = os.path.join(d, "shim.cpp"), os.path.join(d, "shim.so")
        with open(src, "w") as f:
            f.write(SHIM)
        subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tur_b200", "csrc"), src, "-o", so], check=True)
        return ctypes.CDLL(so).requested


@pytest.mark.parametrize("stages", [2, 3])
def test_copies_on_their_way_when_a_wait_runs_out(requested, stages):
    for own in range(12):
        for fails_at in range(own + 1):  # own: none does
            flight, free = {}, set(range(stages))  # stage -> step

            def request(step, stage):
                assert stage in free, "a copy into a stage that another one is on its way to"
                free.discard(stage)
                flight[stage] = step

            for s in range(requested(own, 0, stages)):
                request(s, s)
            n = 0
            while n < own and n != fails_at:
                assert flight.pop(n % stages) == n
                free.add(n % stages)
                if n + stages < own:
                    request(n + stages, n % stages)
                n += 1
            waited = {i % stages: i for i in range(n, requested(own, n, stages))} if n < own else {}
            assert waited == flight
