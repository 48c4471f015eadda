"""Host-side arithmetic of the kernel of single tokens (tur_b200/csrc/attend_plan.h), compiled with g++. A warp's ring of copies: where a
wait runs out, the copies still on their way are exactly those that the warp then waits for, so that none can land in shared memory that is
someone else's by then (the wait that runs out is the simulation's). The plan of a call that also holds tiles of rows."""
import ctypes
import os
import random
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = '#include "attend_plan.h"\nextern "C" int requested(int own, int taken, int stages) { return turq::ring_requested(own, taken, stages); }\n' \
    'extern "C" void tokens(long long pairs, long long ctx, int sms, int ctas, int beside, long long* out) {\n' \
    '  const turq::TokenPlan p = turq::plan_tokens(pairs, ctx, sms, ctas, beside != 0);\n  out[0] = p.chunk; out[1] = p.chunks; out[2] = p.cluster;\n}\n'


@pytest.fixture(scope="module")
def plan():
    with tempfile.TemporaryDirectory() as d:
        src, so = os.path.join(d, "shim.cpp"), os.path.join(d, "shim.so")
        with open(src, "w") as f:
            f.write(SHIM)
        subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tur_b200", "csrc"), src, "-o", so], check=True)
        lib = ctypes.CDLL(so)
    lib.tokens.argtypes = [ctypes.c_longlong] * 2 + [ctypes.c_int] * 3 + [ctypes.POINTER(ctypes.c_longlong)]
    return lib


@pytest.mark.parametrize("stages", [2, 3])
def test_copies_on_their_way_when_a_wait_runs_out(plan, stages):
    requested = plan.requested
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


@pytest.mark.parametrize("ctas", [3, 4])
def test_clusters_beside_tiles_have_room(plan, ctas):
    """All clusters of a call run at once (up to eight chunks), or find an SM for each chunk (more), however the chunks' length was chosen."""
    rng, sms, met = random.Random(9), 148, 0
    for _ in range(4000):
        pairs, ctx = rng.choice([1, 2, 5, 8, 16, 17, 24, 40, 64, 72, 136, 300, 2000]), int(2 ** rng.uniform(4, 17))
        out = (ctypes.c_longlong * 3)()
        plan.tokens(pairs, ctx, sms, ctas, 1, out)
        chunk, chunks, cluster = out
        assert chunk % 128 == 0 and (chunks - 1) * chunk < ctx <= chunks * chunk
        assert not cluster or (2 <= chunks <= 16 and pairs * chunks <= (ctas if chunks <= 8 else 1) * sms)
        met += cluster
    assert met > 100
