"""Index arithmetic of attention over a paged cache (tur_b200/csrc/attend_plan.h), compiled with g++ and checked on the CPU: what the
device arrays say is cut to the call's bounds, chunks cover every context, there are blocks for every tile and room for every piece."""
import ctypes
import os
import random
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r"""
#include "attend_plan.h"
typedef long long ll;
extern "C" void span(ll lo, ll hi, ll ctx, ll n_tokens, ll max_new, ll max_context, ll* out) {
  const turq::Span s = turq::cut_span(lo, hi, ctx, n_tokens, max_new, max_context);
  out[0] = s.first; out[1] = s.n; out[2] = s.ctx; out[3] = s.cut;
}
extern "C" ll seen(ll n, ll ctx, ll t, int causal) { turq::Span s{0, n, ctx, false}; return turq::keys_seen(s, t, causal); }
extern "C" void tokens(ll pairs, ll max_context, int sms, int ctas, ll* out) {
  const turq::TokenPlan p = turq::plan_tokens(pairs, max_context, sms, ctas);
  out[0] = p.chunk; out[1] = p.chunks; out[2] = p.cluster;
}
extern "C" ll blocks(ll n_tokens, ll n_seqs, ll group, ll heads) { return turq::tile_blocks(n_tokens, n_seqs, group, heads); }
extern "C" ll pieces(ll n_tokens, ll n_seqs, ll group, ll heads, ll max_context, int sms) { return turq::plan_tile_pieces(n_tokens, n_seqs, group, heads, max_context, sms); }
extern "C" ll cost(int s, int ctas, int iters, int pieces, int sms) { return turq::tile_split_cost(s, ctas, iters, pieces, sms); }
"""
SMS = 148


@pytest.fixture(scope="module")
def plan():
    with tempfile.TemporaryDirectory() as d:
        src, so = os.path.join(d, "shim.cpp"), os.path.join(d, "shim.so")
        with open(src, "w") as f:
            f.write(SHIM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tur_b200", "csrc"), src, "-o", so], check=True)
        lib = ctypes.CDLL(so)
    q = ctypes.c_longlong
    lib.span.argtypes = [q] * 6 + [ctypes.POINTER(q)]
    lib.seen.argtypes, lib.seen.restype = [q, q, q, ctypes.c_int], q
    lib.tokens.argtypes = [q, q, ctypes.c_int, ctypes.c_int, ctypes.POINTER(q)]
    lib.blocks.argtypes, lib.blocks.restype = [q] * 4, q
    lib.pieces.argtypes, lib.pieces.restype = [q] * 5 + [ctypes.c_int], q
    lib.cost.restype = q
    return lib


def ask(f, *a, n=4):
    out = (ctypes.c_longlong * n)()
    f(*a, out)
    return list(out)


@pytest.mark.parametrize("lo,hi,ctx,want", [
    (3, 10, 50, [3, 7, 50, 0]), (3, 3, 50, [3, 0, 50, 0]), (0, 0, 0, [0, 0, 0, 0]),
    (3, 100, 50, [3, 8, 50, 1]),                        # more than max_new, and behind the last row
    (15, 30, 50, [15, 5, 50, 1]), (25, 30, 50, [20, 0, 50, 1]), (-4, 2, 50, [0, 2, 50, 1]), (9, 4, 50, [9, 0, 50, 1]),
    (0, 1, -1, [0, 1, 0, 1]), (0, 1, 101, [0, 1, 100, 1]), (0, 2 ** 31 - 1, 2 ** 31 - 1, [0, 8, 100, 1]), (-2 ** 31, -2 ** 31, -2 ** 31, [0, 0, 0, 1])])
def test_spans_are_cut_to_the_call(plan, lo, hi, ctx, want):
    got = ask(plan.span, lo, hi, ctx, 20, 8, 100)
    assert got == want
    assert 0 <= got[0] and got[0] + got[1] <= 20 and got[1] <= 8 and 0 <= got[2] <= 100


def test_keys_seen(plan):
    assert [plan.seen(3, 10, t, 1) for t in range(3)] == [8, 9, 10]
    assert [plan.seen(4, 2, t, 1) for t in range(4)] == [0, 0, 1, 2]
    assert [plan.seen(4, 2, t, 0) for t in range(4)] == [2] * 4
    assert plan.seen(1, 0, 0, 1) == 0


@pytest.mark.parametrize("ctas", [3, 4])
def test_chunks_cover_every_context(plan, ctas):
    rng = random.Random(5)
    for _ in range(3000):
        pairs, ctx = rng.choice([1, 2, 8, 40, 64, 512, 5000, 65535 * 8]), int(2 ** rng.uniform(0, 21))
        chunk, chunks, cluster = ask(plan.tokens, pairs, ctx, SMS, ctas, n=3)
        assert chunk % 128 == 0 and 128 <= chunk <= 8192         # whole steps of the kernel; the page list in shared memory
        assert (chunks - 1) * chunk < ctx <= chunks * chunk
        assert not cluster or (2 <= chunks <= 16 and pairs * chunks <= ctas * SMS)
        # few sequences do not leave most of the GPU idle while their context could fill it
        if pairs * ctx >= 128 * SMS * 8 and pairs <= SMS:
            assert pairs * chunks >= SMS // 3


def test_blocks_and_pieces_suffice(plan):
    rng = random.Random(6)
    for _ in range(3000):
        group, heads = rng.choice([1, 2, 3, 5, 8, 17, 32, 100, 128]), rng.choice([1, 2, 8, 10])
        new = [rng.choice([0, 1, 2, 17, 63, 64, 65, 300, 4096]) for _ in range(rng.choice([1, 1, 2, 7, 60]))]
        ctx = [n + rng.choice([0, 1, 100, 9000]) for n in new]
        per_cta = 128 // group * 2
        big = [(n, c) for n, c in zip(new, ctx) if n * group > 16]
        ctas = sum(-(-n // per_cta) for n, _ in big) * heads
        assert plan.blocks(sum(new), len(new), group, heads) >= ctas
        room = plan.pieces(sum(new), len(new), group, heads, max(ctx), SMS)
        iters = max([-(-c // 128) for _, c in big], default=0)
        costs = [min(plan.cost(s, ctas, iters, room, SMS), 0x3FFFFFF) for s in range(1, 33)]
        s = costs.index(min(costs)) + 1
        assert s == 1 or (s * ctas <= room and 2 * s <= iters)
        assert costs[s - 1] <= costs[0] and room <= 3 * SMS
        # one chunk on a long context is spread over the GPU
        if ctas == 8 and iters >= 150:
            assert s * ctas >= 96
