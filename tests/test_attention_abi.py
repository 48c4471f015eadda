"""The cache's geometry and the null checks of the entries between attn_q|k|v and attn_output (no GPU needed)."""
import ctypes

import pytest

import tur_b200 as tq
from tur_b200 import _lib
from tur_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def up(n):
    return (n + 255) // 256 * 256


@pytest.mark.parametrize("pages,page,heads,d", [(1, 16, 1, 64), (7, 32, 3, 128), (100003, 256, 8, 128)])
def test_cache_bytes(lib, pages, page, heads, d):
    rows = pages * page * heads
    for t in (1, 30):
        assert lib.turq_kv_cache_bytes(t, pages, page, heads, d) == 2 * up(rows * d * 2)
    assert lib.turq_kv_cache_bytes(8, pages, page, heads, d) == 2 * up(rows * d) + 2 * up(rows * d // 32 * 2)


@pytest.mark.parametrize("bad", [(0, 4, 16, 2, 64), (12, 4, 16, 2, 64), (1, 0, 16, 2, 64), (1, -1, 16, 2, 64), (1, 4, 15, 2, 64), (1, 4, 8, 2, 64), (1, 4, 512, 2, 64),
                                 (1, 4, 16, 0, 64), (1, 4, 16, 2, 80), (1, 2 ** 31, 16, 1, 64), (1, 2 ** 28, 16, 8, 64)])
def test_shapes_that_no_cache_has(lib, bad):
    assert lib.turq_kv_cache_bytes(*bad) == 0


def test_null_arguments_are_rejected_not_dereferenced(lib):
    h = ctypes.c_void_p()
    assert lib.turq_kv_cache_create(None, 1, 4, 16, 2, 64, None, 0, ctypes.byref(h)) == 1 and not h.value
    assert lib.turq_kv_cache_free(None) == 1
    assert lib.turq_kv_cache_layout(None, None, None) == 1
    assert lib.turq_kv_attention_workspace(None, 1, 1, 8, 1, 100) == 0
    assert lib.turq_rope_table(None, None, 64, 10, 1.0, None, None) == 1
    assert lib.turq_qk_norm_rope(None, None, 0, None, 0, 0, 1, 1, 1, 64, None, None, 0.0, None, 1, 64, 0, None, 0, None, None, None) == 1
    assert lib.turq_kv_append(None, None, None, 0, None, 0, None, 0, 0, 1, 1, None, None, 0.0, None, 1, 64, 0, None, None, 0, None, None) == 1
    assert lib.turq_kv_write(None, None, None, 0, None, 0, 0, 1, None, None) == 1
    assert lib.turq_kv_read(None, None, None, 1, 0, None, None, None) == 1
    assert lib.turq_kv_attention(None, None, None, 0, 1, 1, 1, None, None, None, 1, 1, 1, 1, 1.0, 1, 1, None, None, 0, None) == 1


@pytest.mark.parametrize("kwargs", [{"base": 1.0}, {"base": 0.0}, {"base": -2.0}, {"base": float("nan")}, {"base": float("inf")},
                                    {"scaling": {"type": "linear", "factor": 0.5}}, {"scaling": {"type": "linear", "factor": float("nan")}},
                                    {"scaling": {"type": "yarn", "factor": float("inf"), "original": 100}}, {"scaling": {"type": "yarn", "factor": 2.0}},
                                    {"scaling": {"type": "yarn", "factor": 2.0, "original": 0}}, {"scaling": {"type": "other"}}])
def test_tables_that_no_model_has(kwargs):
    with pytest.raises(tq.TurqError):
        tq.RotaryTable.new(64, 16, **kwargs)


@pytest.mark.parametrize("dim,base,original,factor,ramp", [(64, 1e4, 65536, 8.0, (20, 33)), (128, 1e4, 131072, 4.0, (45, 70)), (64, 1e4, 2048, 4.0, (8, 21)),
                                                           (128, 1e6, 32768, 4.0, (23, 40)), (16, 1e4, 10 ** 9, 2.0, (13, 15))])
def test_yarn_blends_between_its_two_pairs(dim, base, original, factor, ramp, monkeypatch):
    """The pairs that turn beta_fast = 32 and beta_slow = 1 times over the original positions, as numbers between pairs: rounded outwards and held
    to 0 .. dim - 1, which lies behind the last pair (dim / 2 - 1). Frequencies go from kept to divided by the factor linearly in between."""
    import math
    for turns, end, rounded in ((32, ramp[0], math.floor), (1, ramp[1], math.ceil)):
        # base^(-2 p / dim) * original = 2 pi turns
        assert min(dim - 1, max(0, rounded(dim / 2 * math.log(original / (2 * math.pi * turns), base)))) == end
    made = {}
    monkeypatch.setattr(tq.RotaryTable, "from_frequencies", classmethod(lambda cls, freqs, n, interleaved, scale, device, ctx: made.update(freqs=freqs, scale=scale)))
    tq.RotaryTable.new(dim, 16, base=base, scaling={"type": "yarn", "factor": factor, "original": original})
    assert made["scale"] == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-15) and len(made["freqs"]) == dim // 2
    for i, f in enumerate(made["freqs"]):
        kept = 1 - min(1.0, max(0.0, (i - ramp[0]) / (ramp[1] - ramp[0])))
        plain = base ** (-2 * i / dim)
        assert f == pytest.approx(plain * kept + plain / factor * (1 - kept), rel=1e-13), i
        if plain * original > 2 * math.pi:  # more than one turn: not stretched all the way
            assert f > plain / factor * (1 + 1e-9)


@pytest.mark.parametrize("betas", [{"beta_fast": 0}, {"beta_slow": 0.0}, {"beta_fast": -3}, {"beta_slow": float("nan")}, {"beta_fast": float("inf")},
                                   {"beta_fast": 1, "beta_slow": 32}])
def test_yarn_ramps_that_no_table_has(betas):
    with pytest.raises(tq.TurqError) as e:
        tq.RotaryTable.new(64, 16, scaling={"type": "yarn", "factor": 2.0, "original": 100, **betas})
    assert e.value.status == 1
