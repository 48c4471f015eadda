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
