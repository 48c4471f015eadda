"""Attention.forward on quantized linears: padded batches, and how exact a layer is on caches of each type."""
import math

import math

import numpy as np
import pytest
import torch

import oracle
import tur_b200 as tq
from test_gpu_attention import ref_rows

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D = 512, 8, 2, 64


def linear(rng, rows, cols):
    blocks = oracle.quantize(oracle.Q8_0, (rng.standard_normal((rows, cols)) * 0.05).astype(np.float32))
    return tq.LinearX(tq.QMatMul.from_arc(tq.QTensor.new(blocks, tq.GgmlDType.Q8_0, (rows, cols))))


def layer(seed, norms=True, **kw):
    rng = np.random.default_rng(seed)
    q, k, v, o = (linear(rng, *s) for s in ((HQ * D, HIDDEN), (HKV * D, HIDDEN), (HKV * D, HIDDEN), (HIDDEN, HQ * D)))
    w = [torch.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)).cuda() if norms else None for _ in range(2)]
    return tq.Attention(q, k, v, o, D, *w, **kw), rng


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def poison():
    """What the next allocations find is NaN."""
    held = [torch.full((n,), float("nan"), device="cuda") for n in [64, 1024, 16384, 65536, 1 << 18, 1 << 20] for _ in range(8)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("dtype", [tq.GgmlDType.BF16, tq.GgmlDType.F16, tq.GgmlDType.Q8_0])
@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("new", [1, 20])
def test_tokens_of_no_sequence_do_not_read_what_memory_held(dtype, norms, new):
    # a batch padded to 2 + 3 sequences' tokens: the tokens behind the last sequence go to no slot
    block, rng = layer(1, norms)
    n, pad = 2 * new, 3 * new
    x = torch.from_numpy(rng.standard_normal((n + pad, HIDDEN)).astype(np.float32)).cuda()
    table = tq.RotaryTable.new(D, 64, base=1e4)
    pages = ints(*range(8)).view(4, 2)[[0, 1, 0, 0, 0]].contiguous()
    pos = torch.arange(new, dtype=torch.int32, device="cuda").repeat(5)
    slots = torch.cat([p * 16 + torch.arange(new, device="cuda") for p in (0, 2)] + [torch.full((pad,), -1, device="cuda")])
    starts, contexts = ints(0, new, n, n, n, n), ints(new, new, 0, 0, 0)
    for mode in (tq.Mode.AUTO, tq.Mode.EXACT_F32):
        got = []
        for _ in range(2):
            cache = tq.KvCache.new(dtype, 8, 16, HKV, D)
            poison()
            got.append(block.forward(x, cache, table, pos, slots, starts, contexts, pages, max_new=new, max_context=new, mode=mode))
        assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1])
        cache = tq.KvCache.new(dtype, 8, 16, HKV, D)
        alone = block.forward(x[:n], cache, table, pos[:n], slots[:n], starts[:3], contexts[:2], pages[:2], max_new=new, max_context=new, mode=mode)
        # the linears may take another kernel and the contexts another cut: a few roundings to 16 bits (bf16: 2^-8 each)
        assert ((alone - got[0][:n]).norm() / alone.norm()).item() < 2.0 ** -6
    tq.context().poll_status()


@pytest.mark.parametrize("dtype,q_dtype,bound", [(tq.GgmlDType.F16, torch.float16, 2.0 ** -9), (tq.GgmlDType.F16, torch.bfloat16, 2.0 ** -7),
                                                 (tq.GgmlDType.BF16, torch.bfloat16, 2.0 ** -6), (tq.GgmlDType.Q8_0, torch.float16, 2.0 ** -6)])
@pytest.mark.parametrize("cuts", [[0, 150], [0, 140] + list(range(141, 151))])
def test_a_layer_is_as_exact_as_its_types(dtype, q_dtype, bound, cuts):
    # In rms of a row's norm, independent roundings r = eps / 2 / sqrt(3) each (f16 2.8e-4, bf16 2.3e-3; Q8_0, steps of amax / 127 of 32 normal
    # numbers, 5e-3): values r, weights r, and keys and queries, whose normalised heads of 64 move a score by r sqrt(64) / 8, r each. The
    # output is f32. F16: 2 r = 5.6e-4 with f16 queries, 2.4e-3 with bf16 ones; BF16: 2 r = 4.5e-3; Q8_0: sqrt(2) r = 7e-3 of keys and values.
    # The bounds are two to three and a half times that.
    block, rng = layer(2, q_dtype=q_dtype)
    n, mode = 150, tq.Mode.EXACT_F32
    x = torch.from_numpy(rng.standard_normal((n, HIDDEN)).astype(np.float32)).cuda()
    table = tq.RotaryTable.new(D, n, base=1e4)
    freqs = [1e4 ** (-2 * i / D) for i in range(D // 2)]
    q, k, v = (l.forward(x, mode=mode).unflatten(1, (-1, D)) for l in (block.q, block.k, block.v))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    qr = ref_rows(q, block.q_norm, 1e-6, freqs, pos, False)
    kr = ref_rows(k, block.k_norm, 1e-6, freqs, pos, False).repeat_interleave(HQ // HKV, 1)
    z = torch.einsum("nhd,chd->hnc", qr, kr) / D ** 0.5
    z = z.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
    y = torch.einsum("hnc,chd->nhd", torch.softmax(z, -1), v.double().repeat_interleave(HQ // HKV, 1))
    want = block.o.forward(y.float().flatten(1), mode=mode).double()
    pages = torch.randperm(12, device="cuda", dtype=torch.int32)[None, :10].contiguous()
    cache = tq.KvCache.new(dtype, 12, 16, HKV, D)
    got = []
    for a, b in zip(cuts, cuts[1:]):
        t = pos[a:b]
        slots = pages[0].long()[t.long() // 16] * 16 + t.long() % 16
        got.append(block.forward(x[a:b], cache, table, t, slots, ints(0, b - a), ints(b), pages, mode=mode))
    assert ((torch.cat(got).double() - want).norm() / want.norm()).item() < bound
    tq.context().poll_status()


def test_types_of_queries_that_no_layer_has():
    for bad in (torch.float32, torch.int8):
        with pytest.raises(tq.TurqError) as e:
            layer(3, q_dtype=bad)
        assert e.value.status == 3
    block, _ = layer(3, q_dtype=torch.float16)
    cache, table = tq.KvCache.new(tq.GgmlDType.BF16, 1, 16, HKV, D), tq.RotaryTable.new(D, 16)
    with pytest.raises(tq.TurqError) as e:  # a BF16 cache multiplies in bf16
        block.forward(torch.zeros(1, HIDDEN, device="cuda"), cache, table, ints(0), torch.zeros(1, dtype=torch.int64, device="cuda"), ints(0, 1), ints(1),
                      ints(0)[None])
    assert e.value.status == 3
