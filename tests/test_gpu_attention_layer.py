"""Attention.forward on quantized linears: padded batches, and how exact a layer is on caches of each type."""
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
