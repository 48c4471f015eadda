"""Head norms with rotation, the paged cache and attention over it against plain implementations in 64 bits.

Tolerances. A rounding to t is off by at most eps_t / 2 of the value (bf16 2^-8, f16 2^-11, f32 2^-24).
Rows of q and k: everything in f32, rounded once: half a step of the output type, plus what f32 loses on the way
(a sum of 128 squares, a division, a product, two products and a sum: under 2^-18 of the largest element of the pair).
Attention, per element, with w the exact softmax weights and A = sum_j w_j |v_j|:
  a score is a sum of D products, exact products summed in f32 (D 2^-24 of sum |q k|), of keys that Q8_0 rounds to f16
  (2^-11); ds = scale * max_j sum |q k| * (that). A weight is then off by a factor e^(2 ds) with its sum, is rounded to the
  cache's 16-bit type (2^-8 or 2^-11), and comes out of an exponential that is good to 2^-12; values are rounded like keys.
  So |out - exact| <= A (2 ds + 2 e_p + e_v + 2^-11) + half a step of the output type of |exact| + A.
  f16 has no steps finer than 2^-24: what is rounded to it (weights, whose largest is at least 1 before the division by
  their sum; keys and values of Q8_0; outputs) is off by up to 2^-25 however small it is. That adds 2^-25 sum_j |v_j|
  for the weights, 2^-25 for the values, 2^-25 for the output and scale 2^-25 sum |q| to a score.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import tur_b200 as tq
from tur_b200 import _lib

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
GT = {torch.float16: tq.GgmlDType.F16, torch.bfloat16: tq.GgmlDType.BF16, "q8_0": tq.GgmlDType.Q8_0}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


# ---- norms and rotation

def ref_rows(x, w, eps, freqs, positions, interleaved, scale=1.0):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    half = len(freqs)
    ang = (positions.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device=x.device))[:, None, :]
    c, s = ang.cos() * scale, ang.sin() * scale
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def close_rows(got, want, out_dtype):
    # a pair's two elements mix in the rotation: what f32 loses is relative to the larger of a row
    tol = want.abs() * HALF[out_dtype] + want.abs().amax(-1, keepdim=True) * 2.0 ** -18
    bad = ((got.double() - want).abs() > tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {(got.double() - want).abs().max().item()}"


@pytest.mark.parametrize("x_dtype,out_dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (128, 24, True), (128, 8, False), (64, 64, False),
                                               (64, 32, True), (64, 24, False)])
@pytest.mark.parametrize("n,hq,hkv", [(1, 4, 1), (3, 5, 5), (131, 16, 8)])
def test_norm_and_rotation(x_dtype, out_dtype, d, rot, interleaved, n, hq, hkv):
    g = gen(1)
    q, k = (randn(g, n, h, d).mul_(3).to(x_dtype) for h in (hq, hkv))
    wq, wk = 1 + 0.3 * randn(g, d), 1 + 0.3 * randn(g, d)
    freqs = [1e4 ** (-2 * i / rot) for i in range(rot // 2)]
    pos = torch.randint(0, 40000, (n,), device="cuda", generator=g, dtype=torch.int32)
    table = tq.RotaryTable.from_frequencies(freqs, 40000, interleaved)
    qo, ko = tq.qk_norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk, eps=1e-5, out_dtype=out_dtype)
    close_rows(qo, ref_rows(q, wq, 1e-5, freqs, pos, interleaved), out_dtype)
    close_rows(ko, ref_rows(k, wk, 1e-5, freqs, pos, interleaved), out_dtype)
    # one weight, none, in place, into views of one matrix
    qo, ko = tq.qk_norm_rope(q, k, pos, table, k_weight=wk, eps=1e-5, out_dtype=out_dtype)
    close_rows(qo, ref_rows(q, None, 0, freqs, pos, interleaved), out_dtype)
    close_rows(ko, ref_rows(k, wk, 1e-5, freqs, pos, interleaved), out_dtype)
    fused = torch.cat((q.flatten(1), k.flatten(1)), 1)
    qv, kv = fused[:, :hq * d].unflatten(1, (hq, d)), fused[:, hq * d:].unflatten(1, (hkv, d))
    assert all(torch.equal(a, b) for a, b in zip(tq.qk_norm_rope(qv, kv, pos, table, k_weight=wk, eps=1e-5, out_dtype=out_dtype), (qo, ko)))
    want = tq.qk_norm_rope(q, k, pos, table, q_weight=wq, out_dtype=x_dtype)
    q2, k2 = q.clone(), k.clone()
    tq.qk_norm_rope(q2, k2, pos, table, q_weight=wq, out_dtype=x_dtype, q_out=q2, k_out=k2)
    assert torch.equal(q2, want[0]) and torch.equal(k2, want[1])
    tq.context().poll_status()


def test_rotary_tables():
    t = tq.RotaryTable.new(128, 200001, base=1e6)
    want = np.outer([0, 1, 77, 200000], 1e6 ** (-np.arange(64) / 64.0))
    got = t.table[[0, 1, 77, 200000]].cpu().double().numpy()
    assert np.abs(got[..., 0] - np.cos(want)).max() <= 2.0 ** -24 and np.abs(got[..., 1] - np.sin(want)).max() <= 2.0 ** -24
    lin = tq.RotaryTable.new(64, 100, base=1e4, scaling={"type": "linear", "factor": 4.0})
    assert (lin.table[40] - tq.RotaryTable.new(64, 100, base=1e4).table[10]).abs().max() <= 2.0 ** -23
    yarn = tq.RotaryTable.new(64, 9000, base=1e4, scaling={"type": "yarn", "factor": 4.0, "original": 2048})
    m = 0.1 * math.log(4.0) + 1
    plain = tq.RotaryTable.new(64, 9000, base=1e4)
    assert (yarn.table[8000, 0] - plain.table[8000, 0] * m).abs().max() <= 2.0 ** -22      # the fastest pair keeps its angle
    assert (yarn.table[8000, 31] - plain.table[2000, 31] * m).abs().max() <= 2.0 ** -22    # the slowest is stretched


def test_positions_outside_the_table_give_zero_rows():
    g = gen(2)
    table = tq.RotaryTable.new(64, 16)
    pos = torch.tensor([3, 16, -1, 15], dtype=torch.int32, device="cuda")
    q, k, v = randn(g, 4, 2, 64), randn(g, 4, 1, 64), randn(g, 4, 1, 64)
    cache = tq.KvCache.new(tq.GgmlDType.F16, 1, 16, 1, 64)
    cache.memory.fill_(0x11)
    before = cache.k_pages.clone()
    qo = cache.append(q, k, v, pos, table, torch.arange(4, device="cuda"))
    assert not qo[1].any() and not qo[2].any() and qo[0].any() and qo[3].any()
    assert torch.equal(cache.k_pages[:, :, 1:3], before[:, :, 1:3]) and torch.equal(cache.v_pages[:, :, 1:3], before[:, :, 1:3])
    with pytest.raises(tq.TurqError):
        tq.context().poll_status()
    tq.context().poll_status()


# ---- the cache

def ref_q8(x):
    """Quants and f16 scales of Q8_0, numpy in f32 steps."""
    b = x.float().cpu().numpy().reshape(-1, 32)
    top = np.abs(b).max(1)
    d = (top / np.float32(127)).astype(np.float32)
    inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d > 0)
    y = (b * inv[:, None]).astype(np.float64)
    return np.trunc(y + np.copysign(0.5, y)).reshape(x.shape), d.astype(np.float16).reshape(*x.shape[:-1], -1)


def deq(q, d):
    return torch.from_numpy((q.reshape(-1, 32) * d.astype(np.float64).reshape(-1, 1)).reshape(q.shape)).cuda()


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, "q8_0"])
@pytest.mark.parametrize("d,heads,page", [(128, 8, 16), (64, 3, 64), (128, 1, 256)])
@pytest.mark.parametrize("n", [0, 1, 77])
def test_write_and_read(x_dtype, kind, d, heads, page, n):
    g = gen(3)
    cache = tq.KvCache.new(GT[kind], 9, page, heads, d)
    k, v = randn(g, n, heads, d).to(x_dtype), (randn(g, n, heads, d) * 5).to(x_dtype)
    if n > 1:
        k[1, 0] = 0                                # a block of zeros
        v[1] *= 1e-6 if x_dtype != torch.float16 else 1e-2
    slots = torch.randperm(9 * page, device="cuda", generator=g)[:n]
    cache.write(k, v, slots)
    for got, pages, x in zip(cache.read(slots), (cache.k_pages, cache.v_pages), (k, v)):
        if kind == "q8_0":
            assert torch.equal(got.double(), deq(*ref_q8(x)) if n else got.double())
        else:
            assert torch.equal(got, x.to(kind).float())
            assert torch.equal(pages[slots // page, :, slots % page], x.to(kind))
    for t in (torch.bfloat16, torch.float16):
        assert all(torch.equal(a, b.to(t)) for a, b in zip(cache.read(slots, t), cache.read(slots)))
    # padding: skipped on the way in, zeros on the way out; the other slots keep what they hold
    before = cache.memory.clone()
    pad = torch.full((n,), -1, device="cuda", dtype=torch.int64)
    cache.write(k, v, pad)
    assert torch.equal(before, cache.memory) and not any(t.any() for t in cache.read(pad))
    tq.context().poll_status()
    if n:
        bad = slots.clone()
        bad[0] = 9 * page
        cache.write(k, v, bad)
        assert torch.equal(before, cache.memory)
        with pytest.raises(tq.TurqError):
            tq.context().poll_status()
        assert not cache.read(bad)[0][0].any()
        with pytest.raises(tq.TurqError):
            tq.context().poll_status()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, "q8_0"])
@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (128, 64, False), (128, 24, False), (128, 64, True), (64, 64, False), (64, 24, True)])
def test_append_is_rotation_and_write(kind, d, rot, interleaved):
    g = gen(4)
    n, hq, hkv = 45, 6, 3
    fused = randn(g, n, (hq + 2 * hkv) * d)
    q, k, v = (t.unflatten(1, (-1, d)) for t in fused.split([hq * d, hkv * d, hkv * d], 1))
    wq, wk = 1 + 0.2 * randn(g, d), 1 + 0.2 * randn(g, d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda") + 90
    table = tq.RotaryTable.new(rot, 200, base=1e4, interleaved=interleaved)
    a, b = (tq.KvCache.new(GT[kind], 8, 16, hkv, d) for _ in range(2))
    slots = torch.randperm(128, device="cuda", generator=g)[:n]
    slots[7] = -5
    qo = a.append(q, k, v, pos, table, slots, q_weight=wq, k_weight=wk, out_dtype=torch.float16)
    q32, k32 = tq.qk_norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk, out_dtype=torch.float32)
    assert torch.equal(qo, q32.half())
    b.write(k32, v.contiguous(), slots)
    assert torch.equal(a.memory, b.memory) and a.memory.any()
    tq.context().poll_status()


def test_slots_beyond_32_bits():
    """Pages whose elements pass 2^31 in each plane."""
    g = gen(5)
    d, heads, page = 128, 8, 256
    n_pages = 2 ** 31 // (d * heads * page) + 3
    for kind in (torch.float16, "q8_0"):
        cache = tq.KvCache.new(GT[kind], n_pages, page, heads, d)
        n = 300
        k, v, q = randn(g, n, heads, d), randn(g, n, heads, d), randn(g, 40, 2 * heads, d).half()
        table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
        t = torch.arange(n, device="cuda")
        slots = table[0].long()[t // page] * page + t % page
        cache.write(k, v, slots)
        kr, vr = cache.read(slots)
        assert torch.equal(kr.double(), deq(*ref_q8(k)) if kind == "q8_0" else k.half().double())
        for new in (1, 40):
            starts, ctx = torch.tensor([0, new], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
            check_attention(cache.attend(q[:new], starts, ctx, table), q[:new], kr, vr, [(new, n)], kind=kind)
        del cache
        torch.cuda.empty_cache()


# ---- attention

def check_attention(got, q, k, v, spans, *, kind, scale=None, causal=True, out_dtype=None):
    """k, v: what the cache stands for, the contexts of the sequences one behind the other; got [tokens, heads, d]."""
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    out_dtype = out_dtype or got.dtype
    group = q.shape[1] // k.shape[1]
    p16 = torch.bfloat16 if kind is torch.bfloat16 else torch.float16
    e_k = HALF[torch.float16] if kind == "q8_0" else 0.0
    at = kat = 0
    for new, ctx in spans:
        qs = q[at:at + new].double()
        ks, vs = (t[kat:kat + ctx].double().repeat_interleave(group, 1) for t in (k, v))
        if new:
            z = torch.einsum("nhd,chd->hnc", qs, ks) * scale
            za = torch.einsum("nhd,chd->hnc", qs.abs(), ks.abs()) * scale
            if causal:
                last = ctx - new + torch.arange(new, device="cuda")
                hidden = torch.arange(ctx, device="cuda")[None] > last[:, None]
                z = z.masked_fill(hidden, -math.inf)
                za = za.masked_fill(hidden, 0.0)
            w = torch.nan_to_num(torch.softmax(z, -1)) if ctx else z
            want, spread = (torch.einsum("hnc,chd->nhd", w, t) for t in (vs, vs.abs()))
            ds = (za.amax(-1) if ctx else torch.zeros(z.shape[:2], device="cuda")).T[..., None] * (e_k + d * 2.0 ** -24)
            tiny = {True: 2.0 ** -25, False: 0.0}
            if kind == "q8_0":
                ds = ds + scale * 2.0 ** -25 * qs.abs().sum(-1, keepdim=True)
            floor = tiny[p16 is torch.float16] * vs.abs().sum(0)[None] + tiny[kind == "q8_0"] + tiny[out_dtype is torch.float16]
            tol = floor + spread * (2 * ds + 2 * HALF[p16] + e_k + 2.0 ** -11) * (1 + HALF[out_dtype]) + want.abs() * HALF[out_dtype]
            err = (got[at:at + new].double() - want).abs()
            bad = ~(err <= tol + 1e-30)
            assert not bad.any(), f"sequence ({new}, {ctx}): {int(bad.sum())} of {bad.numel()} off, worst {err.max().item()} " \
                                  f"against {tol.flatten()[err.flatten().argmax()].item()}, first {bad.nonzero()[0].tolist()}"
        at, kat = at + new, kat + ctx


def make_case(seed, spans, kind, q_dtype, hq, hkv, d, page, spare=2, stale=float("nan"), sharp=2.0):
    """A cache whose unused slots hold `stale`, its page table, packed queries, and what the contexts stand for."""
    g = gen(seed)
    need = [-(-c // page) for _, c in spans]
    n_pages = sum(need) + spare
    cache = tq.KvCache.new(GT[kind], n_pages, page, hkv, d)
    if kind == "q8_0":
        cache.k_pages.fill_(77), cache.v_pages.fill_(-77)
        cache.k_scales.fill_(stale), cache.v_scales.fill_(stale)
    else:
        cache.k_pages.fill_(stale), cache.v_pages.fill_(stale)
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(spans), max(need + [1])), 2 ** 31 - 1, dtype=torch.int32, device="cuda")   # entries behind a context are not read
    at, slots = 0, []
    for i, (_, c) in enumerate(spans):
        table[i, :need[i]] = order[at:at + need[i]]
        t = torch.arange(c, device="cuda")
        slots.append(table[i].long()[t // page] * page + t % page if c else t)
        at += need[i]
    slots = torch.cat(slots)
    cache.write(randn(g, slots.numel(), hkv, d), randn(g, slots.numel(), hkv, d), slots)
    k, v = cache.read(slots)
    n = sum(s[0] for s in spans)
    starts = torch.tensor(np.cumsum([0] + [s[0] for s in spans]), dtype=torch.int32, device="cuda")
    contexts = torch.tensor([s[1] for s in spans], dtype=torch.int32, device="cuda")
    return cache, table, (randn(g, n, hq, d) * sharp).to(q_dtype), starts, contexts, k, v


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float16, torch.bfloat16), ("q8_0", torch.bfloat16), ("q8_0", torch.float16)]
SPANS = {
    "one": [(1, 1)],
    "token": [(1, 1000)],
    "long": [(1, 5000), (2, 4097)],
    "edges": [(1, c) for c in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513)],
    "empty": [(0, 50), (1, 0), (3, 2), (4, 4), (0, 0), (1, 9)],
    "prompts": [(128, 128), (1, 1), (129, 129), (300, 300)],
    "chunk": [(70, 1000), (257, 700)],
    "mixed": [(40, 333), (1, 70), (1, 1), (130, 900), (2, 600)],
}


@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("spans", list(SPANS))
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (5, 1, 64, 32), (6, 6, 128, 64), (10, 2, 64, 256)])
def test_attention(kind, q_dtype, spans, hq, hkv, d, page):
    spans = SPANS[spans]
    cache, table, q, starts, contexts, k, v = make_case(6, spans, kind, q_dtype, hq, hkv, d, page)
    for causal in (True, False):
        check_attention(cache.attend(q, starts, contexts, table, causal=causal), q, k, v, spans, kind=kind, causal=causal)
    tight = cache.attend(q, starts, contexts, table, max_new=max(s[0] for s in spans), max_context=max(s[1] for s in spans), scale=0.05,
                         out_dtype=torch.float32)
    check_attention(tight, q, k, v, spans, kind=kind, scale=0.05)
    tq.context().poll_status()


@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("group", [1, 3, 7, 8, 16, 17, 32, 33, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_groups_of_query_heads(kind, q_dtype, group, d):
    for spans in ([(1, 300), (1, 1), (1, 2100)], [(3, 77), (9, 400)]):
        cache, table, q, starts, contexts, k, v = make_case(7, spans, kind, q_dtype, 2 * group, 2, d, 16)
        check_attention(cache.attend(q, starts, contexts, table), q, k, v, spans, kind=kind)


@pytest.mark.parametrize("kind,q_dtype", [TYPES[0], TYPES[1], TYPES[3]])
def test_long_contexts_and_many_sequences(kind, q_dtype):
    for spans, heads in (([(1, 70001), (1, 3)], (8, 2, 128)), ([(200, 20011)], (8, 2, 128)), ([(1 + i % 2, 1 + 37 * i % 900) for i in range(300)], (4, 1, 64)),
                         ([(i % 5 * 20, 100 + i) for i in range(60)], (4, 2, 64))):
        cache, table, q, starts, contexts, k, v = make_case(8, spans, kind, q_dtype, *heads, 16)
        check_attention(cache.attend(q, starts, contexts, table, max_new=max(s[0] for s in spans)), q, k, v, spans, kind=kind)


@pytest.mark.parametrize("kind,q_dtype", TYPES)
def test_extreme_scores(kind, q_dtype):
    """Scores that grow along the keys by far more than a running maximum may lag, single keys that take all, all scores alike."""
    spans = [(1, 700), (150, 700), (16, 300)]
    cache, table, q, starts, contexts, _, _ = make_case(9, spans, kind, q_dtype, 4, 2, 128, 16)
    g = gen(10)
    slots = torch.cat([table[i].long()[torch.arange(c, device="cuda") // 16] * 16 + torch.arange(c, device="cuda") % 16 for i, (_, c) in enumerate(spans)])
    for form in ("rising", "falling", "spikes", "flat", "huge"):
        k, v = randn(g, slots.numel(), 2, 128), randn(g, slots.numel(), 2, 128)
        ramp = torch.cat([torch.linspace(0.01, 3, c, device="cuda") for _, c in spans])[:, None, None]
        if form in ("rising", "falling"):
            k = k.sign() * (ramp if form == "rising" else 3.01 - ramp)
        elif form == "spikes":
            k[::97] *= 12
        elif form == "flat":
            k = torch.ones_like(k) * 0.5
        else:
            k *= 60
        cache.write(k, v, slots)
        k, v = cache.read(slots)
        check_attention(cache.attend(q, starts, contexts, table), q, k, v, spans, kind=kind)


def test_rows_outside_the_sequences_stay_and_strides_are_taken():
    spans = [(2, 40), (200, 300)]
    cache, table, q, starts, contexts, k, v = make_case(11, spans, torch.bfloat16, torch.bfloat16, 8, 2, 128, 32)
    want = cache.attend(q, starts, contexts, table)
    n = q.shape[0]
    wide = torch.full((n + 9, 12 * 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[3:3 + n, 256:256 + 1024] = q.flatten(1)
    out = torch.full((n + 9, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = cache.attend(wide[:, 256:1280], starts + 3, contexts, table, out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    assert torch.equal(out[3:3 + n], want) and (out[:3] == 7).all() and (out[3 + n:] == 7).all()
    assert cache.attend(q[:0], torch.zeros(1, dtype=torch.int32, device="cuda"), contexts[:0], table[:0]).shape == (0, 8, 128)
    tq.context().poll_status()


def test_the_same_call_gives_the_same_bits():
    """Also for a sequence whose neighbours' keys, queries and lengths change within the call's bounds."""
    spans = [(1, 1234), (1, 5000), (2, 300), (1, 17), (200, 2600), (1, 5000)]
    for kind in (torch.bfloat16, "q8_0"):
        cache, table, q, starts, contexts, k, v = make_case(12, spans, kind, torch.bfloat16, 8, 2, 128, 16)
        bounds = {"max_new": 200, "max_context": 5000}
        whole = cache.attend(q, starts, contexts, table, **bounds)
        assert torch.equal(cache.attend(q, starts, contexts, table, **bounds), whole)
        for i in (0, 1, 4):
            q2, c2 = torch.randn_like(q), torch.ones_like(contexts) * 3
            a, b = int(starts[i]), int(starts[i + 1])
            q2[a:b], c2[i] = q[a:b], contexts[i]
            assert torch.equal(cache.attend(q2, starts, c2, table, **bounds)[a:b], whole[a:b])


@pytest.mark.parametrize("new", [1, 60])
def test_captured_calls_follow_the_lengths_and_do_not_share_memory(new):
    """Two graphs captured on one context, replayed side by side on two streams while contexts grow."""
    made = [make_case(13 + i, [(new, 400 + 100 * i), (1, 90)], torch.bfloat16, torch.bfloat16, 8, 2, 128, 16, spare=8) for i in range(2)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for (cache, table, q, starts, contexts, k, v), s in zip(made, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            cache.attend(q, starts, contexts, table, max_new=new)
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                outs.append(cache.attend(q, starts, contexts, table, max_new=new))
            graphs.append(gr)
    torch.cuda.synchronize()
    for shrink in (0, 37, 200):
        lengths = [[400 + 100 * i - shrink, max(1, 90 - shrink)] for i in range(2)]
        for m, l in zip(made, lengths):
            m[4].copy_(torch.tensor(l, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(20):
            for gr, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        for i, (cache, table, q, starts, contexts, k, v) in enumerate(made):
            full = 400 + 100 * i
            ks, vs = (torch.cat((t[:lengths[i][0]], t[full:full + lengths[i][1]])) for t in (k, v))
            check_attention(outs[i], q, ks, vs, [(new, lengths[i][0]), (1, lengths[i][1])], kind=torch.bfloat16)
    tq.context().poll_status()


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("kind", [torch.float16, "q8_0"])
def test_lengths_and_pages_outside_their_bounds_are_reported(new, kind):
    spans = [(new, 200), (new, 300)]
    cache, table, q, starts, contexts, k, v = make_case(15, spans, kind, torch.bfloat16, 8, 2, 128, 16)
    ctx = tq.context()

    def reported():
        with pytest.raises(tq.TurqError) as e:
            ctx.poll_status()
        assert e.value.status == 1
        ctx.poll_status()

    bad = table.clone()
    bad[1, 3], bad[1, 4] = cache.n_pages, -7
    got = cache.attend(q, starts, contexts, bad)
    reported()
    check_attention(got[:new], q[:new], k[:200], v[:200], spans[:1], kind=kind)   # the other sequence is as it was
    zeroed = [t.clone() for t in (k[200:], v[200:])]
    for t in zeroed:
        t[48:80] = 0                                                       # such pages read as zeros
    check_attention(got[new:], q[new:], *zeroed, spans[1:], kind=kind)
    for lengths in ([200, 2 ** 30], [200, -4]):
        got = cache.attend(q, starts, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table)
        reported()
        check_attention(got[:new], q[:new], k[:200], v[:200], spans[:1], kind=kind)
    cache.attend(q, starts, contexts, table, max_context=250)
    reported()
    for s in ([0, new, 2 ** 30], [0, new, 0], [-5, new, 2 * new]):
        cache.attend(q, torch.tensor(s, dtype=torch.int32, device="cuda"), contexts, table)
        reported()
    check_attention(cache.attend(q, starts, contexts, table), q, k, v, spans, kind=kind)


def test_calls_on_two_streams():
    made = [make_case(20 + i, [(1, 3000), (90, 1000)], torch.bfloat16, torch.bfloat16, 8, 2, 128, 16) for i in range(2)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            cache, table, q, starts, contexts, _, _ = made[i]
            with torch.cuda.stream(s):
                outs[i].append(cache.attend(q, starts, contexts, table))
    torch.cuda.synchronize()
    for i in range(2):
        _, _, q, _, _, k, v = made[i]
        check_attention(outs[i][0], q, k, v, [(1, 3000), (90, 1000)], kind=torch.bfloat16)
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])


# ---- refusals

def test_refusals():
    g = gen(30)
    n, hq, hkv, d = 4, 4, 2, 64
    q, k, v = randn(g, n, hq, d), randn(g, n, hkv, d), randn(g, n, hkv, d)
    pos, slots = torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n, device="cuda")
    table = tq.RotaryTable.new(64, 32)
    cache = tq.KvCache.new(tq.GgmlDType.BF16, 4, 16, hkv, d)

    def refused(status, f, *a, **kw):
        with pytest.raises(tq.TurqError) as e:
            f(*a, **kw)
        assert e.value.status == status, e.value

    refused(2, tq.RotaryTable.new, 12, 32)
    refused(2, tq.RotaryTable.from_frequencies, [1.0] * 68, 32)
    refused(2, tq.RotaryTable.from_frequencies, [1.0] * 6, 32)
    refused(2, tq.RotaryTable.new, 64, 0)
    refused(1, tq.RotaryTable.new, 64, 32, scaling={"type": "other"})
    refused(1, tq.RotaryTable.new, 64, 32, scaling={"type": "linear", "factor": 0.5})
    for bad in ((tq.GgmlDType.Q4K, 4, 16, 2, 64, 3), (tq.GgmlDType.F16, 4, 8, 2, 64, 2), (tq.GgmlDType.F16, 4, 48, 2, 64, 2), (tq.GgmlDType.F16, 4, 512, 2, 64, 2),
                (tq.GgmlDType.F16, 0, 16, 2, 64, 2), (tq.GgmlDType.F16, 4, 16, 0, 64, 2), (tq.GgmlDType.F16, 4, 16, 2, 96, 2)):
        refused(bad[-1], tq.KvCache.new, *bad[:-1])
    refused(2, tq.qk_norm_rope, q, k, pos, tq.RotaryTable.new(72, 8))          # more than the head
    refused(2, tq.qk_norm_rope, q, k[:3], pos, table)
    refused(2, tq.qk_norm_rope, q, k, pos[:3], table)
    refused(3, tq.qk_norm_rope, q, k, pos.long(), table)
    refused(3, tq.qk_norm_rope, q.double(), k.double(), pos, table)
    refused(3, tq.qk_norm_rope, q, k, pos, table, out_dtype=torch.int8)
    refused(2, tq.qk_norm_rope, q, k, pos, table, q_weight=torch.ones(32, device="cuda"))
    refused(1, tq.qk_norm_rope, q.transpose(0, 1), k, pos, table)
    refused(1, tq.qk_norm_rope, q.cpu(), k, pos, table)
    flat = torch.zeros(n * hq * d + 1, device="cuda")
    refused(4, tq.qk_norm_rope, flat[1:].view(n, hq, d), k, pos, table)       # 4 bytes off
    refused(4, tq.qk_norm_rope, torch.zeros(n, hq * d + 2, device="cuda")[:, :hq * d].unflatten(1, (hq, d)), k, pos, table)
    refused(2, cache.append, q, k, v[:, :1], pos, table, slots)
    refused(3, cache.append, q, k, v, pos, table, slots.int())
    refused(2, cache.write, k[:, :1], v[:, :1], slots)
    refused(2, cache.write, k, v, slots[:2])
    refused(3, cache.read, slots, torch.int32)

    qb = q.bfloat16()
    starts, contexts = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    pages = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    refused(3, cache.attend, q, starts, contexts, pages)                       # f32 queries
    refused(3, cache.attend, q.half(), starts, contexts, pages)                # f16 queries on a bf16 cache
    refused(2, cache.attend, qb[:, :3].contiguous(), starts, contexts, pages)  # 3 heads on 2
    refused(2, cache.attend, qb, starts[:1], contexts, pages)
    refused(2, cache.attend, qb, starts, contexts, pages, max_context=33)      # more than the table holds
    refused(2, cache.attend, qb, starts, contexts, pages, max_new=-1)
    refused(1, cache.attend, qb, starts, contexts, pages, scale=0.0)
    refused(1, cache.attend, qb, starts, contexts, pages, scale=float("inf"))
    refused(3, cache.attend, qb, starts.long(), contexts, pages)
    refused(2, cache.attend, qb, starts, contexts, pages[0])
    refused(2, cache.attend, qb, starts, contexts, pages, out=torch.empty(3, hq, d, dtype=torch.bfloat16, device="cuda"))
    refused(3, cache.attend, qb, starts, contexts, pages, out=torch.empty(n, hq, d, dtype=torch.float16, device="cuda"), out_dtype=torch.float32)
    tq.context().poll_status()
    assert torch.isfinite(cache.attend(qb, starts, contexts, pages)).all()


# ---- together

def test_a_layers_attention_token_by_token_and_at_once(tmp_path):
    """Attention.forward on quantized linears from a GGUF file: a prompt in one call, in chunks, and its last tokens one by one give
    what the same block gives in 64 bits on the same linears' outputs."""
    import gguf
    from gguf.constants import GGMLQuantizationType as T

    import oracle
    from tur_b200.gguf import VarBuilder
    rng = np.random.default_rng(7)
    hidden, hq, hkv, d, n = 512, 8, 2, 64, 150
    path = tmp_path / "block.gguf"
    w = gguf.GGUFWriter(str(path), "qwen3")
    for name, (rows, cols) in {"attn_q": (hq * d, hidden), "attn_k": (hkv * d, hidden), "attn_v": (hkv * d, hidden),
                               "attn_output": (hidden, hq * d)}.items():
        blocks = oracle.quantize(oracle.Q8_0, (rng.standard_normal((rows, cols)) * 0.05).astype(np.float32))
        w.add_tensor(f"blk.0.{name}.weight", blocks, raw_shape=blocks.shape, raw_dtype=T.Q8_0)
    for name in ("attn_q_norm", "attn_k_norm"):
        w.add_tensor(f"blk.0.{name}.weight", (1 + 0.1 * rng.standard_normal(d)).astype(np.float32))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    vb = VarBuilder.from_gguf(str(path)).pp("blk").pp(0)
    block = tq.Attention.new(vb, hidden, hq, hkv, d)
    assert block.q_norm is not None
    x = torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float32)).cuda()
    table = tq.RotaryTable.new(d, n, base=1e4)
    freqs = [1e4 ** (-2 * i / d) for i in range(d // 2)]
    mode = tq.Mode.EXACT_F32
    q, k, v = (l.forward(x, mode=mode).unflatten(1, (-1, d)) for l in (block.q, block.k, block.v))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    qr = ref_rows(q, block.q_norm, 1e-6, freqs, pos, False)
    kr = ref_rows(k, block.k_norm, 1e-6, freqs, pos, False).repeat_interleave(hq // hkv, 1)
    z = torch.einsum("nhd,chd->hnc", qr, kr) / d ** 0.5
    z = z.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
    y = torch.einsum("hnc,chd->nhd", torch.softmax(z, -1), v.double().repeat_interleave(hq // hkv, 1))
    want = block.o.forward(y.float().flatten(1), mode=mode).double()

    def step(cache, a, b, pages):
        t = pos[a:b]
        slots = pages[0].long()[t.long() // 16] * 16 + t.long() % 16
        return block.forward(x[a:b], cache, table, t, slots, torch.tensor([0, b - a], dtype=torch.int32, device="cuda"),
                             torch.tensor([b], dtype=torch.int32, device="cuda"), pages, mode=mode)

    pages = torch.randperm(12, device="cuda", dtype=torch.int32)[None, :10].contiguous()
    for dtype in (tq.GgmlDType.BF16, tq.GgmlDType.F16, tq.GgmlDType.Q8_0):
        # q, k, v and the weights of the softmax are each rounded to 16 bits (bf16: 2^-8, in parts that are independent), or k and v
        # to 8 (a step of amax / 127 on blocks of 32): 2^-6 of the output's norm bounds their sum for every type
        for cuts in ([0, n], [0, 64, 101, n], [0, 140] + list(range(141, n + 1))):
            cache = tq.KvCache.new(dtype, 12, 16, hkv, d)
            got = torch.cat([step(cache, a, b, pages) for a, b in zip(cuts, cuts[1:])]).double()
            assert ((got - want).norm() / want.norm()).item() < 2.0 ** -6, (dtype, cuts)
    tq.context().poll_status()


# ---- calls at the edges of what the header allows

@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("new,ctx", [(1, 300), (1, 3000), (1, 40000), (40, 40), (40, 9000), (300, 300)])
def test_the_output_may_be_the_query(kind, q_dtype, new, ctx):
    cache, table, q, starts, contexts, _, _ = make_case(31, [(new, ctx), (1, 70)], kind, q_dtype, 8, 2, 128, 64)
    want = cache.attend(q, starts, contexts, table)
    same = q.clone()
    assert cache.attend(same, starts, contexts, table, out=same).data_ptr() == same.data_ptr()
    assert torch.equal(same, want)
    tq.context().poll_status()


@pytest.mark.parametrize("kind", [torch.float16, "q8_0"])
@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("exponent", [118, 126, -120])
def test_queries_far_outside_the_range_of_f16(kind, new, exponent):
    # q = +-2^e: divided by its row's power of two it is +-1. At 2^118 the key whose signs it has gets all of the weight (its score leads
    # by 2^118 / sqrt(128) times tens): its values come out as they are. At 2^126 scale brings the score back into f32's range. At 2^-120
    # all scores are 0 within 2^-110: the mean of the keys that a row sees.
    d, ctx = 128, 200
    g = gen(32)
    cache = tq.KvCache.new(GT[kind], 4, 64, 1, d)
    k, v = randn(g, ctx, 1, d), randn(g, ctx, 1, d)
    slots = torch.arange(ctx, device="cuda")
    cache.write(k, v, slots)
    kc, vc = cache.read(slots)
    best = 7
    q = (torch.where(k[best, 0] < 0, -1.0, 1.0) * 2.0 ** exponent).to(torch.bfloat16).expand(new, 1, d).contiguous()
    starts, contexts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, new], [ctx]))
    got = cache.attend(q, starts, contexts, torch.arange(4, dtype=torch.int32, device="cuda")[None], out_dtype=torch.float32,
                       scale=2.0 ** -20 if exponent == 126 else None)
    if exponent > 0:
        scores = (kc[:, 0].double() * torch.sign(q[0, 0].double())).sum(1)
        assert scores.argmax() == best and scores[best] - scores[scores < scores[best]].max() > 1  # of f32 steps below 2^-16: all of the weight
        # Values of Q8_0 go into the product as f16, those of f16 are. The row's one weight, some 2^r, is rounded to f16 for the product (2^-11 of
        # it) and not for the sum that divides it; the f32 product and quotient add 2^-24 each.
        want = vc[best].half().double()
        assert ((got.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -22) * want.abs()).all()
    else:
        vd = vc[:, 0].double()
        for t in range(new):
            seen = vd[:ctx - new + t + 1]
            # weights are exactly 1, values have 11 bits (Q8_0: rounded to f16), sums and quotient are f32's
            tol = (2.0 ** -11 * (kind == "q8_0") + 2.0 ** -15) * seen.abs().mean(0) + 2.0 ** -25
            assert ((got[t, 0].double() - seen.mean(0)).abs() <= tol).all()


@pytest.mark.parametrize("kind,q_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), ("q8_0", torch.bfloat16)])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_that_climb_back_from_far_below(kind, q_dtype, new, d):
    # The first 128 keys point away from every query: scores below -2^22, weights of exactly 0 once an ordinary key is seen. What a row gives is
    # attention over the other 200 alone.
    g = gen(33)
    ctx, far = 328, 128
    cache = tq.KvCache.new(GT[kind], 6, 64, 1, d)
    base = randn(g, 1, 1, d).sign()
    q = (base * (3 + randn(g, new, 1, d).abs())).to(q_dtype)
    k, v = 0.05 * randn(g, ctx, 1, d), randn(g, ctx, 1, d)
    k[:far] = -50000.0 * base
    slots = torch.arange(ctx, device="cuda")
    cache.write(k, v, slots)
    kc, vc = cache.read(slots)
    assert ((q.double() * kc[:1].double()).sum(-1) < -2.0 ** 22).all()
    starts, contexts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, new], [ctx]))
    got = cache.attend(q, starts, contexts, torch.arange(6, dtype=torch.int32, device="cuda")[None], scale=1.0)
    check_attention(got, q, kc[far:], vc[far:], [(new, ctx - far)], kind=kind, scale=1.0)


@pytest.mark.parametrize("new", [1, 30])
def test_no_context_at_all_gives_zeros(new):
    cache = tq.KvCache.new(tq.GgmlDType.BF16, 1, 16, 2, 64)
    starts, contexts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, new], [0]))
    q = torch.ones(new, 4, 64, dtype=torch.bfloat16, device="cuda")
    got = cache.attend(q, starts, contexts, torch.empty(1, 0, dtype=torch.int32, device="cuda"))
    assert not got.any()
    tq.context().poll_status()


def test_a_cache_that_owns_its_memory_and_a_workspace_too_small():
    lib, ctx = _lib.load(), tq.context()
    h = ctypes.c_void_p()
    ctx.check(lib.turq_kv_cache_create(ctx.handle, int(tq.GgmlDType.F16), 600, 16, 1, 64, None, 0, ctypes.byref(h)))
    s = torch.cuda.current_stream().cuda_stream
    try:
        memory, off = ctypes.c_void_p(), (ctypes.c_int64 * 4)()
        ctx.check(lib.turq_kv_cache_layout(h, ctypes.byref(memory), off))
        assert memory.value and off[0] == 0 and off[1] == 600 * 16 * 64 * 2
        slots = torch.arange(600 * 16, device="cuda")
        k, v = (torch.full((600 * 16, 1, 64), 7.0, device="cuda") for _ in range(2))
        ctx.check(lib.turq_kv_read(ctx.handle, h, slots.data_ptr(), 600 * 16, 0, k.data_ptr(), v.data_ptr(), s))
        assert not k.any() and not v.any()
        q = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
        starts, contexts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [9600]))
        table = torch.arange(600, dtype=torch.int32, device="cuda")
        nbytes = lib.turq_kv_attention_workspace(h, 1, 1, 1, 1, 9600)
        assert nbytes > 0
        ws, y = torch.empty(nbytes, dtype=torch.uint8, device="cuda"), torch.full((1, 1, 64), 5.0, device="cuda")
        call = lambda p, n, scale=0.125: lib.turq_kv_attention(ctx.handle, h, q.data_ptr(), 64, 1, 1, 1, starts.data_ptr(), contexts.data_ptr(), table.data_ptr(),
                                                               600, 1, 1, 9600, scale, 1, 0, y.data_ptr(), p, n, s)
        assert call(ws.data_ptr(), nbytes - 1) == 2 and call(None, 0) == 2 and call(None, nbytes) == 1 and call(ws.data_ptr() + 8, nbytes) != 0
        assert call(ws.data_ptr(), nbytes, 3e38) == 1 and call(ws.data_ptr(), nbytes, float("nan")) == 1
        torch.cuda.synchronize()
        assert (y == 5).all()
        ctx.check(call(ws.data_ptr(), nbytes))
        torch.cuda.synchronize()
        assert not y.any()
    finally:
        torch.cuda.synchronize()
        assert lib.turq_kv_cache_free(h) == 0
