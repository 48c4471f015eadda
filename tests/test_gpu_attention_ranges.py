"""Attention over the cache where scores, keys and values leave the ordinary: scores whose steps in f32 are large, NaN among the keys
that a row sees, values of any size among those that it does not, blocks of Q8_0 beyond f16.

Tolerances are those of the definition's roundings (a rounding to t is off by at most eps_t / 2 of the value): see each test."""
import pytest
import torch

import tur_b200 as tq
from test_gpu_attention import GT, HALF, TYPES, check_attention, gen, make_case, randn

pytestmark = pytest.mark.gpu


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def plain_cache(kind, ctx, d, page=64, heads=1):
    """A cache of one sequence whose pages lie in order."""
    pages = -(-ctx // page)
    return tq.KvCache.new(GT[kind], pages, page, heads, d), torch.arange(pages, dtype=torch.int32, device="cuda")[None]


def rows_of(pages, ctx):
    """[n_pages, heads, page, d] -> [ctx, heads, d]"""
    return pages.transpose(1, 2).flatten(0, 1)[:ctx]


@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("new,ctx", [(1, 100), (2, 900), (1, 20000), (40, 300), (40, 9000)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("p", [10, 16, 20, 22, 23, 26, 30])
def test_scores_that_f32_holds_exactly(kind, q_dtype, new, ctx, d, p):
    # q = (2^a, .., step, ..) and k_j = (2^b, .., u_j, ..) with a + b = p and whole u_j: every score, 2^p + step u_j, is a number of f32 (step is at
    # least 2^(p - 23)) and both its products are exact, so the scores carry no error and neither do their differences. What is left: weights
    # (the 16-bit type's half step, an exponential good to 2^-13, their sum) and values (Q8_0 ones rounded to f16).
    step = max(2.0 ** (p - 23), 0.25)
    a, b = (p + 1) // 2, p // 2
    g = gen(41)
    cache, table = plain_cache(kind, ctx, d)
    u = torch.randint(0, 16, (ctx,), device="cuda", generator=g)
    k = torch.zeros(ctx, 1, d, device="cuda")
    k[:, 0, 0], k[:, 0, 32] = 2.0 ** b, u.float()
    v = randn(g, ctx, 1, d)
    slots = torch.arange(ctx, device="cuda")
    cache.write(k, v, slots)
    if kind == "q8_0":  # what quantization would round: 2^b as 64 x 2^(b - 6), u as u x 1
        kp, ks = cache.k_pages.transpose(1, 2).flatten(0, 1), cache.k_scales.transpose(1, 2).flatten(0, 1)
        kp, ks = torch.zeros_like(kp), torch.zeros_like(ks)
        kp[:ctx, 0, 0], kp[:ctx, 0, 32] = 64, u.to(torch.int8)
        ks[:, 0, 0], ks[:, 0, 1] = 2.0 ** (b - 6), 1.0
        n, page = cache.n_pages, cache.page_size
        cache.k_pages.copy_(kp.view(n, page, 1, d).transpose(1, 2))
        cache.k_scales.copy_(ks.view(n, page, 1, d // 32).transpose(1, 2))
    kc, vc = cache.read(slots)
    assert torch.equal(kc, k)
    q = torch.zeros(new, 2, d, device="cuda")
    q[:, 0, 0], q[:, 0, 32] = 2.0 ** a, step
    q[:, 1, 0], q[:, 1, 32] = 2.0 ** a, -step  # the other end of the u's leads (2^p - step u: in f32 too, as step >= 2^(p - 23))
    q = q.to(q_dtype)
    got = cache.attend(q, ints(0, new), ints(ctx), table, scale=1.0, out_dtype=torch.float32).double()
    vd = vc[:, 0].double()
    p16 = torch.bfloat16 if kind is torch.bfloat16 else torch.float16
    for t in range(0, new, 13):
        seen = ctx - new + t + 1
        for h, sign in enumerate((1.0, -1.0)):
            w = torch.softmax(sign * step * u[:seen].double(), 0)
            want, spread = w @ vd[:seen], w @ vd[:seen].abs()
            tol = spread * (2 * HALF[p16] + 2.0 ** -12 + (HALF[torch.float16] if kind == "q8_0" else 0)) + 2.0 ** -25 * (vd.abs().sum(0) + 2)
            err = (got[t, h] - want).abs()
            assert (err <= tol).all(), (t, h, err.max().item(), tol[err.argmax()].item())
    tq.context().poll_status()


@pytest.mark.parametrize("kind", [torch.float16, "q8_0"])
@pytest.mark.parametrize("new", [1, 2, 40])
def test_scores_that_vanish_leave_the_mean(kind, new):
    # a query of zeros, or of its type's smallest numbers, and a scale that takes the rest: every score is 0 within 2^-100
    g = gen(48)
    ctx, d = 300, 64
    cache, table = plain_cache(kind, ctx, d)
    v = randn(g, ctx, 1, d)
    slots = torch.arange(ctx, device="cuda")
    cache.write(randn(g, ctx, 1, d), v, slots)
    vd = cache.read(slots)[1][:, 0].double()
    q = torch.zeros(new, 2, d, dtype=torch.bfloat16, device="cuda")
    q[:, 1] = 1e-38
    got = cache.attend(q, ints(0, new), ints(ctx), table, scale=1e-20, out_dtype=torch.float32).double()
    for t in range(new):
        seen = vd[:ctx - new + t + 1]
        # weights are 1; values of Q8_0 are rounded to f16; sums and quotient are f32's
        assert ((got[t] - seen.mean(0)).abs() <= (2.0 ** -11 * (kind == "q8_0") + 2.0 ** -15) * seen.abs().mean(0) + 2.0 ** -25).all()
    tq.context().poll_status()


@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", ["tokens", "tiles"])
def test_a_key_that_is_not_a_number_is_seen_by_every_row_behind_it(kind, q_dtype, d, rows):
    # Rows that see the key are NaN throughout, the others what they are without it; at every place that a key can have among the 32
    # that a thread takes at a time, and at the ends of the tiles.
    g = gen(42)
    ctx, new = (200, 40) if rows == "tiles" else (200, 2)
    cache, table = plain_cache(kind, ctx, d)
    k, v, q = randn(g, ctx, 1, d), randn(g, ctx, 1, d), randn(g, new, 4, d).to(q_dtype)
    slots = torch.arange(ctx, device="cuda")
    cache.write(k, v, slots)
    want = cache.attend(q, ints(0, new), ints(ctx), table)
    assert torch.isfinite(want).all()
    for at in list(range(32)) + [63, 64, 126, 127, 128, 129, ctx - new, ctx - 1]:
        plane = cache.k_scales if kind == "q8_0" else cache.k_pages
        old = plane[at // 64, 0, at % 64].clone()
        plane[at // 64, 0, at % 64] = float("nan")
        got = cache.attend(q, ints(0, new), ints(ctx), table)
        plane[at // 64, 0, at % 64] = old
        first = max(0, at - (ctx - new))  # the first row that sees it
        assert torch.isnan(got[first:]).all(), at
        assert torch.equal(got[:first], want[:first]), at
    assert torch.equal(cache.attend(q, ints(0, new), ints(ctx), table), want)
    cache_status()


def cache_status():
    try:
        tq.context().poll_status()
    except tq.TurqError:
        pass


@pytest.mark.parametrize("kind,q_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [2, 40, 300])
def test_values_that_a_row_does_not_see_have_no_weight(kind, q_dtype, d, new):
    # every value is as large as its type goes, but for the first: the row that sees nothing else gives it. Its one weight, whatever the
    # exponential makes of 0, is rounded to the 16-bit type for the product and not for the sum that divides it: half a step of it, and
    # what f32 loses in product and quotient (2^-22 is four half steps).
    g = gen(43)
    ctx = new
    cache, table = plain_cache(kind, ctx, d)
    v = torch.full((ctx, 1, d), 3e38 if kind is torch.bfloat16 else 65504.0, device="cuda")
    v[0] = randn(g, 1, d)
    cache.write(torch.zeros(ctx, 1, d, device="cuda"), v, torch.arange(ctx, device="cuda"))
    q = randn(g, new, 8, d).to(q_dtype)
    got = cache.attend(q, ints(0, new), ints(ctx), table, out_dtype=torch.float32)
    first = v[0].to(kind).float().expand(8, d)
    assert ((got[0] - first).abs() <= (HALF[kind] + 2.0 ** -22) * first.abs()).all()
    tq.context().poll_status()


@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_maxima_that_grow_from_tile_to_tile(kind, q_dtype, d):
    """Every tile of 128 keys has scores far above the one before, so that sums and products are scaled again at each of them."""
    g = gen(44)
    for spans in ([(1, 900), (150, 900)], [(40, 6000), (1, 6000)]):
        cache, table, q, starts, contexts, _, _ = make_case(45, spans, kind, q_dtype, 4, 2, d, 16)
        n = sum(c for _, c in spans)
        slots = torch.cat([table[i].long()[torch.arange(c, device="cuda") // 16] * 16 + torch.arange(c, device="cuda") % 16 for i, (_, c) in enumerate(spans)])
        ramp = torch.cat([torch.arange(c, device="cuda") // 128 * 1.5 for _, c in spans])[:, None, None]
        k, v = randn(g, n, 2, d).sign() * (0.01 + ramp), randn(g, n, 2, d)
        for keys in (k, k.flip(0)):
            cache.write(keys, v, slots)
            kc, vc = cache.read(slots)
            check_attention(cache.attend(q, starts, contexts, table), q, kc, vc, spans, kind=kind)
    tq.context().poll_status()


@pytest.mark.parametrize("kind,q_dtype", [TYPES[0], TYPES[1], TYPES[3]])
@pytest.mark.parametrize("new,contexts", [(1, [333]), (1, [4096]), (1, [20011]), (1, [5000, 9000, 70001]), (2, [40000]), (40, [300]), (40, [9001]),
                                          (40, [20000, 6000]), (300, [5000])])
@pytest.mark.parametrize("d", [64, 128])
def test_every_border_of_a_long_context(kind, q_dtype, new, contexts, d):
    # Two keys on either side of a border of 16 keys share all of the weight of a row of their own (scores of 64 against 0: e^-64 for the
    # rest), so that one lost, doubled or taken from elsewhere moves the row by a third of their values. Chunks, steps, pieces and tiles all
    # begin at multiples of 16; those of 128, where pieces can begin, are all tried, the others by a stride.
    g = gen(46)
    hkv, group = 2, 4
    page = 64
    need = [-(-c // page) for c in contexts]
    cache = tq.KvCache.new(GT[kind], sum(need), page, hkv, d)
    order = torch.randperm(sum(need), device="cuda", generator=g)
    table = torch.zeros(len(contexts), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    slots = [table[i].long()[torch.arange(c, device="cuda") // page] * page + torch.arange(c, device="cuda") % page for i, c in enumerate(contexts)]
    values = [randn(g, c, hkv, d) for c in contexts]
    for s, v in zip(slots, values):
        cache.write(torch.zeros_like(v), v, s)
    held = [cache.read(s)[1].double() for s in slots]
    seq = max(range(len(contexts)), key=lambda i: contexts[i])
    ctx = contexts[seq]
    last = ctx - new  # behind it rows see different keys
    borders = [b for b in range(128, last, 128)] + [b for b in range(16, last, 16 * (1 + last // 2000)) if b % 128] + ([last] if last > 1 else [])
    rows = min(d, new * group)
    zero = torch.zeros(ctx, hkv, d, device="cuda")
    p16 = torch.bfloat16 if kind is torch.bfloat16 else torch.float16
    # the two weights are equal, the sum is of f32: value roundings (Q8_0 ones to f16), the weights' own rounding (the same for both, not in
    # the sum), what f32 sums and e^-64 x values leave
    rel = HALF[p16] + (HALF[torch.float16] if kind == "q8_0" else 0) + 2.0 ** -20
    spare = []  # a key pair is used by one row only if no other border of the same call lies next to it
    queue = list(borders)
    while queue or spare:
        take, spare, used = [], [], set()
        for b in queue:
            if len(take) < rows * hkv and not {b - 1, b} & used:
                take.append(b)
                used |= {b - 1, b}
            else:
                spare.append(b)
        queue, spare = spare, []
        k = zero.clone()
        q = torch.zeros(len(contexts) * new, hkv * group, d, device="cuda")
        for i, b in enumerate(take):
            h, r = divmod(i, rows)
            k[b - 1:b + 1, h, r] = 8.0
            q[seq * new + r // group, h * group + r % group, r] = 8.0
        cache.write(k, values[seq], slots[seq])
        starts = ints(*[i * new for i in range(len(contexts) + 1)])
        got = cache.attend(q.to(q_dtype), starts, ints(*contexts), table, max_new=new, max_context=ctx, scale=1.0, out_dtype=torch.float32).double()
        for i, b in enumerate(take):
            h, r = divmod(i, rows)
            pair = held[seq][b - 1:b + 1, h]
            y = got[seq * new + r // group, h * group + r % group]
            assert ((y - pair.mean(0)).abs() <= rel * pair.abs().mean(0) + 2.0 ** -24).all(), (b, (y - pair.mean(0)).abs().max().item())
    tq.context().poll_status()


@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("which", ["k", "v"])
def test_blocks_of_q8_0_up_to_what_f16_holds_and_beyond(q_dtype, d, new, which):
    # 127 x 515.5 is the largest product of a quant and a scale that f16 holds (65468.5, rounded to 65472)
    g = gen(47)
    ctx = 150
    cache, table = plain_cache("q8_0", ctx, d)
    k, v = 0.01 * randn(g, ctx, 1, d), randn(g, ctx, 1, d)
    big = 65400.0
    (k if which == "k" else v)[70, 0, 5] = big
    slots = torch.arange(ctx, device="cuda")
    cache.write(k, v, slots)
    kc, vc = cache.read(slots)
    q = (0.001 * randn(g, new, 4, d)).to(q_dtype)
    spans = [(new, ctx)]
    check_attention(cache.attend(q, ints(0, new), ints(ctx), table, scale=1.0, out_dtype=torch.float32), q, kc, vc, spans, kind="q8_0", scale=1.0)
    tq.context().poll_status()
    (k if which == "k" else v)[70, 0, 5] = 66000.0
    cache.write(k, v, slots)
    tq.context().poll_status()  # the cache holds and returns it
    kc, vc = cache.read(slots)
    assert abs((kc if which == "k" else vc)[70, 0, 5].item() - 66000.0) <= 2.0 ** -8 * 66000
    cache.attend(q, ints(0, new), ints(ctx), table, scale=1.0)
    with pytest.raises(tq.TurqError) as e:
        tq.context().poll_status()
    assert e.value.status == 1
    # behind a context's end it does not matter
    short = 70
    check_attention(cache.attend(q, ints(0, new), ints(short), table, scale=1.0, out_dtype=torch.float32), q, kc[:short], vc[:short], [(new, short)],
                    kind="q8_0", scale=1.0)
    tq.context().poll_status()


@pytest.mark.parametrize("kind,q_dtype", TYPES)
@pytest.mark.parametrize("d,group", [(128, 128), (128, 3), (64, 64), (64, 17)])
def test_many_rows_that_see_no_key(kind, q_dtype, d, group):
    # Tiles without a key, by hundreds, on the SMs beside tiles with some and behind one another: zeros, exactly, whatever the queries are.
    spans = [(1 + i % 9 * (40 // group + 1), 0) for i in range(60)] + [(300, 300)] + [(20 + i, 0) for i in range(60)]
    cache, table, q, starts, contexts, k, v = make_case(49, spans, kind, q_dtype, 2 * group, 2, d, 16)
    full = slice(int(starts[60]), int(starts[61]))
    out = torch.empty_like(q)
    for _ in range(30):
        out.fill_(7.0)
        cache.attend(q, starts, contexts, table, out=out)
        assert not out[:full.start].any() and not out[full.stop:].any()
    check_attention(out[full], q[full], k, v, [(300, 300)], kind=kind)
    tq.context().poll_status()
