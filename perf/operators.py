"""The operators between attn_q|k|v and attn_output, and how their speed is measured: per-head norms of
queries and keys with the position rotation, the paged cache of keys and values (16 bits, or quantized to
Q8_0 as it is written), and attention of new tokens over that cache, from one token to whole prompts.

A case is one call as a serving program makes it. Its kind says which:

  "rotate"  norm and rotation of q and k into dense tensors
  "append"  the same, with keys and values written into their pages in the same pass
  "store"   keys and values written into a quantized cache and read back
  "attend"  attention of the new tokens of several sequences over their pages

Head counts and head dimensions are those of the decoders whose linears this repository runs: 32 and 64
query heads over 8 of 128, 16 over 8 of 128, 40 over 10 of 64. Scores have the spread that normalised heads
give; pages lie in a pool in no order, and slots that no sequence uses hold what an earlier one left there.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def _rows(name, kind, tokens, heads, x, cache, norm=True, rotary=None, interleaved=False, stretch=1.0, first=0, page=16):
    hq, hkv, d = heads
    return {"name": name, "kind": kind, "tokens": tokens, "q_heads": hq, "kv_heads": hkv, "head_dim": d, "x": x, "cache": cache,
            "norm": norm, "rotary": rotary or d, "interleaved": interleaved, "stretch": stretch, "first": first, "page": page}


def _attend(name, heads, q, cache, page, spans, spread=0):
    """spans: "new tokens:context" of each sequence, or "count*new:shortest-longest" for a batch of ragged contexts."""
    hq, hkv, d = heads
    return {"name": name, "kind": "attend", "q_heads": hq, "kv_heads": hkv, "head_dim": d, "q": q, "cache": cache, "page": page,
            "spans": spans, "spread": spread}


def listed():
    return [
        # one token of a decoding 8B model: nothing but latency
        _rows("append_8b_token", "append", 1, (32, 8, 128), "f32", "bf16", first=4095),
        # a decode batch of a 32B model
        _rows("append_32b_batch64", "append", 64, (64, 8, 128), "f32", "f16", first=20000, page=32),
        # a prompt that a program rotates into tensors of its own
        _rows("rotate_8b_prompt8192", "rotate", 8192, (32, 8, 128), "f32", "none"),
        # a 3B model without head norms, part of the head rotated in neighbouring pairs, positions stretched
        _rows("append_3b_prompt2049", "append", 2049, (40, 10, 64), "bf16", "f16", norm=False, rotary=32, interleaved=True, stretch=4.0,
              first=30000),
        # a few tokens and a prompt through the quantized cache
        _rows("store_3b_17", "store", 17, (40, 10, 64), "f32", "q8_0"),
        _rows("store_8b_prompt4099", "store", 4099, (32, 8, 128), "bf16", "q8_0", page=64),
        # the single-user decode step at a usual context
        _attend("decode_8b_ctx4096", (32, 8, 128), "bf16", "bf16", 16, "1:4096"),
        # continuous batching: 64 users with contexts of any length, quantized cache
        _attend("decode_32b_batch64_q8", (64, 8, 128), "bf16", "q8_0", 32, "64*1:100-8192", spread=1),
        # two users with very long contexts
        _attend("decode_8b_long", (32, 8, 128), "f16", "f16", 64, "1:131072,1:100001"),
        # one scheduler step: a chunk of a long prompt, a short tail of another, users that decode
        _attend("mixed_3b_chunk512", (40, 10, 64), "bf16", "f16", 16, "512:8000,33:1000,1:77,1:2500,1:1,1:6001"),
        # several prompts packed into one prefill
        _attend("prompts_8b_packed8192", (32, 8, 128), "bf16", "bf16", 16, "4096:4096,2777:2777,1000:1000,319:319"),
        # one long prompt
        _attend("prompt_8b_16384", (32, 8, 128), "bf16", "bf16", 16, "16384:16384"),
    ]


def draw(rng):
    """Any kind and type over the listed sizes: tokens from one to thousands, contexts to over a hundred
    thousand, one query head or many to a key head, pages of 16 to 128."""
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8, 8, 10])
    heads = (hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), hkv, d)
    page = rng.choice([16, 16, 32, 64, 128])
    kind = rng.choice(["rotate", "append", "store", "attend", "attend", "attend"])
    if kind != "attend":
        x = rng.choice(["f32", "f32", "bf16", "f16"])
        if kind == "store":
            c = _rows("", kind, log(1, 6000), heads, x, "q8_0", page=page)
        else:
            c = _rows("", kind, log(1, 6000), heads, x, "none" if kind == "rotate" else rng.choice(["bf16", "f16"]),
                      norm=rng.random() < 0.7, rotary=rng.choice([d, d, d // 2, 24]), interleaved=rng.random() < 0.4,
                      stretch=rng.choice([1.0, 1.0, 8.0]), first=log(1, 100000), page=page)
    else:
        cache = rng.choice(["bf16", "f16", "q8_0"])
        q = "bf16" if cache == "bf16" else rng.choice(["bf16", "f16"])
        while True:
            form = rng.choice(["decode", "decode", "chunk", "prompt", "mixed"])
            if form == "decode":
                n = log(1, 128)
                top = log(16, max(64, 200000 // n))
                spans = f"{n}*{rng.choice([1, 1, 1, 2, 4])}:{max(4, top // rng.choice([1, 2, 30]))}-{max(8, top)}"
            elif form == "chunk":
                new = log(2, 2048)
                spans = f"{new}:{new + log(1, 30000)}"
            elif form == "prompt":
                spans = ",".join(f"{n}:{n}" for n in (log(1, 6000) for _ in range(rng.randint(1, 6))))
            else:
                new = log(16, 1024)
                spans = f"{new}:{new + log(1, 9000)}," + ",".join(f"1:{log(1, 9000)}" for _ in range(rng.randint(1, 40)))
            c = _attend("", heads, q, cache, page, spans, spread=rng.randrange(1 << 30))
            w = work(c)
            if w["flops"] <= 2.1e12 and w["bytes"] <= 9e8:
                break
    del c["name"]
    return c


def _spans(case):
    """(new tokens, context) of each sequence."""
    rng = random.Random(case["spread"])
    out = []
    for part in case["spans"].split(","):
        new, ctx = part.split(":")
        if "*" in new:
            count, new = (int(v) for v in new.split("*"))
            lo, hi = (int(v) for v in ctx.split("-"))
            out += [(new, max(new, rng.randint(lo, hi))) for _ in range(count)]
        else:
            out.append((int(new), int(ctx)))
    return out


def work(case):
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "attend":
        per = 2.0 if case["cache"] != "q8_0" else 34 / 32
        spans = _spans(case)
        tokens = sum(n for n, _ in spans)
        seen = sum(n * c - n * (n - 1) // 2 for n, c in spans)
        return {"bytes": int(2 * tokens * hq * d * 2 + sum(c for _, c in spans) * 2 * hkv * d * per), "flops": 4 * d * hq * seen}
    t = case["tokens"]
    xb = 4 if case["x"] == "f32" else 2
    if case["kind"] == "store":  # read both, write the pages, read them, write what they hold in 32 bits
        return {"bytes": int(t * 2 * hkv * d * (xb + 2 * 34 / 32 + 4)), "flops": t * 2 * hkv * d * 4}
    table = t * case["rotary"] * 4
    if case["kind"] == "rotate":
        return {"bytes": t * (hq + hkv) * d * (xb + 2) + table, "flops": t * (hq + hkv) * d * 7}
    return {"bytes": t * (hq + 2 * hkv) * d * (xb + 2) + table, "flops": t * (hq + hkv) * d * 7}


# ---- inputs: the same tensors for both sides

def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _frequencies(case):
    """Angle of a pair per position, in 64 bits on the host; stretched positions are divided."""
    i = np.arange(case["rotary"] // 2, dtype=np.float64)
    return 1e6 ** (-2.0 * i / case["rotary"]) / case["stretch"]


def _slots(gen, tokens, page, spare):
    """Slots of a run of tokens on pages that lie anywhere in the pool."""
    pages = -(-tokens // page)
    order = torch.randperm(pages + spare, device="cuda", generator=gen)[:pages]
    t = torch.arange(tokens, device="cuda")
    return order[t // page] * page + t % page, pages + spare


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 9176 + 5)
    hq, hkv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["kind"] != "attend":
        t, x = case["tokens"], TYPES[case["x"]]
        s = {"q": (_randn(gen, t, hq, d) * 1.7).to(x), "k": (_randn(gen, t, hkv, d) * 1.3 + 0.2).to(x), "v": _randn(gen, t, hkv, d).to(x)}
        s["slots"], n_pages = _slots(gen, t, page, 4)
        if case["kind"] == "store":
            s["pool"] = n_pages
            return s
        # a prompt goes on from its first position; the users of a batch are each at one of their own
        s["positions"] = (torch.arange(t, device="cuda") + case["first"]).to(torch.int32)
        s["wq"], s["wk"] = (1.0 + 0.2 * _randn(gen, d), 1.0 + 0.2 * _randn(gen, d)) if case["norm"] else (None, None)
        if case["kind"] == "append":
            c = TYPES[case["cache"]]
            s["k_pages"], s["v_pages"] = (_randn(gen, n_pages, hkv, page, d).to(c) for _ in range(2))
        return s
    spans = _spans(case)
    need = [-(-c // page) for _, c in spans]
    n_pages = sum(need) + 4
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((len(spans), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    tokens = sum(n for n, _ in spans)
    starts = np.cumsum([0] + [n for n, _ in spans])
    s = {"q": (_randn(gen, tokens, hq, d) * 2.0).to(TYPES[case["q"]]), "table": table,
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "contexts": torch.tensor([c for _, c in spans], dtype=torch.int32, device="cuda")}
    src = TYPES["bf16" if case["cache"] == "q8_0" else case["cache"]]
    s["k_pages"], s["v_pages"] = (_randn(gen, n_pages, hkv, page, d).to(src) for _ in range(2))
    return s


def _quantized(x):
    """Q8_0: blocks of 32, a 16-bit scale amax / 127, values rounded half away from zero. Whole numbers and scales."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    d = top / torch.full_like(top, 127.0)  # a tensor divided by a number is multiplied by its rounded reciprocal
    inv = torch.where(d > 0, torch.ones_like(d) / d, torch.zeros_like(d))
    scaled = (b * inv).double()
    q = torch.sign(scaled) * torch.floor(scaled.abs() + 0.5)
    return q.to(torch.int8), d.half()


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    s["case"] = case
    if kind in ("rotate", "append"):
        angles = torch.arange(case["first"] + case["tokens"], device="cuda", dtype=torch.float64)[:, None] \
            * torch.from_numpy(_frequencies(case)).cuda()
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    if kind == "attend":
        spans = _spans(case)
        s["spans"], s["max_new"], s["max_context"] = spans, max(n for n, _ in spans), max(c for _, c in spans)
    if not own:
        if kind == "attend" and case["cache"] == "q8_0":
            s["k_pages"], s["v_pages"] = _quantized(s["k_pages"]), _quantized(s["v_pages"])
        return s
    import tur_b200 as tq
    dtype = {"bf16": tq.GgmlDType.BF16, "f16": tq.GgmlDType.F16, "q8_0": tq.GgmlDType.Q8_0, "none": None}[case["cache"]]
    if kind in ("rotate", "append"):
        s["rotary"] = tq.RotaryTable.from_frequencies(_frequencies(case), case["first"] + case["tokens"], interleaved=case["interleaved"])
    if dtype is not None:
        n_pages = s["pool"] if kind == "store" else s["k_pages"].shape[0]
        cache = s["cache"] = tq.KvCache.new(dtype, n_pages, case["page"], case["kv_heads"], case["head_dim"])
        if kind == "attend" and case["cache"] == "q8_0":
            rows = [p.transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"]).contiguous() for p in (s["k_pages"], s["v_pages"])]
            cache.write(*rows, torch.arange(rows[0].shape[0], device="cuda"))
        elif kind != "store":
            cache.k_pages.copy_(s["k_pages"])
            cache.v_pages.copy_(s["v_pages"])
        s.pop("k_pages", None), s.pop("v_pages", None)
    return s


# ---- one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import tur_b200 as tq
    case = s["case"]
    kind = case["kind"]
    if kind == "rotate":
        return tq.qk_norm_rope(s["q"], s["k"], s["positions"], s["rotary"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                               out_dtype=torch.bfloat16)
    cache = s["cache"]
    if kind == "append":
        q = cache.append(s["q"], s["k"], s["v"], s["positions"], s["rotary"], s["slots"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                         out_dtype=torch.bfloat16)
        return q, cache.k_pages, cache.v_pages
    if kind == "store":
        cache.write(s["k"], s["v"], s["slots"])
        return cache.read(s["slots"])
    return cache.attend(s["q"], s["starts"], s["contexts"], s["table"], max_new=s["max_new"], max_context=s["max_context"])


def _normed_rotated(x, w, cos, sin, case):
    x = x.float()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    rot, rest = x[..., :case["rotary"]], x[..., case["rotary"]:]
    if case["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = rot.chunk(2, -1)
        rot = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((rot, rest), -1)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("rotate", "append"):
        cos, sin = (t[s["positions"].long()][:, None, :] for t in (s["cos"], s["sin"]))
        q = _normed_rotated(s["q"], s["wq"], cos, sin, case).to(torch.bfloat16)
        k = _normed_rotated(s["k"], s["wk"], cos, sin, case)
        if kind == "rotate":
            return q, k.to(torch.bfloat16)
        page, off = s["slots"] // case["page"], s["slots"] % case["page"]
        s["k_pages"][page, :, off] = k.to(s["k_pages"].dtype)
        s["v_pages"][page, :, off] = s["v"].to(s["v_pages"].dtype)
        return q, s["k_pages"], s["v_pages"]
    if kind == "store":
        page, off, out = s["slots"] // case["page"], s["slots"] % case["page"], []
        for x in (s["k"], s["v"]):
            hkv, d = x.shape[1:]
            quants = torch.zeros((s["pool"], hkv, case["page"], d // 32, 32), dtype=torch.int8, device="cuda")
            scales = torch.zeros((s["pool"], hkv, case["page"], d // 32, 1), dtype=torch.float16, device="cuda")
            quants[page, :, off], scales[page, :, off] = _quantized(x)
            out.append((quants[page, :, off].float() * scales[page, :, off].float()).flatten(-2))
        return tuple(out)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    group = hq // hkv
    out = torch.zeros_like(s["q"])
    at = 0
    for i, (new, ctx) in enumerate(s["spans"]):
        pages = s["table"][i, :-(-ctx // case["page"])].long()
        k, v = (_context(p, pages, ctx) for p in (s["k_pages"], s["v_pages"]))
        step = max(1, int(2.5e8 / (hq * ctx)))  # rows whose scores are held at a time
        for r in range(0, new, step):
            n = min(step, new - r)
            seen = ctx - new + r + n             # keys that the last of these rows sees
            q = s["q"][at + r:at + r + n].float().reshape(n, hkv, group, d).permute(1, 2, 0, 3).reshape(hkv, group * n, d)
            scores = q @ k[:, :seen].transpose(1, 2) * (1.0 / math.sqrt(d))
            if n > 1:
                hidden = torch.arange(seen, device="cuda")[None, :] > (ctx - new + r + torch.arange(n, device="cuda"))[:, None]
                scores.view(hkv, group, n, seen).masked_fill_(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            o = p @ v[:, :seen] / p.sum(-1, keepdim=True)
            out[at + r:at + r + n] = o.view(hkv, group, n, d).permute(2, 0, 1, 3).reshape(n, hq, d).to(out.dtype)
        at += new
    return out


def _context(pages, index, ctx):
    """[heads, ctx, dim] of one sequence in 32 bits."""
    if isinstance(pages, tuple):
        x = (pages[0][index].float() * pages[1][index].float()).flatten(-2)
    else:
        x = pages[index].float()
    return x.transpose(0, 1).flatten(1, 2)[:, :ctx]


# ---- the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    d = case["head_dim"]
    if case["kind"] == "store":
        # the format's own steps are in 32 bits (scale and its reciprocal); what they give is exact in 64
        out = []
        for name in ("k", "v"):
            x = s[name].float().cpu().numpy().reshape(-1, 32)
            top = np.abs(x).max(axis=1).astype(np.float32)
            scale = (top / np.float32(127)).astype(np.float32)
            inv = np.divide(np.float32(1), scale, out=np.zeros_like(scale), where=scale > 0)
            y = (x * inv[:, None]).astype(np.float64)
            n = np.trunc(y + np.copysign(0.5, y))
            out.append(torch.from_numpy((n * scale.astype(np.float16).astype(np.float64)[:, None]).reshape(tuple(s[name].shape))).cuda())
        return tuple(out)
    if case["kind"] in ("rotate", "append"):
        freq = torch.from_numpy(_frequencies(case)).cuda()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * freq)[:, None, :]
        done = []
        for name, w in (("q", s["wq"]), ("k", s["wk"])):
            x = s[name].double()
            if w is not None:
                x = x * (x.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * w.double()
            half = case["rotary"] // 2
            first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            done.append(y)
        if case["kind"] == "rotate":
            return tuple(done)
        pools = []
        for pool, rows in ((s["k_pages"], done[1]), (s["v_pages"], s["v"].double())):
            flat = pool.double().transpose(1, 2).flatten(0, 1)
            flat[s["slots"]] = rows
            pools.append(flat.view(pool.shape[0], case["page"], case["kv_heads"], d).transpose(1, 2).contiguous())
        return done[0], pools[0], pools[1]
    group = case["q_heads"] // case["kv_heads"]
    held = []
    for pool in (s["k_pages"], s["v_pages"]):
        if case["cache"] == "q8_0":
            n, scale = _quantized(pool)
            pool = (n.double() * scale.double()).flatten(-2)
        held.append(pool)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (new, ctx) in enumerate(_spans(case)):
        where = torch.arange(ctx, device="cuda")
        page, off = s["table"][i].long()[where // case["page"]], where % case["page"]
        for h in range(case["kv_heads"]):
            k, v = (pool[page, h, off].double() for pool in held)
            for r in range(0, new, 1024):
                q = s["q"][at + r:at + min(new, r + 1024), h * group:(h + 1) * group].double()
                z = torch.einsum("ngd,cd->ngc", q, k) / d ** 0.5
                last = ctx - new + r + torch.arange(q.shape[0], device="cuda")
                z = torch.where((where <= last[:, None])[:, None, :], z, torch.full_like(z, -math.inf))
                out[at + r:at + r + q.shape[0], h * group:(h + 1) * group] = torch.einsum("ngc,cd->ngd", torch.softmax(z, -1), v)
        at += new
    return out
