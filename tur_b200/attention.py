"""Between attn_q|k|v and attn_output: head norms with the position rotation, the paged cache of keys and
values, and attention over it (include/turq.h, "Between attn_q|k|v and attn_output").

tur does these in Qwen3Attention::forward (src/models/qwen3.rs:263-505; without head norms in
src/models/granite_41.rs) on a PagedKvCache (src/models/kv_cache.rs:288-525). Tensors are packed: the new
tokens of all sequences of a call stand one behind the other, [n_tokens, heads, head_dim] (or
[n_tokens, heads * head_dim]); views with a longer stride between tokens are taken as they are.
Every call runs on the current stream of the cache's device, allocates its outputs and workspace from
torch and can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import torch

from . import _lib
from .linear import LinearX, linear
from .quantized import (_TORCH_TO_GGML, GgmlDType, Mode, QMatMul, TurqError, _check_operand, _Context, _stream_ptr, context)

_ROW_CODE = {t: int(c) for t, c in _TORCH_TO_GGML.items()}


def _rows(x: torch.Tensor, what: str, device: int, head_dim: int) -> tuple[int, int, int]:
    """(tokens, heads, elements from one token to the next) of a packed operand; refuses what the kernels cannot read."""
    # A token's calls take a few microseconds on the GPU: what is in order passes with as few questions as possible.
    if x.dim() == 3 and x.get_device() == device and x.dtype in _ROW_CODE:
        n, heads, d = x.shape
        s0, s1, s2 = x.stride()
        if d == head_dim and s2 == 1 and (s1 == d or heads == 1):
            return n, heads, s0 if n > 1 else heads * d
    return _rows_checked(x, what, device, head_dim)


def _rows_checked(x: torch.Tensor, what: str, device: int, head_dim: int) -> tuple[int, int, int]:
    if not x.is_cuda or x.get_device() != device:
        raise TurqError(1, f"{what} lives on {x.device}, expected cuda:{device}")
    if x.dtype not in _ROW_CODE:
        raise TurqError(3, f"{what} has dtype {x.dtype}, expected float32, float16 or bfloat16")
    if x.dim() == 3:
        n, heads, d = x.shape
        dense = x.stride(2) == 1 and (heads == 1 or x.stride(1) == d)
    elif x.dim() == 2:
        n, d = x.shape[0], head_dim
        heads = x.shape[1] // head_dim
        if heads * head_dim != x.shape[1]:
            raise TurqError(2, f"{what} has {x.shape[1]} columns, not whole heads of {head_dim}")
        dense = x.stride(1) == 1
    else:
        raise TurqError(2, f"{what} must be [n_tokens, heads, head_dim] or [n_tokens, heads * head_dim], got {tuple(x.shape)}")
    if d != head_dim:
        raise TurqError(2, f"{what} has heads of {d}, expected {head_dim}")
    if not dense:
        raise TurqError(1, f"{what} must hold the heads of a token side by side")
    return n, heads, x.stride(0) if n > 1 else heads * head_dim


def _vector(x: torch.Tensor, what: str, device: int, dtype: torch.dtype, n: Optional[int]) -> int:
    if x.dtype is dtype and x.get_device() == device and x.is_contiguous() and (n is None or x.numel() == n):
        return x.data_ptr()
    _check_operand(x, what, device, (dtype,))
    raise TurqError(2, f"{what} has {x.numel()} elements, expected {n}")


def _out(x: Optional[torch.Tensor], what: str, shape: tuple, dtype: torch.dtype, like: torch.Tensor) -> torch.Tensor:
    """The output given, or a new one on the device of `like`."""
    if x is None:
        return like.new_empty(shape, dtype=dtype)
    device = like.get_device()
    _check_operand(x, what, device, (dtype,))
    if x.numel() != math.prod(shape):
        raise TurqError(2, f"{what} has {x.numel()} elements, expected {shape}")
    return x


class RotaryTable:
    """cos and sin of every position a program will use, [n_positions, rotary_dim / 2, 2] f32 on the device, computed in 64
    bits (tur keeps the same table, src/models/qwen3.rs:64-78)."""

    def __init__(self, table: torch.Tensor, rotary_dim: int, interleaved: bool, ctx: _Context):
        self.table, self.rotary_dim, self.interleaved, self._ctx = table, rotary_dim, interleaved, ctx
        self._device = table.get_device()
        self._args = (table.data_ptr(), table.shape[0], rotary_dim, int(interleaved))

    @property
    def n_positions(self) -> int:
        return self.table.shape[0]

    @classmethod
    def new(cls, rotary_dim: int, n_positions: int, base: float = 1e6, interleaved: bool = False, scaling: Optional[dict] = None,
            device: int | torch.device | None = None, ctx: Optional[_Context] = None) -> "RotaryTable":
        """Frequencies base^(-2i / rotary_dim). `scaling`: {"type": "linear", "factor": f} divides every position by f;
        {"type": "yarn", "factor": f, "original": n} does so for the slow pairs only, keeps the fast ones (pairs that turn more
        than beta_fast = 32 times, fewer than beta_slow = 1 times over n positions, blended in between) and lengthens both by
        0.1 ln f + 1 (the YaRN paper's rule)."""
        if rotary_dim <= 0 or rotary_dim % 8:
            raise TurqError(2, f"rotary_dim {rotary_dim} must be a positive multiple of 8")
        if not 1.0 < base < math.inf:
            raise TurqError(1, f"base {base} must be finite and above 1")
        half = rotary_dim // 2
        freqs = [base ** (-2.0 * i / rotary_dim) for i in range(half)]
        scale = 1.0
        if scaling is not None:
            kind, factor = scaling.get("type"), float(scaling.get("factor", 1.0))
            if not 1.0 <= factor < math.inf:
                raise TurqError(1, f"scaling factor {factor} must be finite and at least 1")
            if kind == "linear":
                freqs = [f / factor for f in freqs]
            elif kind == "yarn":
                n = float(scaling.get("original", 0.0))
                if not 0.0 < n < math.inf:
                    raise TurqError(1, f"yarn scaling needs the original number of positions, got {scaling.get('original')}")

                fast, slowest = float(scaling.get("beta_fast", 32)), float(scaling.get("beta_slow", 1))
                if not 0.0 < slowest <= fast < math.inf:
                    raise TurqError(1, f"yarn scaling needs 0 < beta_slow <= beta_fast, got {slowest} and {fast}")

                def pair_of(turns: float) -> float:
                    return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

                low = max(0, math.floor(pair_of(fast)))
                high = min(rotary_dim - 1, math.ceil(pair_of(slowest)))
                for i in range(half):
                    slow = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
                    freqs[i] *= 1.0 - slow + slow / factor
                scale = 0.1 * math.log(factor) + 1.0
            else:
                raise TurqError(1, f"unknown scaling type {kind!r} (linear, yarn)")
        return cls.from_frequencies(freqs, n_positions, interleaved, scale, device, ctx)

    @classmethod
    def from_frequencies(cls, freqs: Sequence[float], n_positions: int, interleaved: bool = False, scale: float = 1.0,
                         device: int | torch.device | None = None, ctx: Optional[_Context] = None) -> "RotaryTable":
        """Angle of pair i at a position: position * freqs[i]; cos and sin times `scale`."""
        ctx = ctx or context(device)
        n = len(freqs)
        if n == 0 or n_positions <= 0:
            raise TurqError(2, f"a table of {n} frequencies and {n_positions} positions")
        table = torch.empty((n_positions, n, 2), dtype=torch.float32, device=torch.device("cuda", ctx.device))
        ctx.check(_lib.load().turq_rope_table(ctx.handle, (ctypes.c_double * n)(*[float(f) for f in freqs]), n, n_positions, float(scale),
                                              table.data_ptr(), _stream_ptr(ctx.device)))
        return cls(table, 2 * n, bool(interleaved), ctx)


def _weights(table: RotaryTable, head_dim: int, dev: int, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor]) -> tuple:
    if table._device != dev:
        raise TurqError(1, f"the rotary table lives on {table.table.device}, q on cuda:{dev}")
    return (None if q_weight is None else _vector(q_weight, "q_weight", dev, torch.float32, head_dim),
            None if k_weight is None else _vector(k_weight, "k_weight", dev, torch.float32, head_dim))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: RotaryTable, *, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None,
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm of every head (where a weight is given) and rotation of q [n, heads, d] and k [n, kv_heads, d] in one pass, into
    dense tensors of out_dtype (default: q's). positions: int32 [n]."""
    if q.dim() != 3 or k.dim() != 3:
        raise TurqError(2, "q and k must be [n_tokens, heads, head_dim]")
    ctx, d = table._ctx, q.shape[-1]
    dev = ctx.device
    n, hq, qs = _rows(q, "q", dev, d)
    nk, hkv, ks = _rows(k, "k", dev, d)
    if nk != n or k.dtype != q.dtype:
        raise TurqError(2, f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must agree in tokens and type")
    out_dtype = out_dtype or q.dtype
    if out_dtype not in _ROW_CODE:
        raise TurqError(3, f"out_dtype {out_dtype} is none of float32, float16, bfloat16")
    qo, ko = _out(q_out, "q_out", (n, hq, d), out_dtype, q), _out(k_out, "k_out", (n, hkv, d), out_dtype, q)
    wq, wk = _weights(table, d, dev, q_weight, k_weight)
    st = _lib.load().turq_qk_norm_rope(ctx.handle, q.data_ptr(), qs, k.data_ptr(), ks, _ROW_CODE[q.dtype], n, hq, hkv, d, wq, wk, eps, *table._args,
                                       _vector(positions, "positions", dev, torch.int32, n), _ROW_CODE[out_dtype], qo.data_ptr(), ko.data_ptr(),
                                       _stream_ptr(dev))
    if st != 0:
        ctx.check(st)
    return qo, ko


class KvCache:
    """One layer's keys and values in pages of `page_size` tokens, 16 bits (F16, BF16) or Q8_0. A slot is page * page_size +
    offset; which pages a sequence has is the caller's table. The memory is a torch tensor; `k_pages`, `v_pages`
    [n_pages, n_kv_heads, page_size, head_dim] (int8 for Q8_0, with `k_scales`, `v_scales` [..., head_dim / 32]) are views of it."""

    def __init__(self, handle: ctypes.c_void_p, memory: torch.Tensor, dtype: GgmlDType, shape: tuple, ctx: _Context):
        self._h, self.memory, self.dtype, self._ctx, self._device = handle, memory, dtype, ctx, ctx.device
        lib = _lib.load()
        self._append, self._write, self._read = lib.turq_kv_append, lib.turq_kv_write, lib.turq_kv_read
        self._attention, self._workspace = lib.turq_kv_attention, lib.turq_kv_attention_workspace
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = shape
        self._scale = 1.0 / math.sqrt(self.head_dim)
        off = (ctypes.c_int64 * 4)()
        ctx.check(_lib.load().turq_kv_cache_layout(handle, None, off))
        elem = {GgmlDType.F16: torch.float16, GgmlDType.BF16: torch.bfloat16, GgmlDType.Q8_0: torch.int8}[dtype]

        def plane(o, t, last):
            n = math.prod(shape[:3]) * last * t.itemsize
            return memory[o:o + n].view(t).view(*shape[:3], last)

        self.k_pages, self.v_pages = plane(off[0], elem, shape[3]), plane(off[1], elem, shape[3])
        self.k_scales = self.v_scales = None
        if dtype == GgmlDType.Q8_0:
            self.k_scales, self.v_scales = plane(off[2], torch.float16, shape[3] // 32), plane(off[3], torch.float16, shape[3] // 32)

    @classmethod
    def new(cls, dtype: GgmlDType, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device: int | torch.device | None = None,
            ctx: Optional[_Context] = None) -> "KvCache":
        ctx = ctx or context(device)
        lib = _lib.load()
        nbytes = lib.turq_kv_cache_bytes(int(dtype), n_pages, page_size, n_kv_heads, head_dim)
        memory = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=torch.device("cuda", ctx.device))
        h = ctypes.c_void_p()
        ctx.check(lib.turq_kv_cache_create(ctx.handle, int(dtype), n_pages, page_size, n_kv_heads, head_dim, memory.data_ptr(), nbytes,
                                           ctypes.byref(h)))
        return cls(h, memory, GgmlDType(dtype), (n_pages, n_kv_heads, page_size, head_dim), ctx)

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                _lib.load().turq_kv_cache_free(h)
            except Exception:
                pass

    def device(self) -> torch.device:
        return torch.device("cuda", self._ctx.device)

    def _kv(self, k: torch.Tensor, v: torch.Tensor) -> tuple:
        dev, d = self._device, self.head_dim
        n, hk, ks = _rows(k, "k", dev, d)
        nv, hv, vs = _rows(v, "v", dev, d)
        if hk != self.n_kv_heads or hv != self.n_kv_heads or nv != n or v.dtype != k.dtype:
            raise TurqError(2, f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} must agree, with {self.n_kv_heads} heads of {d}")
        return n, ks, vs

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, table: RotaryTable, slots: torch.Tensor, *,
               q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
               out_dtype: torch.dtype = torch.bfloat16, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """What attn_q|k|v gave for n new tokens: norms (where a weight is given) and rotation of q and k, k and v into their
        slots (int64 [n]; a negative one is skipped: padding), all in one pass. Returns q [n, heads, d] of out_dtype."""
        dev, d = self._device, self.head_dim
        n, ks, vs = self._kv(k, v)
        nq, hq, qs = _rows(q, "q", dev, d)
        dtype = q.dtype
        if nq != n or dtype is not k.dtype:
            raise TurqError(2, f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must agree in tokens and type")
        if out_dtype not in _ROW_CODE:
            raise TurqError(3, f"out_dtype {out_dtype} is none of float32, float16, bfloat16")
        if table._device != dev:
            raise TurqError(1, f"the rotary table lives on {table.table.device}, the cache on cuda:{dev}")
        wq = _vector(q_weight, "q_weight", dev, torch.float32, d) if q_weight is not None else None
        wk = _vector(k_weight, "k_weight", dev, torch.float32, d) if k_weight is not None else None
        p_positions, p_slots = _vector(positions, "positions", dev, torch.int32, n), _vector(slots, "slots", dev, torch.int64, n)
        qo = q.new_empty((n, hq, d), dtype=out_dtype) if q_out is None else _out(q_out, "q_out", (n, hq, d), out_dtype, q)
        t_ptr, t_n, t_dim, t_pairs = table._args
        st = self._append(self._ctx.handle, self._h, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, _ROW_CODE[dtype], n, hq, wq, wk, eps,
                          t_ptr, t_n, t_dim, t_pairs, p_positions, p_slots, _ROW_CODE[out_dtype], qo.data_ptr(), _stream_ptr(dev))
        if st != 0:
            self._ctx.check(st)
        return qo

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Keys and values as they are into their slots, rounded to the cache's type or quantized."""
        dev = self._device
        n, ks, vs = self._kv(k, v)
        st = self._write(self._ctx.handle, self._h, k.data_ptr(), ks, v.data_ptr(), vs, _ROW_CODE[k.dtype], n,
                         _vector(slots, "slots", dev, torch.int64, n), _stream_ptr(dev))
        if st != 0:
            self._ctx.check(st)

    def read(self, slots: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of the slots, [n, n_kv_heads, d] each; a negative slot reads as zeros."""
        dev, n = self._device, slots.numel()
        p_slots = _vector(slots, "slots", dev, torch.int64, None)
        if out_dtype not in _ROW_CODE:
            raise TurqError(3, f"out_dtype {out_dtype} is none of float32, float16, bfloat16")
        k = slots.new_empty((n, self.n_kv_heads, self.head_dim), dtype=out_dtype)
        v = torch.empty_like(k)
        st = self._read(self._ctx.handle, self._h, p_slots, n, _ROW_CODE[out_dtype], k.data_ptr(), v.data_ptr(), _stream_ptr(dev))
        if st != 0:
            self._ctx.check(st)
        return k, v

    def attend(self, q: torch.Tensor, starts: torch.Tensor, contexts: torch.Tensor, page_table: torch.Tensor, *, max_new: Optional[int] = None,
               max_context: Optional[int] = None, scale: Optional[float] = None, causal: bool = True,
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q K^T) V of the new tokens of n_seqs sequences over their pages: q [n, heads, d] packed, rows
        starts[i] .. starts[i + 1] (int32 [n_seqs + 1]) of sequence i, whose context of contexts[i] tokens (int32 [n_seqs], the new
        ones last) lies in the pages page_table[i] (int32 [n_seqs, pages]). scale: 1 / sqrt(d) by default. `out` may be q. Single tokens,
        chunks and whole prompts go together; max_new and max_context are the longest of each that the call may meet (the
        values on the device are not read here), by default all tokens and the whole page table. How the work is cut goes by them,
        so they are worth giving, and as small as they are: 64 users of one token each (Q8_0, contexts to 8000) take 154 us without
        max_new=1 and 115 with it, one user at 4096 keys 34 us with max_context=131072 and 8.6 with 4096.
        Q8_0 blocks of a context with scales above 515.5 (values beyond 65500, which f16 does not hold) are infinities to the
        products, and context().poll_status() reports them. `out` keeps its rows that belong to no sequence; without `out` they
        hold anything."""
        dev, d = self._device, self.head_dim
        n, hq, qs = _rows(q, "q", dev, d)
        p_table = _vector(page_table, "page_table", dev, torch.int32, None)
        if page_table.dim() != 2:
            raise TurqError(2, f"page_table must be [n_seqs, pages], got {tuple(page_table.shape)}")
        n_seqs, pages = page_table.shape
        p_starts = _vector(starts, "starts", dev, torch.int32, n_seqs + 1)
        p_contexts = _vector(contexts, "contexts", dev, torch.int32, n_seqs)
        max_new = n if max_new is None else int(max_new)
        max_context = pages * self.page_size if max_context is None else int(max_context)
        out_dtype = (out.dtype if out is not None else q.dtype) if out_dtype is None else out_dtype
        if out_dtype not in _ROW_CODE:
            raise TurqError(3, f"out_dtype {out_dtype} is none of float32, float16, bfloat16")
        if out is not None:
            y = _out(out, "out", (n, hq, d), out_dtype, q)
        elif out_dtype is q.dtype and q.dim() == 3 and q.is_contiguous():
            y = torch.empty_like(q)
        else:
            y = q.new_empty((n, hq, d), dtype=out_dtype)
        nbytes = self._workspace(self._h, n, n_seqs, hq, max_new, max_context)
        ws = y.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        st = self._attention(self._ctx.handle, self._h, q.data_ptr(), qs, _ROW_CODE[q.dtype], n, hq, p_starts, p_contexts, p_table, pages, n_seqs,
                             max_new, max_context, self._scale if scale is None else scale, causal, _ROW_CODE[out_dtype], y.data_ptr(),
                             ws.data_ptr() if nbytes else None, nbytes, _stream_ptr(dev))
        if st != 0:
            self._ctx.check(st)
        return y if y.dim() == 3 else y.view(n, hq, d)


class Attention:
    """tur's attention block on a quantized layer (Qwen3Attention, src/models/qwen3.rs:205-222, 263-505; Granite's without
    head norms): attn_q|k|v in one call, norms, rotation and cache write in one pass, attention, attn_output. q_dtype: the type of the
    queries between them, bfloat16 by default; float16 for F16 and Q8_0 caches keeps three bits more of queries below 65504. What
    goes to attn_output is bfloat16, with float16 queries or mode EXACT_F32 float32."""

    def __init__(self, q: LinearX, k: LinearX, v: LinearX, o: LinearX, head_dim: int, q_norm: Optional[torch.Tensor] = None,
                 k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, scale: Optional[float] = None,
                 q_dtype: torch.dtype = torch.bfloat16):
        if q_dtype not in (torch.bfloat16, torch.float16):
            raise TurqError(3, f"q_dtype {q_dtype} is neither bfloat16 nor float16")
        self.q, self.k, self.v, self.o = q, k, v, o
        self.head_dim, self.q_norm, self.k_norm, self.eps, self.scale, self.q_dtype = head_dim, q_norm, k_norm, eps, scale, q_dtype

    @classmethod
    def new(cls, vb, hidden: int, n_heads: int, n_kv_heads: int, head_dim: int, eps: float = 1e-6, scale: Optional[float] = None,
            q_dtype: torch.dtype = torch.bfloat16) -> "Attention":
        """From the tensors of one block (`vb.pp("blk").pp(i)`): attn_q, attn_k, attn_v, attn_output, and attn_q_norm /
        attn_k_norm where the file has them."""
        def norm(name):
            return vb.pp(name).get(head_dim, "weight").dequantize().reshape(head_dim) if vb.pp(name).contains_key("weight") else None

        return cls(linear(hidden, n_heads * head_dim, vb.pp("attn_q")), linear(hidden, n_kv_heads * head_dim, vb.pp("attn_k")),
                   linear(hidden, n_kv_heads * head_dim, vb.pp("attn_v")), linear(n_heads * head_dim, hidden, vb.pp("attn_output")),
                   head_dim, norm("attn_q_norm"), norm("attn_k_norm"), eps, scale, q_dtype)

    def forward(self, x: torch.Tensor, cache: KvCache, table: RotaryTable, positions: torch.Tensor, slots: torch.Tensor, starts: torch.Tensor,
                contexts: torch.Tensor, page_table: torch.Tensor, *, max_new: Optional[int] = None, max_context: Optional[int] = None,
                mode: Mode = Mode.AUTO) -> torch.Tensor:
        """x [n_tokens, hidden] (f32 or bf16), the packed new tokens of all sequences -> [n_tokens, hidden] f32. The other
        arguments are those of KvCache.append and KvCache.attend. Rows of tokens that belong to no sequence (the padding of a
        captured batch) follow from x alone and mean nothing."""
        linears = (self.q, self.k, self.v)
        biases = [l.bias for l in linears] if any(l.bias is not None for l in linears) else None
        q, k, v = QMatMul.forward_multi([l.qmatmul for l in linears], x, biases=biases, mode=mode)
        q = cache.append(q, k, v, positions, table, slots, q_weight=self.q_norm, k_weight=self.k_norm, eps=self.eps, out_dtype=self.q_dtype)
        # Into q's own memory, or into zeros: rows of tokens of no sequence hold their queries then, and not what the memory held before.
        # f32 where its bits are asked for: it costs 2 us a call, and twice the bytes (2048 tokens 5 % of a layer's time).
        wide = mode == Mode.EXACT_F32 or q.dtype is not torch.bfloat16
        y = cache.attend(q, starts, contexts, page_table, max_new=max_new, max_context=max_context, scale=self.scale,
                         out=torch.zeros_like(q, dtype=torch.float32) if wide else q)
        return self.o.forward(y.view(y.shape[0], -1), mode=mode)

    __call__ = forward
