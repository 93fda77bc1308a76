"""A paged key / value cache in 8-bit floating point: pages of a step, writes, and the decode that reads it.

The reference's serving call reads a 16-bit paged cache that its caller fills (core/template/cute_template_kvshared/
flash_mla_interface.py:73-113); here the cache is half as large, and the two steps in front of the attention, handing out pages and writing
the new tokens, are operators as well:

    cache = PagedCache8(num_pages, page_size, n_kv_heads, head_dim)
    plan = plan_pages(lens, new_lens, block_table, free_pages, free_head, page_size, n_tokens)   # once per step
    cache.write(k, v, plan.segments)                                                             # k, v [n_tokens, Hkv, D], every layer
    o = engine.decode_cache8(q, cache, plan.block_table, plan.seq_lens)                          # engine built with cache_dtype

Nothing of a step is read back to the host, so it can be captured into a CUDA graph.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from .. import runtime as rt
from ..lower.cuda_lower import lower_attention
from ..lower.torch_eval import evaluate

E4M3 = torch.float8_e4m3fn
MAX_ROWS = 4096        # rows of a step (AE_PLAN_ROWS of plan_pages.cuh)
PAGE_SIZES = (16, 32, 64, 128)
STATUS_TEXT = {1: "the free pages ran out", 2: "a row needs more pages than block_table has columns",
               4: "the new lengths add up to more than n_tokens", 8: "a length is negative"}


class PagePlan(NamedTuple):
    """What ``plan_pages`` makes; every field is a tensor on the lengths' device."""
    block_table: torch.Tensor  #: the caller's, with the new pages entered
    cu_seqlens: torch.Tensor   #: int32 [B + 1]: row b's new tokens are cu_seqlens[b] ... of the packed axis
    positions: torch.Tensor    #: int32 [n_tokens]: position of each new token in its row (-1 behind the last one)
    slots: torch.Tensor        #: int64 [n_tokens]: page * page_size + offset (-1 without a page)
    seq_lens: torch.Tensor     #: int32 [B]: old + new
    free_head: torch.Tensor    #: int32 [1]: pages taken from free_pages so far
    segments: torch.Tensor     #: int32 [n, 4]: (page, first slot, first token, tokens) of every page that gets tokens, then zeros
    status: torch.Tensor       #: int32 [1]: 0, or bits of STATUS_TEXT

    def check(self):
        """Raise if the plan does not hold all tokens (reads the status word: waits for the GPU)."""
        code = int(self.status.item())
        if code:
            raise ValueError("plan_pages: " + "; ".join(t for bit, t in STATUS_TEXT.items() if code & bit))


@functools.lru_cache(maxsize=None)
def _plan_kernel():
    smem = 3 * (MAX_ROWS + 1) * 4 + 4 + 2 * 8 * 8 + 8
    cfg = rt.KernelConfig(kind=rt.KIND_PLAN_PAGES, threads=256, smem_bytes=smem)
    return rt.compile_module(rt.kernel_source("plan_pages.cuh", prelude=f"#define AE_PLAN_ROWS {MAX_ROWS}\n"), "ae_plan_pages", cfg)


def plan_pages(old_lens, new_lens, block_table, free_pages, free_head, page_size: int, n_tokens: int) -> PagePlan:
    """Pages, slots and segments of a step in which row b, with ``old_lens[b]`` tokens in its pages, gets ``new_lens[b]`` more.

    All int32 tensors on one GPU: ``old_lens``, ``new_lens`` [B]; ``block_table`` [B, max_pages], whose new entries are written in place;
    ``free_pages`` [n] of which the first ``free_head[0]`` are taken.  Pages are handed out in the order of the rows.  ``n_tokens`` is the
    length of the packed axis, at least the sum of ``new_lens``.  Lengths are not read on the host: what does not fit is left out and
    reported in ``status``.  ``old_lens`` and ``free_head`` are not changed; the next step's are ``plan.seq_lens`` and ``plan.free_head``.
    Pages come back through ``plan_forks`` (a row that has ended: parent -1), or by the caller's hand: a row that has ended gets a length of 0, and the next step a
    ``free_pages`` with its pages behind those not yet taken, and a head of 0."""
    if isinstance(page_size, bool) or not isinstance(page_size, int) or isinstance(n_tokens, bool) or not isinstance(n_tokens, int):
        raise TypeError("page_size and n_tokens are ints")
    r = rt.host().plan_pages(_plan_kernel().handle.value, old_lens, new_lens, block_table, free_pages, free_head, page_size, n_tokens)
    if r is None:
        _refuse_plan(old_lens, new_lens, block_table, free_pages, free_head, page_size, n_tokens)
    return PagePlan(*r)


def _ints(name, t, dim, device):
    if not t.is_cuda:
        raise rt.AeError(f"{name} must be a CUDA tensor: this back end has no CPU path")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dtype != torch.int32 or t.dim() != dim or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be int32 with {dim} dimension(s), the last contiguous")


def refuse_gradients(what: str, named):
    """Raise if one of ``named``, (name, tensor) pairs, wants a gradient of a call that has none, or carries a tangent."""
    for name, t in named:
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{name} requires a gradient: {what} forward only")
        if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has a tangent: {what} without derivatives")


def _refuse_plan(old_lens, new_lens, block_table, free_pages, free_head, page_size, n_tokens):
    for name, t, dim in (("old_lens", old_lens, 1), ("new_lens", new_lens, 1), ("block_table", block_table, 2),
                         ("free_pages", free_pages, 1), ("free_head", free_head, 1)):
        _ints(name, t, dim, old_lens.device)
    B = old_lens.shape[0]
    if not 1 <= B <= MAX_ROWS or new_lens.shape[0] != B or block_table.shape[0] != B or block_table.shape[1] < 1:
        raise ValueError(f"1 to {MAX_ROWS} rows, as many in old_lens, new_lens and block_table, and a column at least")
    if free_head.shape[0] != 1:
        raise ValueError("free_head has one element")
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError(f"page_size {page_size}: a power of two")
    raise ValueError(f"n_tokens = {n_tokens} or the number of free pages is outside 0 ... 2^31 - 1")


class PagedCache8:
    """Keys and values of one layer in e4m3: ``k`` [num_pages, page_size, Hkv, D], ``v`` [..., DV], and a fp32 scale for each page and
    head, ``k_scale`` and ``v_scale`` [num_pages, Hkv]: a value is its code times its page's scale for the head.

    ``page_size`` 16, 32, 64 or 128; head dims 64 or 128.  Scales that ``write`` makes are powers of two; a cache filled elsewhere may hold
    any positive ones."""

    def __init__(self, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, head_dim_v: int | None = None, device="cuda"):
        dv = head_dim if head_dim_v is None else head_dim_v

        def pool(d):
            return torch.zeros(num_pages, page_size, n_kv_heads, d, dtype=torch.uint8, device=device).view(E4M3)

        self._hold(pool(head_dim), pool(dv), *(torch.ones(num_pages, n_kv_heads, dtype=torch.float32, device=device) for _ in "kv"))

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale):
        """A cache over the caller's tensors, which stay the caller's to read and write."""
        self = cls.__new__(cls)
        self._hold(k, v, k_scale, v_scale)
        return self

    def _hold(self, k, v, k_scale, v_scale):
        for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            if not t.is_cuda:
                raise rt.AeError(f"{name} must be a CUDA tensor: this back end has no CPU path")
            if t.device != k.device:
                raise ValueError(f"{name} is on {t.device}, k on {k.device}")
        for name, t in (("k", k), ("v", v)):
            if t.dtype != E4M3:
                raise TypeError(f"{name} has dtype {t.dtype}: codes are torch.float8_e4m3fn")
            if t.dim() != 4 or t.stride(3) != 1 or t.shape[:3] != k.shape[:3]:
                raise ValueError(f"{name} must be [num_pages, page_size, Hkv, D] with a contiguous last dimension, k and v alike")
            if t.shape[1] not in PAGE_SIZES:
                raise ValueError(f"page size {t.shape[1]}: one of {PAGE_SIZES}")
            if t.shape[3] not in (64, 128):
                raise NotImplementedError(f"head dim {t.shape[3]}: 64 and 128 are supported")
            if t.shape[0] < 1 or not 1 <= t.shape[2] <= 65535:
                raise ValueError("a cache has a page and a head at least")
            if t.data_ptr() % 16 or any(s % 16 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
                raise ValueError(f"{name} and its strides must be multiples of 16 bytes")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or t.shape != (k.shape[0], k.shape[2]) or (t.shape[1] > 1 and t.stride(1) != 1):
                raise ValueError(f"{name} must be float32 [num_pages, Hkv] with contiguous heads")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.page_size, self.n_kv_heads = k.shape[:3]
        self.head_dim, self.head_dim_v = k.shape[3], v.shape[3]
        self._native = rt.host().Cache8(k, v, k_scale, v_scale)
        self._write = _write_kernel(self.page_size, self.head_dim, self.head_dim_v)
        self._write_handle = self._write.handle.value

    def write(self, k, v, segments):
        """Round the new keys and values ``k`` [n, Hkv, D], ``v`` [n, Hkv, DV] (fp16 or bf16) into the pages that ``segments``
        (``plan_pages(...).segments``) names.

        A page's scale for a head is the smallest power of two that keeps its largest finite value at most 448; a page that goes on
        keeps its scale or takes the coarser one that the new tokens need, and its codes are rounded again.  Infinities and NaN
        become NaN.  No two segments of a call name the same page."""
        if not rt.host().cache8_write(self._write_handle, self._native, k, v, segments):
            self._refuse(k, v, segments)

    def _refuse(self, k, v, segments):
        for name, t, d in (("k", k, self.head_dim), ("v", v, self.head_dim_v)):
            if not t.is_cuda:
                raise rt.AeError(f"{name} must be a CUDA tensor: this back end has no CPU path")
            if t.device != self.k.device:
                raise ValueError(f"{name} is on {t.device}, the cache on {self.k.device}")
            if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != k.dtype:
                raise TypeError(f"{name} has dtype {t.dtype}: fp16 or bf16, k and v alike")
            if t.dim() != 3 or tuple(t.shape) != (k.shape[0], self.n_kv_heads, d) or t.stride(2) != 1:
                raise ValueError(f"{name} must be [n, {self.n_kv_heads}, {d}] with a contiguous last dimension, got {tuple(t.shape)}")
            if t.requires_grad and torch.is_grad_enabled():
                raise NotImplementedError(f"{name} requires a gradient: a write into the cache has none")
        _ints("segments", segments, 2, self.k.device)
        if segments.shape[1] != 4 or (segments.shape[0] > 1 and segments.stride(0) != 4):
            raise ValueError("segments must be contiguous [n, 4]")
        raise NotImplementedError("a write into the cache takes no forward-mode gradients and is not traced")


@functools.lru_cache(maxsize=None)
def _write_kernel(page: int, D: int, DV: int):
    threads = max(32, page * max(D, DV) // 64)  # 64 values each: the kernel's comment
    cfg = rt.KernelConfig(kind=rt.KIND_CACHE8_WRITE, head_dim=D, head_dim_v=DV, threads=threads)
    src = rt.kernel_source("cache8_write.cuh", defines={"AE_PAGE": page, "AE_D": D, "AE_DV": DV, "AE_W_THREADS": threads})
    return rt.compile_module(src, "ae_cache8_write", cfg)


def is_softmax(online_func) -> bool:
    """Whether the traced recurrence is that of a softmax: tile by tile over random scores, some of them -inf, it gives
    softmax(scores) V."""
    from ..core.transform.core import SymbolicArray, SymbolScalar, Var
    try:
        g = torch.Generator().manual_seed(11)
        R, N, T, DV = 8, 16, 4, 4
        scores = [torch.randn(R, N, generator=g, dtype=torch.float64) * (1 + 2 * t) for t in range(T)]
        for t in range(T):
            scores[t][t, 3:9] = -torch.inf
        vals = [torch.randn(N, DV, generator=g, dtype=torch.float64) for _ in range(T)]
        rs = {k: SymbolScalar(k, Var(k), shape_idx=["block_M"]) for k in online_func.online_rowscales}
        state = {k: torch.full((R, 1), float(str(v.code.name if v.code.type == "Var" else v.code.value).replace("inf", "1e30")),
                               dtype=torch.float64) for k, v in online_func.online_rowscales.items()}
        x = SymbolicArray("scores", Var("scores"), shape_idx=["block_M", "block_N"])
        idx = [SymbolScalar(n, Var(n), require_grad=False) for n in ("b", "h", "q_idx")]
        p_sym, rs_new, osc_sym = online_func.online_fwd(x, dict(rs), *idx)
        o = torch.zeros(R, DV, dtype=torch.float64)
        for s, v in zip(scores, vals):
            env, cache = {id(rs[k]): state[k] for k in rs}, {}
            env[id(x)] = s
            p, osc = torch.as_tensor(evaluate(p_sym, env, cache)), evaluate(osc_sym, env, cache)
            state = {k: torch.as_tensor(evaluate(e, env, cache), dtype=torch.float64).expand(R, 1) for k, e in rs_new.items()}
            o = o * osc + p @ v
        o_sym = SymbolicArray("o", Var("o"), shape_idx=["block_M", "dimv"])
        o_new, _ = online_func.online_fwd_epilogue(o_sym, rs, *idx)
        env = {id(rs[k]): state[k] for k in rs}
        env[id(o_sym)] = o
        want = torch.softmax(torch.cat(scores, 1), -1) @ torch.cat(vals)
        return torch.allclose(torch.as_tensor(evaluate(o_new, env)), want, rtol=1e-9, atol=1e-9)
    except Exception:  # what the evaluator cannot run is not taken for a softmax
        return False


class CacheDecode8:
    """The 8-bit side of a decode engine: traced ``score_mod`` and ``mask_mod``, softmax rows."""

    def __init__(self, score_mod, mask_mod, online_func, custom_fwd_inputs, Hq, Hkv, Sq, D, DV, dtype, mask_value="-inf"):
        if Hq % Hkv:
            raise ValueError("query heads must be a multiple of kv heads")
        if Hq > Hkv and Sq != 1:
            raise NotImplementedError("decode with grouped query heads takes q_len == 1 (as the reference does)")
        if D not in (64, 128) or DV not in (64, 128):
            raise NotImplementedError(f"head dims D={D}, DV={DV}: 64 and 128 are supported over an 8-bit cache")
        if mask_mod is not None and str(mask_value).strip() not in ("-inf", "-float('inf')"):
            raise NotImplementedError("an 8-bit cache is read with the mask value -inf")
        if not is_softmax(online_func):
            raise NotImplementedError("an 8-bit cache is read with the softmax recurrence: the value scales go into its exponent")
        self.rows = Hq // Hkv if Hq > Hkv else Sq
        self.Hq, self.Hkv, self.Sq, self.D, self.DV, self.dtype = Hq, Hkv, Sq, D, DV, dtype
        bf16 = dtype == torch.bfloat16
        self.low = lower_attention(score_mod, mask_mod, online_func, custom_fwd_inputs, D=D, DV=DV, bf16=bf16,
                                   mask_mode=0 if mask_mod is None else 3, mask_value=mask_value)
        if any(d > 1 for sp in self.low.custom for d in sp.dim_slots):
            raise NotImplementedError("custom inputs over positions are not read beside an 8-bit cache: batch and heads only")
        self.rt = 8 if self.rows <= 8 else 16
        self.kernel, self.merge = self._build()
        customs = [(sp.slot, bool(sp.is_16bit), [int(d) for d in sp.dim_slots]) for sp in self.low.custom]
        self.plan = rt.host().Decode8Plan(self.kernel.handle.value, self.merge.handle.value, bf16, Hq, Hkv, Sq, D, DV, customs)

    def _build(self):
        # 32 keys a tile at 128 dims, 64 at 64: 8 KB; eight warps with three tiles under way each (two where the partials of 16 query rows need
        # the room) fill an SM's shared memory, and four warps fetch.  In a graph: 64 ragged rows of up to 16384 keys, 8 heads of 128 dims: 125 us, with
        # two tiles under way 135; 16 rows of 4096 keys 34.8 and 36.0.  A team takes two tiles at least: one row of 2000 keys 12.0, one at least
        # 10.0, four 15.9; 24 rows of up to 1500 keys, 16 heads of 64 dims 15.9, 15.9 and 17.1; the others within 1 %.  A unit of up to four tiles a
        # warp is a CTA's (`single`): one row of 700 keys 8.2 instead of 11.2, 16 rows of 1000 keys 13.0 instead of 18.0; up to eight tiles a warp, 16 rows of 2000 keys take
        # 19.1 instead of 21.7, one row of them 15.7 instead of 12.0.  Other numbers of warps were compared on an earlier form alone, in which each warp copied its own
        # tiles.
        tile, warps, fetch, slots, least, single = 4096 // max(self.D, self.DV), 8, 4, 3 if self.rt == 8 else 2, 2, 4
        smem = warps * slots * (tile * (self.D + self.DV) + tile // 8 * 4 + 16) + warps * (self.rt * (self.DV + 2) * 4 + 64) + 208 + 1024
        cfg = rt.KernelConfig(kind=rt.KIND_CACHE8_DECODE, dtype=rt.DTYPE_BF16 if self.dtype == torch.bfloat16 else rt.DTYPE_F16,
                              head_dim=self.D, head_dim_v=self.DV, threads=32 * (warps + fetch), smem_bytes=smem, stages=slots,
                              mask_mode=self.low.defines["AE_MASK_MODE"])
        cfg.reserved[0], cfg.reserved[2], cfg.reserved[3], cfg.reserved[4] = self.rt, tile, warps, single
        self.src = rt.kernel_source("cache8_decode.cuh", prelude=self.low.prelude_fwd, defines={
            "AE_RT": self.rt, "AE_T": tile, "AE_T_LOG2": tile.bit_length() - 1, "AE_WARPS": warps, "AE_FETCH": fetch, "AE_C8_SLOTS": slots, "AE_MIN_TILES": least})
        merge_cfg = rt.KernelConfig(kind=rt.KIND_CACHE8_MERGE, dtype=cfg.dtype, head_dim=self.D, head_dim_v=self.DV, threads=128)
        merge_cfg.reserved[0] = warps
        self.merge_src = rt.kernel_source("cache8_merge.cuh", defines={
            "AE_BF16": int(self.dtype == torch.bfloat16), "AE_DV": self.DV, "AE_RT": self.rt, "AE_WARPS": warps})
        return rt.compile_module(self.src, "ae_cache8_decode", cfg), rt.compile_module(self.merge_src, "ae_cache8_merge", merge_cfg)

    @property
    def status(self):
        return self.plan.status

    def __call__(self, q, cache, block_table, seq_lens, *custom):
        if not isinstance(cache, PagedCache8):
            raise TypeError(f"expected a PagedCache8, got {type(cache).__name__}")
        o = rt.host().decode8(self.plan, cache._native, q, block_table, seq_lens, custom)
        if o is None:
            self._refuse(q, cache, block_table, seq_lens, custom)
        return o

    def _refuse(self, q, cache, block_table, seq_lens, custom):
        """The native path did not take these tensors: raise what is wrong with them."""
        if not q.is_cuda:
            raise rt.AeError("q must be a CUDA tensor: this back end has no CPU path")
        if q.dtype != self.dtype:
            raise TypeError(f"q has dtype {q.dtype}, engine was built for {self.dtype}")
        if q.dim() != 4 or q.stride(3) != 1 or tuple(q.shape[1:]) != (self.Sq, self.Hq, self.D):
            raise ValueError(f"q must be [B, {self.Sq}, {self.Hq}, {self.D}] with a contiguous last dimension, got {tuple(q.shape)}")
        if (cache.n_kv_heads, cache.head_dim, cache.head_dim_v) != (self.Hkv, self.D, self.DV):
            raise ValueError(f"the cache has (Hkv, D, DV) = {(cache.n_kv_heads, cache.head_dim, cache.head_dim_v)}, the engine "
                             f"{(self.Hkv, self.D, self.DV)}")
        if q.device != cache.k.device:
            raise ValueError(f"q is on {q.device}, the cache on {cache.k.device}")
        _ints("block_table", block_table, 2, q.device)
        _ints("seq_lens", seq_lens, 1, q.device)
        B = q.shape[0]
        if block_table.shape[0] != B or block_table.shape[1] < 1 or seq_lens.shape[0] != B:
            raise ValueError(f"block_table must be [{B}, pages] and seq_lens [{B}]")
        if len(custom) != len(self.low.custom):
            raise TypeError(f"expected {len(self.low.custom)} custom input(s) {[s.name for s in self.low.custom]}, got {len(custom)}")
        refuse_gradients("decode over a cache is", [("q", q)] + [(f"custom input {sp.name}", t) for sp, t in zip(self.low.custom, custom)])
        raise ValueError("tensors do not fit this engine")
