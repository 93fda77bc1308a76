"""Pages of a cache that rows share, give back and move, as plans on the GPU and copies of what they name:

    fork = plan_forks(parents, seq_lens, block_table, free_pages, free_head, page_size, num_pages)   # rows go on from others, or end
    copy_pages(caches, fork.copies)                                                                  # every layer's cache, one launch
    pack = plan_compaction(seq_lens, block_table, page_size, num_pages)                              # pages in use to the front of the pool
    copy_pages(caches, pack.copies)

``plan_pages`` goes on from either's ``block_table``, ``free_pages`` and ``free_head``.  Nothing is read back to the host, and nothing that a plan reads is
changed, so every call can be captured into a CUDA graph.  (The reference's block tables are its caller's, core/template/cute_template_kvshared/
flash_mla_interface.py:73-113.)
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from .. import runtime as rt
from .cache8 import MAX_ROWS, PagedCache8, _ints

STATUS_TEXT = {1: "the free pages ran out", 2: "a length is beyond block_table's columns", 4: "more pages came back than free_head says are taken",
               8: "a parent is no row, a length is negative, or more tokens are kept than there are", 16: "a page is outside the pool"}
LIST_THREADS, LIST_BATCH = (1024, 512), 4  # threads of the kernel of all phases, and of those of one
LIST_SMEM = 16 * 1024 + 12 * 512 + 6 * 16384 + 16  # 1024 rows, 16384 pages
COPY_THREADS, COPY_UNROLL, COPY_CTAS, COPY_PART = 64, (8, 16), 32, 32768  # threads, reads of each on their way, CTAs of an SM, bytes of a part


def _check(what, status):
    code = int(status.item())
    if code:
        raise ValueError(f"{what}: " + "; ".join(t for bit, t in STATUS_TEXT.items() if code & bit))


class ForkPlan(NamedTuple):
    """What ``plan_forks`` makes; every field is a new tensor on the lengths' device."""
    block_table: torch.Tensor  #: int32 [B, max_pages]: the rows' pages, then 0
    seq_lens: torch.Tensor     #: int32 [B]
    free_pages: torch.Tensor   #: int32 [n]: the list with the pages that came back
    free_head: torch.Tensor    #: int32 [1]: how many of it are taken
    copies: torch.Tensor       #: int32 [B, 4]: (page, new page, slots, 0) for ``copy_pages``, then zeros
    status: torch.Tensor       #: int32 [1]: 0, or bits of STATUS_TEXT

    def check(self):
        """Raise if something did not fit (reads the status word: waits for the GPU)."""
        _check("plan_forks", self.status)


class CompactionPlan(NamedTuple):
    """What ``plan_compaction`` makes; every field is a new tensor on the lengths' device."""
    block_table: torch.Tensor  #: int32 [B, max_pages]: the rows' pages by their new numbers, then 0
    free_pages: torch.Tensor   #: int32 [num_pages]: all pages in order
    free_head: torch.Tensor    #: int32 [1]: how many are in use; the pool may be cut behind them
    copies: torch.Tensor       #: int32 [num_pages // 2, 4]: (page, new page, slots in use, 0) for ``copy_pages``, then zeros
    status: torch.Tensor       #: int32 [1]: 0, or bits of STATUS_TEXT

    def check(self):
        """Raise if something did not fit (reads the status word: waits for the GPU)."""
        _check("plan_compaction", self.status)


def _list_source(file: str, phase: int) -> str:
    return rt.kernel_source("page_lists.cuh", file, defines={"AE_LIST_THREADS": LIST_THREADS[phase > 0], "AE_LIST_BATCH": LIST_BATCH, "AE_PHASE": phase})


def _list_kernels(kind: int, file: str, name: str, phases: int):
    """The kernel that runs all phases in one CTA, then one for each phase."""
    out = []
    for phase in range(phases + 1):
        cfg = rt.KernelConfig(kind=kind, threads=LIST_THREADS[phase > 0], smem_bytes=0 if phase else LIST_SMEM)
        cfg.reserved[1] = phase
        out.append(rt.compile_module(_list_source(file, phase), name, cfg))
    return tuple(out), [m.handle.value for m in out]


@functools.lru_cache(maxsize=None)
def _forks_kernels():
    return _list_kernels(rt.KIND_PLAN_FORKS, "plan_forks.cuh", "ae_plan_forks", 3)


@functools.lru_cache(maxsize=None)
def _compaction_kernels():
    return _list_kernels(rt.KIND_PLAN_COMPACTION, "plan_compaction.cuh", "ae_plan_compaction", 4)


def _copy_source(runs: bool) -> str:
    return rt.kernel_source("copy_pages.cuh", defines={"AE_COPY_THREADS": COPY_THREADS, "AE_COPY_UNROLL": COPY_UNROLL[runs], "AE_COPY_RUNS": int(runs)})


@functools.lru_cache(maxsize=None)
def _copy_kernels():
    """For pools of any layout, and for those whose slots lie behind each other."""
    out = []
    for runs in (False, True):
        cfg = rt.KernelConfig(kind=rt.KIND_COPY_PAGES, threads=COPY_THREADS)
        cfg.reserved[0], cfg.reserved[1], cfg.reserved[2] = COPY_PART, COPY_CTAS, int(runs)
        out.append(rt.compile_module(_copy_source(runs), "ae_copy_pages", cfg))
    return tuple(out), [m.handle.value for m in out]


def _sizes(page_size, num_pages):
    for n in (page_size, num_pages):
        if isinstance(n, bool) or not isinstance(n, int):
            raise TypeError("page_size and num_pages are ints")


def plan_forks(parents, seq_lens, block_table, free_pages, free_head, page_size: int, num_pages: int, keep_lens=None) -> ForkPlan:
    """Pages of a step in which row b goes on from row ``parents[b]`` (itself: nothing happens; -1: the row ends), of which it keeps the first
    ``keep_lens[b]`` tokens (None: all).

    All int32 tensors on one GPU: ``parents``, ``seq_lens``, ``keep_lens`` [B]; ``block_table`` [B, max_pages] of pages below ``num_pages``; ``free_pages`` [n]
    of which the first ``free_head[0]`` are taken.  Whole pages are shared between the rows that have them in common.  A begun page stays with
    one row, and only if none holds it whole; the others take a free page each, in the order of the rows, which ``copy_pages`` fills from
    ``copies``.  Pages that no row holds any more go back to the free list, lowest on top; where the list does not last, they serve the rows behind it,
    lowest first.  So a sampled prompt is B rows with one parent, a beam search's step its parents, and a cut (speculation that failed) a row that keeps less
    of itself.

    Rows are shortened through ``keep_lens`` alone: a length that a caller lowers by itself would let ``plan_pages`` put new tokens into a page that other rows hold.
    Pages that something beside the table's rows is to keep (a prefix for later requests) need a row of their own in it.  What does not fit is left
    out and reported in ``status``."""
    _sizes(page_size, num_pages)
    r = rt.host().plan_forks(_forks_kernels()[1], parents, seq_lens, block_table, free_pages, free_head, page_size, num_pages, keep_lens)
    if r is None:
        named = [("parents", parents, 1), ("seq_lens", seq_lens, 1), ("block_table", block_table, 2), ("free_pages", free_pages, 1),
                 ("free_head", free_head, 1)] + ([("keep_lens", keep_lens, 1)] if keep_lens is not None else [])
        _refuse(named, seq_lens, block_table, page_size, num_pages)
        if free_head.shape[0] != 1:
            raise ValueError("free_head has one element")
        B = seq_lens.shape[0]
        raise ValueError(f"1 to {MAX_ROWS} rows, as many in parents, seq_lens, keep_lens and block_table, got {B}")
    return ForkPlan(*r)


def plan_compaction(seq_lens, block_table, page_size: int, num_pages: int) -> CompactionPlan:
    """Moves that bring the pages in use to the front of a pool of ``num_pages``: with U of them, those from U on go into the unused ones below U, both in ascending
    order.  ``seq_lens`` [B] and ``block_table`` [B, max_pages] int32; rows may share pages.

    Every page that no row holds counts as unused, so all of a pool's rows have to be in the table.  ``copy_pages(caches, plan.copies)`` has to
    follow before the new table is used."""
    _sizes(page_size, num_pages)
    r = rt.host().plan_compaction(_compaction_kernels()[1], seq_lens, block_table, page_size, num_pages)
    if r is None:
        _refuse([("seq_lens", seq_lens, 1), ("block_table", block_table, 2)], seq_lens, block_table, page_size, num_pages)
        raise ValueError("seq_lens [B] and block_table [B, max_pages] of a row at least")
    return CompactionPlan(*r)


def _refuse(named, seq_lens, block_table, page_size, num_pages):
    for name, t, dim in named:
        _ints(name, t, dim, seq_lens.device)
    if page_size < 1 or page_size > 2 ** 30 or page_size & (page_size - 1):
        raise ValueError(f"page_size {page_size}: a power of two")
    if not 1 <= num_pages <= 0x3fffffff:
        raise ValueError(f"num_pages {num_pages}: 1 to 2^30 - 1")
    if block_table.shape[0] != seq_lens.shape[0] or block_table.shape[1] < 1 or block_table.numel() > 0x7fffffff:
        raise ValueError(f"block_table must be [{seq_lens.shape[0]}, max_pages] with a column at least and fewer than 2^31 entries, got {tuple(block_table.shape)}")


def copy_pages(pools, copies) -> None:
    """Copy, for every entry (page, new page, slots, 0) of ``copies`` int32 [n, 4], the first ``slots`` slots of a page into another, in all ``pools``: a list of
    ``PagedCache8`` (their pages' scales too) and tensors [num_pages, page_size, ...] of any type, of up to four dimensions with the last one
    contiguous, all of one pool size and page size.

    ``copies`` of ``plan_forks`` and ``plan_compaction`` fit as they are.  It ends at its first entry without slots; entries with pages outside the pools or more
    slots than a page has are passed over.  New pages are distinct, and none is another entry's source.  48 pools (24 caches) a launch, those whose slots
    do not lie behind each other apart."""
    pools = list(pools) if isinstance(pools, (list, tuple)) else [pools]
    if not rt.host().copy_pages(*_copy_kernels()[1], [p._native if isinstance(p, PagedCache8) else p for p in pools], copies):
        _refuse_copies(pools, copies)


def _refuse_copies(pools, copies):
    _ints("copies", copies, 2, copies.device)
    if copies.shape[1] != 4 or (copies.shape[0] > 1 and copies.stride(0) != 4) or copies.data_ptr() % 16:
        raise ValueError("copies must be contiguous [n, 4] at a multiple of 16 bytes")
    for p in pools:
        if not isinstance(p, (PagedCache8, torch.Tensor)):
            raise TypeError(f"a pool is a PagedCache8 or a tensor, got {type(p).__name__}")
    tensors = [t for p in pools for t in ((p.k, p.v) if isinstance(p, PagedCache8) else (p,))]
    for t in tensors:
        if not t.is_cuda:
            raise rt.AeError("a pool must be a CUDA tensor: this back end has no CPU path")
        if t.device != copies.device:
            raise ValueError(f"a pool is on {t.device}, copies on {copies.device}")
        if t.dim() < 2 or t.shape[:2] != tensors[0].shape[:2]:
            raise ValueError(f"pools must be [num_pages, page_size, ...], all alike, got {tuple(t.shape)} and {tuple(tensors[0].shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("a pool requires a gradient: copies of pages have none")
    raise ValueError("a pool has at most four dimensions, the last one contiguous, positive strides, and pages below 2 GB; copies of pages take no "
                     "forward-mode gradients and are not traced")
