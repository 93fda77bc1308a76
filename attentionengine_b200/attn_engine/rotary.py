"""Norm of each query and key head and its rotation by the token's position, in one pass, in front of any attention call:

    rope = QKNormRope(head_dim, base=1e6)                        # held by a model; its weights are the caller's
    q, k = rope(q, k, positions, q_weight, k_weight)             # [B, S, H, D] or [T, H, D], with gradients
    o = engine(q, k, v)

In a serving step ``positions`` is ``plan_pages(...).positions``.  The reference's scripts take queries and keys as they come (attn_script/mha.py); models
norm and rotate them first.
"""
from __future__ import annotations

import functools
import math
from fractions import Fraction

import torch

from .. import runtime as rt

HEAD_DIMS = (32, 64, 128, 256)
_PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def turns_of(frequency: float) -> int:
    """The fraction of a turn that one position makes at ``frequency`` radians, in units of 2^-64."""
    t = Fraction(frequency) / (2 * _PI)
    return round((t - math.floor(t)) * 2 ** 64) % 2 ** 64


SHAPES = ((4, 4), (8, 3), (32, 1))  # of each kernel: warps of a CTA, CTAs of an SM
BWD_HEADS = 1  # of a team on their way together in the backward (the forward takes four, two or one)


def _defines(D: int, R: int, norm: bool, interleaved: bool, which: int) -> dict:
    warps, ctas = SHAPES[which]
    return {"AE_D": D, "AE_R": R, "AE_NORM": int(norm), "AE_NEXT": int(interleaved), "AE_ROPE_KERNEL": which, "AE_ROPE_WARPS": warps,
            "AE_ROPE_CTAS": ctas, **({"AE_ROPE_U": BWD_HEADS} if which == 1 else {})}


@functools.lru_cache(maxsize=None)
def _kernels(D: int, R: int, norm: bool, interleaved: bool):
    out = []
    for i, name in enumerate(("ae_qk_rope_fwd", "ae_qk_rope_bwd", "ae_qk_rope_dw")):
        cfg = rt.KernelConfig(kind=rt.KIND_QK_ROPE, head_dim=D, threads=32 * SHAPES[i][0])
        cfg.reserved[1], cfg.reserved[3] = SHAPES[min(i, 1)]  # the sums: the backward's
        out.append(rt.compile_module(rt.kernel_source("qk_norm_rope.cuh", defines=_defines(D, R, norm, interleaved, i)), name, cfg))
    return tuple(out)


class QKNormRope:
    """Root-mean-square norm over the dims of each head, times a weight of ``head_dim`` values, then the rotation of ``rotary_dim`` dims.

    ``head_dim`` 32, 64, 128 or 256; ``rotary_dim`` a multiple of 16 up to it (default: all), the dims behind it are normed alone.  Pair i is (i, i +
    rotary_dim / 2), with ``interleaved`` (2i, 2i + 1).  Its frequency is ``base ** (-2 i / rotary_dim)`` radians a position, or ``inv_freq[i]``
    (rotary_dim / 2 values: scaled contexts).  ``rotary_scale`` multiplies the rotated dims.  ``norm=False``: the rotation alone.

    Everything is computed in fp32 and rounded once, angles in 64-bit fixed point.  With the frequencies as 64-bit floats, an angle is off by 2^-26 of a turn, as any in fp32, and
    by 2^-65 of one for each position: nothing beside the former up to position 2^39 (so for every int32), an eighth of a turn at 2^62.  A row's squares are summed
    in fp32, so values beyond 1e18 make it overflow as they do in any fp32 norm: finite ones become 0."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0, inv_freq=None, interleaved: bool = False, norm: bool = True,
                 eps: float = 1e-6, rotary_scale: float = 1.0):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if type(head_dim) is not int or head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"head dim {head_dim}: one of {HEAD_DIMS}")
        if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int) or rotary_dim % 16 or not 16 <= rotary_dim <= head_dim:
            raise ValueError(f"rotary_dim {rotary_dim}: a multiple of 16 up to head_dim = {head_dim}")
        if inv_freq is None:
            if not (math.isfinite(base) and base > 0):
                raise ValueError(f"base {base}: a positive number")
            freq = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
        else:
            freq = [float(f) for f in (inv_freq.tolist() if isinstance(inv_freq, torch.Tensor) else inv_freq)]
        if len(freq) != rotary_dim // 2 or not all(math.isfinite(f) for f in freq):
            raise ValueError(f"inv_freq: {rotary_dim // 2} finite frequencies, one for each pair")
        if not (math.isfinite(eps) and eps >= 0) or not math.isfinite(rotary_scale):
            raise ValueError("eps is a finite number, 0 at least; rotary_scale a finite one")
        self.head_dim, self.rotary_dim, self.interleaved, self.norm = head_dim, rotary_dim, bool(interleaved), bool(norm)
        self.eps, self.rotary_scale, self.inv_freq = float(eps), float(rotary_scale), freq
        self._modules = _kernels(head_dim, rotary_dim, self.norm, self.interleaved)
        self._plan = rt.host().RopePlan(*(m.handle.value for m in self._modules), head_dim, self.norm, self.eps, self.rotary_scale,
                                        [turns_of(f) for f in freq])

    def __call__(self, q, k, positions, q_weight=None, k_weight=None):
        """``q`` [B, S, Hq, D] and ``k`` [B, S, Hkv, D], or [T, H, D] of packed tokens, fp16 or bf16 with contiguous heads (views of a joint
        projection are fine); ``k`` may be None.  ``positions`` int32 or int64, [B, S] or [S] ([T]).  ``q_weight`` and ``k_weight`` [D], fp32 or
        the type of q; without one, 1.  Returns new contiguous tensors (q, k).

        A token with a negative position is none (``plan_pages`` marks those behind the last one so): zeros, and no gradient.  Gradients: q, k and
        the weights, the same bits every time; no second derivatives."""
        r = rt.host().qk_rope(self._plan, q, k, positions, q_weight, k_weight)
        if r is None:
            self._refuse(q, k, positions, q_weight, k_weight)
        return r

    def _refuse(self, q, k, positions, q_weight, k_weight):
        heads = [("q", q)] + ([("k", k)] if k is not None else [])
        weights = [(n, w) for n, w in (("q_weight", q_weight), ("k_weight", k_weight)) if w is not None]
        for name, t in heads + weights + [("positions", positions)]:
            if not t.is_cuda:
                raise rt.AeError(f"{name} must be a CUDA tensor: this back end has no CPU path")
            if t.device != q.device:
                raise ValueError(f"{name} is on {t.device}, q on {q.device}")
        for name, t in heads:
            if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != q.dtype:
                raise TypeError(f"{name} has dtype {t.dtype}: fp16 or bf16, q and k alike")
            if t.dim() not in (3, 4) or t.dim() != q.dim() or t.shape[-1] != self.head_dim or t.stride(-1) != 1 or t.shape[:-2] != q.shape[:-2]:
                raise ValueError(f"{name} must be [B, S, H, {self.head_dim}] or [T, H, {self.head_dim}] with a contiguous last dimension, q and k of the same "
                                 f"tokens, got {tuple(t.shape)}")
            if not 1 <= t.shape[-2] <= 65535:
                raise ValueError(f"{name} has {t.shape[-2]} heads")
            if t.numel() and (t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:-1], t.shape) if n > 1)):
                raise ValueError(f"{name} and its strides must be multiples of 16 bytes")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions have dtype {positions.dtype}: int32 or int64")
        if tuple(positions.shape) not in ((q.shape[0],),) if q.dim() == 3 else tuple(positions.shape) not in ((q.shape[1],), tuple(q.shape[:2]), (1, q.shape[1])):
            raise ValueError(f"positions must be [T], or [S] or [B, S], of q's tokens, got {tuple(positions.shape)}")
        if weights and not self.norm:
            raise ValueError("weights belong to the norm: this object was built with norm=False")
        if k is None and k_weight is not None:
            raise ValueError("k_weight without k")
        for name, w in weights:
            if w.dtype not in (torch.float32, q.dtype) or w.dtype != weights[0][1].dtype:
                raise TypeError(f"{name} has dtype {w.dtype}: fp32 or the type of q, both alike")
            if tuple(w.shape) != (self.head_dim,) or w.stride(0) != 1 or w.data_ptr() % 16:
                raise ValueError(f"{name} must be [{self.head_dim}], contiguous, at a multiple of 16 bytes")
        raise NotImplementedError("norm and rotation take no forward-mode gradients and are not traced")
