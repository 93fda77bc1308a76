"""The reference's example programs written against this package: the OnlineFunc definitions and engine
factories of attn_script/mha.py, gqa.py, sigmoidattn.py, reluattn.py, retention.py, mla_decode.py,
gqa_inference.py and mamba2_ngroup1.py, plus seeded input generators with the benchmark's distributions.
The benchmark, the build step and the tests all take their engines from here."""
import math

import torch

from .attn_engine import (AttentionEngine, LinearAttentionEngine, OnlineFunc, PagedCache8, copy_pages, plan_compaction, plan_forks,
                          plan_pages)
from .core import CustomIO, SymbolScalar, Var, meta_tensor


class OnlineSoftmax(OnlineFunc):
    """attn_script/mha.py:27-84."""

    def __init__(self):
        super().__init__({"m": SymbolScalar("m", Var("-inf")), "r": SymbolScalar("r", Var("0.0"))},
                         {"lse": SymbolScalar("lse", Var("0.0"))}, CustomIO())

    @staticmethod
    def online_fwd(scores, online_rowscales, b, h, q_idx):
        m, r = online_rowscales["m"], online_rowscales["r"]
        m_new = m.max(scores.get_reduce("max"))
        scale_tmp = (m - m_new).exp()
        r = r * scale_tmp
        scores = (scores - m_new).exp()
        r = r + scores.get_reduce("sum")
        return scores, {"m": m_new, "r": r}, scale_tmp

    @staticmethod
    def online_fwd_epilogue(o, online_rowscales, b, h, q_idx):
        o_new = o / online_rowscales["r"]
        lse = (online_rowscales["r"]).log() + online_rowscales["m"]
        return o_new, {"lse": lse}

    @staticmethod
    def forward(scores, final_rowscales, b, h, q_idx, kv_idx):
        return (scores - final_rowscales["lse"]).exp()

    @staticmethod
    def backward(dp, scores, final_rowscales, doosum_rowscales, b, h, q_idx, kv_idx):
        return (dp - doosum_rowscales) * scores


class OnlineIdentity(OnlineFunc):
    """attn_script/sigmoidattn.py:24-49, reluattn.py:21-46."""

    def __init__(self):
        super().__init__({}, {}, CustomIO())

    @staticmethod
    def online_fwd(scores, online_rowscales, b, h, q_idx):
        return scores, online_rowscales, SymbolScalar("o_scale", Var("1"))

    @staticmethod
    def online_fwd_epilogue(o, online_rowscales, b, h, q_idx):
        return o, {}

    @staticmethod
    def forward(scores, final_rowscales, b, h, q_idx, kv_idx):
        return scores

    @staticmethod
    def backward(dp, scores, final_rowscales, doosum_rowscales, b, h, q_idx, kv_idx):
        return dp


def causal_mask(b, h, q_idx, kv_idx):
    return q_idx >= kv_idx


def metas(B, Hq, Hkv, S, D, DV, dtype):
    return (meta_tensor(B, Hq, S, D, dtype=dtype), meta_tensor(B, Hkv, S, D, dtype=dtype),
            meta_tensor(B, Hkv, S, DV, dtype=dtype))


class OnlineSoftmaxSplit(OnlineSoftmax):
    """Online softmax with the split-KV merge of attn_script/gqa_inference.py:72-80 / mla_decode.py."""

    @staticmethod
    def combine(final_rowscales):
        lse = final_rowscales["lse"]
        lse_max = lse.get_reduce("max")
        row_sum = (lse - lse_max).exp()
        row_sum_sum = row_sum.get_reduce("sum")
        lse_sum = row_sum_sum.log() + lse_max
        return (lse - lse_sum).exp()


def decode_engine(B, Hq, Hkv, Sq, Skv, D, dtype, scale=None, online=None, **kw):
    """q_len != kv_len: the split-KV decode path (reference scripts gqa_inference.py / mha_inference.py)."""
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    metas_ = (meta_tensor(B, Hq, Sq, D, dtype=dtype), meta_tensor(B, Hkv, Skv, D, dtype=dtype),
              meta_tensor(B, Hkv, Skv, D, dtype=dtype))
    return AttentionEngine(metas_, CustomIO({}), score_mod=lambda s, c, b, h, q, kv: s * scale, mask_mod=None,
                           online_func=online if online is not None else OnlineSoftmaxSplit(), **kw)


def softmax_engine(B, Hq, Hkv, S, D, DV, dtype, causal, scale=None, **kw):
    scale = 1.0 / math.sqrt(D) if scale is None else scale

    def score_mod(score, custom_fwd_inputs, b, h, q_idx, kv_idx):
        return score * scale

    return AttentionEngine(metas(B, Hq, Hkv, S, D, DV, dtype), CustomIO({}), score_mod=score_mod,
                           mask_mod=causal_mask if causal else None, online_func=OnlineSoftmax(), **kw)


def sigmoid_engine(B, H, S, D, dtype, causal, scale=None):
    """P = sigmoid(score * scale + bias) in the reference's tanh form (attn_script/sigmoidattn.py:14-18);
    bias arrives as the custom input ``softmax_bias`` of shape (1,)."""
    scale = 1.0 / math.sqrt(D) if scale is None else scale

    def score_mod(score, custom_fwd_inputs, b, h, q_idx, kv_idx):
        softmax_bias = custom_fwd_inputs.input_tensors["softmax_bias"]
        score = score * scale + softmax_bias
        return ((score * 0.5).tanh() + 1) * 0.5

    return AttentionEngine(metas(B, H, H, S, D, D, dtype), CustomIO({"softmax_bias": (1,)}), score_mod=score_mod,
                           mask_mod=causal_mask if causal else None, online_func=OnlineIdentity())


def relu_engine(B, H, S, D, dtype, causal=False, scale=None, post_scale=1.0):
    """P = relu(score * scale) * post_scale (attn_script/reluattn.py:14-17)."""
    scale = 1.0 / math.sqrt(D) if scale is None else scale

    def score_mod(score, custom_fwd_inputs, b, h, q_idx, kv_idx):
        score = (score * scale).max(0)
        return score * post_scale if post_scale != 1.0 else score

    return AttentionEngine(metas(B, H, H, S, D, D, dtype), CustomIO({}), score_mod=score_mod,
                           mask_mod=causal_mask if causal else None, online_func=OnlineIdentity())


def seeded_qkv(B, Hq, Hkv, S, D, DV, dtype, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, S, Hq, D, generator=g).to(dtype)
    k = torch.randn(B, S, Hkv, D, generator=g).to(dtype)
    v = torch.randn(B, S, Hkv, DV, generator=g).to(dtype)
    d_o = torch.randn(B, S, Hq, DV, generator=g).to(dtype)
    return [t.to(device) for t in (q, k, v, d_o)]


def mla_engine(B, H, S, dtype, scale):
    """attn_script/mla_decode.py:88-118 with the scale chosen by the caller's score_mod."""
    def score_mod(score, custom_fwd_inputs, b, h, q_idx, kv_idx):
        return score * scale

    qkv = (meta_tensor(B, H, 1, 576, dtype=dtype), meta_tensor(B, 1, S, 576, dtype=dtype),
           meta_tensor(B, 1, S, 512, dtype=dtype))
    return AttentionEngine(qkv, CustomIO({}), score_mod=score_mod, mask_mod=None, online_func=OnlineSoftmaxSplit(),
                           kv_shared=True)


def mamba2_engine(B, H, T, DK, DV, dtype, d_skip=False):
    """attn_script/mamba2_ngroup1.py:26-63: decay_mod = decay * A, v_mod = v * dt, one q / k head (ngroups = 1).
    ``d_skip``: add the benchmark configuration's skip connection o += D[h] * x as an ``o_mod`` over a fourth custom
    input D [1, heads] (the reference's harness runs without it, benchmark/bench_utils.py:304-308)."""
    def decay_mod(decay, custom_io):
        return decay * custom_io.input_tensors["A"]

    def v_mod(v, custom_io):
        return v * custom_io.input_tensors["dt"]

    def o_mod(o, v, custom_io):
        return o + v * custom_io.input_tensors["D"]

    metas_ = (meta_tensor(B, 1, T, DK, dtype=dtype), meta_tensor(B, 1, T, DK, dtype=dtype), meta_tensor(B, H, T, DV, dtype=dtype))
    customs = {"A": (1, "heads"), "dt": ("batch", "heads", "seq_len")}
    if d_skip:
        customs["D"] = (1, "heads")
    return LinearAttentionEngine(metas_, decay_mod=decay_mod, v_mod=v_mod, custom_io=CustomIO(customs),
                                 o_mod=o_mod if d_skip else None)


def mamba2_inputs(B, H, T, DK, DV, dtype, seed=0):
    """The benchmark's distributions: x, B, C ~ N(0,1); dt = softplus(N(0,1) - 4); A = -exp(U(ln 1, ln 16))."""
    import math
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, DV, generator=g).to(dtype)
    Bm = torch.randn(B, 1, T, DK, generator=g).to(dtype)
    Cm = torch.randn(B, 1, T, DK, generator=g).to(dtype)
    dt = torch.nn.functional.softplus(torch.randn(B, H, T, generator=g) - 4.0)
    A = -torch.exp(torch.rand(H, generator=g) * math.log(16.0))
    return x, dt, A, Bm, Cm


class OnlineRetention(OnlineFunc):
    """Row normaliser max(sum |score|, 1), the recurrence of attn_script/retention.py:19-71."""

    def __init__(self):
        super().__init__({"r_wo_clamp": SymbolScalar("r_wo_clamp", Var("0.0")), "r": SymbolScalar("r", Var("0.0"))},
                         {"r": SymbolScalar("r", Var("0.0"))}, CustomIO())

    @staticmethod
    def online_fwd(scores, online_rowscales, b, h, q_idx):
        r_wo_clamp = online_rowscales["r_wo_clamp"] + scores.get_reduce("abssum")
        r_new = r_wo_clamp.max(1.0)
        o_scale = online_rowscales["r"] / r_new
        return scores / r_new, {"r_wo_clamp": r_wo_clamp, "r": r_new}, o_scale

    @staticmethod
    def online_fwd_epilogue(o, online_rowscales, b, h, q_idx):
        return o, {"r": online_rowscales["r"]}

    @staticmethod
    def forward(scores, final_rowscales, b, h, q_idx, kv_idx):
        return scores / final_rowscales["r"]

    @staticmethod
    def backward(dp, scores, final_rowscales, doosum_rowscales, b, h, q_idx, kv_idx):
        return dp / final_rowscales["r"]


def retention_engine(B, H, S, D, DV, dtype):
    """Parallel retention (attn_script/retention.py:14-17, 93-104): the decay mask is a tile-shaped custom input
    [1, heads, seq_len, seq_len_kv] multiplied into the scores; causal mask with additive mask value 0."""

    def score_mod(score, custom_fwd_inputs, b, h, q_idx, kv_idx):
        return score * custom_fwd_inputs.input_tensors["mask"]

    return AttentionEngine(metas(B, H, H, S, D, DV, dtype), CustomIO({"mask": (1, "heads", "seq_len", "seq_len_kv")}),
                           score_mod=score_mod, mask_mod=causal_mask, online_func=OnlineRetention(), mask_value="0")


class PagedLayers:
    """The attention of a server's layers over paged 8-bit caches: ``prompts`` admits a batch of requests of different lengths, ``tokens``
    takes one more token for each.  The layers share the pages' numbers, so one plan serves a step; nothing is read back.  A prompt attends to itself
    alone, so ``prompts`` is the first step: rows that hold tokens cannot get another one (a later turn, a part of a long prompt).

    ``rope``: a ``QKNormRope`` that norms and rotates the queries and keys of every step by the plan's positions, with ``weights`` (q_weight, k_weight) of
    every layer.  ``fork`` lets rows go on from others (samples of one prompt, beams), cuts and ends them; ``compact`` brings the pages in use to the
    front of the pools."""

    def __init__(self, n_layers, Hq, Hkv, D, dtype, rows, num_pages, page_size, max_len, device="cuda", rope=None, weights=None):
        self.page_size, self.rows, self.num_pages = page_size, rows, num_pages
        if weights is not None and (rope is None or len(weights) != n_layers):
            raise ValueError(f"weights are (q_weight, k_weight) of each of the {n_layers} layers, for a rope")
        self.rope, self.weights = rope, weights if weights is not None else [(None, None)] * n_layers
        self.caches = [PagedCache8(num_pages, page_size, Hkv, D, device=device) for _ in range(n_layers)]
        self.prompt = softmax_engine("B", Hq, Hkv, "S", D, D, dtype, True, packed=True)
        self.token = decode_engine("B", Hq, Hkv, 1, "S", D, dtype, cache_dtype=torch.float8_e4m3fn)
        ints = dict(dtype=torch.int32, device=device)
        self.free, self.head = torch.arange(num_pages, **ints), torch.zeros(1, **ints)
        self.table, self.lens = torch.zeros(rows, -(-max_len // page_size), **ints), torch.zeros(rows, **ints)
        self.one = torch.ones(rows, **ints)
        self.status, self.moved = torch.zeros(1, **ints), torch.zeros(1, **ints)
        self.begun = False

    def _plan(self, new_lens, n_tokens):
        self.begun = True
        plan = plan_pages(self.lens, new_lens, self.table, self.free, self.head, self.page_size, n_tokens)
        self.lens, self.head = plan.seq_lens, plan.free_head
        self.status |= plan.status
        return plan

    def _rotated(self, layers, plan):
        for (q, k, v), w in zip(layers, self.weights):
            yield (q, k, v) if self.rope is None else (*self.rope(q, k, plan.positions, *w), v)

    def prompts(self, layers, new_lens):
        """``layers``: (q, k, v) of every layer, [T, heads, D] with the requests' tokens behind each other; returns the layers' outputs."""
        if self.begun:
            raise NotImplementedError("rows hold tokens already: new prompts would attend to themselves alone, without what is cached")
        plan = self._plan(new_lens, layers[0][0].shape[0])
        out = []
        for cache, (q, k, v) in zip(self.caches, self._rotated(layers, plan)):
            cache.write(k, v, plan.segments)
            out.append(self.prompt.prefill_packed(q, k, v, plan.cu_seqlens))
        return out

    def tokens(self, layers):
        """``layers``: (q, k, v) of every layer, [rows, heads, D]."""
        plan = self._plan(self.one, self.rows)
        out = []
        for cache, (q, k, v) in zip(self.caches, self._rotated(layers, plan)):
            cache.write(k, v, plan.segments)
            out.append(self.token.decode_cache8(q.unsqueeze(1), cache, plan.block_table, plan.seq_lens).squeeze(1))
        return out

    def fork(self, parents, keep_lens=None):
        """Row b goes on from the first ``keep_lens[b]`` tokens (None: all) of row ``parents[b]``; -1: it ends, and its pages are free again.  A row that has
        ended takes part in ``tokens`` from position 0."""
        plan = plan_forks(parents, self.lens, self.table, self.free, self.head, self.page_size, self.num_pages, keep_lens)
        self._moved(plan)
        self.lens = plan.seq_lens

    def compact(self):
        """The pages in use to the front of every layer's pool; the number of them stays on the GPU, in ``head``."""
        self._moved(plan_compaction(self.lens, self.table, self.page_size, self.num_pages))

    def _moved(self, plan):
        copy_pages(self.caches, plan.copies)
        self.table, self.free, self.head = plan.block_table, plan.free_pages, plan.free_head
        self.moved |= plan.status

    def check(self):
        """Raise if a step did not fit the pages or a kernel reported something (waits for the GPU)."""
        if int(self.status.item()):
            raise ValueError(f"plan_pages reported 0x{int(self.status.item()):x}")
        if int(self.moved.item()):
            raise ValueError(f"plan_forks or plan_compaction reported 0x{int(self.moved.item()):x}")
        self.prompt.check_status()
        self.token.check_status()
