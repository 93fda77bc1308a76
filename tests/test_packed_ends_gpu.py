"""Packed sequences that end inside a tile of 128 keys, under scores and recurrences for which a key that is not there could count: scores that
stay finite at -inf, factors of 0, functions that are not a softmax.  Against 64 bits; two roundings before the result (P and the stored
output), as in test_packed_gpu.py."""
import math

import pytest
import torch

import parity
from attentionengine_b200 import AttentionEngine, CustomIO, OnlineFunc, SymbolScalar, Var, examples, meta_tensor
from test_packed_gpu import causal, inputs, offsets, plain

pytestmark = pytest.mark.gpu

LENS = [1, 65, 129, 128, 2, 250]


class OnlineShare(OnlineFunc):
    """P is the score over the row's sum of scores."""

    def __init__(self):
        super().__init__({"r": SymbolScalar("r", Var("0.0"))}, {"r": SymbolScalar("r", Var("0.0"))}, CustomIO())

    @staticmethod
    def online_fwd(scores, online_rowscales, b, h, q_idx):
        return scores, {"r": online_rowscales["r"] + scores.get_reduce("sum")}, SymbolScalar("o_scale", Var("1"))

    @staticmethod
    def online_fwd_epilogue(o, online_rowscales, b, h, q_idx):
        return o / online_rowscales["r"], {"r": online_rowscales["r"]}

    @staticmethod
    def forward(scores, final_rowscales, b, h, q_idx, kv_idx):
        return scores / final_rowscales["r"]

    @staticmethod
    def backward(dp, scores, final_rowscales, doosum_rowscales, b, h, q_idx, kv_idx):
        return dp


class OnlineSoftmaxOne(examples.OnlineSoftmax):
    """A softmax with one more score, 0, that has no value."""

    def __init__(self):
        OnlineFunc.__init__(self, {"m": SymbolScalar("m", Var("0.0")), "r": SymbolScalar("r", Var("1.0"))},
                            {"lse": SymbolScalar("lse", Var("0.0"))}, CustomIO())


class OnlinePeak(OnlineShare):
    """P is the score; the output is divided by the row's largest score (at least 0.001)."""

    def __init__(self):
        OnlineFunc.__init__(self, {"r": SymbolScalar("r", Var("0.001"))}, {"r": SymbolScalar("r", Var("0.0"))}, CustomIO())

    @staticmethod
    def online_fwd(scores, online_rowscales, b, h, q_idx):
        return scores, {"r": online_rowscales["r"].max(scores.get_reduce("max"))}, SymbolScalar("o_scale", Var("1"))


def engine(score, online, mask=None, customs=None, Hq=4, Hkv=2, D=64, **kw):
    m = [meta_tensor("B", h, "S", D, dtype=torch.float16) for h in (Hq, Hkv, Hkv)]
    return AttentionEngine(m, CustomIO(customs or {}), score_mod=score, mask_mod=mask, online_func=online, packed=True, **kw)


def compare(eng, p_of, keep=None, customs=(), lens=LENS, Hq=4, Hkv=2, D=64, seed=3):
    q, k, v = inputs(lens, Hq, Hkv, D, D, torch.float16, seed=seed)
    o = eng.prefill_packed(q, k, v, offsets(lens), *customs)
    eng.check_status()
    want, at = plain(q, k, v, lens, p_of, keep), 0
    for n in lens:
        parity.check(f"o[{n}]", o[at:at + n], want[at:at + n], torch.float16, stages=2)
        at += n


def softmax_of(score):
    return lambda s, kept, b: torch.softmax(score(s).masked_fill(~kept, -math.inf), -1)


MASKS = {"none": (None, None), "causal": (examples.causal_mask, causal),
         "window": (lambda b, h, q, kv: (q >= kv) & (q - kv < 40), lambda b, i, j: (i >= j) & (i - j < 40))}


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("cap,D", [(1.0, 64), (2.0, 128), (30.0, 64)])
def test_capped_scores(cap, D, mask):
    fn, keep = MASKS[mask]
    scale = 1 / (cap * math.sqrt(D))
    eng = engine(lambda s, c, b, h, q, kv: (s * scale).tanh() * cap, examples.OnlineSoftmax(), fn, D=D)
    compare(eng, softmax_of(lambda s: cap * torch.tanh(s * scale)), keep, D=D)


@pytest.mark.parametrize("mask", list(MASKS))
def test_a_factor_of_the_caller_s(mask):
    """0 and negative ones: 0 * -inf is NaN, and a negative factor would make the largest score of a key that is not there."""
    fn, keep = MASKS[mask]
    factor = torch.tensor([0.0, 0.125, -0.125, 0.3], device="cuda")
    eng = engine(lambda s, c, b, h, q, kv: s * c.input_tensors["factor"], examples.OnlineSoftmax(), fn, {"factor": ("heads",)})
    compare(eng, softmax_of(lambda s: s * factor.double()[:, None, None]), keep, (factor,))


@pytest.mark.parametrize("mask", list(MASKS))
def test_a_slope_over_positions(mask):
    fn, keep = MASKS[mask]
    eng = engine(lambda s, c, b, h, q, kv: s * 0.125 - (q - kv) * 0.02, examples.OnlineSoftmax(), fn)

    def score(s):
        i = torch.arange(s.shape[-1], device="cuda", dtype=torch.float64)
        return s * 0.125 - (i[:, None] - i[None, :]) * 0.02

    compare(eng, softmax_of(score), keep)


@pytest.mark.parametrize("mask", list(MASKS))
def test_a_softmax_with_a_term_of_its_own(mask):
    fn, keep = MASKS[mask]
    eng = engine(lambda s, c, b, h, q, kv: (s * 0.125).tanh() * 2.0, OnlineSoftmaxOne(), fn)

    def p_of(s, kept, b):
        e = torch.exp(2 * torch.tanh(s * 0.125)) * kept
        return e / (1 + e.sum(-1, keepdim=True))

    compare(eng, p_of, keep)


@pytest.mark.parametrize("shift", [0.0, 0.25])
def test_shares_of_scores(shift):
    """Not a softmax: what is not there is in no sum.  With a shift, a raw score of -inf would be worth 0.25."""
    eng = engine(lambda s, c, b, h, q, kv: ((s * 0.125).tanh() + 1.0) * 0.5 + shift, OnlineShare())
    p = lambda s, kept, b: (lambda x: x / x.sum(-1, keepdim=True))((torch.tanh(s * 0.125) + 1) * 0.5 + shift)  # noqa: E731
    compare(eng, p)


def test_largest_scores():
    """A maximum over scores that are all below what a key with a raw score of 0 would have."""
    eng = engine(lambda s, c, b, h, q, kv: 1.5 - ((s * 0.01).tanh() + 1.1) * 0.5 * (kv * 0.005 + 0.3), OnlinePeak())

    def p_of(s, kept, b):
        kv = torch.arange(s.shape[-1], device="cuda", dtype=torch.float64)
        x = 1.5 - (torch.tanh(s * 0.01) + 1.1) * 0.5 * (kv * 0.005 + 0.3)
        return x / x.amax(-1, keepdim=True)

    q, k, v = inputs(LENS, 4, 2, 64, 64, torch.float16, seed=3)
    o = eng.prefill_packed(q, k, v, offsets(LENS))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, LENS, p_of, None), torch.float16, stages=2, unnormalised=True)


@pytest.mark.parametrize("mask_value", ["-inf", "0"])
def test_retention_s_normaliser(mask_value):
    """max(sum |score|, 1) with scores that are not 0 where the raw score is."""
    eng = engine(lambda s, c, b, h, q, kv: s * 0.02 + 0.01, examples.OnlineRetention(), mask_value=mask_value)
    p = lambda s, kept, b: (lambda x: x / x.abs().sum(-1, keepdim=True).clamp(min=1))(s * 0.02 + 0.01)  # noqa: E731
    compare(eng, p)


@pytest.mark.parametrize("which", ["capped", "shares"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_sequences_do_not_meet(which, value):
    """A sequence full of infinities or NaN between two others leaves them bit for bit as they are."""
    if which == "capped":
        eng = engine(lambda s, c, b, h, q, kv: (s * 0.125).tanh(), examples.OnlineSoftmax())
    else:
        eng = engine(lambda s, c, b, h, q, kv: ((s * 0.125).tanh() + 1.0) * 0.5, OnlineShare())
    lens = [130, 60, 200]
    q, k, v = inputs(lens, 4, 2, 64, 64, torch.float16)
    a = eng.prefill_packed(q, k, v, offsets(lens))
    for t in (q, k, v):
        t[130:190] = value
    b = eng.prefill_packed(q, k, v, offsets(lens))
    assert torch.equal(a[:130], b[:130]) and torch.equal(a[190:], b[190:]) and a.isfinite().all()


def test_a_call_allocates_its_output_alone():
    eng = engine(lambda s, c, b, h, q, kv: s * 0.125, examples.OnlineSoftmax(), examples.causal_mask)
    q, k, v = inputs(LENS, 4, 2, 64, 64, torch.float16)
    cu = offsets(LENS)
    eng.prefill_packed(q, k, v, cu)  # the status word and the counters are the engine's
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    o = eng.prefill_packed(q, k, v, cu)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == 1 and o.shape == q.shape
