"""Which masks an engine of unknown lengths takes for plain causal attention: those whose expression is that comparison, and no other,
however it looks on a short sequence."""
import pytest
import torch

from attentionengine_b200 import AttentionEngine, CustomIO, examples, meta_tensor


def make(mask, packed=True, **kw):
    m = [meta_tensor("B", 2, "S", 64, dtype=torch.float16) for _ in range(3)]
    return AttentionEngine(m, CustomIO({}), score_mod=lambda s, c, b, h, q, kv: s, mask_mod=mask, online_func=examples.OnlineSoftmax(),
                           packed=packed, **kw)


LIKE_CAUSAL = {  # equal to causal attention on 1024 positions, not beyond
    "window_1024": lambda b, h, q, kv: (q >= kv) & (q - kv < 1024),
    "window_4096": lambda b, h, q, kv: (q >= kv) & (q - kv < 4096),
    "sinks": lambda b, h, q, kv: (q >= kv) & ((q - kv < 1500) | (kv < 4)),
    "chunks": lambda b, h, q, kv: (q >= kv) & (q // 8192 == kv // 8192),
    "late_rows": lambda b, h, q, kv: (q >= kv) | (q > 5000),
}


@pytest.mark.parametrize("name", list(LIKE_CAUSAL))
def test_a_mask_that_looks_causal_is_applied_everywhere(name):
    assert make(LIKE_CAUSAL[name]).mask_mode == 3


@pytest.mark.parametrize("mask", [
    lambda b, h, q, kv: q >= kv, lambda b, h, q, kv: kv <= q, lambda b, h, q, kv: ~(q < kv), lambda b, h, q, kv: q - kv >= 0,
    lambda b, h, q, kv: kv - q <= 0, lambda b, h, q, kv: q + 1 > kv, lambda b, h, q, kv: kv - 1 < q, lambda b, h, q, kv: 0 <= q - kv,
    lambda b, h, q, kv: torch.logical_not(kv > q)])
def test_the_causal_comparison_in_its_spellings(mask):
    assert make(mask).mask_mode == 1


@pytest.mark.parametrize("mask", [
    lambda b, h, q, kv: q > kv, lambda b, h, q, kv: q >= kv + 1, lambda b, h, q, kv: kv >= q, lambda b, h, q, kv: q + 3 >= kv,
    lambda b, h, q, kv: q >= 2 * kv, lambda b, h, q, kv: q + b >= kv, lambda b, h, q, kv: kv >= 0, lambda b, h, q, kv: q + q >= kv])
def test_other_comparisons(mask):
    assert make(mask).mask_mode == 3


def test_no_inference_when_the_caller_asks_for_none():
    assert make(examples.causal_mask, infer_mask=False).mask_mode == 3


@pytest.mark.parametrize("name", list(LIKE_CAUSAL))
def test_padded_batches_of_named_lengths(name):
    """Engines of named dims: tile lists for the length of the call, which see what a mask does there."""
    eng = make(LIKE_CAUSAL[name], packed=False)
    assert eng.mask_mode == 2 and make(examples.causal_mask, packed=False).mask_mode == 1
    if name == "window_1024":
        count, index = (x.tolist() for x in eng._ensure_lists("cpu", None, 1, 2, 1536, 1536)[:2])
        assert count[0][0] == [min(i + 1, 9) for i in range(12)] and [x & 0xffff for x in index[0][0][11][:9]] == list(range(3, 12))


def test_a_mask_that_would_not_be_applied_is_refused():
    with pytest.raises(NotImplementedError, match="-inf"):
        make(examples.causal_mask, mask_value="0")
    make(None, mask_value="0")
