"""How a packed engine leaves out what stands behind a sequence's end: by its score_mod and its recurrence."""
import pytest
import torch

from attentionengine_b200 import AttentionEngine, CustomIO, examples, meta_tensor
from attentionengine_b200.lower.cuda_lower import drops_neg_inf
from test_cache8_cpu import Plain


def way(score, online=None, customs=None, packed=True):
    m = [meta_tensor("B", 2, "S", 64, dtype=torch.float16) for _ in range(3)]
    src = AttentionEngine(m, CustomIO(customs or {}), score_mod=score, mask_mod=examples.causal_mask,
                          online_func=online or examples.OnlineSoftmax(), packed=packed).tl_code
    at = src.find("#define AE_PACK_SCORES ")
    return int(src[at + 23]) if at >= 0 else None


def test_scores_that_keep_minus_infinity():
    assert way(lambda s, c, b, h, q, kv: s) == 0 and way(lambda s, c, b, h, q, kv: s * 0.125) == 0
    assert way(lambda s, c, b, h, q, kv: s * 0.5 / 4.0 + 3.0) == 0
    assert way(lambda s, c, b, h, q, kv: s * 0.125 + c.input_tensors["x"], customs={"x": ("batch", "heads")}) == 0


def test_scores_that_may_not():
    assert way(lambda s, c, b, h, q, kv: s.tanh()) == 1 and way(lambda s, c, b, h, q, kv: s.max(0)) == 1
    assert way(lambda s, c, b, h, q, kv: s * -1.0) == 1 and way(lambda s, c, b, h, q, kv: s * 0.0) == 1
    assert way(lambda s, c, b, h, q, kv: s * c.input_tensors["x"], customs={"x": ("heads",)}) == 1
    assert way(lambda s, c, b, h, q, kv: s + kv * 0.1) == 1  # not taken for one: a sum of two tiles


def test_recurrences():
    assert drops_neg_inf(examples.OnlineSoftmax()) and drops_neg_inf(examples.OnlineSoftmaxSplit()) and drops_neg_inf(Plain())
    assert not drops_neg_inf(examples.OnlineIdentity()) and not drops_neg_inf(examples.OnlineRetention())
    assert way(lambda s, c, b, h, q, kv: s.tanh(), examples.OnlineIdentity()) == 2


def test_padded_batches_are_as_they_were():
    assert way(lambda s, c, b, h, q, kv: s.tanh(), packed=False) is None
