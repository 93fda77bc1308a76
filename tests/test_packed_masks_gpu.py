"""Packed prompts under masks that look causal on a short sequence, against 64 bits.  Two roundings before the result: P and the stored
output, as in test_packed_gpu.py."""
import math

import pytest
import torch

import parity
from attentionengine_b200 import AttentionEngine, CustomIO, examples, meta_tensor
from test_packed_gpu import inputs, offsets, plain, softmax

pytestmark = pytest.mark.gpu

MASKS = {
    "window_1024": lambda b, h, q, kv: (q >= kv) & (q - kv < 1024),
    "window_1500": lambda b, h, q, kv: (q >= kv) & (q - kv < 1500),
    "sinks": lambda b, h, q, kv: (q >= kv) & ((q - kv < 1100) | (kv < 4)),
    "chunks": lambda b, h, q, kv: (q >= kv) & (q // 1024 == kv // 1024),
    "causal": lambda b, h, q, kv: kv <= q,
}


@pytest.mark.parametrize("infer", [True, False])
@pytest.mark.parametrize("name", list(MASKS))
def test_sequences_longer_than_the_window(name, infer):
    mask, lens = MASKS[name], [2600, 90, 1700, 1025]
    m = [meta_tensor("B", h, "S", 64, dtype=torch.float16) for h in (2, 1, 1)]
    eng = AttentionEngine(m, CustomIO({}), score_mod=lambda s, c, b, h, q, kv: s * 0.125, mask_mod=mask, online_func=examples.OnlineSoftmax(),
                          packed=True, infer_mask=infer)
    q, k, v = inputs(lens, 2, 1, 64, 64, torch.float16, seed=9)
    o = eng.prefill_packed(q, k, v, offsets(lens))
    eng.check_status()
    want = plain(q, k, v, lens, softmax(0.125), lambda b, i, j: mask(b, 0, i, j))
    at = 0
    for n in lens:  # each sequence by itself: a long one does not hide a short one's error
        parity.check("o", o[at:at + n], want[at:at + n], torch.float16, stages=2)
        at += n
