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


@pytest.mark.parametrize("name", list(MASKS))
def test_padded_batches_of_named_lengths(name):
    """The same masks in an engine of named dims, forward and gradients (stages: P, output; for the gradients P and dS beside)."""
    mask, S = MASKS[name], 1700
    m = [meta_tensor("B", "H", "S", 64, dtype=torch.float16) for _ in range(3)]
    eng = AttentionEngine(m, CustomIO({}), score_mod=lambda s, c, b, h, q, kv: s * 0.125, mask_mod=mask, online_func=examples.OnlineSoftmax())
    g = torch.Generator().manual_seed(2)
    q, k, v, d_o = (torch.randn(1, S, 2, 64, generator=g).half().cuda() for _ in range(4))
    got = [t.clone().requires_grad_() for t in (q, k, v)]
    o = eng(*got)
    grads = torch.autograd.grad(o, got, d_o)
    eng.check_status()
    i = torch.arange(S, device="cuda")
    ref = [t.double().requires_grad_() for t in (q, k, v)]
    x, y, z = (t.transpose(1, 2) for t in ref)
    s = (x @ y.transpose(2, 3) * 0.125).masked_fill(~mask(0, 0, i[:, None], i[None, :]), -math.inf)
    want = (torch.softmax(s, -1) @ z).transpose(1, 2)
    parity.check("o", o, want, torch.float16, stages=2)
    for name, a, b in zip(("dq", "dk", "dv"), grads, torch.autograd.grad(want, ref, d_o.double())):
        parity.check(name, a, b, torch.float16, stages=3)
