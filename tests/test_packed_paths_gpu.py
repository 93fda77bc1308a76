"""Packed prompts with more items than SMs: a CTA takes several, of many steps each, from the counter.  Each way of pairing the q tiles, against 64 bits;
two roundings before the result (P and the stored output), as in test_packed_gpu.py."""
import math

import pytest
import torch

import parity
from attentionengine_b200 import AttentionEngine, CustomIO, examples, meta_tensor
from test_packed_ends_gpu import OnlineShare, softmax_of
from test_packed_gpu import DT, causal, inputs, offsets, plain, softmax

pytestmark = pytest.mark.gpu

LENS = [1500, 100, 1024, 777, 1, 640, 1409, 333, 129, 900, 1280, 0, 511, 128]  # 9732


def items(lens, Hq, Hkv):
    """(items, how the two q tiles of a CTA are chosen), by the rule of the launch."""
    T, n = sum(lens), min(len(lens), sum(lens))
    blocks = lambda rows: T // rows + n  # noqa: E731
    mode = 2 if blocks(128) * Hq <= 148 else 1 if Hq // Hkv % 2 == 0 else 0
    return blocks(256 if mode == 0 else 128) * (Hq // 2 if mode == 1 else Hq), mode


@pytest.mark.parametrize("Hq,Hkv,D,DV,dtype,mode", [
    (6, 2, 64, 64, "fp16", 0), (4, 4, 128, 128, "bf16", 0), (5, 1, 64, 128, "bf16", 0), (9, 3, 128, 64, "fp16", 0),
    (32, 8, 128, 128, "bf16", 1), (16, 4, 64, 64, "fp16", 1), (8, 1, 128, 64, "fp16", 1), (12, 6, 64, 128, "bf16", 1)])
@pytest.mark.parametrize("mask", [True, False])
def test_many_items(Hq, Hkv, D, DV, dtype, mode, mask):
    n, m = items(LENS, Hq, Hkv)
    assert m == mode and n > 148
    eng = examples.softmax_engine("B", Hq, Hkv, "S", D, DV, DT[dtype], mask, packed=True)
    q, k, v = inputs(LENS, Hq, Hkv, D, DV, DT[dtype], seed=Hq)
    cu = offsets(LENS)
    first = eng.prefill_packed(q, k, v, cu)
    again = [eng.prefill_packed(q, k, v, cu) for _ in range(8)]
    torch.cuda.synchronize()
    eng.check_status()
    parity.check("o", first, plain(q, k, v, LENS, softmax(1 / math.sqrt(D)), causal if mask else None), DT[dtype], stages=2)
    assert all(torch.equal(first, x) for x in again)


@pytest.mark.parametrize("Hq,Hkv,mode", [(3, 3, 2), (4, 2, 2)])
def test_one_tile_a_cta(Hq, Hkv, mode):
    """As many items as SMs at most, of many steps."""
    lens = [2500, 300, 1100]
    n, m = items(lens, Hq, Hkv)
    assert m == mode and n <= 148
    eng = examples.softmax_engine("B", Hq, Hkv, "S", 128, 128, torch.float16, True, packed=True)
    q, k, v = inputs(lens, Hq, Hkv, 128, 128, torch.float16, seed=Hq)
    o = eng.prefill_packed(q, k, v, offsets(lens))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, lens, softmax(1 / math.sqrt(128)), causal), torch.float16, stages=2)


@pytest.mark.parametrize("Hq,Hkv", [(6, 2), (8, 2)])
@pytest.mark.parametrize("kind", ["window", "capped", "shares"])
def test_other_masks_and_scores(kind, Hq, Hkv):
    assert items(LENS, Hq, Hkv)[0] > 148
    m = [meta_tensor("B", h, "S", 64, dtype=torch.float16) for h in (Hq, Hkv, Hkv)]
    make = lambda score, mask, online: AttentionEngine(m, CustomIO({}), score_mod=score, mask_mod=mask, online_func=online, packed=True)  # noqa: E731
    if kind == "window":
        eng = make(lambda s, c, b, h, q, kv: s * 0.125, lambda b, h, q, kv: (q >= kv) & (q - kv < 1100), examples.OnlineSoftmax())
        p_of, keep = softmax(0.125), lambda b, i, j: (i >= j) & (i - j < 1100)
    elif kind == "capped":
        eng = make(lambda s, c, b, h, q, kv: (s * 0.125).tanh() * 2.0, examples.causal_mask, examples.OnlineSoftmax())
        p_of, keep = softmax_of(lambda s: 2 * torch.tanh(s * 0.125)), causal
    else:
        eng = make(lambda s, c, b, h, q, kv: ((s * 0.125).tanh() + 1.0) * 0.5 + 0.25, None, OnlineShare())
        p_of, keep = lambda s, kept, b: (lambda x: x / x.sum(-1, keepdim=True))((torch.tanh(s * 0.125) + 1) * 0.5 + 0.25), None
    q, k, v = inputs(LENS, Hq, Hkv, 64, 64, torch.float16, seed=2)
    o = eng.prefill_packed(q, k, v, offsets(LENS))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, LENS, p_of, keep), torch.float16, stages=2)


@pytest.mark.parametrize("Hq,Hkv", [(6, 2), (8, 2)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_sequences_do_not_meet(Hq, Hkv, value):
    eng = examples.softmax_engine("B", Hq, Hkv, "S", 128, 128, torch.bfloat16, True, packed=True)
    q, k, v = inputs(LENS, Hq, Hkv, 128, 128, torch.bfloat16)
    cu, at = offsets(LENS), offsets(LENS).tolist()
    a = eng.prefill_packed(q, k, v, cu)
    bad = torch.zeros(sum(LENS), dtype=torch.bool, device="cuda")
    for i in (1, 3, 8):
        bad[at[i]:at[i + 1]] = True
    for t in (q, k, v):
        t[bad] = value
    b = eng.prefill_packed(q, k, v, cu)
    assert torch.equal(a[~bad], b[~bad]) and a.isfinite().all()


def test_streams_and_graphs():
    Hq, Hkv, D = 6, 2, 64
    eng = examples.softmax_engine("B", Hq, Hkv, "S", D, D, torch.float16, True, packed=True)
    q, k, v = inputs(LENS, Hq, Hkv, D, D, torch.float16)
    cu = offsets(LENS)
    first = eng.prefill_packed(q, k, v, cu)
    sides = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):  # calls on several streams, each with its own counter
        for s in sides:
            with torch.cuda.stream(s):
                out.append(eng.prefill_packed(q, k, v, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [eng.prefill_packed(q, k, v, cu) for _ in range(2)]
    cu.copy_(offsets(LENS[::-1]))  # the lengths of the replay
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want = eng.prefill_packed(q, k, v, cu)
    assert all(torch.equal(want, x) for x in held)
    eng.check_status()
