"""Packed prompts against 64 bits, sequence by sequence.  Two roundings before the result: P and the stored output (stages = 2 of
tests/parity.py for bf16; 2 x 2^-11 inside its 1e-3 for fp16)."""
import math

import pytest
import torch

import parity
from attentionengine_b200 import AttentionEngine, CustomIO, examples, meta_tensor
from attentionengine_b200.runtime import AeError

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def inputs(lens, Hq, Hkv, D, DV, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    return [torch.randn(T, h, d, generator=g).to(dtype).cuda() for h, d in ((Hq, D), (Hkv, D), (Hkv, DV))]


def plain(q, k, v, lens, p_of, keep):
    """p_of(scores [Hq, n, n], kept) -> weights, in 64 bits."""
    out, at = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device="cuda"), 0
    G = q.shape[1] // k.shape[1]
    for b, n in enumerate(lens):
        x, y, z = (t[at:at + n].double().transpose(0, 1) for t in (q, k, v))
        y, z = y.repeat_interleave(G, 0), z.repeat_interleave(G, 0)
        i = torch.arange(n, device="cuda")
        kept = keep(b, i[:, None], i[None, :]) if keep else torch.ones(n, n, dtype=torch.bool, device="cuda")
        out[at:at + n] = (p_of(x @ y.transpose(1, 2), kept, b) @ z).transpose(0, 1)
        at += n
    return out


def softmax(scale):
    return lambda s, kept, b: torch.softmax((s * scale).masked_fill(~kept, -math.inf), -1)


def causal(b, i, j):
    return i >= j


LENS = [1, 0, 127, 128, 129, 2, 255, 256, 257, 0, 500, 1]


@pytest.mark.parametrize("Hq,Hkv,D,DV,dtype", [(4, 2, 128, 128, "bf16"), (6, 2, 64, 64, "fp16"), (4, 4, 64, 128, "bf16"), (8, 1, 128, 64, "fp16"),
                                               (2, 1, 64, 256, "fp16")])
def test_causal(Hq, Hkv, D, DV, dtype):
    eng = examples.softmax_engine("B", Hq, Hkv, "S", D, DV, DT[dtype], True, packed=True)
    q, k, v = inputs(LENS, Hq, Hkv, D, DV, DT[dtype])
    o = eng.prefill_packed(q, k, v, offsets(LENS))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, LENS, softmax(1 / math.sqrt(D)), causal), DT[dtype], stages=2)


@pytest.mark.parametrize("lens", [[1], [128], [3001], [1] * 200, [700, 5], [0, 0, 300], [20] * 40 + [600]])
def test_lengths(lens):
    eng = examples.softmax_engine("B", 4, 2, "S", 64, 64, torch.float16, True, packed=True)
    q, k, v = inputs(lens, 4, 2, 64, 64, torch.float16, seed=len(lens))
    o = eng.prefill_packed(q, k, v, offsets(lens))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, lens, softmax(0.125), causal), torch.float16, stages=2)


def test_many_sequences():
    lens = [(7 * i) % 50 for i in range(4096)]
    eng = examples.softmax_engine("B", 2, 1, "S", 64, 64, torch.bfloat16, True, packed=True)
    q, k, v = inputs(lens, 2, 1, 64, 64, torch.bfloat16)
    o = eng.prefill_packed(q, k, v, offsets(lens))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, lens, softmax(0.125), causal), torch.bfloat16, stages=2)


@pytest.mark.parametrize("mask", ["none", "window", "row"])
def test_other_masks(mask):
    """No mask, a window, and one that depends on the sequence's number."""
    fn = {"none": None, "window": lambda b, h, q, kv: (q >= kv) & (q - kv < 100), "row": lambda b, h, q, kv: (kv % 3 == b % 3) | (q == kv)}[mask]
    keep = {"none": None, "window": lambda b, i, j: (i >= j) & (i - j < 100), "row": lambda b, i, j: (j % 3 == b % 3) | (i == j)}[mask]
    m = [meta_tensor("B", h, "S", 64, dtype=torch.float16) for h in (4, 2, 2)]
    eng = AttentionEngine(m, CustomIO({}), score_mod=lambda s, c, b, h, q, kv: s * 0.125, mask_mod=fn, online_func=examples.OnlineSoftmax(), packed=True)
    lens = [300, 1, 140, 128]
    q, k, v = inputs(lens, 4, 2, 64, 64, torch.float16)
    o = eng.prefill_packed(q, k, v, offsets(lens))
    eng.check_status()
    parity.check("o", o, plain(q, k, v, lens, softmax(0.125), keep), torch.float16, stages=2)


def test_sigmoid_scores_and_customs():
    """An online function without row state, and a bias for each sequence and head."""
    m = [meta_tensor("B", 4, "S", 64, dtype=torch.bfloat16) for _ in range(3)]
    eng = AttentionEngine(m, CustomIO({"bias": ("batch", "heads")}), mask_mod=examples.causal_mask, online_func=examples.OnlineIdentity(), packed=True,
                          score_mod=lambda s, c, b, h, q, kv: (((s * 0.125 + c.input_tensors["bias"]) * 0.5).tanh() + 1) * 0.5)
    lens, bias = [200, 33], torch.randn(2, 4, device="cuda")
    q, k, v = inputs(lens, 4, 4, 64, 64, torch.bfloat16)
    o = eng.prefill_packed(q, k, v, offsets(lens), bias)
    eng.check_status()
    want = plain(q, k, v, lens, lambda s, kept, b: torch.sigmoid(s * 0.125 + bias[b].double()[:, None, None]) * kept, causal)
    parity.check("o", o, want, torch.bfloat16, stages=2, unnormalised=True)
    with pytest.raises(ValueError):
        eng.prefill_packed(q, k, v, offsets(lens), bias[:1, :3])
    with pytest.raises(TypeError):
        eng.prefill_packed(q, k, v, offsets(lens))


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("causal_mask", [True, False])
def test_sequences_do_not_meet(value, causal_mask):
    """A sequence full of infinities or NaN between two others leaves them bit for bit as they are."""
    lens = [130, 60, 200]
    eng = examples.softmax_engine("B", 4, 2, "S", 128, 128, torch.bfloat16, causal_mask, packed=True)
    q, k, v = inputs(lens, 4, 2, 128, 128, torch.bfloat16)
    a = eng.prefill_packed(q, k, v, offsets(lens))
    for t in (q, k, v):
        t[130:190] = value
    b = eng.prefill_packed(q, k, v, offsets(lens))
    assert torch.equal(a[:130], b[:130]) and torch.equal(a[190:], b[190:]) and a.isfinite().all()


def test_equal_lengths_as_a_batch():
    """Packed sequences of one length and the padded call of the same engine kind: the same tiles, the same bits."""
    B, S, Hq, Hkv, D = 3, 384, 4, 2, 128
    q, k, v = inputs([S] * B, Hq, Hkv, D, D, torch.float16)
    packed = examples.softmax_engine("B", Hq, Hkv, "S", D, D, torch.float16, True, packed=True)
    batch = examples.softmax_engine("B", Hq, Hkv, "S", D, D, torch.float16, True)
    a = packed.prefill_packed(q, k, v, offsets([S] * B))
    b = batch(*(t.view(B, S, t.shape[1], D) for t in (q, k, v)))
    assert torch.equal(a.view_as(b), b)


def test_strides_streams_and_graphs():
    lens = [90, 300, 7]
    T, Hq, Hkv, D = sum(lens), 4, 2, 64
    eng = examples.softmax_engine("B", Hq, Hkv, "S", D, D, torch.float16, True, packed=True)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, device="cuda").half()
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
    v = torch.randn(Hkv, T, D, device="cuda").half().transpose(0, 1)  # heads outermost
    cu = offsets(lens)
    first = eng.prefill_packed(q, k, v, cu)
    parity.check("o", first, plain(q, k, v, lens, softmax(0.125), causal), torch.float16, stages=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eng.prefill_packed(q, k, v, cu)
    torch.cuda.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = eng.prefill_packed(q, k, v, cu)
    cu.copy_(offsets([200, 100, 97]))  # the lengths of the replay
    graph.replay()
    torch.cuda.synchronize()
    eng.check_status()
    assert torch.equal(held, eng.prefill_packed(q, k, v, cu))


@pytest.mark.parametrize("cu", [[0, 50, 120], [0, 50, 90], [3, 50, 100], [0, 60, 50, 100], [-4, 50, 100]])
def test_bad_offsets_are_reported(cu):
    """Offsets that do not run from 0 to T: cut to the tensors, and the status says so."""
    eng = examples.softmax_engine("B", 2, 1, "S", 64, 64, torch.float16, True, packed=True)
    q, k, v = inputs([100], 2, 1, 64, 64, torch.float16)
    eng.prefill_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    with pytest.raises(AeError, match="0x2000"):
        eng.check_status()


def test_refusals():
    eng = examples.softmax_engine("B", 4, 2, "S", 64, 64, torch.float16, True, packed=True)
    q, k, v = inputs([20], 4, 2, 64, 64, torch.float16)
    cu = offsets([20])
    for args, err in (((q.float(), k, v, cu), TypeError), ((q.cpu(), k, v, cu), AeError), ((q[None], k, v, cu), ValueError),
                      ((q[:, :3], k, v, cu), ValueError), ((q, k[:10], v[:10], cu), ValueError), ((q, k, v[..., :32], cu), ValueError),
                      ((q, k, v, cu.long()), ValueError), ((q, k, v, cu[:1]), ValueError), ((q, k, v, cu.cpu()), AeError),
                      ((q.clone().requires_grad_(), k, v, cu), NotImplementedError)):
        with pytest.raises(err):
            eng.prefill_packed(*args)
    with torch.no_grad():
        eng.prefill_packed(q.clone().requires_grad_(), k, v, cu)
    with pytest.raises(NotImplementedError):
        eng(q[None], k[None], v[None])
    with pytest.raises(NotImplementedError):
        examples.softmax_engine("B", 4, 2, "S", 64, 64, torch.float16, True).prefill_packed(q, k, v, cu)
    assert tuple(eng.prefill_packed(q[:0], k[:0], v[:0], offsets([0])).shape) == (0, 4, 64)
