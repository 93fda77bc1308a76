"""The decode over an 8-bit cache where it splits its work: intervals of tiles between the SMs, teams of one to eight warps, cut rows and their
merge.  Against 64 bits, tolerances as in test_cache8_gpu.py.  ``team`` is the size that the lengths ask for, so that a test says which form it runs."""
import math

import pytest
import torch

import cache8_ref as ref
import parity
from attentionengine_b200 import PagedCache8
from attentionengine_b200.runtime import AeError
from test_cache8_gpu import DT, E4M3, engine, filled, ints, run, tables

pytestmark = pytest.mark.gpu

# lengths of a few hundred up to 1300 keys, with rows of 0, 1 and a few keys: sums of about 12, 6, 3 and 1 times the longest
MANY = [1300, 1, 700, 0, 1299, 33, 1024, 900, 1300, 640, 1, 1250, 31, 1100, 990, 0, 1290, 777, 1001, 1111, 64, 65, 1200, 128]
SOME = [1300, 0, 1299, 1, 1290, 1000, 17, 1100, 1200, 555]
PAIR = [1300, 1, 1299, 40, 0, 1024]
LONE = [4100, 5]
LONG = [2200, 2100, 1, 2000, 1800, 0, 900, 2199, 17]  # more than 32 tiles of 64 keys


def team(lens, Hkv, Hq, D, DV, Sq=1):
    """Warps that take the same tiles, and whether each unit is a CTA's."""
    tile = 4096 // max(D, DV)
    tiles = [max(1, -(-n // tile)) for n in lens]
    rows = Hq // Hkv if Hq > Hkv else Sq
    row_tiles = -(-rows // (8 if rows <= 8 else 16))
    best = 0
    for i in range(1, 4):
        if Hkv % (1 << i) == 0 and max(tiles) * 148 <= 16 * sum(tiles) * (Hkv >> i) * row_tiles:
            best = i
    single = len(lens) * Hkv * row_tiles <= 148 and -(-max(lens) // tile) <= 32
    return 0 if single else 1 << best


@pytest.mark.parametrize("lens,Hq,Hkv,page,D,DV,dtype,size", [
    (MANY, 32, 8, 64, 128, 128, "bf16", 8), (MANY, 32, 8, 16, 128, 128, "fp16", 8), (MANY, 16, 8, 128, 64, 128, "bf16", 8),
    (MANY, 8, 8, 32, 128, 64, "fp16", 8), (MANY, 16, 16, 16, 64, 64, "fp16", 8), (SOME, 32, 8, 32, 128, 128, "bf16", 4),
    (MANY, 8, 4, 128, 128, 128, "fp16", 4), (LONG, 24, 8, 16, 64, 64, "bf16", 4), (PAIR, 32, 8, 128, 128, 128, "fp16", 2),
    (MANY, 8, 2, 16, 128, 128, "bf16", 2), (LONE, 32, 8, 64, 128, 128, "bf16", 1), (MANY, 4, 1, 32, 128, 128, "fp16", 1),
    (LONG, 9, 3, 64, 64, 64, "bf16", 1),
    # more than 8 query rows of a kv head: tiles of 16, one and several of them
    (MANY, 128, 8, 64, 128, 128, "bf16", 8), (MANY, 40, 4, 16, 128, 128, "fp16", 4), (LONE, 32, 2, 128, 128, 128, "bf16", 1),
    (LONG, 16, 1, 32, 64, 64, "fp16", 1), (MANY, 80, 4, 64, 64, 128, "bf16", 4)])
def test_teams(lens, Hq, Hkv, page, D, DV, dtype, size):
    assert team(lens, Hkv, Hq, D, DV) == size
    o, want = run(Hq, Hkv, lens, page, D, DV, dtype, seed=len(lens) + Hq)
    parity.check("o", o, want, DT[dtype])
    for i, n in enumerate(lens):
        assert n > 0 or (o[i] == 0).all()


@pytest.mark.parametrize("Hkv,Sq,size", [(4, 3, 4), (2, 11, 2), (8, 20, 8)])
def test_positions(Hkv, Sq, size):
    assert team(MANY, Hkv, Hkv, 128, 128, Sq) == size
    o, want = run(Hkv, Hkv, MANY, 32, 128, 128, "fp16", Sq=Sq, seed=Sq)
    parity.check("o", o, want, torch.float16)


@pytest.mark.parametrize("B,Hkv,D,page", [(60, 8, 128, 32), (48, 4, 64, 16), (47, 4, 64, 16), (3000, 1, 64, 16)])
def test_many_rows(B, Hkv, D, page):
    """On both sides of the number of rows whose places are held apart from the tiles, and far beyond."""
    lens = [(37 * i) % 61 * (B < 100) * 5 + i % 40 for i in range(B)]
    assert team(lens, Hkv, Hkv, D, D) > 0
    o, want = run(Hkv, Hkv, lens, page, D, D, "fp16", seed=B)
    parity.check("o", o, want, torch.float16)


@pytest.mark.parametrize("lens,Hkv,G", [(MANY, 8, 4), (SOME, 4, 16), (LONE, 2, 4)])
def test_any_positive_scales(lens, Hkv, G):
    assert team(lens, Hkv, Hkv * G, 128, 128) > 0
    o, want = run(Hkv * G, Hkv, lens, 32, 128, 128, "bf16", pow2=False, spread=3.0, seed=3)
    parity.check("o", o, want, torch.bfloat16, unnormalised=True)


def setup(lens, page, Hkv, D, seed):
    rows, pages = tables(lens, page, seed)
    return rows, pages, filled(pages, page, Hkv, D, D, seed)


@pytest.mark.parametrize("lens,Hkv,G", [(MANY, 8, 2), (SOME, 4, 12), (LONE, 2, 4), (MANY, 1, 4)])
def test_masks_and_customs(lens, Hkv, G):
    """A window that leaves short rows without keys and cuts the first tiles off the others, a slope for each head, a bias for each row."""
    D, Hq, B = 128, Hkv * G, len(lens)
    assert team(lens, Hkv, Hq, D, D) > 0
    rows, _, (k, v, ks, vs) = setup(lens, 16, Hkv, D, 1)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(B, 1, Hq, D, generator=g).half().cuda()
    slope, bias = torch.rand(1, Hq, generator=g).cuda() * 0.01, torch.randn(B, generator=g).cuda()
    eng = engine(Hq, Hkv, 1, D, D, torch.float16, customs={"slope": (1, "heads"), "bias": ("batch",)}, mask=lambda b, h, qi, kv: kv >= 100,
                 score=lambda s, c, b, h, qi, kv: s * 0.08 + kv * c.input_tensors["slope"] + c.input_tensors["bias"])
    o = eng.decode_cache8(q, PagedCache8.from_tensors(k, v, ks, vs), ints(rows), ints(lens), slope, bias)
    eng.check_status()
    want = ref.decode(q, k, v, ks, vs, rows, lens, 0.08, keep=lambda b, h, i, kv: kv >= 100,
                      score=lambda s, b, h: s + torch.arange(len(s)) * slope[0, h].item() + bias[b].item())
    parity.check("o", o, want, torch.float16)
    for i, n in enumerate(lens):
        assert n > 100 or (o[i] == 0).all()


@pytest.mark.parametrize("lens,Hkv,G", [(MANY, 8, 4), (SOME, 4, 16), (LONE, 2, 4)])
def test_pages_outside_the_pool_count_as_zeros(lens, Hkv, G):
    """Reported, and the keys of such a page are zeros: the other rows are as they were, bit for bit."""
    D, page, Hq = 128, 32, Hkv * G
    assert team(lens, Hkv, Hq, D, D) > 0
    rows, pages, (k, v, ks, vs) = setup(lens, page, Hkv, D, 2)
    q = torch.randn(len(lens), 1, Hq, D, device="cuda").half()
    eng, cache = engine(Hq, Hkv, 1, D, D, torch.float16), PagedCache8.from_tensors(k, v, ks, vs)
    good = eng.decode_cache8(q, cache, ints(rows), ints(lens))
    eng.check_status()
    bad = [list(r) for r in rows]
    bad[0][1], bad[0][17] = pages, -1
    o = eng.decode_cache8(q, cache, ints(bad), ints(lens))
    with pytest.raises(AeError, match="0x1000"):
        eng.check_status()
    assert torch.equal(o[1:], good[1:])
    zeros = [torch.cat([t.view(torch.uint8), t.view(torch.uint8)[:1] * 0]).view(E4M3) for t in (k, v)]
    ones = [torch.cat([t, torch.ones_like(t[:1])]) for t in (ks, vs)]
    want = ref.decode(q[:1], *zeros, *ones, [[p if 0 <= p < pages else pages for p in bad[0]]], lens[:1], 1 / math.sqrt(D))
    parity.check("o", o[:1], want, torch.float16)


@pytest.mark.parametrize("which", ["k", "v", "q", "behind"])
@pytest.mark.parametrize("lens,Hkv,G", [(MANY, 8, 4), (SOME, 4, 16), (PAIR, 8, 1)])
def test_nan_stays_in_its_row(which, lens, Hkv, G):
    D, page, Hq = 128, 16, Hkv * G
    assert team(lens, Hkv, Hq, D, D) > 0
    rows, pages, (k, v, ks, vs) = setup(lens, page, Hkv, D, 5)
    q = torch.randn(len(lens), 1, Hq, D, device="cuda", dtype=torch.float16)
    eng = engine(Hq, Hkv, 1, D, D, torch.float16)
    cache = PagedCache8.from_tensors(k, v, ks, vs)
    good = eng.decode_cache8(q, cache, ints(rows), ints(lens))
    bad, hit = torch.zeros(len(lens), 1, Hq, D, dtype=torch.bool), 2
    heads = slice(G, 2 * G)  # of kv head 1
    if which == "q":
        q[hit, 0, G, 5] = math.nan
        bad[hit, 0, G] = True
    elif which == "behind":  # codes behind each row's last key, and the scales of pages that are no row's
        used = set()
        for row, n in zip(rows, lens):
            used |= set(row[:-(-n // page)])
            if n % page:
                for t in (k, v):
                    t.view(torch.uint8)[row[n // page], n % page:] = 0x7f
        for p in set(range(pages)) - used:
            ks[p] = vs[p] = math.nan
    else:
        (k if which == "k" else v).view(torch.uint8)[rows[hit][lens[hit] // page // 2], 4, 1, 9] = 0x7f
        bad[hit, 0, heads] = True
        if which == "v":
            bad[hit, 0, heads] = (torch.arange(D) == 9)
    o = eng.decode_cache8(q, cache, ints(rows), ints(lens))
    eng.check_status()
    assert torch.equal(o.isnan().cpu(), bad)
    keep = ~bad.cuda()
    assert torch.equal(o[keep], good[keep]) or which == "q"


@pytest.mark.parametrize("lens,Hkv,G", [(MANY, 8, 4), (SOME, 4, 16), (LONE, 1, 8)])
def test_repeats_and_graphs(lens, Hkv, G):
    D, page, Hq = 128, 64, Hkv * G
    rows, pages, (k, v, ks, vs) = setup(lens, page, Hkv, D, 6)
    q = torch.randn(len(lens), 1, Hq, D, device="cuda").to(torch.bfloat16)
    eng, cache = engine(Hq, Hkv, 1, D, D, torch.bfloat16), PagedCache8.from_tensors(k, v, ks, vs)
    t, n = ints(rows), ints(lens)
    first = eng.decode_cache8(q, cache, t, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [eng.decode_cache8(q, cache, t, n) for _ in range(10)]
    again = [eng.decode_cache8(q, cache, t, n) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in other + again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = eng.decode_cache8(q, cache, t, n)
    n.copy_(ints([max(0, x - 300) for x in lens]))  # a graph reads the lengths of its replay
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, eng.decode_cache8(q, cache, t, n))
    eng.check_status()
