"""The paged 8-bit cache: writes bit for bit against 64 bits, decode against 64 bits on the cached values.

Tolerances of the decode: e4m3 codes are exact in fp16 and the query rows too, so what is rounded is P (fp16, a step of 2^-11) and the stored
output.  bf16 outputs: one rounding to bf16 and P's, an eighth of it: sqrt(1 + 1/64) of the floor, inside the 1.15 of tests/parity.py at one
stage.  fp16 outputs: two roundings of 2^-11, rel-L2 about 1.4 x 2^-11 / sqrt(3) = 4e-4 against the 1e-3 of tests/parity.py.
"""
import math

import numpy as np
import pytest
import torch

import cache8_ref as ref
import parity
from attentionengine_b200 import AttentionEngine, CustomIO, PagedCache8, examples, meta_tensor, plan_pages
from attentionengine_b200.runtime import AeError

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def values(shape, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(shape[0], shape[1], 1, generator=g))).to(dtype)


def both(cache):
    """The cache's contents as float64 arrays."""
    return {n: getattr(cache, n).double().cpu().numpy().copy() for n in ("k", "v", "k_scale", "v_scale")}


def write_and_compare(cache, k, v, segments):
    want = both(cache)
    ref.write(want["k"], want["k_scale"], k.double().cpu().numpy(), segments)
    ref.write(want["v"], want["v_scale"], v.double().cpu().numpy(), segments)
    cache.write(k.cuda(), v.cuda(), ints(segments))
    got = both(cache)
    for n in want:
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)


@pytest.mark.parametrize("page,H,D,DV,dtype", [(16, 1, 64, 64, "bf16"), (32, 3, 128, 64, "fp16"), (64, 8, 128, 128, "bf16"),
                                               (128, 2, 64, 128, "fp16"), (128, 1, 128, 128, "bf16")])
def test_write(page, H, D, DV, dtype):
    cache = PagedCache8(9, page, H, D, DV)
    # full pages, one token, a part; then pages that go on, some at a coarser scale, and a segment without tokens
    first = [[3, 0, 0, page], [5, 0, page, 1], [0, 0, page + 1, page - 3], [8, 0, 2 * page - 2, 2]]
    n = sum(s[3] for s in first)
    write_and_compare(cache, values((n, H, D), DT[dtype], 1), values((n, H, DV), DT[dtype], 2), first)
    more = [[5, 1, 0, page - 1], [0, 0, 0, 0], [0, page - 3, page - 1, 3], [8, 2, page + 2, 1]]
    n = sum(s[3] for s in more)
    write_and_compare(cache, values((n, H, D), DT[dtype], 3), values((n, H, DV), DT[dtype], 4), more)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_write_special_values(dtype):
    """Infinities, NaN, zeros, the ends of the type's range, and the scale's own edge 448 x 2^e."""
    cache = PagedCache8(4, 16, 2, 64)
    fin = torch.finfo(DT[dtype])
    x = torch.zeros(20, 2, 64, dtype=DT[dtype])
    x[0, 0, :8] = torch.tensor([math.inf, -math.inf, math.nan, 1.0, -3.5, 448.0, 1e-3, 0.0]).to(DT[dtype])
    x[1, 1, :3] = torch.tensor([fin.max, fin.tiny, -fin.max])
    x[16, 0, :4] = torch.tensor([3.5, 3.25, 2.0 ** -9, 2.0 ** -10])
    x[17, 1, :2] = torch.tensor([fin.smallest_normal, fin.smallest_normal / 4])
    segments = [[1, 0, 0, 16], [2, 0, 16, 4]]
    write_and_compare(cache, x, x.flip(0), segments)
    write_and_compare(cache, x * 0, x * 0, [[1, 0, 0, 1]])  # inf * 0: NaN everywhere it was infinite
    assert cache.k_scale[1].tolist() == [2.0 ** -64] * 2


@pytest.mark.parametrize("dtype,exponents", [("fp16", [13, 0, -6, -7, -8, -9, -14, -20]), ("bf16", [100, 20, 0, -7, -9, -40, -70, -110])])
def test_write_magnitudes(dtype, exponents):
    """Pages from the top of the type's range to its bottom, small values beside large ones in each: where a scale's reciprocal is a number of
    the type and where it is not, and scales at their lower bound."""
    cache = PagedCache8(len(exponents), 32, 2, 64)
    x = torch.cat([values((32, 2, 64), torch.float32, 50 + i, spread=3.0).clamp(-3, 3) * 2.0 ** e for i, e in enumerate(exponents)]).to(DT[dtype])
    assert x.isfinite().all()
    write_and_compare(cache, x, -x.flip(1), [[i, 0, 32 * i, 32] for i in range(len(exponents))])


def test_a_page_that_grows_token_by_token():
    """Sixteen steps into one page, each larger than the last: the codes that are there are rounded again each time."""
    cache = PagedCache8(2, 16, 1, 64)
    for i in range(16):
        k = values((1, 1, 64), torch.bfloat16, 100 + i, spread=0.0) * 2.0 ** (i - 8)
        write_and_compare(cache, k, -k, [[1, i, 0, 1]])


def test_write_takes_slices_and_strided_pools():
    """k and v as parts of one projection's output, and pools that share one tensor."""
    page, H, D = 32, 2, 64
    pool = torch.zeros(5, page, 2 * H, D, dtype=torch.uint8, device="cuda").view(E4M3)
    scale = torch.ones(5, 2 * H, device="cuda")
    cache = PagedCache8.from_tensors(pool[:, :, :H], pool[:, :, H:], scale[:, :H], scale[:, H:])
    qkv = values((40, 3 * H, D), torch.bfloat16, 7).cuda()
    seg = [[4, 0, 0, 32], [2, 0, 32, 8]]
    want = both(cache)
    ref.write(want["k"], want["k_scale"], qkv[:, H:2 * H].double().cpu().numpy(), seg)
    ref.write(want["v"], want["v_scale"], qkv[:, 2 * H:].double().cpu().numpy(), seg)
    cache.write(qkv[:, H:2 * H], qkv[:, 2 * H:], ints(seg))
    for n, x in both(cache).items():
        np.testing.assert_array_equal(x, want[n])


def test_write_passes_over_segments_outside():
    """A page, a slot range or tokens that are not there: nothing is written."""
    cache = PagedCache8(3, 16, 1, 64)
    before = both(cache)
    x = values((4, 1, 64), torch.float16, 1).cuda()
    cache.write(x, x, ints([[3, 0, 0, 1], [-1, 0, 0, 1], [1, 15, 0, 2], [1, 0, 3, 2], [1, 0, -1, 1], [1, 16, 0, 1], [2, 0, 0, -5]]))
    cache.write(x[:0], x[:0], ints([[0, 0, 0, 1]]))
    cache.write(x, x, ints([[0, 0, 0, 1]])[:0])
    for n, y in both(cache).items():
        np.testing.assert_array_equal(y, before[n])


# ------------------------------------------------------------------------------------------------------------ decode
def filled(pages, page, H, D, DV, seed, pow2=True, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    out = []
    for d in (D, DV):
        x = torch.randn(pages, page, H, d, generator=g) * torch.exp(spread * torch.randn(pages, 1, H, 1, generator=g))
        s = x.abs().amax(dim=(1, 3)) / 448
        s = torch.exp2(torch.ceil(torch.log2(s))) if pow2 else s * (1 + torch.rand(pages, H, generator=g))
        out += [(x / s[:, None, :, None]).to(E4M3).cuda(), s.float().cuda()]
    return out[0], out[2], out[1], out[3]  # k, v, k_scale, v_scale


def tables(lens, page, seed, wide=0):
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [10 ** 9] * (max(max(need), 1) + wide - n))  # entries behind a row's pages are not read
        at += n
    return rows, sum(need) + 3


def run(Hq, Hkv, lens, page, D, DV, dtype, Sq=1, seed=0, pow2=True, spread=0.5, q_scale=1.0):
    rows, pages = tables(lens, page, seed)
    k, v, ks, vs = filled(pages, page, Hkv, D, DV, seed, pow2, spread)
    q = (torch.randn(len(lens), Sq, Hq, D, generator=torch.Generator().manual_seed(seed + 1)) * q_scale).to(DT[dtype]).cuda()
    eng = engine(Hq, Hkv, Sq, D, DV, DT[dtype])
    o = eng.decode_cache8(q, PagedCache8.from_tensors(k, v, ks, vs), ints(rows), ints(lens))
    eng.check_status()
    return o, ref.decode(q, k, v, ks, vs, rows, lens, 1 / math.sqrt(D))


def engine(Hq, Hkv, Sq, D, DV, dtype, score=None, mask=None, customs=None, online=None):
    m = (meta_tensor("B", Hq, Sq, D, dtype=dtype), meta_tensor("B", Hkv, "S", D, dtype=dtype), meta_tensor("B", Hkv, "S", DV, dtype=dtype))
    scale = 1 / math.sqrt(D)
    return AttentionEngine(m, CustomIO(customs or {}), score_mod=score or (lambda s, c, b, h, q, kv: s * scale), mask_mod=mask,
                           online_func=online or examples.OnlineSoftmaxSplit(), cache_dtype=E4M3)


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("D,DV,dtype", [(128, 128, "bf16"), (64, 64, "fp16"), (128, 64, "fp16"), (64, 128, "bf16")])
def test_lengths_and_pages(page, D, DV, dtype):
    o, want = run(4, 2, EDGES, page, D, DV, dtype, seed=page)
    parity.check("o", o, want, DT[dtype])
    assert (o[0] == 0).all()


@pytest.mark.parametrize("Hq,Hkv,Sq", [(1, 1, 1), (3, 3, 1), (10, 2, 1), (16, 2, 1), (18, 2, 1), (32, 2, 1), (40, 1, 1), (2, 2, 3), (2, 2, 11), (1, 1, 37)])
def test_groups_and_positions(Hq, Hkv, Sq):
    o, want = run(Hq, Hkv, [70, 1, 200], 16, 128, 128, "bf16", Sq=Sq, seed=Hq)
    parity.check("o", o, want, torch.bfloat16)


@pytest.mark.parametrize("lens", [[5000], [3000, 1, 40, 2500], [700] * 40, [1] * 300, [4000] * 3, [0] * 5])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (12, 6)])
def test_many_splits(lens, Hq, Hkv):
    """Few long rows, many short ones, both."""
    o, want = run(Hq, Hkv, lens, 64, 64, 64, "fp16", seed=len(lens))
    parity.check("o", o, want, torch.float16)


def test_any_positive_scales():
    o, want = run(8, 2, [300, 90], 32, 128, 128, "bf16", pow2=False, spread=3.0, seed=3)
    parity.check("o", o, want, torch.bfloat16, unnormalised=True)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-4, 30.0, 1e30])
def test_query_magnitudes(q_scale):
    """bf16 queries far outside fp16's range: scores that vanish, a softmax that picks one key, scores of 1e30."""
    o, want = run(8, 2, [150, 40], 16, 64, 64, "bf16", q_scale=q_scale, seed=5)
    parity.check("o", o, want, torch.bfloat16)


def test_masks_and_customs():
    """A window that leaves a row without keys, a slope for each head, a bias for each row."""
    lens, D = [100, 33, 260], 64
    rows, pages = tables(lens, 16, 1)
    k, v, ks, vs = filled(pages, 16, 2, D, D, 1)
    q = torch.randn(3, 1, 4, D, dtype=torch.float16, device="cuda")
    slope, bias = torch.tensor([[0.1, 0.02, 0.3, 0.0]], device="cuda"), torch.tensor([0.5, -1.0, 2.0], device="cuda")
    eng = engine(4, 2, 1, D, D, torch.float16, customs={"slope": (1, "heads"), "bias": ("batch",)}, mask=lambda b, h, qi, kv: kv >= 40,
                 score=lambda s, c, b, h, qi, kv: s * 0.125 + kv * c.input_tensors["slope"] + c.input_tensors["bias"])
    o = eng.decode_cache8(q, PagedCache8.from_tensors(k, v, ks, vs), ints(rows), ints(lens), slope, bias)
    eng.check_status()
    want = ref.decode(q, k, v, ks, vs, rows, lens, 0.125, keep=lambda b, h, i, kv: kv >= 40,
                      score=lambda s, b, h: s + torch.arange(len(s)) * slope[0, h].item() + bias[b].item())
    parity.check("o", o, want, torch.float16)
    assert (o[1] == 0).all()
    for bad in ((slope,), (slope[:, :3], bias), (slope, bias[:2]), (slope.cpu(), bias)):
        with pytest.raises((TypeError, ValueError, AeError)):
            eng.decode_cache8(q, PagedCache8.from_tensors(k, v, ks, vs), ints(rows), ints(lens), *bad)


def test_what_lies_behind_the_keys_is_not_read():
    """Old codes behind a row's last key, NaN among them, and NaN scales of pages that are not its own."""
    lens, page, D = [5, 70, 33], 16, 128
    rows, pages = tables(lens, page, 2)
    k, v, ks, vs = filled(pages, page, 2, D, D, 2)
    clean = PagedCache8.from_tensors(k.clone(), v.clone(), ks.clone(), vs.clone())
    eng = engine(8, 2, 1, D, D, torch.bfloat16)
    q = torch.randn(3, 1, 8, D, device="cuda").to(torch.bfloat16)
    a = eng.decode_cache8(q, clean, ints(rows), ints(lens))
    used = set()
    for row, n in zip(rows, lens):
        used |= set(row[:-(-n // page)])
        for t in (k, v):
            t.view(torch.uint8)[row[(n - 1) // page], (n - 1) % page + 1:] = 0x7f
    for p in set(range(pages)) - used:
        k.view(torch.uint8)[p] = v.view(torch.uint8)[p] = 0x7f
        ks[p] = vs[p] = math.nan
    b = eng.decode_cache8(q, PagedCache8.from_tensors(k, v, ks, vs), ints(rows), ints(lens))
    assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_nan_stays_in_its_row(which):
    lens, page, D = [90, 90, 90], 16, 64
    rows, pages = tables(lens, page, 3)
    k, v, ks, vs = filled(pages, page, 2, D, D, 3)
    q = torch.randn(3, 1, 4, D, device="cuda", dtype=torch.float16)
    if which == "q":
        q[1, 0, 2, 5] = math.nan
    else:
        (k if which == "k" else v).view(torch.uint8)[rows[1][3], 4, 1, 9] = 0x7f
    eng = engine(4, 2, 1, D, D, torch.float16)
    o = eng.decode_cache8(q, PagedCache8.from_tensors(k, v, ks, vs), ints(rows), ints(lens)).cpu()
    bad = torch.zeros(3, 1, 4, D, dtype=torch.bool)
    if which == "q":
        bad[1, 0, 2] = True
    elif which == "k":
        bad[1, 0, 2:] = True
    else:
        bad[1, 0, 2:, 9] = True
    assert torch.equal(o.isnan(), bad)


def test_offsets_past_32_bits():
    """A pool of 4.8e9 bytes: pages on both sides of 2^31 and 2^32."""
    page, H, D, pages = 128, 8, 128, 36_700
    k = torch.empty(pages, page, H, D, dtype=torch.uint8, device="cuda").view(E4M3)
    v, ks, vs = torch.empty_like(k), torch.full((pages, H), math.nan, device="cuda"), torch.full((pages, H), math.nan, device="cuda")
    assert k.numel() > 2 ** 32
    rows, lens = [[36_699, 16_390, 32_770], [32_767, 5, 0]], [300, 259]
    cache = PagedCache8.from_tensors(k, v, ks, vs)
    seg, tok = [], 0
    for row, n in zip(rows, lens):
        for i, p in enumerate(row):
            seg.append([p, 0, tok, min(page, n - i * page)])
            tok += seg[-1][3]
    new_k, new_v = values((tok, H, D), torch.bfloat16, 1, 0.3).cuda(), values((tok, H, D), torch.bfloat16, 2, 0.3).cuda()
    cache.write(new_k, new_v, ints(seg))
    q = torch.randn(2, 1, 16, D, device="cuda", dtype=torch.float16)
    eng = engine(16, 8, 1, D, D, torch.float16)
    o = eng.decode_cache8(q, cache, ints(rows), ints(lens))
    used = [p for row in rows for p in row]
    at = {p: i for i, p in enumerate(used)}
    small = [t[used] for t in (k.view(torch.uint8), v.view(torch.uint8))]
    want = ref.decode(q, small[0].view(E4M3), small[1].view(E4M3), ks[used], vs[used], [[at[p] for p in r] for r in rows], lens, 1 / math.sqrt(D))
    parity.check("o", o, want, torch.float16)


def test_strided_queries_other_streams_graphs_and_repeats():
    lens, page, D = [500, 3, 0, 77], 32, 128
    rows, pages = tables(lens, page, 4, wide=3)
    k, v, ks, vs = filled(pages, page, 4, D, D, 4)
    cache = PagedCache8.from_tensors(k, v, ks, vs)
    eng = engine(16, 4, 1, D, D, torch.bfloat16)
    wide = torch.randn(16, 4, 3 * D, device="cuda").to(torch.bfloat16)
    q = wide[:, :, D:2 * D].permute(1, 0, 2).unsqueeze(1)  # [4, 1, 16, D], heads outermost, rows of a wider tensor
    t, n = ints(rows)[:, :-2], ints(lens)
    want = ref.decode(q, k, v, ks, vs, rows, lens, 1 / math.sqrt(D))
    first = eng.decode_cache8(q, cache, t, n)
    parity.check("o", first, want, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [eng.decode_cache8(q, cache, t, n) for _ in range(20)]
    again = [eng.decode_cache8(q, cache, t, n) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in other + again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = eng.decode_cache8(q, cache, t, n)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, held)
    n.copy_(ints([10, 500, 40, 1])[:4].clamp(max=t.shape[1] * page))  # a graph reads the lengths of its replay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, eng.decode_cache8(q, cache, t, n))


def test_bad_lengths_and_pages_are_reported():
    page, D = 16, 64
    k, v, ks, vs = filled(4, page, 1, D, D, 1)
    cache, eng = PagedCache8.from_tensors(k, v, ks, vs), engine(2, 1, 1, D, D, torch.float16)
    q = torch.randn(2, 1, 2, D, device="cuda", dtype=torch.float16)
    eng.decode_cache8(q, cache, ints([[0, 1], [2, 3]]), ints([32, 17]))
    eng.check_status()
    for rows, lens in (([[0, 1], [2, 3]], [33, 1]), ([[0, 1], [2, 3]], [3, -1]), ([[0, 4], [2, 3]], [17, 1]), ([[0, -1], [2, 3]], [17, 1])):
        eng.decode_cache8(q, cache, ints(rows), ints(lens))
        with pytest.raises(AeError, match="status"):
            eng.check_status()
        eng.check_status()


def test_refusals():
    k, v, ks, vs = filled(4, 16, 2, 64, 64, 1)
    good = PagedCache8.from_tensors(k, v, ks, vs)
    for args, err in (((k.cpu(), v, ks, vs), AeError), ((k.float(), v, ks, vs), TypeError), ((k[0], v, ks, vs), ValueError),
                      ((k[:, :8], v[:, :8], ks, vs), ValueError), ((k, v[:3], ks, vs), ValueError), ((k, v, ks[:3], vs), ValueError),
                      ((k, v, ks.double(), vs), ValueError), ((k[..., :32], v, ks, vs), (ValueError, NotImplementedError)),
                      ((k[:0], v[:0], ks[:0], vs[:0]), ValueError)):
        with pytest.raises(err):
            PagedCache8.from_tensors(*args)
    x, seg = torch.randn(3, 2, 64, device="cuda").half(), ints([[0, 0, 0, 3]])
    for args, err in (((x.float(), x.float(), seg), TypeError), ((x, x.bfloat16(), seg), TypeError), ((x[:, :1], x, seg), ValueError),
                      ((x, x[:2], seg), ValueError), ((x.cpu(), x, seg), AeError), ((x, x, seg.long()), ValueError),
                      ((x, x, ints([0, 0, 0, 3])), ValueError), ((x.clone().requires_grad_(), x, seg), NotImplementedError)):
        with pytest.raises(err):
            good.write(*args)
    with torch.no_grad():
        good.write(x.clone().requires_grad_(), x, seg)
    eng = engine(4, 2, 1, 64, 64, torch.float16)
    q, t, n = torch.randn(2, 1, 4, 64, device="cuda").half(), ints([[0], [1]]), ints([5, 9])
    eng.decode_cache8(q, good, t, n)
    for args, err in (((q.float(), good, t, n), TypeError), ((q.cpu(), good, t, n), AeError), ((q[:, :, :2], good, t, n), ValueError),
                      ((q, k, t, n), TypeError), ((q, good, t[:1], n), ValueError), ((q, good, t.long(), n), ValueError),
                      ((q, good, t, n[:1]), ValueError), ((q, good, t, n.cpu()), AeError), ((q, good, t[:, :0], n), ValueError),
                      ((q, PagedCache8(2, 16, 1, 64), t, n), ValueError), ((q, good, t, n, n), TypeError),
                      ((q.clone().requires_grad_(), good, t, n), NotImplementedError)):
        with pytest.raises(err):
            eng.decode_cache8(*args)
    with pytest.raises(NotImplementedError):
        eng(q, k, v)
    with pytest.raises(NotImplementedError):
        examples.decode_engine(2, 4, 2, 1, 64, 64, torch.float16).decode_cache8(q, good, t, n)
    empty = eng.decode_cache8(q[:0], good, t[:0], n[:0])
    assert tuple(empty.shape) == (0, 1, 4, 64)


# ------------------------------------------------------------------------------------------------------------ a serving loop
def test_a_step_in_a_graph():
    """Plan, write and decode of a step captured as one graph, each brought up under the one in front; replayed with other lengths, keys and queries
    it gives what the calls give."""
    Hq, Hkv, D, page, B, dtype = 16, 4, 128, 32, 5, torch.bfloat16
    g = torch.Generator().manual_seed(3)
    k, v, ks, vs = filled(60, page, Hkv, D, D, 9)
    eng = engine(Hq, Hkv, 1, D, D, dtype)
    free, head, one = ints(list(range(40, 60))), ints([0]), ints([1] * B)
    table, lens = ints([[8 * b + i if i < 7 else 0 for i in range(10)] for b in range(B)]), ints([1] * B)
    q, nk, nv = (torch.zeros(B, h, D, dtype=dtype, device="cuda") for h in (Hq, Hkv, Hkv))

    def step(cache, table):
        plan = plan_pages(lens, one, table, free, head, page, B)
        cache.write(nk, nv, plan.segments)
        return plan, eng.decode_cache8(q.unsqueeze(1), cache, plan.block_table, plan.seq_lens)

    def fresh():
        return PagedCache8.from_tensors(*(t.clone() for t in (k, v, ks, vs)))

    in_graph, its_table = fresh(), table.clone()
    step(in_graph, its_table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, o = step(in_graph, its_table)
    for now in ([1, 31, 32, 95, 200], [224, 223, 1, 64, 63], [96, 128, 7, 33, 160]):
        lens.copy_(ints(now))
        for t in (q, nk, nv):
            t.copy_(torch.randn(t.shape, generator=g))
        for a, b in zip((in_graph.k, in_graph.v, in_graph.k_scale, in_graph.v_scale), (k, v, ks, vs)):
            a.copy_(b)
        its_table.copy_(table)
        graph.replay()
        apart, want_table = fresh(), table.clone()
        want_plan, want = step(apart, want_table)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(its_table, want_table)
        assert all(torch.equal(x, y) for x, y in zip(plan, want_plan))
        for a, b in zip((in_graph.k, in_graph.v, in_graph.k_scale, in_graph.v_scale), (apart.k, apart.v, apart.k_scale, apart.v_scale)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        plan.check()
    eng.check_status()


def test_a_served_layer_from_prompts_to_tokens():
    """examples.PagedLayers: prompts of different lengths, then tokens one by one, the pages running over several times; two layers share the
    pages.  Prompts against 64 bits on the 16-bit keys, tokens on the cached ones."""
    Hq, Hkv, D, page, dtype = 8, 2, 64, 16, torch.bfloat16
    lens = [37, 1, 16, 90]
    serve = examples.PagedLayers(2, Hq, Hkv, D, dtype, rows=len(lens), num_pages=40, page_size=page, max_len=200)
    g = torch.Generator().manual_seed(1)
    new = lambda n: [torch.randn(n, h, D, generator=g).to(dtype).cuda() for h in (Hq, Hkv, Hkv)]  # noqa: E731
    layers = [new(sum(lens)) for _ in range(2)]
    outs = serve.prompts(layers, ints(lens))
    for (q, k, v), o in zip(layers, outs):
        at = 0
        for n in lens:
            x, y, z = (t[at:at + n].double().transpose(0, 1).repeat_interleave(Hq // t.shape[1], 0) for t in (q, k, v))
            s = (x @ y.transpose(1, 2) / 8).masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
            parity.check("prompt", o[at:at + n], (torch.softmax(s, -1) @ z).transpose(0, 1), dtype, stages=2)
            at += n
    for step in range(20):
        layers = [new(len(lens)) for _ in range(2)]
        outs = serve.tokens(layers)
        now = [n + step + 1 for n in lens]
        assert serve.lens.tolist() == now
        if step in (0, 1, 15, 19):
            for (q, k, v), o, c in zip(layers, outs, serve.caches):
                want = ref.decode(q[:, None], c.k, c.v, c.k_scale, c.v_scale, serve.table.tolist(), now, 1 / 8)
                parity.check("token", o, want[:, 0], dtype)
    serve.check()
