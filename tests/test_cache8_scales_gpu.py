"""Writes into pages whose scales are not powers of two (a cache that was filled elsewhere), bit for bit against 64 bits: a page that goes on
keeps such a scale while it is the coarser one, or is rounded again at the power of two that the new tokens need."""
import math

import numpy as np
import pytest
import torch

from attentionengine_b200 import PagedCache8
from test_cache8_gpu import E4M3, write_and_compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,D,dtype", [(16, 64, torch.float16), (32, 128, torch.bfloat16), (128, 128, torch.float16), (64, 64, torch.bfloat16)])
def test_pages_that_came_with_any_scale(page, D, dtype):
    H, pages = 4, 12
    g = torch.Generator().manual_seed(page)

    def pool():
        x = torch.randn(pages, page, H, D, generator=g)
        s = x.abs().amax(dim=(1, 3)) / 448 * (1 + torch.rand(pages, H, generator=g))
        return (x / s[:, None, :, None]).to(E4M3).cuda(), s.cuda()

    (k, ks), (v, vs) = pool(), pool()
    cache = PagedCache8.from_tensors(k, v, ks, vs)
    # pages that go on with tokens a quarter to 64 times as large as theirs; head by head some keep their scale and some do not
    seg, tok, size = [], 0, []
    for p in range(pages - 2):
        n = page // 2 - p % 3
        seg.append([p, page // 2, tok, n])
        size += [2.0 ** (p % 9 - 2)] * n
        tok += n
    new = [(torch.randn(tok, H, D, generator=g) * torch.tensor(size)[:, None, None] * torch.exp(torch.randn(1, H, 1, generator=g))).to(dtype) for _ in "kv"]
    kept = ks.cpu().clone()
    write_and_compare(cache, *new, seg)
    same = (cache.k_scale.cpu() == kept)[:pages - 2]
    assert same.any() and not same.all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quotients_beside_a_tie(dtype):
    """Values whose quotient by the scale lies next to the middle of two codes, on either side: x = s t (1 + d) for the middles t, as near as the
    type and a fp32 scale can come."""
    page, D, H = 64, 128, 1
    steps = torch.tensor([t * 2.0 ** e for e in range(-6, 8) for t in (1.0625, 1.1875, 1.3125, 1.4375, 1.5625, 1.6875, 1.8125, 1.9375)])
    x = torch.cat([torch.linspace(1, 2, 257)[:-1] * 2.0 ** e for e in (-3, 0, 3)]).to(dtype).double()
    scales, rows = [], []
    for i in range(len(steps) // 4):
        t = steps[4 * i].double()
        s = (x[7 + 5 * i] / t).float()  # the quotient of x[7 + 5 i] is t but for the rounding of s
        scales.append(s.item())
        near = (steps.double() * s.double()).to(dtype)
        rows.append(torch.cat([near, -near])[:D] if len(near) * 2 >= D else torch.cat([near, -near, near])[:D])
    n = len(scales)
    new = torch.stack(rows).view(n, 1, D)
    limit = torch.exp2(torch.tensor(scales).double().log2().floor()).view(n, 1, 1) * 448  # no value asks for a coarser scale
    new = torch.where(new.double().abs() <= limit, new, 0).to(dtype)
    codes = torch.zeros(n, page, H, D, dtype=torch.uint8, device="cuda").view(E4M3)
    s = torch.tensor(scales, device="cuda").view(n, 1)
    cache = PagedCache8.from_tensors(codes, codes.view(torch.uint8).clone().view(E4M3), s, s.clone())
    write_and_compare(cache, new, -new, [[i, 1, i, 1] for i in range(n)])
    assert cache.k_scale.flatten().tolist() == [np.float32(x) for x in scales]


def test_special_values_beside_such_a_scale():
    k = torch.full((2, 16, 1, 64), 1.0, device="cuda").to(E4M3)
    k.view(torch.uint8)[0, 0, 0, 5] = 0x7f
    s = torch.tensor([[0.3], [3e-20]], device="cuda")
    cache = PagedCache8.from_tensors(k, k.view(torch.uint8).clone().view(E4M3), s, s.clone())
    x = torch.zeros(4, 1, 64, dtype=torch.float16)
    x[0, 0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 100.0, 0.15, 6e-8])
    x[2, 0, :3] = torch.tensor([6e-8, -1e-3, math.inf])
    write_and_compare(cache, x, -x, [[0, 1, 0, 2], [1, 3, 2, 2]])
    assert cache.k_scale[0, 0].item() == np.float32(0.3)
