"""QKNormRope on rows of the type's largest values: their squares' sum is infinite in fp32, the norm's factor 0, and every finite value becomes 0 (an infinity or NaN: NaN),
as with x * rsqrt(mean(x^2) + eps) * w in fp32; nothing before the factor may overflow by itself."""
import pytest
import torch

from attentionengine_b200 import QKNormRope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,R,interleaved", [(32, 32, False), (64, 64, True), (128, 128, False), (128, 64, True), (256, 144, False)])
@pytest.mark.parametrize("weight", [None, 1.0, 100.0])
def test_rows_of_the_type_s_largest_values(D, R, interleaved, weight):
    g = torch.Generator().manual_seed(D + R)
    rope = QKNormRope(D, rotary_dim=R, interleaved=interleaved, rotary_scale=1.2)
    low = torch.finfo(torch.bfloat16).min
    x = torch.randn(40, 6, D, generator=g).bfloat16()
    rows = torch.rand(40, 6, generator=g) < 0.4
    big = torch.where(torch.rand(40, 6, D, generator=g) < 0.5, low, -low).bfloat16()
    big[::2] = low
    mixed = torch.where(rows[..., None], big, x)
    mixed[3, 2], mixed[3, 2, 1::2], rows[3, 2] = low, 0.5, True  # small values beside them
    w = None if weight is None else (weight * (1 + 0.2 * torch.rand(D, generator=g))).cuda()
    pos = torch.randint(0, 10000, (40,), generator=g).cuda()
    q = mixed.cuda().requires_grad_()
    k = mixed[:, :1].contiguous().cuda()
    out = rope(q, k, pos, w, w)
    clean = rope(x.cuda(), x[:, :1].contiguous().cuda(), pos, w, w)
    for y, c, r in ((out[0], clean[0], rows.cuda()), (out[1], clean[1], rows[:, :1].cuda())):
        assert (y[r] == 0).all() and torch.equal(y[~r], c[~r])
    grad = torch.randn(40, 6, D, generator=g).bfloat16().cuda()
    (dq,) = torch.autograd.grad(out[0], q, grad)
    assert (dq[rows.cuda()] == 0).all() and dq.isfinite().all()


def test_what_is_not_finite_beside_them():
    rope = QKNormRope(64)
    x = torch.full((2, 1, 64), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device="cuda")
    x[0, 0, 5], x[1, 0, 40] = float("inf"), float("nan")
    y = rope(x, None, torch.tensor([3, 4], device="cuda"))[0][:, 0]
    pair = torch.zeros(64, dtype=torch.bool, device="cuda")
    pair[[5, 37]] = True
    assert y[0][pair].isnan().all() and (y[0][~pair] == 0).all() and y[1].isnan().all()
