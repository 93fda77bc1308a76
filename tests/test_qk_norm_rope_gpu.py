"""QKNormRope against 64 bits: forward, gradients (the formula's and differences), layouts, positions, refusals.

Bounds, from the arithmetic: a value of the output is two products of three fp32 factors each, times the norm's factor.  The norm's factor is off by at most
(D + 4) 2^-24 for the sum of D squares one after the other (16 in a row, then a tree: 22 2^-24), half of that behind the root, and 2^-22 for
rsqrtf; cos and sin by 2^-22 (a rounding of the angle, 2^-24 of half a turn at most, and the function's own 2 units): under 2^-20 of the magnitudes together.  A gradient is
two such steps and a mean of D values: under 2^-18.  A weight's sum has at most 512 values in a row for a thread at these sizes: 2^-14."""
import pytest
import torch

import rope_ref as ref
from attentionengine_b200 import QKNormRope, examples, plan_pages
from attentionengine_b200 import runtime as rt

pytestmark = pytest.mark.gpu
FWD, BWD, SUM = 2.0 ** -20, 2.0 ** -18, 2.0 ** -14


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


CASES = [  # tokens (packed T or (B, S)), Hq, Hkv, D, R, interleaved, norm, dtype, weight
    (1, 1, 1, 128, 128, False, True, torch.bfloat16, torch.bfloat16),
    (1, 32, 8, 128, 128, False, True, torch.bfloat16, torch.float32),
    (7, 5, 1, 64, 64, True, True, torch.float16, torch.float16),
    (33, 40, 8, 128, 64, False, True, torch.float16, torch.float32),
    (130, 3, 2, 64, 16, True, True, torch.bfloat16, None),
    (19, 9, 3, 32, 32, False, True, torch.bfloat16, torch.float32),
    (6, 2, 2, 256, 256, False, True, torch.float16, torch.float32),
    (5, 6, 6, 256, 144, True, True, torch.bfloat16, torch.bfloat16),
    (21, 128, 1, 64, 64, True, False, torch.bfloat16, None),
    (11, 4, 4, 128, 128, False, False, torch.float16, None),
    (11, 7, 1, 32, 16, True, False, torch.float16, None),
    ((3, 111), 12, 4, 64, 64, False, True, torch.float16, torch.float16),
    ((2, 300), 8, 2, 128, 128, False, True, torch.bfloat16, torch.float32),
    ((1, 1000), 16, 16, 64, 32, True, True, torch.bfloat16, torch.float32),
]


def make(case, seed=0, far=200000):
    tokens, Hq, Hkv, D, R, inter, norm, dtype, wt = case
    g = gen(seed)
    lead = (tokens,) if isinstance(tokens, int) else tokens
    rope = QKNormRope(D, rotary_dim=R, base=1e6, interleaved=inter, norm=norm)
    q, k = randn(g, *lead, Hq, D, dtype=dtype), randn(g, *lead, Hkv, D, dtype=dtype)
    pos = torch.randint(0, far, lead, generator=g).cuda()
    w = [None if wt is None else (1 + 0.3 * randn(g, D)).to(wt) for _ in "qk"]
    grads = [randn(g, *lead, h, D, dtype=dtype) for h in (Hq, Hkv)]
    return rope, q, k, pos, w, grads, (R, inter, norm)


@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case):
    rope, q, k, pos, w, grads, (R, inter, norm) = make(case)
    leaves = [t.requires_grad_() for t in (q, k, *w) if t is not None]
    out = rope(q, k, pos, *w)
    got = torch.autograd.grad(out, leaves, grads)
    again = torch.autograd.grad(rope(q, k, pos.int(), *w), leaves, grads)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for i, x in enumerate((q, k)):
        assert out[i].dtype == x.dtype and out[i].is_contiguous() and out[i].shape == x.shape
        y, size = ref.forward(x, w[i], pos, rope.inv_freq, R, inter, norm, 1e-6)
        ref.close(out[i], y, size, FWD)
        dx, dx_size, dw, dw_size = ref.backward(x, w[i], pos, rope.inv_freq, R, inter, norm, 1e-6, grads[i])
        ref.close(got[i], dx, dx_size, BWD)
        if w[i] is not None:
            assert got[2 + i].dtype == w[i].dtype
            ref.close(got[2 + i], dw, dw_size, SUM)


def test_gradients_against_differences():
    """(loss(x + h d) - loss(x - h d)) / 2 h of the 64-bit forward for a random direction, against the kernels' gradients.  The difference's own error is h^2 / 6
    of a third derivative of order one: 1e-6 of the gradient's size; the kernels' are rounded to fp16: 2^-11 of each value, in quadrature well below 1e-3 of their norm."""
    rope, q, k, pos, w, grads, (R, inter, norm) = make((40, 4, 2, 64, 64, False, True, torch.float16, torch.float32), seed=5)
    leaves = [t.requires_grad_() for t in (q, k, *w)]
    got = torch.autograd.grad(rope(q, k, pos, *w), leaves, grads)
    base = [t.detach().double().cpu() for t in leaves]

    def loss(v):
        return sum((ref.forward(v[i], v[2 + i], pos, rope.inv_freq, R, inter, norm, 1e-6)[0] * grads[i].double().cpu()).sum() for i in range(2))

    g, h = gen(9), 1e-4
    for i in range(4):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        ends = [loss([b + s * h * d if j == i else b for j, b in enumerate(base)]) for s in (1, -1)]
        want = (ends[0] - ends[1]) / (2 * h)
        here = (got[i].double().cpu() * d).sum()
        assert abs(here - want) <= 1e-3 * got[i].double().norm().cpu() * 2, (i, here, want)


@pytest.mark.parametrize("pos", [0, 1, 2 ** 20 - 1, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 40 + 12345, 2 ** 62])
def test_far_positions(pos):
    """Any position: the angle modulo a turn from whole numbers (frequencies that are binary fractions of a turn times 2 pi are not floats, so the reference reduces
    p f exactly with the same rational 2 pi)."""
    from fractions import Fraction
    import math
    from attentionengine_b200.attn_engine.rotary import _PI
    rope = QKNormRope(64, base=1e4, norm=False)
    x = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    got = rope(x, None, torch.tensor([pos], device="cuda"))[0].double().cpu().flatten()
    for i, f in enumerate(rope.inv_freq):
        t = Fraction(pos) * Fraction(f) / (2 * _PI)
        a = float((t - math.floor(t)) * 2 * _PI)
        # the frequency is held to 2^-65 of a turn
        off = 2 * math.pi * min(1.0, pos * 2.0 ** -65) + 2.0 ** -20
        for v, want in ((got[i], math.cos(a) - math.sin(a)), (got[32 + i], math.cos(a) + math.sin(a))):
            assert abs(v - want) <= 2 * off + 2.0 ** -11 * abs(want), (i, v, want)


def test_layouts():
    """Views of a joint projection, transposed heads, positions of one row for all, [1, S], strided positions, fewer dims, k left out."""
    g = gen(3)
    rope = QKNormRope(64)
    w = [1 + 0.2 * randn(g, 64) for _ in "qk"]
    qkv = randn(g, 2, 50, 4 + 2 * 2, 64, dtype=torch.bfloat16)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    pos = torch.arange(7, 57, device="cuda")
    want = rope(q.contiguous(), k.contiguous(), pos.expand(2, 50).contiguous(), *w)
    turned = qkv.transpose(1, 2).contiguous().transpose(1, 2)  # [B, H, S, D] in memory
    for a, b, p in ((q, k, pos), (q, k, pos[None]), (q, k, pos.int()), (turned[:, :, :4], turned[:, :, 4:6], pos),
                    (q, k, pos.repeat_interleave(2)[::2])):
        got = rope(a, b, p, *w)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    flat = rope(q.flatten(0, 1), k.flatten(0, 1), pos.repeat(2), *w)
    assert all(torch.equal(x, y.flatten(0, 1)) for x, y in zip(flat, want))
    alone = rope(q, None, pos, w[0])
    assert torch.equal(alone[0], want[0]) and alone[1] is None
    assert torch.equal(rope(k, None, pos, w[1])[0], want[1])
    one = rope(q, k, pos, w[0], None)
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], rope(q, k, pos, None, torch.ones(64, device="cuda"))[1])


def test_gradients_of_views_and_of_one_output():
    """A leaf that both are views of; a gradient that is expanded, transposed or missing; k without a gradient; weights alone."""
    g = gen(4)
    rope = QKNormRope(64, interleaved=True)
    qkv = randn(g, 30, 6, 64, dtype=torch.float16)
    w = [1 + 0.2 * randn(g, 64) for _ in "qk"]
    pos = torch.arange(30, device="cuda")
    gq = randn(g, 30, 4, 64, dtype=torch.float16)
    q, k = qkv[:, :4].contiguous().requires_grad_(), qkv[:, 4:5].contiguous().requires_grad_()
    want = torch.autograd.grad(rope(q, k, pos, *w)[0], (q, k), gq)
    assert (want[1] == 0).all()
    leaf = qkv.clone().requires_grad_()
    rope(leaf[:, :4], leaf[:, 4:5], pos, *w)[0].backward(gq)
    assert torch.equal(leaf.grad[:, :4], want[0]) and (leaf.grad[:, 4:] == 0).all()
    other = gq.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(torch.autograd.grad(rope(q, k.detach(), pos, *w)[0], q, other)[0], want[0])
    odd = torch.zeros(30 * 4 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(30, 4, 64).copy_(gq)  # not at a multiple of 16 bytes
    assert torch.equal(torch.autograd.grad(rope(q, None, pos, w[0])[0], q, odd)[0], want[0])
    ones = torch.autograd.grad(rope(q, k, pos, *w)[0].sum(), q)[0]
    assert torch.equal(ones, torch.autograd.grad(rope(q, k, pos, *w)[0], q, torch.ones_like(gq))[0])
    ws = [t.clone().requires_grad_() for t in w]
    dw = torch.autograd.grad(rope(q.detach(), k.detach(), pos, *ws)[0], ws, gq)
    assert torch.equal(dw[0], torch.autograd.grad(rope(q, k, pos, *ws)[0], ws[0], gq)[0]) and (dw[1] == 0).all()
    with torch.no_grad():
        assert not rope(q, k, pos, *ws)[0].requires_grad


def test_tokens_that_are_none():
    """Negative positions: zeros whatever stands there, no gradient, nothing in the weights' sums."""
    g = gen(6)
    rope = QKNormRope(128)
    q, k = randn(g, 9, 4, 128, dtype=torch.bfloat16), randn(g, 9, 1, 128, dtype=torch.bfloat16)
    w = [(1 + 0.2 * randn(g, 128)).requires_grad_() for _ in "qk"]
    pos = torch.tensor([5, 0, 3, -1, 9, 9, 2, -1, -7], dtype=torch.int32, device="cuda")
    keep = pos >= 0
    q[~keep] = float("nan")
    k[~keep] = float("inf")
    q.requires_grad_(), k.requires_grad_()
    grads = [randn(g, 9, h, 128, dtype=torch.bfloat16) for h in (4, 1)]
    out = rope(q, k, pos, *w)
    got = torch.autograd.grad(out, (q, k, *w), grads)
    few = [t.detach()[keep].requires_grad_() for t in (q, k)]
    want_out = rope(*few, pos[keep], *w)
    want = torch.autograd.grad(want_out, (*few, *w), [t[keep] for t in grads])
    for i in range(2):
        assert (out[i][~keep] == 0).all() and torch.equal(out[i][keep], want_out[i])
        assert (got[i][~keep] == 0).all() and torch.equal(got[i][keep], want[i])
        ref.close(got[2 + i], want[2 + i].double().cpu(), want[2 + i].double().cpu().abs() + 1, SUM)


def test_rows_of_zeros_and_what_is_not_finite():
    rope = QKNormRope(64, eps=1e-6)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    x[1, 0, 3], x[2, 1, 5] = float("inf"), float("nan")
    y = rope(x, None, torch.arange(3, device="cuda"))[0]
    assert (y[0] == 0).all() and (y[1, 1] == 0).all() and (y[2, 0] == 0).all() and y[2, 1].isnan().all() and not y[1, 0].isfinite().all()
    none = QKNormRope(64, eps=0.0)
    v = torch.ones(5, 3, 64, dtype=torch.bfloat16, device="cuda").requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    out = none(v, None, torch.zeros(5, dtype=torch.int32, device="cuda"), w)[0]
    dv, dw = torch.autograd.grad(out, (v, w), torch.ones_like(out))
    assert (out == 1).all() and (dw == 15).all() and (dv == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_dims_that_are_not_rotated_keep_to_themselves(interleaved, norm):
    """An infinity or NaN in one of them reaches no other dim, forward or backward, but through the norm's factor (which it makes 0 or NaN)."""
    g = gen(15)
    rope = QKNormRope(128, rotary_dim=64, interleaved=interleaved, norm=norm)
    pos = torch.arange(6, device="cuda")
    for bad in (float("inf"), float("nan")):
        x, grad = randn(g, 6, 3, 128, dtype=torch.float16), randn(g, 6, 3, 128, dtype=torch.float16)
        clean = rope(x, None, pos)[0]
        for d in (64, 71, 72, 80, 127):
            y = x.clone()
            y[2, 1, d] = bad
            out = rope(y, None, pos)[0]
            rest = torch.arange(128, device="cuda") != d
            assert not out[2, 1, d].isfinite()
            want = clean[2, 1] if not norm else torch.zeros_like(clean[2, 1]) if bad == float("inf") else torch.full_like(clean[2, 1], bad)
            assert torch.equal(out[2, 1][rest].nan_to_num(7.0), want[rest].nan_to_num(7.0))
            out[2, 1] = clean[2, 1]
            assert torch.equal(out, clean)
            if not norm:
                leaf, gr = x.clone().requires_grad_(), grad.clone()
                gr[2, 1, d] = bad
                got, fine = (torch.autograd.grad(rope(leaf, None, pos)[0], leaf, t)[0] for t in (gr, grad))
                assert not got[2, 1, d].isfinite() and torch.equal(got[2, 1][rest], fine[2, 1][rest])


def test_nothing_to_do():
    rope = QKNormRope(64)
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    out = rope(q, q[:, :1], torch.zeros(0, dtype=torch.int32, device="cuda"), w, w)
    dq, dw = torch.autograd.grad(out, (q, w), [torch.zeros_like(t) for t in out])
    assert out[0].shape == (0, 4, 64) and out[1].shape == (0, 1, 64) and dq.shape == q.shape and (dw == 0).all()
    assert rope(torch.zeros(0, 5, 2, 64, dtype=torch.float16, device="cuda"), None, torch.arange(5, device="cuda"))[0].shape == (0, 5, 2, 64)


def test_scaled_frequencies_and_rotary_scale():
    g = gen(8)
    f = torch.rand(16, generator=g, dtype=torch.float32)
    q, pos = randn(g, 20, 3, 64, dtype=torch.float16), torch.randint(0, 100000, (20,), generator=g).cuda()
    rope = QKNormRope(64, rotary_dim=32, inv_freq=f, rotary_scale=1.25, norm=False)
    y, size = ref.forward(q, None, pos, [float(x) for x in f], 32, False, False, 0.0, m=1.25)
    ref.close(rope(q, None, pos)[0], y, size, FWD)
    leaf = q.clone().requires_grad_()
    gr = randn(g, 20, 3, 64, dtype=torch.float16)
    dx, dx_size, _, _ = ref.backward(q, None, pos, [float(x) for x in f], 32, False, False, 0.0, gr, m=1.25)
    ref.close(torch.autograd.grad(rope(leaf, None, pos)[0], leaf, gr)[0], dx, dx_size, BWD)


def test_second_derivatives_are_refused_when_asked_for():
    rope = QKNormRope(64)
    q = torch.randn(3, 2, 64, device="cuda").half().requires_grad_()
    out = rope(q, None, torch.arange(3, device="cuda"))[0]
    (dq,) = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    assert dq.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        dq.float().sum().backward()


def test_saved_inputs_that_change_are_noticed():
    rope = QKNormRope(64)
    q = torch.randn(3, 2, 64, device="cuda").half()
    w = torch.ones(64, device="cuda", requires_grad=True)
    out = rope(q, None, torch.arange(3, device="cuda"), w)[0]
    q.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_streams_and_graphs():
    """A side stream; a captured forward and backward, replayed on new values, beside eager calls."""
    g = gen(12)
    rope = QKNormRope(128, base=5e5)
    q, k = randn(g, 70, 8, 128, dtype=torch.bfloat16), randn(g, 70, 2, 128, dtype=torch.bfloat16)
    w = [(1 + 0.2 * randn(g, 128)) for _ in "qk"]
    pos = torch.arange(70, dtype=torch.int32, device="cuda")
    grads = [randn(g, 70, h, 128, dtype=torch.bfloat16) for h in (8, 2)]

    def step(q, k, w, pos):
        leaves = [t.detach().requires_grad_() for t in (q, k, *w)]
        out = rope(leaves[0], leaves[1], pos, *leaves[2:])
        return [*out, *torch.autograd.grad(out, leaves, grads)]

    want = step(q, k, w, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(q, k, w, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, k, w, pos)
    for seed in (1, 2):
        h = gen(seed)
        q.copy_(randn(h, 70, 8, 128)), k.copy_(randn(h, 70, 2, 128)), pos.copy_(torch.randint(0, 9999, (70,), generator=h))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step(q, k, w, pos)))


def test_positions_of_a_plan():
    """plan_pages' positions as they are: int32, -1 behind the last token."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    plan = plan_pages(i32(3, 20), i32(2, 1), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32(*range(9)), i32(0), 16, 5)
    rope = QKNormRope(64)
    q = torch.randn(5, 4, 64, device="cuda").half()
    out = rope(q, q[:, :2], plan.positions)[0]
    assert torch.equal(out[:3], rope(q[:3], None, i32(3, 4, 20))[0]) and (out[3:] == 0).all()


def test_in_front_of_attention():
    """Gradients through rotation and attention together, against the same chain in 64 bits: 1e-2 of the gradient's norm holds the roundings of a bf16 chain of six
    stages (2^-9 rms each against the norm) with room, and a wrong term does not pass it."""
    g = gen(20)
    B, S, Hq, Hkv, D = 1, 200, 4, 2, 64
    rope, eng = QKNormRope(D, base=1e4), examples.softmax_engine(B, Hq, Hkv, S, D, D, torch.bfloat16, True)
    q, k, v = (randn(g, B, S, h, D, dtype=torch.bfloat16).requires_grad_() for h in (Hq, Hkv, Hkv))
    w = [(1 + 0.2 * randn(g, D)).requires_grad_() for _ in "qk"]
    pos, d_o = torch.arange(S, device="cuda"), randn(g, B, S, Hq, D, dtype=torch.bfloat16)
    rq, rk = rope(q, k, pos, *w)
    got = torch.autograd.grad(eng(rq, rk, v), (q, k, v, *w), d_o)
    leaves = [t.detach().double().cpu().requires_grad_() for t in (q, k, v, *w)]
    angle = pos.cpu().double()[:, None] * torch.tensor(rope.inv_freq, dtype=torch.float64)

    def plain(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = x.chunk(2, -1)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    pq, pk = plain(leaves[0], leaves[3]), plain(leaves[1], leaves[4])
    s = torch.einsum("bihd,bjhd->bhij", pq, pk.repeat_interleave(2, 2)) / 8.0
    p = torch.softmax(s.masked_fill(~torch.ones(S, S, dtype=torch.bool).tril(), -torch.inf), -1)
    o = torch.einsum("bhij,bjhd->bihd", p, leaves[2].repeat_interleave(2, 2))
    want = torch.autograd.grad(o, leaves, d_o.double().cpu())
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).norm() <= 1e-2 * b.norm()


def test_refusals():
    rope, plain = QKNormRope(64), QKNormRope(64, norm=False)
    q, k = torch.zeros(2, 5, 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 5, 2, 64, dtype=torch.float16, device="cuda")
    pos, w = torch.arange(5, device="cuda"), torch.ones(64, device="cuda")
    ok = dict(q=q, k=k, positions=pos, q_weight=w, k_weight=w)
    rope(**ok)
    for change, err in (({"q": q.float()}, TypeError), ({"k": k.bfloat16()}, TypeError), ({"k": k[:1]}, ValueError), ({"k": k[:, :4]}, ValueError),
                        ({"q": q[..., :32]}, ValueError), ({"q": q.transpose(2, 3)}, ValueError), ({"k": k[0]}, ValueError),
                        ({"q": torch.zeros(2, 5, 4, 72, dtype=torch.float16, device="cuda")[..., 4:68]}, ValueError),
                        ({"q": torch.zeros(2, 5, 4, 68, dtype=torch.float16, device="cuda")[..., :64]}, ValueError),
                        ({"positions": pos.float()}, TypeError), ({"positions": pos[:4]}, ValueError), ({"positions": pos.expand(3, 5)}, ValueError),
                        ({"positions": pos.cpu()}, rt.AeError), ({"q_weight": w.half()}, TypeError), ({"q_weight": w.bfloat16(), "k_weight": w.bfloat16()}, TypeError),
                        ({"q_weight": w[:32]}, ValueError), ({"k_weight": torch.ones(65, device="cuda")[1:]}, ValueError), ({"k": None}, ValueError),
                        ({"q_weight": w.expand(1, 64)}, ValueError), ({"q": q[:, :, :0]}, ValueError)):
        with pytest.raises(err):
            rope(**{**ok, **change})
    with pytest.raises(ValueError, match="norm=False"):
        plain(q, k, pos, w)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError):
        rope(fwd.make_dual(q, q), k, pos)


@pytest.mark.parametrize("inter", [False, True])
def test_offsets_beyond_32_bits(inter):
    """The last of 4.6 GB of heads: as in a call of their own."""
    rope = QKNormRope(256, interleaved=inter)
    T, last = 70001, 37
    q = torch.zeros(T, 128, 256, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(T, 1, 256, dtype=torch.bfloat16, device="cuda")
    gq, gk = torch.zeros_like(q), torch.zeros_like(k)
    g = gen(31)
    for t in (q, k, gq, gk):
        t[-last:] = randn(g, last, *t.shape[1:], dtype=torch.bfloat16)
    pos = torch.arange(T, device="cuda")
    own = [t[-last:].clone().requires_grad_() for t in (q, k)]
    want = rope(*own, pos[-last:])
    dwant = torch.autograd.grad(want, own, [gq[-last:], gk[-last:]])
    leaves = [t.requires_grad_() for t in (q, k)]
    out = rope(*leaves, pos)
    for a, b in zip(out, want):
        assert torch.equal(a[-last:], b) and not a[:-last].any()
    got = torch.autograd.grad(out, leaves, [gq, gk])
    for a, b in zip(got, dwant):
        assert torch.equal(a[-last:], b) and not a[:-last].any()
