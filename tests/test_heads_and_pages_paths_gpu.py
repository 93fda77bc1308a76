"""What depends on how a call is split: the forms of the planners on both sides of the rule, shares of a token's heads, offsets beyond 32 bits, calls of
two threads, and calls whose first one is captured."""
import os
import random
import subprocess
import sys
import threading

import pytest
import torch

import pages_ref as ref
import rope_ref
from attentionengine_b200 import QKNormRope, copy_pages, plan_compaction, plan_forks
from attentionengine_b200 import runtime as rt
from test_pages_gpu import check_forks, ints, pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,cols,pages,launches", [
    (1024, 8, 16384, 0), (1025, 7, 9000, 1), (64, 128, 16000, 0), (64, 129, 16000, 1), (3, 9, 16384, 0), (3, 9, 16385, 1), (1, 8192, 8300, 0), (2, 5000, 12000, 1)])
def test_both_forms_of_the_planners(B, cols, pages, launches):
    """One CTA up to 1024 rows, 16384 pages and 8192 table entries, a launch for each phase beyond."""
    assert rt.lib().ae_plan_lists_phases(B, cols, pages) == launches
    P, rng = 16, random.Random(B + cols)
    share = max(1, pages // (2 * B))
    lens = [rng.randrange(P * min(cols, share) + 1) for _ in range(B)]
    table, free, head, N = pool(rng, lens, P, 0, groups=3 if B > 2 else 0, extra_cols=0)
    table = [row + [0] * (cols - len(row)) for row in table]
    rest = list(range(N, pages))
    rng.shuffle(rest)
    parents = [rng.choice((-1, i, i, rng.randrange(B))) for i in range(B)]
    keep = [0 if p < 0 else rng.randrange(lens[p] + 1) for p in parents]
    p = check_forks(parents, lens, table, free + rest, head, P, pages, keep)
    c = plan_compaction(p.seq_lens, p.block_table, P, pages)
    c.check()
    for name, w in ref.compaction(p.seq_lens.tolist(), p.block_table.tolist(), P, pages).items():
        assert getattr(c, name).tolist() == w, name


@pytest.mark.parametrize("T,Hq,Hkv,D", [(1, 300, 20, 32), (2, 300, 1, 64), (700, 130, 6, 64), (1, 65, 65, 256), (3000, 1, 1, 128), (5, 2, 1, 256)])
def test_shares_of_heads(T, Hq, Hkv, D):
    """Few tokens of many heads, many tokens of few; each row's bits are those of the same row alone."""
    g = torch.Generator().manual_seed(T + Hq)
    rope = QKNormRope(D, base=1e5)
    q, k = (torch.randn(T, h, D, generator=g).half().cuda().requires_grad_() for h in (Hq, Hkv))
    w = [(1 + 0.2 * torch.randn(D, generator=g)).cuda().requires_grad_() for _ in "qk"]
    grads = [torch.randn(T, h, D, generator=g).half().cuda() for h in (Hq, Hkv)]
    pos = torch.randint(0, 100000, (T,), generator=g).cuda()
    out = rope(q, k, pos, *w)
    got = torch.autograd.grad(out, (q, k, *w), grads)
    for i, x in enumerate((q, k)):
        y, size = rope_ref.forward(x, w[i], pos, rope.inv_freq, D, False, True, 1e-6)
        rope_ref.close(out[i], y, size, 2.0 ** -20)
        dx, dx_size, dw, dw_size = rope_ref.backward(x, w[i], pos, rope.inv_freq, D, False, True, 1e-6, grads[i])
        rope_ref.close(got[i], dx, dx_size, 2.0 ** -18)
        rope_ref.close(got[2 + i], dw, dw_size, 2.0 ** -14)
        one = x.detach()[T // 2:T // 2 + 1, :1].contiguous().requires_grad_()
        alone = rope(one, None, pos[T // 2:T // 2 + 1], w[i])[0]
        assert torch.equal(alone[0, 0], out[i][T // 2, 0])
        assert torch.equal(torch.autograd.grad(alone, one, grads[i][T // 2:T // 2 + 1, :1])[0][0, 0], got[i][T // 2, 0])


def test_offsets_beyond_32_bits():
    """430,000 tokens of 40 heads of 128 dims: 2.2e9 values each way."""
    T, H, D = 430_000, 40, 128
    rope = QKNormRope(D)
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda").normal_().requires_grad_()
    grad = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda").normal_()
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    out = rope(q, None, pos)[0]
    (dq,) = torch.autograd.grad(out, q, grad)
    few = q.detach()[-3:].contiguous().requires_grad_()
    want = rope(few, None, pos[-3:])[0]
    assert torch.equal(out[-3:], want) and torch.equal(dq[-3:], torch.autograd.grad(want, few, grad[-3:])[0])
    few = q.detach()[:3].contiguous().requires_grad_()
    want = rope(few, None, pos[:3])[0]
    assert torch.equal(out[:3], want) and torch.equal(dq[:3], torch.autograd.grad(want, few, grad[:3])[0])


def test_two_threads():
    rope = QKNormRope(64)
    w = torch.ones(64, device="cuda")
    rng = random.Random(2)
    lens = [rng.randrange(90) for _ in range(40)]
    table, free, head, N = pool(rng, lens, 16, 60)
    args = [ints([rng.randrange(40) for _ in lens]), ints(lens), ints(table), ints(free), ints([head])]
    q = torch.randn(300, 6, 64, device="cuda").half()
    data = torch.randn(N, 16, 24, device="cuda")
    pos = torch.arange(300, device="cuda")

    def work():
        leaf, wl, mine = q.clone().requires_grad_(), w.clone().requires_grad_(), data.clone()
        out = rope(leaf, leaf[:, :2], pos, wl, wl)
        grads = torch.autograd.grad(out, (leaf, wl), [torch.ones_like(t) for t in out])
        p = plan_forks(*args, 16, N)
        copy_pages([mine], p.copies)
        c = plan_compaction(p.seq_lens, p.block_table, 16, N)
        copy_pages([mine], c.copies)
        return [*[t.detach() for t in out], *grads, *p, *c, mine]

    want, bad = work(), []
    torch.cuda.synchronize()

    def loop():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = work()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    bad.append(1)

    threads = [threading.Thread(target=loop) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


FIRST = """
import torch
from attentionengine_b200 import QKNormRope, copy_pages, plan_compaction, plan_forks
B, W, P = 600, 40, 16
i32 = dict(dtype=torch.int32, device="cuda")
table, lens, parents = torch.arange(B * W, **i32).view(B, W), torch.full((B,), W * P - 3, **i32), torch.zeros(B, **i32)
N = B * W + 700
free, head, data = torch.arange(N, **i32), torch.full((1,), B * W, **i32), torch.zeros(N, P, 4, device="cuda")
rope, q, pos = QKNormRope(64), torch.ones(50, 4, 64, device="cuda", dtype=torch.float16), torch.arange(50, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    p = plan_forks(parents, lens, table, free, head, P, N)
    copy_pages([data], p.copies)
    c = plan_compaction(p.seq_lens, p.block_table, P, N)
    y = rope(q, None, pos)[0]
graph.replay()
torch.cuda.synchronize()
assert p.status.item() == 0 and c.free_head.item() == W - 1 + B and torch.equal(y, rope(q, None, pos)[0])
print("as it should")
"""


def test_a_first_call_that_is_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300, cwd=root)
    assert out.returncode == 0 and "as it should" in out.stdout, out.stderr[-2000:]


def test_other_things_than_pools():
    for pools in ([3], ["cache"], [None], [[torch.zeros(2, 16, 4, device="cuda")]]):
        with pytest.raises(TypeError, match="pool"):
            copy_pages(pools, ints([[0, 1, 3, 0]]))
    with pytest.raises(NotImplementedError):
        QKNormRope(64.0)
