"""Forks in pools whose free pages do not last: pages that the step itself gives back are handed out behind them, and only then do rows end early."""
import random

import pytest
import torch

from attentionengine_b200 import QKNormRope, copy_pages, examples, plan_forks
from attentionengine_b200 import runtime as rt
from test_pages_gpu import ints

pytestmark = pytest.mark.gpu


def forks(parents, lens, table, free, head, P, keep=None):
    """As pages_ref.forks, for pools of any fill: (block_table, seq_lens, free_pages, free_head, copies, status)."""
    B, W = len(lens), len(table[0])
    n = [0 if p < 0 else lens[p] if keep is None else keep[i] for i, p in enumerate(parents)]
    whole, begun = set(), {}
    for i, p in enumerate(parents):
        whole |= {table[p][c] for c in range(n[i] // P)}
    for i, p in sorted(enumerate(parents), key=lambda x: (x[1] != x[0], x[0])):
        if n[i] % P:
            begun.setdefault(table[p][n[i] // P], i)
    held = {table[i][c] for i in range(B) for c in range(-(-lens[i] // P))}
    back = sorted(held - whole - set(begun))
    out, copies, status, free = [], [], 0, list(free)
    for i, p in enumerate(parents):
        row = [table[p][c] for c in range(n[i] // P)]
        if n[i] % P:
            page = table[p][n[i] // P]
            if page in whole or begun[page] != i:
                new = None
                if head < len(free):
                    new, head = free[head], head + 1
                elif back:
                    new = back.pop(0)
                if new is None:
                    n[i], status = n[i] // P * P, 1
                else:
                    copies.append([page, new, n[i] % P, 0])
                    row.append(new)
            else:
                row.append(page)
        out.append(row + [0] * (W - len(row)))
    if len(back) > head:
        back, status = back[:head], status | 4
    head -= len(back)
    free[head:head + len(back)] = back
    return out, n, free, [head], copies + [[0] * 4] * (B - len(copies)), status


@pytest.mark.parametrize("B,P,longest,cols,seed", [
    (2, 16, 60, 0, 0), (8, 16, 300, 0, 1), (40, 64, 900, 0, 2), (200, 16, 200, 0, 3), (1024, 16, 90, 0, 4), (1500, 16, 60, 0, 5), (4096, 32, 100, 0, 6),
    (300, 16, 100, 60, 7), (64, 128, 20000, 0, 8)])
@pytest.mark.parametrize("spare", [0, 1, 3, 0.1, 1.5])
def test_pages_that_a_step_gives_back_serve_it(B, P, longest, cols, seed, spare):
    """Both forms of the planner; `spare` free pages, or a share of the rows.  Some steps fit by what they give back, some do not."""
    rng = random.Random(seed)
    lens = [rng.randrange(1, longest + 1) for _ in range(B)]
    need = [-(-n // P) for n in lens]
    N = sum(need) + (spare if isinstance(spare, int) else int(spare * B))
    ids, at, table, W = rng.sample(range(N), N), 0, [], max(max(need), cols)
    for k in need:
        table.append(ids[at:at + k] + [-9] * (W - k))
        at += k
    for kind in range(3):
        if kind == 0:  # beams of four
            parents = [i - i % 4 + rng.randrange(min(4, B - (i - i % 4))) for i in range(B)]
        else:
            parents = [rng.choice((-1, i, rng.randrange(B), rng.randrange(B))) for i in range(B)]
        keep = [0 if p < 0 else rng.randrange(lens[p] + 1) for p in parents] if kind == 2 else None
        args = [ints(parents), ints(lens), ints(table), ints(ids), ints([at])]
        got = plan_forks(*args, P, N, keep_lens=None if keep is None else ints(keep))
        want = forks(parents, lens, table, ids, at, P, keep)
        for name, w in zip(("block_table", "seq_lens", "free_pages", "free_head", "copies"), want):
            assert getattr(got, name).tolist() == w, name
        assert got.status.item() == want[5]
        rows = [row[:-(-n // P)] for row, n in zip(want[0], want[1])]
        held = {p for row in rows for p in row}
        assert held | set(want[2][want[3][0]:]) == set(range(N)) and len(held) + N - want[3][0] == N  # each page in a row or free, none lost
        if want[5] == 0:
            data = torch.randn(N, P, 3, device="cuda")
            first = data.clone()
            copy_pages([data], got.copies)
            for i in range(0, B, max(1, B // 50)):
                if want[1][i]:
                    old = table[parents[i]][:len(rows[i])]
                    assert torch.equal(data[rows[i]].flatten(0, 1)[:want[1][i]], first[old].flatten(0, 1)[:want[1][i]])


def test_a_step_without_any_free_page():
    """Two rows change their last tokens, the third ends: its pages are the ones that the copies go to, in both forms."""
    P = 16
    for cols in (4, 3000):
        assert rt.lib().ae_plan_lists_phases(3, cols, 8) == (cols > 4)
        table = [row + [0] * (cols - 4) for row in ([6, 2, 0, 0], [4, 0, 0, 0], [7, 5, 3, 0])]
        p = plan_forks(ints([0, 0, 0]), ints([20, 5, 40]), ints(table), ints([6, 2, 4, 7, 5, 3]), ints([6]), P, 8)
        p.check()
        assert p.block_table[:, :3].tolist() == [[6, 2, 0], [6, 3, 0], [6, 4, 0]] and p.seq_lens.tolist() == [20, 20, 20]
        assert p.copies.tolist() == [[2, 3, 4, 0], [2, 4, 4, 0], [0] * 4]
        assert p.free_head.item() == 4 and p.free_pages.tolist() == [6, 2, 4, 7, 5, 7]


def test_more_pages_back_than_taken_and_none_on_the_list():
    """A list without entries: copies take what comes back, the rest has no room (status 4)."""
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    p = plan_forks(ints([0, 0]), ints([20, 40]), ints([[6, 2, 0], [7, 5, 3]]), empty, ints([0]), 16, 8)
    assert p.status.item() == 4 and p.block_table.tolist() == [[6, 2, 0], [6, 3, 0]] and p.seq_lens.tolist() == [20, 20]
    assert p.copies.tolist() == [[2, 3, 4, 0], [0] * 4] and p.free_head.item() == 0


def test_beams_of_a_full_pool():
    """A server whose pool has no page left goes on from one of its rows: no token is lost."""
    serve = examples.PagedLayers(2, 2, 1, 64, torch.float16, 4, 12, 16, 64, rope=QKNormRope(64))
    x = [tuple(torch.randn(4 * 40, h, 64, device="cuda").half() for h in (2, 1, 1)) for _ in range(2)]
    serve.prompts(x, ints([40] * 4))
    assert serve.head.item() == 12
    old = [[c.k.view(torch.uint8)[serve.table[1, :3].long()].flatten(0, 1)[:40] for c in serve.caches], [c.k_scale[serve.table[1, :3].long()] for c in serve.caches]]
    serve.fork(ints([1, 1, 1, 1]))
    serve.check()
    assert serve.lens.tolist() == [40] * 4 and serve.head.item() == 6
    for row in serve.table[:, :3].long():
        for c, codes, scales in zip(serve.caches, *old):
            assert torch.equal(c.k.view(torch.uint8)[row].flatten(0, 1)[:40], codes) and torch.equal(c.k_scale[row], scales)
    token = [tuple(torch.randn(4, h, 64, device="cuda").half() for h in (2, 1, 1)) for _ in range(2)]
    serve.tokens(token)
    serve.check()
