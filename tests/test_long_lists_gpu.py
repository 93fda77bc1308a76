"""Lists of more entries than one step of a search takes, with the data that they copy; compactions of pages that rows hold to different lengths.  Whole numbers and
bytes, equal."""
import random

import pytest
import torch

import pages_ref as ref
from attentionengine_b200 import copy_pages, plan_compaction, plan_forks
from attentionengine_b200 import runtime as rt
from test_pages_gpu import ints

pytestmark = pytest.mark.gpu


def copied(t, copies):
    """`t` after the entries (page, new page, slots, 0), a tensor on the CPU."""
    t = t.clone()
    src, dst, n, _ = copies.unbind(1)
    keep = (torch.arange(t.shape[1]) < n[:, None]).view(-1, t.shape[1], *[1] * (t.dim() - 2))
    t[dst] = torch.where(keep, t[src], t[dst])
    return t


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 255, 256, 257, 511, 512, 513, 3000])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("behind", [0, 1, 300])
def test_where_a_list_ends(n, heads_first, behind):
    """n entries, one without slots, and `behind` more that have some; without one (0) the list ends with its tensor."""
    g = torch.Generator().manual_seed(n + behind)
    P, pages = 8, 2 * (n + behind + 1)
    data = torch.randint(-2 ** 15, 2 ** 15, (pages, P, 3, 8), generator=g, dtype=torch.int16)
    ids, slots = torch.randperm(pages, generator=g), torch.randint(1, P + 1, (n + behind + 1,), generator=g)
    copies = torch.stack([ids[0::2], ids[1::2], slots, torch.zeros_like(slots)], 1)
    copies[n, 2] = -1 if n % 2 else 0
    listed = copies if behind else copies[:n]
    pool = data.cuda()
    if heads_first:
        pool = pool.transpose(1, 2).contiguous().transpose(1, 2)
    copy_pages([pool], listed.int().cuda())
    assert torch.equal(pool.cpu(), copied(data, copies[:n]))


def test_samples_of_one_prompt():
    """600 rows with one parent: every one reads its tokens, from whole pages that all share and a begun one of its own."""
    B, W, P, n = 600, 5, 16, 5 * 16 - 3
    N = B * W + 700
    ids = torch.randperm(N, generator=torch.Generator().manual_seed(1))
    table, lens = ids[:B * W].view(B, W).int().cuda(), torch.full((B,), n, dtype=torch.int32, device="cuda")
    data = torch.randn(N, P, 2, 6, device="cuda")
    want = data[table[77].long()].flatten(0, 1)[:n]
    p = plan_forks(torch.full_like(lens, 77), lens, table, ids.int().cuda(), ints([B * W]), P, N)
    copy_pages([data], p.copies)
    p.check()
    rows = p.block_table.long()
    assert (p.copies[:, 2] > 0).sum() == B - 1 and rows[:, -1].unique().numel() == B and (rows[:, :-1] == table[77, :-1].long()).all()
    assert torch.equal(data[rows].flatten(1, 2)[:, :n], want.expand(B, *want.shape))


@pytest.mark.parametrize("pages,rows,longest", [(9000, 200, 500), (40000, 300, 1500)])
def test_a_compaction_s_moves(pages, rows, longest):
    """Thousands of moves, and what every row reads behind them."""
    rng, P = random.Random(pages), 16
    lens = [rng.randrange(longest + 1) for _ in range(rows)]
    need = [-(-n // P) for n in lens]
    ids, at, table = rng.sample(range(pages), sum(need)), 0, []
    for k in need:
        table.append(ids[at:at + k] + [0] * (max(need) - k))
        at += k
    data = torch.randint(-2 ** 31, 2 ** 31, (pages, P, 3), generator=torch.Generator().manual_seed(2)).int()
    pool = data.cuda()
    c = plan_compaction(ints(lens), ints(table), P, pages)
    copy_pages([pool], c.copies)
    c.check()
    want = ref.compaction(lens, table, P, pages)
    moves = torch.tensor([e for e in want["copies"] if e[2]])
    assert len(moves) > 2000 and c.copies.tolist() == want["copies"] and c.block_table.tolist() == want["block_table"]
    assert torch.equal(pool.cpu(), copied(data, moves))


@pytest.mark.parametrize("pages,launches", [(60, 0), (16000, 0), (20000, 1)])
def test_compaction_of_pages_held_to_different_lengths(pages, launches):
    """A page that one row has begun and another holds whole, or that two have begun: all of its slots that some row reads go along.  Pages with nothing that
    anybody reads behind a row's length stay out of it."""
    P = 16
    far = [pages - 1 - i for i in range(12)]
    lens = [20, 32, 20, 17, 5, 11, 16, 3, 0, 16]
    table = [[far[0], far[1], -9], [far[0], far[1], 3],     # begun in the first, whole in the second
             [far[2], far[3], 1], [far[2], far[3], far[11]],  # begun in both, to 4 and to 1
             [far[4], -9, -9], [far[4], 2, 2],              # begun in both, the longer one behind
             [far[5], 0, 0], [far[5], -9, -9],              # whole, then begun
             [far[6], far[7], 0],                           # nothing
             [2, far[8], far[9]]]                           # stays where it is
    assert rt.lib().ae_plan_lists_phases(len(lens), 3, pages) == launches
    c = plan_compaction(ints(lens), ints(table), P, pages)
    c.check()
    want = ref.compaction(lens, table, P, pages)
    for name, w in want.items():
        assert getattr(c, name).tolist() == w, name
    moved = {e[0]: e[2] for e in want["copies"] if e[2]}
    assert moved == {far[0]: 16, far[1]: 16, far[2]: 16, far[3]: 4, far[4]: 11, far[5]: 16}
    data = torch.randn(pages, P, 4, device="cuda")
    first = data.clone()
    copy_pages([data], c.copies)
    for old, new, n in zip(table, c.block_table.tolist(), lens):
        k = -(-n // P)
        assert torch.equal(data[new[:k]].flatten(0, 1)[:n], first[old[:k]].flatten(0, 1)[:n])
