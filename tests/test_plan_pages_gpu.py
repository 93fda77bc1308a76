"""plan_pages against a loop over rows and tokens: whole numbers, equal."""
import pytest
import torch

import cache8_ref as ref
from attentionengine_b200 import plan_pages

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def case(B, P, seed, longest_old, longest_new, spare=0):
    g = torch.Generator().manual_seed(seed)
    old = [int(x) for x in torch.randint(0, longest_old + 1, (B,), generator=g)]
    new = [int(x) for x in torch.randint(0, longest_new + 1, (B,), generator=g)]
    need = [-(-(o + n) // P) for o, n in zip(old, new)]
    have = [-(-o // P) for o in old]
    ids = torch.randperm(sum(need) + 9, generator=g).tolist()
    table, at = [], 0
    for h in have:
        table.append(ids[at:at + h] + [-7] * (max(need) + 1 - h))
        at += h
    return old, new, table, ids[at:], sum(new) + spare


def check(old, new, table, free, head, P, T):
    dev = ints(table)
    lens, h0 = ints(old), ints([head])
    p = plan_pages(lens, ints(new), dev, ints(free), h0, P, T)
    want = ref.plan(old, new, table, free, head, P, T)
    assert p.block_table is dev and dev.tolist() == table
    for name, got in (("cu", p.cu_seqlens), ("positions", p.positions), ("slots", p.slots), ("lens", p.seq_lens), ("head", p.free_head),
                      ("segments", p.segments)):
        assert got.tolist() == want[name], name
    assert p.slots.dtype == torch.int64 and p.status.item() == 0
    assert lens.tolist() == old and h0.tolist() == [head]
    p.check()
    return p


@pytest.mark.parametrize("B,P,longest_old,longest_new,spare", [
    (1, 16, 0, 1, 0), (1, 64, 63, 130, 0), (3, 16, 40, 40, 5), (31, 1, 5, 3, 0), (255, 64, 500, 1, 0), (256, 128, 500, 1, 3),
    (257, 32, 70, 70, 0), (700, 16, 100, 9, 1000), (4096, 64, 300, 2, 0), (5, 16, 20, 9000, 0)])
def test_plan(B, P, longest_old, longest_new, spare):
    check(*case(B, P, B + P, longest_old, longest_new, spare)[:4], 0, P, sum(case(B, P, B + P, longest_old, longest_new)[1]) + spare)


@pytest.mark.parametrize("old,new,head", [
    ([0], [0], 0),                    # nothing comes
    ([16, 32, 0], [1, 0, 16], 2),     # a full page goes on in a new one, an empty row takes exactly one
    ([15, 15], [1, 2], 1),            # the page's last slot
    ([0, 0, 0, 7], [0, 0, 0, 1], 0),  # rows without tokens in front of the one that has them
])
def test_edges(old, new, head):
    P = 16
    table = [[100 * b + i for i in range(-(-o // P))] + [-7] * (6 - -(-o // P)) for b, o in enumerate(old)]
    check(old, new, table, list(range(900, 920)), head, P, sum(new))


def test_the_same_call_again_gives_the_same():
    old, new, table, free, T = case(40, 16, 5, 90, 90)
    dev = ints(table)
    a = plan_pages(ints(old), ints(new), dev, ints(free), ints([0]), 16, T)
    first = [t.clone() for t in a]
    b = plan_pages(ints(old), ints(new), dev, ints(free), ints([0]), 16, T)
    assert all(torch.equal(x, y) for x, y in zip(first, b))


def test_steps_go_on_from_one_another():
    """Three steps, each from the plan of the one before; a table that is a slice of a wider one."""
    P, free = 16, list(range(50, 90))
    wide = ints([[-7] * 40 for _ in range(3)])
    table, lens, head = [[-7] * 20 for _ in range(3)], [0, 0, 0], 0
    t_lens, t_head = ints(lens), ints([0])
    for new in ([20, 0, 33], [1, 1, 1], [12, 300, 0]):
        p = plan_pages(t_lens, ints(new), wide[:, 10:30], ints(free), t_head, P, sum(new))
        want = ref.plan(lens, new, table, free, head, P, sum(new))
        assert wide[:, 10:30].tolist() == table and p.slots.tolist() == want["slots"] and p.segments.tolist() == want["segments"]
        t_lens, t_head, lens, head = p.seq_lens, p.free_head, want["lens"], want["head"][0]
    assert (wide[:, :10] == -7).all() and (wide[:, 30:] == -7).all()


@pytest.mark.parametrize("what,code", [("free", 1), ("table", 2), ("tokens", 4), ("negative", 8)])
def test_what_does_not_fit_is_reported_and_left_out(what, code):
    P, old, new = 16, [5, 0, 16], [20, 40, 2]
    free, cols, T = list(range(60, 80)), 8, sum(new)
    if what == "free":
        free = free[:3]  # the rows need 1 + 3 + 1
    elif what == "table":
        cols = 2
    elif what == "tokens":
        T = 30
    else:
        old = [-3, 0, 16]
    table = ints([[100 * b + i if i < -(-o // P) else -7 for i in range(cols)] for b, o in enumerate(old)])
    guard = torch.cat([table, torch.full((3, 4), -9, dtype=torch.int32, device="cuda")], 1)
    p = plan_pages(ints(old), ints(new), guard[:, :cols], ints(free), ints([0]), P, T)
    assert p.status.item() == code and (guard[:, cols:] == -9).all()
    with pytest.raises(ValueError, match="plan_pages"):
        p.check()
    slots, seg = p.slots.tolist(), [s for s in p.segments.tolist() if s[3]]
    if what == "free":
        assert slots[-2:] == [-1, -1] and slots[52:60] == [-1] * 8 and p.free_head.item() == 3  # the last pages of rows 1 and 2
        assert sum(s[3] for s in seg) == 62 - 10
    elif what == "table":
        assert slots[20 + 32:20 + 40] == [-1] * 8 and min(slots[:52] + slots[60:]) >= 0
    elif what == "tokens":
        assert p.cu_seqlens.tolist() == [0, 20, 30, 30] and p.seq_lens.tolist() == [25, 10, 16] and min(slots) >= 0
    else:
        assert p.seq_lens.tolist() == [20, 40, 18] and p.positions.tolist()[:20] == list(range(20))


def test_refusals():
    ok = dict(old_lens=ints([3]), new_lens=ints([1]), block_table=ints([[0]]), free_pages=ints([1]), free_head=ints([0]), page_size=16,
              n_tokens=1)
    plan_pages(**ok).check()
    for change, err in (({"page_size": 24}, ValueError), ({"page_size": 0}, ValueError), ({"page_size": 16.0}, TypeError),
                        ({"n_tokens": -1}, ValueError), ({"new_lens": ints([1, 1])}, ValueError),
                        ({"old_lens": ints([3]).long()}, ValueError), ({"block_table": ints([0])}, ValueError),
                        ({"free_head": ints([0, 0])}, ValueError), ({"free_pages": ints([[1]])}, ValueError),
                        ({"old_lens": torch.zeros(5000, dtype=torch.int32, device="cuda")}, ValueError),
                        ({"block_table": ints([[0], [1]]).t()[:, ::2]}, None)):
        if err is None:
            plan_pages(**{**ok, **change})
        else:
            with pytest.raises(err):
                plan_pages(**{**ok, **change})
