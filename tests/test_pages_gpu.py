"""plan_forks, plan_compaction and copy_pages against loops over rows and pages: whole numbers and bytes, equal."""
import random

import pytest
import torch

import pages_ref as ref
from attentionengine_b200 import PagedCache8, copy_pages, examples, plan_compaction, plan_forks, plan_pages
from attentionengine_b200 import runtime as rt

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(rng, lens, P, spare, groups=0, extra_cols=1):
    """A pool in use: (table, free list, head, pages); with `groups` rows have whole pages in common with the first of their group."""
    need = [-(-n // P) for n in lens]
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    W, table, at = max(need) + extra_cols, [], 0
    for i, n in enumerate(need):
        first = i - i % groups if groups else i
        common = rng.randrange(min(lens[i], lens[first]) // P + 1) if first != i else 0
        row = (table[first][:common] if common else []) + ids[at:at + n - common]
        at += n - common
        table.append(row + [-9] * (W - n))
    return table, ids, at, len(ids)


def check_forks(parents, lens, table, free, head, P, N, keep=None):
    args = [ints(parents), ints(lens), ints(table), ints(free), ints([head])]
    before = [t.clone() for t in args]
    p = plan_forks(*args, P, N, keep_lens=None if keep is None else ints(keep))
    want = ref.forks(parents, lens, table, free, head, P, keep)
    p.check()
    for name, w in want.items():
        assert getattr(p, name).tolist() == w, name
    assert all(torch.equal(a, b) for a, b in zip(args, before))
    return p


@pytest.mark.parametrize("B,P,longest,groups,seed", [
    (1, 16, 40, 0, 0), (2, 1, 9, 0, 1), (3, 64, 64, 0, 2), (8, 16, 300, 4, 3), (33, 16, 90, 2, 4), (64, 128, 5000, 8, 5), (257, 32, 400, 4, 6),
    (513, 64, 700, 3, 7), (1500, 16, 50, 5, 8), (4096, 16, 33, 2, 9), (5, 16, 20000, 0, 10)])
@pytest.mark.parametrize("kind", ["any", "keep", "same", "end", "one"])
def test_forks(B, P, longest, groups, seed, kind):
    rng = random.Random(seed)
    lens = [rng.randrange(longest + 1) for _ in range(B)]
    if kind == "one":  # a prompt is sampled B times
        parents, keep = [rng.randrange(B)] * B, None
    elif kind == "same":
        parents, keep = list(range(B)), None
    elif kind == "end":
        parents, keep = [-1 if rng.random() < 0.7 else i for i in range(B)], None
    else:
        parents = [rng.choice((-1, i, i, rng.randrange(B))) for i in range(B)]
        keep = [0 if p < 0 else rng.randrange(lens[p] + 1) for p in parents] if kind == "keep" else None
    table, free, head, N = pool(rng, lens, P, B + 3, groups)
    check_forks(parents, lens, table, free, head, P, N, keep)


@pytest.mark.parametrize("parents,lens,keep", [
    ([0], [0], None), ([-1], [17], None), ([0], [17], [16]), ([0], [32], [17]), ([0], [16], [0]),
    ([1, 0], [5, 40], None),              # two rows change places
    ([0, 0], [40, 3], [40, 35]),          # a whole page for one row, a begun one for the other
    ([0, 0, 0], [40, 0, 0], [35, 33, 40]),  # three ways to hold one page
    ([1, 1, 1], [0, 37, 0], [36, 34, 36]),  # the row itself is the last to keep it, and keeps it
    ([1, 2, 0], [16, 32, 48], None), ([0, 0], [16, 16], None), ([-1, 0], [37, 0], None)])
def test_edges(parents, lens, keep):
    P, at, table = 16, 0, []
    for n in lens:
        need = -(-n // P)
        table.append(list(range(at, at + need)) + [-9] * (5 - need))
        at += need
    check_forks(parents, lens, table, list(range(at + 6)), at, P, at + 6, keep)


def test_steps_that_go_on_from_one_another():
    """Forks, ends and cuts in a row, with plan_pages between them; every page is either in a row or free, and never in both."""
    rng, P, B, N = random.Random(3), 16, 12, 200
    lens, table, free, head = ints([0] * B), ints([[0] * 30 for _ in range(B)]), ints(rng.sample(range(N), N)), ints([0])
    for step in range(12):
        new = [rng.randrange(40) if rng.random() < 0.6 else 0 for _ in range(B)]
        plan = plan_pages(lens, ints(new), table, free, head, P, sum(new))
        plan.check()
        lens, head = plan.seq_lens, plan.free_head
        L = lens.tolist()
        parents = [rng.choice((-1, i, i, i, rng.randrange(B))) for i in range(B)]
        keep = [0 if p < 0 else L[p] if rng.random() < 0.7 else rng.randrange(L[p] + 1) for p in parents]
        fork = check_forks(parents, L, table.tolist(), free.tolist(), head.item(), P, N, keep)
        table, lens, free, head = fork.block_table, fork.seq_lens, fork.free_pages, fork.free_head
        held = {p for row, n in zip(table.tolist(), lens.tolist()) for p in row[:-(-n // P)]}
        assert held | set(free.tolist()[head.item():]) == set(range(N)) and len(held) + N - head.item() == N
        begun = [row[n // P] for row, n in zip(table.tolist(), lens.tolist()) if n % P]
        assert len(set(begun)) == len(begun)  # what is written next is nobody else's


@pytest.mark.parametrize("what,code", [("free", 1), ("table", 2), ("back", 4), ("parent", 8), ("keep", 8), ("negative", 8), ("page", 16), ("list", 16)])
def test_what_does_not_fit_is_reported_and_left_out(what, code):
    P, N = 16, 40
    parents, lens, keep = [0, 0, 0, 3], [20, 0, 0, 16], [20, 20, 18, 16]
    table, free, head = [[5, 6, 0, 0], [0] * 4, [0] * 4, [7, 0, 0, 0]], [5, 6, 7, 30, 31, 32], 3
    if what == "free":
        free = free[:4]
    elif what == "table":
        lens[0] = keep[0] = 70
        table[0] = [5, 6, 8, 9]
        keep[0] = 64
    elif what == "back":
        parents[3], head, free = -1, 0, [30, 31]
        parents[0] = parents[1] = parents[2] = -1
    elif what == "parent":
        parents[3] = 9
    elif what == "keep":
        keep[3] = 17
    elif what == "negative":
        lens[1] = -4
    elif what == "page":
        table[3][0] = 99
    else:
        free[3] = 77
    guard = torch.full((4, 8), -9, dtype=torch.int32, device="cuda")
    guard[:, :4] = ints(table)
    p = plan_forks(ints(parents), ints(lens), guard[:, :4], ints(free), ints([head]), P, N, keep_lens=ints(keep))
    assert p.status.item() == code
    with pytest.raises(ValueError, match="plan_forks"):
        p.check()
    out, n = p.block_table.tolist(), p.seq_lens.tolist()
    if what == "free":
        assert out == [[5, 6, 0, 0], [5, 30, 0, 0], [5, 0, 0, 0], [7, 0, 0, 0]] and n == [20, 20, 16, 16]
        assert p.copies.tolist() == [[6, 30, 4, 0]] + [[0] * 4] * 3 and p.free_head.item() == 4
    elif what == "table":
        assert n[0] == 64 and out[0] == [5, 6, 8, 9]
    elif what == "back":
        assert n == [0] * 4 and p.free_head.item() == 0 and p.free_pages.tolist() == [30, 31]
    elif what == "parent":
        assert n[3] == 0 and p.free_pages.tolist()[p.free_head.item()] == 7
    elif what == "keep":
        assert n[3] == 16
    elif what == "negative":
        assert n == [20, 20, 18, 16]
    elif what == "page":
        assert out[3][0] == 99 and n[3] == 16
    else:  # the free list names a page outside the pool: that row ends with its whole pages, the next one takes the next page
        assert out == [[5, 6, 0, 0], [5, 0, 0, 0], [5, 31, 0, 0], [7, 0, 0, 0]] and n == [20, 16, 18, 16]
        assert p.copies.tolist() == [[6, 6, 4, 0], [6, 31, 2, 0]] + [[0] * 4] * 2


@pytest.mark.parametrize("B,P,longest,spare,groups,seed", [
    (1, 16, 1, 0, 0, 0), (1, 16, 40, 5, 0, 1), (2, 1, 30, 40, 0, 2), (9, 64, 900, 33, 3, 3), (64, 16, 200, 1000, 0, 4), (300, 32, 3000, 9000, 4, 5),
    (4096, 16, 20, 100, 0, 6), (5000, 16, 20, 100, 2, 7), (3, 128, 100000, 3, 0, 8)])
def test_compaction(B, P, longest, spare, groups, seed):
    rng = random.Random(seed)
    lens = [rng.randrange(longest + 1) for _ in range(B)]
    table, ids, _, N = pool(rng, lens, P, spare, groups)
    t, n = ints(table), ints(lens)
    p = plan_compaction(n, t, P, N)
    p.check()
    for name, w in ref.compaction(lens, table, P, N).items():
        assert getattr(p, name).tolist() == w, name
    assert t.tolist() == table and n.tolist() == lens


@pytest.mark.parametrize("B,W,N", [(1, 8, 5001), (7, 13, 20), (40, 300, 9000), (3, 2, 20000), (2000, 3, 64)])
def test_compaction_of_rows_without_tokens(B, W, N):
    dirt = torch.full((1 << 18,), 0x7f7f7f7f, dtype=torch.int32, device="cuda")  # what a plan's memory may hold before it
    del dirt
    c = plan_compaction(ints([0] * B), torch.full((B, W), -9, dtype=torch.int32, device="cuda"), 16, N)
    c.check()
    for name, w in ref.compaction([0] * B, [[-9] * W] * B, 16, N).items():
        assert getattr(c, name).tolist() == w, name


def test_compaction_reports():
    for lens, table, code in (([-1, 3], [[0], [1]], 8), ([17, 3], [[0], [1]], 2), ([3, 3], [[9], [1]], 16), ([3, 3], [[-1], [1]], 16)):
        p = plan_compaction(ints(lens), ints(table), 16, 4)
        assert p.status.item() == code
        with pytest.raises(ValueError, match="plan_compaction"):
            p.check()
    assert p.block_table.tolist() == [[-1], [0]]


def test_a_pool_of_one_page():
    p = plan_compaction(ints([3]), ints([[0]]), 16, 1)
    assert p.copies.shape == (0, 4) and p.free_head.item() == 1
    copy_pages(torch.zeros(1, 16, 4, device="cuda"), p.copies)


def plain_copy(t, copies, per_page=False):
    for src, dst, n, _ in copies:
        if per_page:
            t[dst] = t[src]
        else:
            t[dst, :n] = t[src, :n]


POOLS = {  # [pages, slots, ...] tensors of 24 pages of 16 slots
    "codes": lambda: torch.randint(0, 256, (24, 16, 8, 128), dtype=torch.uint8, device="cuda"),
    "halves": lambda: torch.randn(24, 16, 2, 64, device="cuda").half(),
    "latent": lambda: torch.randn(24, 16, 1, 576, device="cuda").bfloat16(),
    "heads first": lambda: torch.randn(24, 4, 16, 64, device="cuda").half().transpose(1, 2),
    "some heads": lambda: torch.randn(24, 16, 6, 64, device="cuda").half()[:, :, 1:4],
    "odd rows": lambda: torch.randn(24, 16, 3, 5, device="cuda").half(),
    "odd place": lambda: torch.randint(0, 256, (24 * 16 * 33 + 1,), dtype=torch.uint8, device="cuda")[1:].view(24, 16, 33),
    "words": lambda: torch.randn(24, 16, 7, device="cuda"),
    "one each": lambda: torch.randint(-9, 9, (24, 16), device="cuda"),
    "every other page": lambda: torch.randn(48, 16, 40, device="cuda")[::2],
    "large slots": lambda: torch.randn(24, 16, 80, 128, device="cuda"),
    "no values": lambda: torch.zeros(24, 16, 0, 4, device="cuda"),
}


@pytest.mark.parametrize("name", POOLS)
def test_copies(name):
    t = POOLS[name]()
    rng = random.Random(5)
    ids = rng.sample(range(24), 24)
    copies = [[ids[2 * i], ids[2 * i + 1], n, 0] for i, n in enumerate((16, 1, 7, 16, 15, 8, 2, 16, 9))]
    want = t.clone()
    plain_copy(want, copies)
    whole = t._base if t._base is not None else t
    outside = whole.clone()
    copy_pages(t, ints(copies + [[0] * 4] * 3 + [[ids[20], ids[21], 16, 0]]))  # behind the end of the list
    assert torch.equal(t, want)
    if t._base is not None and name in ("some heads", "every other page"):  # nothing beside the view
        cut = (slice(None), slice(None), [0, 4, 5]) if name == "some heads" else (slice(1, None, 2),)
        assert torch.equal(whole[cut], outside[cut])


def test_copies_of_many_caches():
    """More pools than a launch takes, caches and tensors mixed; scales go along; the list is on the device alone."""
    def cache(over):
        codes = [torch.randint(0, 120, (9, 32, 4, 64), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "kv"]
        scales = [torch.rand(9, 6, device="cuda")[:, 1:5] if over else torch.rand(9, 4, device="cuda") for _ in "kv"]
        return PagedCache8.from_tensors(*codes, *scales)

    pools = [cache(i % 2) if i % 3 else torch.randn(9, 32, 5, device="cuda") for i in range(70)]
    copies = [[3, 7, 32, 0], [0, 1, 5, 0], [8, 2, 31, 0]]
    want = []
    for p in pools:
        parts = [(p, False)] if isinstance(p, torch.Tensor) else [(p.k.view(torch.uint8), False), (p.v.view(torch.uint8), False), (p.k_scale, True), (p.v_scale, True)]
        for t, per_page in parts:
            w = t.clone()
            plain_copy(w, copies, per_page)
            want.append((t, w))
    copy_pages(pools, ints(copies))
    assert all(torch.equal(t, w) for t, w in want)


def test_entries_that_do_not_fit_are_passed_over():
    t = torch.randn(6, 16, 8, device="cuda")
    want = t.clone()
    want[2, :4] = want[1, :4]
    copy_pages([t], ints([[9, 0, 3, 0], [0, -1, 3, 0], [-5, 0, 3, 0], [0, 6, 16, 0], [0, 3, 17, 0], [4, 4, 9, 0], [1, 2, 4, 0]]))
    assert torch.equal(t, want)
    copy_pages([t], ints([[1, 0, -3, 0], [1, 0, 3, 0]]))  # ends the list
    assert torch.equal(t, want)
    copy_pages([t], ints([[0] * 4]))
    copy_pages([t], torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
    copy_pages([], ints([[0] * 4]))
    assert torch.equal(t, want)


def test_offsets_beyond_32_bits():
    """Pages that lie more than 4 GB into a pool."""
    t = torch.zeros(9000, 64, 8192, dtype=torch.uint8, device="cuda")
    t[8999] = torch.randint(1, 256, (64, 8192), dtype=torch.uint8, device="cuda")
    t[2] = 7
    copy_pages([t], ints([[8999, 8990, 64, 0], [2, 8500, 63, 0]]))
    assert torch.equal(t[8990], t[8999]) and (t[8500, :63] == 7).all() and (t[8500, 63] == 0).all() and (t[8501] == 0).all()


def test_the_largest_pages():
    """A byte short of the limit, and of bytes, so that a loop's last step comes as near to 2^31 as it can; one more is refused."""
    t = torch.zeros(2, 0x7fff0001, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="below 2 GB"):
        copy_pages([t], ints([[0, 1, 1, 0]]))
    for pool in (t[:, 1:], t[:, None, 1:]):
        t.zero_()
        pool[0, ..., -40000:] = 5
        n = pool.shape[1]
        copy_pages([pool], ints([[0, 1, n, 0]]))
        assert torch.equal(pool[0], pool[1]) and t[1, 0] == 0
    t.zero_()
    wide = t.view(-1)[:2 * 0x7fff0000].view(2, 0x3fff8000, 2)[:, :, :1]  # bytes that do not lie behind each other
    wide[0, -40000:] = 6
    copy_pages([wide], ints([[0, 1, wide.shape[1], 0]]))
    assert torch.equal(wide[0], wide[1]) and (t.view(-1)[:2 * 0x7fff0000].view(2, 0x3fff8000, 2)[:, :, 1] == 0).all()


def test_plans_and_copies_in_a_graph():
    """Captured once, replayed on other lengths and parents; a call on another stream beside it."""
    rng, P, N, B = random.Random(8), 16, 120, 6
    lens = [rng.randrange(100) for _ in range(B)]
    table, free, head, _ = pool(rng, lens, P, N - sum(-(-n // P) for n in lens), extra_cols=8)
    t = [ints(x) for x in ([0] * B, lens, table, free, [head])]
    data = torch.randn(N, P, 4, 8, device="cuda")
    first = data.clone()
    plan_forks(*t, P, N)
    copy_pages([data], ints([[0] * 4]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = plan_forks(*t, P, N)
        copy_pages([data], p.copies)
        c = plan_compaction(p.seq_lens, p.block_table, P, N)
        copy_pages([data], c.copies)
    for seed in range(3):
        rng = random.Random(seed)
        parents = [rng.choice((-1, i, rng.randrange(B))) for i in range(B)]
        t[0].copy_(ints(parents))
        data.copy_(first)
        graph.replay()
        want = first.clone()
        f = ref.forks(parents, lens, table, free, head, P)
        plain_copy(want, f["copies"])
        r = ref.compaction(f["seq_lens"], f["block_table"], P, N)
        plain_copy(want, r["copies"])
        assert p.block_table.tolist() == f["block_table"] and c.block_table.tolist() == r["block_table"] and torch.equal(data, want)
        for i, (row, n) in enumerate(zip(r["block_table"], f["seq_lens"])):  # every row reads its parent's tokens
            if n:
                old = first[table[parents[i]][:-(-n // P)]].flatten(0, 1)[:n]
                assert torch.equal(data[row[:-(-n // P)]].flatten(0, 1)[:n], old)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = plan_forks(*t, P, N)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_refusals():
    ok = dict(parents=ints([0, 1]), seq_lens=ints([3, 0]), block_table=ints([[0], [0]]), free_pages=ints([0, 1]), free_head=ints([1]), page_size=16, num_pages=4)
    plan_forks(**ok).check()
    for change, err in (({"page_size": 24}, ValueError), ({"page_size": True}, TypeError), ({"num_pages": 0}, ValueError), ({"num_pages": 2.0}, TypeError),
                        ({"parents": ints([0])}, ValueError), ({"parents": ints([0, 1]).long()}, ValueError), ({"keep_lens": ints([1])}, ValueError),
                        ({"block_table": ints([[0]])}, ValueError), ({"free_head": ints([0, 0])}, ValueError), ({"free_head": ints([0]).cpu()}, rt.AeError),
                        ({"seq_lens": torch.zeros(5000, dtype=torch.int32, device="cuda")}, ValueError)):
        with pytest.raises(err):
            plan_forks(**{**ok, **change})
    two = dict(seq_lens=ok["seq_lens"], block_table=ok["block_table"], page_size=16, num_pages=4)
    for change, err in (({"page_size": 0}, ValueError), ({"num_pages": -1}, ValueError), ({"block_table": ints([0, 0])}, ValueError),
                        ({"seq_lens": ints([1])}, ValueError)):
        with pytest.raises(err):
            plan_compaction(**{**two, **change})
    t, c = torch.zeros(4, 16, 8, device="cuda"), ints([[0, 1, 3, 0]])
    for pools, copies, err in (([t, t[:3]], c, ValueError), ([t.cpu()], c, rt.AeError), ([t], c.long(), ValueError), ([t], c[0], ValueError),
                               ([t], ints([[0] * 8])[:, :4].expand(2, 4), ValueError), ([t[..., ::2]], c, ValueError), ([t[0, 0]], c, ValueError),
                               ([t[:, :1].expand(4, 16, 8)], c, ValueError), ([torch.zeros(2, 16, 1, 1, 8, device="cuda")], c, ValueError),
                               ([t.clone().requires_grad_()], c, NotImplementedError), ([t], c.cpu(), rt.AeError)):
        with pytest.raises(err):
            copy_pages(pools, copies)
