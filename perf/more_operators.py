"""Norm and rotation of query and key heads, and the pages of a cache that is forked, freed and compacted, as cases that can be timed.

A case names one of five operators and its sizes:

* ``rope``: queries and keys normed head by head and rotated by their positions, in one pass (``QKNormRope``)
* ``train``: the same with the gradients of queries, keys and both weights
* ``fork``: the pages of a step in which rows go on from others, are cut or end (``plan_forks``)
* ``compact``: every page in use moved to the front of the pool (``plan_compaction``)
* ``copy``: the pages that such plans name, in the caches of several layers (``copy_pages``)

``own`` false: the operators in elementary torch operations, in 32 bits (angles in 64), rounded once at the end; true: the framework's
calls.  Lengths follow from the case alone; values are made on the GPU from the seed.
"""
import functools
import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_DEV = "cuda"
_E4M3 = torch.float8_e4m3fn
_EPS = 1e-6
_KEPT, _OLD, _NEVER = 0, 2 ** 31 - 2, 2 ** 31 - 1  # what the plain fork notes of a page


def listed():
    return [
        # a decode step: one token for each of 64 requests, far into their contexts, heads as the projection left them
        dict(name="rope_step_64", op="rope", rows=64, new=1, old=100000, Hq=32, Hkv=8, D=128, R=128, base=1e6, norm=True, pairs="half", dtype="bf16",
             weight="bf16", packed=True, mix=1),
        # prompts behind each other, on their way into packed attention
        dict(name="rope_prompts_16k", op="rope", rows=8, new=4096, old=0, Hq=32, Hkv=8, D=128, R=128, base=1e6, norm=True, pairs="half", dtype="bf16",
             weight="bf16", packed=True, mix=13),
        # a padded batch of small heads, neighbouring pairs, half of the dims rotated
        dict(name="rope_batch_d64", op="rope", rows=3, new=1111, old=0, Hq=16, Hkv=16, D=64, R=32, base=1e4, norm=True, pairs="next", dtype="fp16",
             weight="fp32", packed=False, mix=3),
        # no norm: the rotary part of 128 heads of a latent-cache model, one token for each request
        dict(name="rope_pe_128", op="rope", rows=128, new=1, old=8192, Hq=128, Hkv=1, D=64, R=64, base=1e4, norm=False, pairs="next", dtype="bf16",
             weight="bf16", packed=True, mix=4),
        # training at the sizes of the framework's benchmark, two of its eight sequences
        dict(name="train_gqa_8k", op="train", rows=2, new=8192, old=0, Hq=32, Hkv=8, D=128, R=128, base=1e6, norm=True, pairs="half", dtype="bf16",
             weight="fp32", packed=False, mix=5),
        # a small training step of odd sizes
        dict(name="train_odd_1001", op="train", rows=3, new=1001, old=0, Hq=12, Hkv=4, D=64, R=64, base=1e4, norm=True, pairs="half", dtype="fp16",
             weight="fp16", packed=False, mix=6),
        # beams: 8 requests of four rows each, every row goes on from one of the four
        dict(name="fork_beams_32", op="fork", rows=32, longest=1500, page=16, group=4, kind="beams", mix=7),
        # a server's batch: some rows end, new ones take over the prompt of another
        dict(name="fork_server_512", op="fork", rows=512, longest=16384, page=64, group=4, kind="server", mix=8),
        # a pool of half-empty rows closes its gaps
        dict(name="compact_48", op="compact", rows=48, longest=2000, page=64, spare=0.6, mix=9),
        # a large pool of small pages
        dict(name="compact_60k", op="compact", rows=300, longest=9000, page=16, spare=0.4, mix=10),
        # the begun pages of 96 forked rows, in the caches of eight layers
        dict(name="copy_tails_96", op="copy", n=96, layers=8, page=64, Hkv=8, D=128, whole=False, mix=11),
        # a compaction's moves, four layers
        dict(name="copy_moves_1500", op="copy", n=1500, layers=4, page=64, Hkv=8, D=128, whole=True, mix=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, mix = rng.choice(("rope", "rope", "train", "fork", "compact", "copy")), rng.randrange(1 << 20)
    page = rng.choice((16, 32, 64, 128))
    if op in ("rope", "train"):
        D = rng.choice((64, 128, 128))
        Hkv, G = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 5, 8))
        c = dict(op=op, old=rng.choice((0, _log_int(rng, 1, 500000))), Hq=min(40, Hkv * G), Hkv=Hkv, D=D, R=rng.choice((D, D, D // 2, 16)),
                 base=rng.choice((1e4, 5e5, 1e6)), norm=rng.random() < 0.8, pairs=rng.choice(("half", "next")), dtype=rng.choice(("fp16", "bf16")),
                 mix=mix)
        c["weight"] = rng.choice((c["dtype"], "fp32"))
        if op == "rope" and rng.random() < 0.4:
            return dict(c, rows=_log_int(rng, 1, 300), new=1, packed=True)
        new = _log_int(rng, 1, 8000)
        return dict(c, rows=_log_int(rng, 1, max(1, 16000 // new)), new=new, packed=op == "rope" and rng.random() < 0.6)
    if op == "fork":
        longest = _log_int(rng, 20, 16384)
        rows = _log_int(rng, 1, max(1, min(512, 2 ** 18 // (longest // page + 1))))
        return dict(op=op, rows=rows, longest=longest, page=page, group=rng.choice((1, 2, 4, 8)), kind=rng.choice(("beams", "server")), mix=mix)
    if op == "compact":
        longest = _log_int(rng, 20, 16384)
        rows = _log_int(rng, 1, max(1, min(300, 2 ** 17 // (longest // page + 1))))
        return dict(op=op, rows=rows, longest=longest, page=page, spare=round(rng.uniform(0.05, 0.8), 2), mix=mix)
    Hkv, D, layers = rng.choice((1, 2, 4, 8, 12)), rng.choice((64, 128)), rng.choice((1, 2, 5, 8))
    return dict(op=op, n=_log_int(rng, 1, min(1500, 2 ** 29 // (2 * page * Hkv * D * layers))), layers=layers, page=page, Hkv=Hkv, D=D,
                whole=rng.random() < 0.5, mix=mix)


# ---------------------------------------------------------------------------------------------------- sizes
@functools.lru_cache(maxsize=64)
def _spread(n, most, mix):
    """n lengths of 1 to `most`, the first of them `most`: as in earnest, many short ones and a few long ones."""
    rng = random.Random(mix)
    out = [max(1, int(most * rng.random() ** 2)) for _ in range(n)]
    out[0] = most
    return tuple(out)


def _tokens(c):
    if c["packed"]:
        return sum(_spread(c["rows"], c["new"], c["mix"])) if c["new"] > 1 else c["rows"]
    return c["rows"] * c["new"]


def _pages(n, page):
    return -(-n // page)


def _copy_slots(c):
    rng = random.Random(c["mix"])
    return [c["page"] if c["whole"] and i % 16 else rng.randrange(1, c["page"] + (c["page"] == 1)) for i in range(c["n"])]


@functools.lru_cache(maxsize=16)
def _fork_case(rows, longest, page, group, kind, mix):
    """(lengths, whole pages that row i has in common with the first of its group, parents, kept lengths)."""
    rng = random.Random(mix)
    lens = list(_spread(rows, longest, mix + 1))
    shared = [0] * rows
    for i in range(rows):
        first = i - i % group
        if i != first:
            if kind == "beams":  # of one length, all but the last pages in common
                lens[i] = lens[first]
                shared[i] = max(0, lens[first] // page - rng.randrange(3))
            else:
                shared[i] = min(lens[i], lens[first]) // page // 2
    if kind == "beams":
        parents = [i - i % group + rng.randrange(min(group, rows - (i - i % group))) for i in range(rows)]
        keep = [lens[p] for p in parents]
    else:  # a tenth of the rows end, a tenth become another row's prompt
        parents, keep = [], []
        for i in range(rows):
            u = rng.random()
            p = -1 if u < 0.1 else rng.randrange(rows) if u < 0.2 else i
            parents.append(p)
            keep.append(0 if p < 0 else lens[p] if p == i else rng.randrange(lens[p] + 1))
    return lens, shared, parents, keep


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=_DEV).manual_seed(seed * 16 + salt)


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=_DEV, dtype=torch.float32).to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=_DEV)


def _frequencies(c):
    return [c["base"] ** (-2.0 * i / c["R"]) for i in range(c["R"] // 2)]


def prepare(case, seed):
    return {"rope": _prepare_rope, "train": _prepare_rope, "fork": _prepare_fork, "compact": _prepare_compact, "copy": _prepare_copy}[case["op"]](case, seed)


def _prepare_rope(c, seed):
    g, rng, s = _gen(seed, 1), random.Random(seed), {"case": c}
    dtype, Hq, Hkv, D = _DTYPES[c["dtype"]], c["Hq"], c["Hkv"], c["D"]
    if c["packed"]:
        lens = list(_spread(c["rows"], c["new"], c["mix"])) if c["new"] > 1 else [1] * c["rows"]
        rng.shuffle(lens)
        old = [rng.randrange(c["old"] + 1) for _ in lens]
        s["positions"] = torch.cat([torch.arange(o, o + n, dtype=torch.int32) for o, n in zip(old, lens)]).to(_DEV)
        # heads as they come out of the projection of queries, keys and values
        qkv = _normal(g, (sum(lens), Hq + 2 * Hkv, D), dtype)
        s["q"], s["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
    else:
        B, S = c["rows"], c["new"]
        s["positions"] = _ints([[o + i for i in range(S)] for o in (rng.randrange(c["old"] + 1) for _ in range(B))])
        s["q"], s["k"] = _normal(g, (B, S, Hq, D), dtype), _normal(g, (B, S, Hkv, D), dtype)
    s["wq"], s["wk"] = ((1 + 0.2 * _normal(g, (D,))).to(_DTYPES[c["weight"]]) if c["norm"] else None for _ in "qk")
    if c["op"] == "train":
        s["gq"], s["gk"] = _normal(g, s["q"].shape, dtype), _normal(g, s["k"].shape, dtype)
        s["leaves"] = [t for t in (s["q"], s["k"], s["wq"], s["wk"]) if t is not None]
        for t in s["leaves"]:
            t.requires_grad_()
    s["frequencies"] = torch.tensor(_frequencies(c), dtype=torch.float64, device=_DEV)
    if own:
        s["rope"] = _rope(D, c["R"], c["base"], c["pairs"], c["norm"])
    return s


@functools.lru_cache(maxsize=None)
def _rope(D, R, base, pairs, norm):
    import attentionengine_b200 as ae
    return ae.QKNormRope(D, rotary_dim=R, base=base, interleaved=pairs == "next", norm=norm, eps=_EPS)


def _prepare_fork(c, seed):
    rng, page = random.Random(seed), c["page"]
    lens, shared, parents, keep = _fork_case(c["rows"], c["longest"], page, c["group"], c["kind"], c["mix"])
    need = [_pages(n, page) - s for n, s in zip(lens, shared)]
    used, spare = sum(need), c["rows"] + 5
    ids = list(range(used + spare))
    rng.shuffle(ids)
    wide = max(_pages(n, page) for n in lens) + 1
    table, at = [], 0
    for i, (n, sh) in enumerate(zip(need, shared)):
        own_pages = ids[at:at + n]
        at += n
        row = (table[i - i % c["group"]][:sh] if sh else []) + own_pages
        table.append(row + [0] * (wide - len(row)))
    free = ids  # a pool in use: what has been taken stands in front of what is free
    return {"case": c, "parents": _ints(parents), "keep": _ints(keep), "lens": _ints(lens), "table": _ints(table), "free": _ints(free),
            "head": _ints([used]), "page": page, "pages": used + spare}


def _prepare_compact(c, seed):
    rng, page = random.Random(seed), c["page"]
    lens = list(_spread(c["rows"], c["longest"], c["mix"]))
    need = [_pages(n, page) for n in lens]
    pages = sum(need) + max(1, int(sum(need) * c["spare"]))
    ids = rng.sample(range(pages), sum(need))
    wide, table, at = max(need), [], 0
    for n in need:
        table.append(ids[at:at + n] + [0] * (wide - n))
        at += n
    return {"case": c, "lens": _ints(lens), "table": _ints(table), "page": page, "pages": pages}


def _prepare_copy(c, seed):
    g, rng = _gen(seed, 2), random.Random(seed)
    slots = _copy_slots(c)
    pages = 2 * c["n"] + 3
    ids = list(range(pages))
    rng.shuffle(ids)
    s = {"case": c, "copies": _ints([[ids[2 * i], ids[2 * i + 1], n, 0] for i, n in enumerate(slots)]), "layers": []}
    for _ in range(c["layers"]):
        pools = []
        for _ in "kv":
            codes = torch.randint(0, 256, (pages, c["page"], c["Hkv"], c["D"]), generator=g, device=_DEV, dtype=torch.uint8)
            codes[(codes & 127) == 127] = 8  # no NaN
            pools.append(codes.view(_E4M3))
        scales = [torch.exp2(torch.randint(-9, 3, (pages, c["Hkv"]), generator=g, device=_DEV).float()) for _ in "kv"]
        s["layers"].append((*pools, *scales))
    if own:
        import attentionengine_b200 as ae
        s["caches"] = [ae.PagedCache8.from_tensors(*t) for t in s["layers"]]
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"rope": _run_rope, "train": _run_train, "fork": _run_fork, "compact": _run_compact, "copy": _run_copy}[state["case"]["op"]](state)


def _run_rope(s):
    if own:
        return s["rope"](s["q"], s["k"], s["positions"], s["wq"], s["wk"])
    cos, sin = _cos_sin(s)
    return _plain_rope(s["q"], s["wq"], cos, sin, s["case"]), _plain_rope(s["k"], s["wk"], cos, sin, s["case"])


def _cos_sin(s):
    angle = (s["positions"].double()[..., None] * s["frequencies"])[..., None, :]  # [..., 1, R / 2]
    return angle.cos().float(), angle.sin().float()


def _plain_rope(x, w, cos, sin, c):
    z, R = x.float(), c["R"]
    if c["norm"]:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + _EPS) * w.float()
    if c["pairs"] == "half":
        a, b = z[..., :R // 2], z[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = z[..., 0:R:2], z[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, z[..., R:]], -1).to(x.dtype)


def _run_train(s):
    if own:
        q, k = s["rope"](s["q"], s["k"], s["positions"], s["wq"], s["wk"])
    else:
        cos, sin = _cos_sin(s)
        q, k = _plain_rope(s["q"], s["wq"], cos, sin, s["case"]), _plain_rope(s["k"], s["wk"], cos, sin, s["case"])
    grads = torch.autograd.grad((q, k), s["leaves"], (s["gq"], s["gk"]))
    return [q.detach(), k.detach(), *grads]


def _run_fork(s):
    if own:
        from attentionengine_b200 import plan_forks
        p = plan_forks(s["parents"], s["lens"], s["table"], s["free"], s["head"], s["page"], s["pages"], keep_lens=s["keep"])
        return {"table": p.block_table, "lens": p.seq_lens, "free": p.free_pages, "head": p.free_head, "copies": p.copies}
    P, N, table = s["page"], s["pages"], s["table"].long()
    B, wide = table.shape
    lens, col, row = s["lens"].long(), torch.arange(wide, device=_DEV), torch.arange(B, device=_DEV)
    parent = s["parents"].long()
    goes_on, p = parent >= 0, parent.clamp(min=0)
    n = torch.where(goes_on, torch.minimum(s["keep"].long(), lens[p]), 0)
    whole, part = n.div(P, rounding_mode="floor"), n % P
    pages = table[p]
    last = pages.gather(1, whole.clamp(max=wide - 1)[:, None])[:, 0]
    key = 1 + row + torch.where(parent == row, 0, B)  # a row that goes on from itself first, then the lowest
    # what the rows hold: before, in part, whole; page N takes what is not there
    note = torch.full((N + 1,), _NEVER, dtype=torch.int64, device=_DEV)
    note[torch.where(col < (lens + P - 1).div(P, rounding_mode="floor")[:, None], table, N)] = _OLD
    note.scatter_reduce_(0, torch.where(part > 0, last, N), key, "amin")
    note[torch.where(col < whole[:, None], pages, N)] = _KEPT
    copy = (part > 0) & (note[last] != key)
    order = copy.long().cumsum(0) - 1
    head, taken = s["head"].long(), copy.sum()
    fresh = s["free"].long()[(head + order).clamp(0, s["free"].numel() - 1)]
    at_last = (col == whole[:, None]) & (part > 0)[:, None]
    out = torch.where(col < whole[:, None], pages, torch.where(at_last, torch.where(copy, fresh, last)[:, None], 0))
    copies = torch.zeros(B + 1, 4, dtype=torch.int64, device=_DEV)
    copies[torch.where(copy, order, B)] = torch.stack([last, fresh, part, torch.zeros_like(part)], 1)
    freed = note[:N] == _OLD
    top = head + taken - freed.sum()
    free = torch.cat([s["free"], s["free"][:1]])
    free[torch.where(freed, top + freed.long().cumsum(0) - 1, s["free"].numel())] = torch.arange(N, dtype=torch.int32, device=_DEV)
    return {"table": out.int(), "lens": n.int(), "free": free[:-1], "head": top.int(), "copies": copies[:B].int()}


def _run_compact(s):
    if own:
        from attentionengine_b200 import plan_compaction
        p = plan_compaction(s["lens"], s["table"], s["page"], s["pages"])
        return {"table": p.block_table, "free": p.free_pages, "head": p.free_head, "copies": p.copies}
    P, N, table = s["page"], s["pages"], s["table"].long()
    lens, col = s["lens"].long()[:, None], torch.arange(table.shape[1], device=_DEV)
    there = col * P < lens
    slots = torch.zeros(N + 1, dtype=torch.int64, device=_DEV)
    slots.scatter_reduce_(0, torch.where(there, table, N).flatten(), (lens - col * P).clamp(0, P).flatten(), "amax")
    slots = slots[:N]
    used, page = slots > 0, torch.arange(N, device=_DEV)
    in_use = used.sum()
    moves, holes = used & (page >= in_use), ~used & (page < in_use)
    room = N // 2
    copies = torch.zeros(room + 1, 4, dtype=torch.int64, device=_DEV)
    number, hole = moves.long().cumsum(0) - 1, holes.long().cumsum(0) - 1
    copies[torch.where(moves, number, room), 0] = page
    copies[torch.where(holes, hole, room), 1] = page
    copies[torch.where(moves, number, room), 2] = slots
    to = torch.where(moves, copies[:, 1][number.clamp(0, room)], page)
    return {"table": torch.where(there, to[table], 0).int(), "free": torch.arange(N, dtype=torch.int32, device=_DEV), "head": in_use.int()[None],
            "copies": copies[:room].int()}


def _run_copy(s):
    if own:
        from attentionengine_b200 import copy_pages
        copy_pages(s["caches"], s["copies"])
        return s["layers"]
    src, dst, n, _ = s["copies"].long().unbind(1)
    keep = (torch.arange(s["case"]["page"], device=_DEV) < n[:, None])[..., None, None]
    for layer in s["layers"]:
        for codes in (t.view(torch.uint8) for t in layer[:2]):
            codes[dst] = torch.where(keep, codes[src], codes[dst])
        for scales in layer[2:]:
            scales[dst] = scales[src]
    return s["layers"]


# ---------------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    c = case
    if c["op"] in ("rope", "train"):
        T = _tokens(c)
        values, weights = T * (c["Hq"] + c["Hkv"]) * c["D"], 2 * c["D"] * (4 if c["weight"] == "fp32" else 2) * c["norm"]
        if c["op"] == "rope":
            return {"bytes": 4 * values + 4 * T + weights, "flops": 7 * values}
        return {"bytes": 8 * values + 4 * T + 2 * weights, "flops": 22 * values}  # values and gradients read, both written
    P = c.get("page")
    if c["op"] == "fork":
        lens, shared, parents, keep = _fork_case(c["rows"], c["longest"], P, c["group"], c["kind"], c["mix"])
        wide = max(_pages(n, P) for n in lens) + 1
        pages = sum(_pages(n, P) - s for n, s in zip(lens, shared)) + c["rows"] + 5
        # entries in use and the whole new table, four numbers a row, the free list in and out, a copy a row
        return {"bytes": 4 * sum(_pages(n, P) for n in lens) + 4 * c["rows"] * wide + 16 * c["rows"] + 8 * pages + 16 * c["rows"], "flops": 0}
    if c["op"] == "compact":
        need = [_pages(n, P) for n in _spread(c["rows"], c["longest"], c["mix"])]
        pages = sum(need) + max(1, int(sum(need) * c["spare"]))
        return {"bytes": 4 * sum(need) + 4 * c["rows"] * max(need) + 4 * c["rows"] + 4 * pages + 16 * (pages // 2), "flops": 0}
    return {"bytes": c["layers"] * 2 * 2 * (sum(_copy_slots(c)) * c["Hkv"] * c["D"] + 4 * c["n"] * c["Hkv"]) + 16 * c["n"], "flops": 0}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Heads as complex numbers, turned by unit numbers; pools page by page; None where the outputs are whole numbers."""
    c = case
    if c["op"] in ("fork", "compact"):
        return None
    s = prepare(c, seed)
    if c["op"] == "copy":
        for src, dst, n, _ in s["copies"].tolist():
            for layer in s["layers"]:
                for t in layer:
                    t[dst][:n if t.dim() == 4 else None].view(torch.uint8).copy_(t[src][:n if t.dim() == 4 else None].view(torch.uint8))
        return s["layers"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=_DEV), s["positions"].double()[..., None, None] * s["frequencies"])
    out, grads, weights = [], [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        x = x.detach().double()
        length = torch.sqrt(x.square().sum(-1, keepdim=True) / c["D"] + _EPS) if c["norm"] else torch.ones((), dtype=torch.float64, device=_DEV)
        n = x / length
        z = n * w.detach().double() if c["norm"] else n
        out.append(_as_real(_as_complex(z, c) * turn, z, c))
        if c["op"] == "train":
            g = g.double()
            dz = _as_real(_as_complex(g, c) * turn.conj(), g, c)
            if c["norm"]:
                weights.append((dz * n).flatten(0, -2).sum(0))
                dz = dz * w.detach().double()
                dz = (dz - n * (dz * n).mean(-1, keepdim=True)) / length
            grads.append(dz)
    return [*out, *grads, *weights] if c["op"] == "train" else tuple(out)


def _as_complex(z, c):
    h = c["R"] // 2
    return torch.complex(z[..., :h].contiguous(), z[..., h:2 * h].contiguous()) if c["pairs"] == "half" else torch.view_as_complex(
        z[..., :2 * h].unflatten(-1, (h, 2)).contiguous())


def _as_real(u, z, c):
    out, h = z.clone(), c["R"] // 2
    if c["pairs"] == "half":
        out[..., :h], out[..., h:2 * h] = u.real, u.imag
    else:
        out[..., 0:2 * h:2], out[..., 1:2 * h:2] = u.real, u.imag
    return out
