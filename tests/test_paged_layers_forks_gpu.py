"""A server's steps as they are used: prompts, forks, tokens, cuts, ends and a compaction over several layers, with normed and rotated heads, against plain attention in
64 bits over the tokens that each row has seen.

Bounds: keys and values are held in e4m3 (half a step: 2^-4 of the value; 2^-5 rms and less), so an output is off by about 2^-5 / sqrt(keys that count) of
the values' size beside the value's own rounding, and a score by 2^-5 of |q| |k| / sqrt(D).  The plain form takes the codes as the cache rounds them: with the same scales it
is exact, without (a forked page keeps the coarser scale of the page it was copied from) codes differ by nothing but subnormals.  What is left are the 16-bit
roundings of rotated heads, probabilities and outputs: four of 2^-9 (fp16: 2^-12) rms of the output's norm; 2^-7 (2^-10) holds them."""
import random

import pytest
import torch

import cache8_ref
import rope_ref
from attentionengine_b200 import QKNormRope, copy_pages, examples, plan_compaction, plan_forks

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Plain:
    """The rows' tokens as lists, one layer: rotated 16-bit heads in, attention over rounded keys and values out."""

    def __init__(self, rows, Hkv, D, page):
        self.rows, self.page = [[] for _ in range(rows)], page

    def codes(self, x):
        """The tokens' values as a page holds them: x [n, Hkv, D] in pages of `page`."""
        out = x.clone()
        for at in range(0, x.shape[0], self.page):
            for h in range(x.shape[1]):
                part = x[at:at + self.page, h].numpy()
                s = cache8_ref.scale_of(part)
                out[at:at + self.page, h] = torch.from_numpy(cache8_ref.e4m3(part / s) * s)
        return out

    def attend(self, q, row, last):
        """q [n, Hq, D] of the row's last n tokens; a prompt's own keys and values are not rounded (it attends before the cache)."""
        k, v = (torch.stack([t[i] for t in self.rows[row]]) for i in (0, 1))
        if not last:
            k, v = self.codes(k), self.codes(v)
        n, Hq, D = q.shape
        G, S = Hq // k.shape[1], k.shape[0]
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(G, 1)) / D ** 0.5
        s = s.masked_fill(~torch.ones(S, S, dtype=torch.bool).tril()[S - n:], -torch.inf)
        return torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v.repeat_interleave(G, 1))


@pytest.mark.parametrize("dtype,page,D", [(torch.bfloat16, 16, 128), (torch.float16, 32, 64)])
def test_a_server_s_steps(dtype, page, D):
    L, Hq, Hkv, rows, N = 3, 4, 2, 5, 40
    g = torch.Generator().manual_seed(7)
    rope = QKNormRope(D, base=1e4)
    weights = [tuple((1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in "qk") for _ in range(L)]
    serve = examples.PagedLayers(L, Hq, Hkv, D, dtype, rows, N, page, 160, rope=rope, weights=weights)
    plain = [Plain(rows, Hkv, D, page) for _ in range(L)]
    bound = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -10

    def heads(n):
        return [tuple(torch.randn(n, h, D, generator=g).to(dtype).cuda() for h in (Hq, Hkv, Hkv)) for _ in range(L)]

    def step(call, news, prompt):
        layers = heads(sum(news))
        pos = torch.tensor([len(plain[0].rows[r]) + i for r, n in enumerate(news) for i in range(n)])
        out = call(layers)
        for layer, (q, k, v), w, o in zip(plain, layers, weights, out):
            rq, rk = (rope_ref.forward(x, ww, pos, rope.inv_freq, D, False, True, 1e-6)[0].to(dtype).double() for x, ww in ((q, w[0]), (k, w[1])))
            at = 0
            for r, n in enumerate(news):
                layer.rows[r] += [(rk[at + i], v[at + i].double().cpu()) for i in range(n)]
                want = layer.attend(rq[at:at + n], r, prompt)
                assert (o[at:at + n].double().cpu() - want).norm() <= bound * want.norm(), (r, n)
                at += n

    def fork(parents, keep=None):
        serve.fork(ints(parents), None if keep is None else ints(keep))
        for layer in plain:
            layer.rows = [[] if p < 0 else list(layer.rows[p][:None if keep is None else keep[i]]) for i, p in enumerate(parents)]

    tokens = lambda: step(serve.tokens, [1] * rows, False)  # noqa: E731
    step(lambda x: serve.prompts(x, ints([37, 9, 1, 50, 16])), [37, 9, 1, 50, 16], True)
    fork([0, 0, 0, 3, 4])           # three samples of one prompt
    tokens(), tokens()
    fork([1, 2, 2, 0, 4])           # beams
    tokens()
    fork([0, 1, -1, 3, 4], [20, len(plain[0].rows[1]), 0, len(plain[0].rows[3]), 5])  # cuts and an end
    tokens()
    serve.compact()
    tokens()
    fork([0, 0, 4, 3, 3], [21, 18, 6, len(plain[0].rows[3]), 33])
    serve.compact()
    tokens(), tokens()
    serve.check()
    used = {p for row, n in zip(serve.table.tolist(), serve.lens.tolist()) for p in row[:-(-n // page)]}
    assert used | set(serve.free.tolist()[serve.head.item():]) == set(range(N)) and len(used) == serve.head.item()


def test_what_does_not_fit_is_reported():
    serve = examples.PagedLayers(1, 2, 1, 64, torch.float16, 3, 4, 16, 64)
    x = [tuple(torch.randn(21, h, 64, device="cuda").half() for h in (2, 1, 1))]
    serve.prompts(x, ints([21, 0, 0]))
    serve.fork(ints([0, 0, 0]))
    serve.check()
    serve.fork(ints([0, 0, 7]))
    with pytest.raises(ValueError, match="plan_forks"):
        serve.check()


def test_weights_of_other_layers_are_refused():
    w = [(None, None)]
    for kw in (dict(rope=QKNormRope(64), weights=w), dict(weights=w * 2)):
        with pytest.raises(ValueError, match="weights"):
            examples.PagedLayers(2, 2, 1, 64, torch.float16, 3, 4, 16, 64, **kw)


@pytest.mark.parametrize("kind", ["grouped heads", "latent"])
def test_16_bit_pools(kind):
    """Forks, cuts, a compaction and their copies in the pools of the 16-bit decodes: each row's output is bit for bit that of its tokens in an untouched pool."""
    rng = random.Random(4)
    g = torch.Generator().manual_seed(3)
    randn = lambda *s: torch.randn(*s, generator=g).half().cuda()  # noqa: E731
    page, B, N = 128 if kind == "grouped heads" else 64, 5, 60
    lens = [rng.randrange(1, 7 * page) for _ in range(B)]
    ids, table, at = rng.sample(range(N), N), [], 0
    for n in lens:
        need = -(-n // page)
        table.append(ids[at:at + need] + [0] * (8 - need))
        at += need
    if kind == "grouped heads":
        eng = examples.decode_engine("B", 8, 2, 1, "S", 64, torch.float16)
        pools, q = [randn(N, page, 2, 64), randn(N, page, 2, 64)], randn(1, 1, 8, 64).expand(B, -1, -1, -1).contiguous()

        def decode(pools, table, lens):
            return eng.decode_varlen(q, *pools, lens, block_table=table)
    else:
        eng = examples.mla_engine("B", 16, "S", torch.float16, 0.1)
        pools, q = [randn(N, page, 1, 576)], randn(1, 1, 16, 576).expand(B, -1, -1, -1).contiguous()

        def decode(pools, table, lens):
            return torch.cat([t.float().flatten(1) for t in eng.decode_paged(q, *pools, table, lens, num_split=1)], 1)

    parents, keep = [2, 2, 2, 0, 4], [lens[2], lens[2], lens[2] // 2 + 1, lens[0], lens[4] // 3 + 1]
    want = decode([p.clone() for p in pools], ints([table[p] for p in parents]), ints(keep))
    f = plan_forks(ints(parents), ints(lens), ints(table), ints(ids), ints([at]), page, N, keep_lens=ints(keep))
    copy_pages(pools, f.copies)
    f.check()
    assert torch.equal(decode(pools, f.block_table, f.seq_lens), want)
    c = plan_compaction(f.seq_lens, f.block_table, page, N)
    copy_pages(pools, c.copies)
    c.check()
    held = c.free_head.item()
    assert torch.equal(decode([p[:held].contiguous() for p in pools], c.block_table, f.seq_lens), want)
