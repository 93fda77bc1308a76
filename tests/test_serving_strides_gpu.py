"""Dimensions of one element have any stride: one request, one token, one kv head, one page, out of a buffer whose rows are not a multiple of 16
bytes apart.  The calls give what they give for contiguous tensors."""
import pytest
import torch

from attentionengine_b200 import PagedCache8, examples
from test_cache8_gpu import engine, filled, ints

pytestmark = pytest.mark.gpu


def odd(t):
    """The same values with strides of 1001, 1003 ... elements where a dimension has one."""
    st = [1001 + 2 * i if n == 1 else s for i, (n, s) in enumerate(zip(t.shape, t.stride()))]
    return torch.as_strided(t, t.shape, st)


@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (4, 2), (1, 1)])
def test_one_request(Hq, Hkv):
    D, page = 64, 16
    q, k, v = (torch.randn(1, h, D, device="cuda").half() for h in (Hq, Hkv, Hkv))
    prompt = examples.softmax_engine("B", Hq, Hkv, "S", D, D, torch.float16, True, packed=True)
    cu = ints([0, 1])
    assert torch.equal(prompt.prefill_packed(odd(q), odd(k), odd(v), cu), prompt.prefill_packed(q, k, v, cu))
    kc, vc, ks, vs = filled(1, page, Hkv, D, D, 1)
    caches = []
    for change in (lambda t: t, odd):
        parts = [t.clone() for t in (kc, vc, ks, vs)]
        c = PagedCache8.from_tensors(*(change(t) for t in parts[:2]), *parts[2:])
        c.write(change(k), change(v), ints([[0, 7, 0, 1]]))
        caches.append((c, parts))
    for a, b in zip(*(parts for _, parts in caches)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    eng = engine(Hq, Hkv, 1, D, D, torch.float16)
    q = q.unsqueeze(1)
    want = eng.decode_cache8(q, caches[0][0], ints([[0]]), ints([8]))
    assert torch.equal(eng.decode_cache8(odd(q), caches[1][0], ints([[0]]), ints([8])), want)
    prompt.check_status()
    eng.check_status()
