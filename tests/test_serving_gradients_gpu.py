"""The serving calls are forward only: a custom input that wants a gradient, or carries a tangent, is refused as q, k and v are."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from attentionengine_b200 import AttentionEngine, CustomIO, PagedCache8, examples, meta_tensor

pytestmark = pytest.mark.gpu


def prompt():
    m = [meta_tensor("B", 2, "S", 64, dtype=torch.float16) for _ in range(3)]
    eng = AttentionEngine(m, CustomIO({"slope": (1, "heads"), "bias": ("batch",)}), mask_mod=examples.causal_mask, online_func=examples.OnlineSoftmax(),
                          score_mod=lambda s, c, b, h, q, kv: s * 0.125 + c.input_tensors["slope"] + c.input_tensors["bias"], packed=True)
    q, k, v = (torch.randn(30, 2, 64, device="cuda").half() for _ in range(3))
    cu = torch.tensor([0, 10, 30], dtype=torch.int32, device="cuda")
    return lambda *c: eng.prefill_packed(q, k, v, cu, *c)


def token():
    m = [meta_tensor("B", 2, n, 64, dtype=torch.float16) for n in (1, "S", "S")]
    eng = AttentionEngine(m, CustomIO({"slope": (1, "heads"), "bias": ("batch",)}), mask_mod=None, online_func=examples.OnlineSoftmaxSplit(),
                          score_mod=lambda s, c, b, h, q, kv: s * 0.125 + c.input_tensors["slope"] + c.input_tensors["bias"], cache_dtype=torch.float8_e4m3fn)
    q, cache = torch.randn(2, 1, 2, 64, device="cuda").half(), PagedCache8(4, 16, 2, 64)
    table, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0], [1]], [5, 9]))
    return lambda *c: eng.decode_cache8(q, cache, table, lens, *c)


@pytest.mark.parametrize("call", [prompt, token])
def test_custom_inputs(call):
    run = call()
    slope, bias = torch.randn(1, 2, device="cuda"), torch.randn(2, device="cuda")
    want = run(slope, bias)
    for i, name in enumerate(("slope", "bias")):
        c = [slope.clone(), bias.clone()]
        c[i].requires_grad_()
        with pytest.raises(NotImplementedError, match=name):
            run(*c)
        with torch.no_grad():
            assert torch.equal(run(*c), want)
        with fwd.dual_level():
            c = [slope, bias]
            c[i] = fwd.make_dual(c[i], torch.ones_like(c[i]))
            with pytest.raises(NotImplementedError, match=name):
                run(*c)
    with pytest.raises(TypeError):
        run(slope)
