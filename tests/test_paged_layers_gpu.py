"""examples.PagedLayers takes prompts into empty rows alone: attention of new tokens over a cached prefix is not there."""
import pytest
import torch

from attentionengine_b200 import examples

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", ["prompts", "tokens"])
def test_rows_that_hold_tokens_get_no_prompt(first):
    Hq, Hkv, D, dtype = 4, 2, 64, torch.float16
    serve = examples.PagedLayers(1, Hq, Hkv, D, dtype, rows=2, num_pages=12, page_size=16, max_len=90)
    new = lambda n: [tuple(torch.randn(n, h, D, device="cuda").to(dtype) for h in (Hq, Hkv, Hkv))]  # noqa: E731
    lens = torch.tensor([20, 5], dtype=torch.int32, device="cuda")
    if first == "prompts":
        serve.prompts(new(25), lens)
    else:
        serve.tokens(new(2))
    before = serve.lens.tolist()
    with pytest.raises(NotImplementedError, match="cached"):
        serve.prompts(new(25), lens)
    assert serve.lens.tolist() == before  # nothing of the refused step has happened
    serve.tokens(new(2))
    assert serve.lens.tolist() == [n + 1 for n in before]
    serve.check()
