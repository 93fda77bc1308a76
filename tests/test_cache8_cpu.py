"""The serving operators without a GPU: parameter blocks, what the engines refuse when they are made, CPU tensors, entry points."""
import ctypes as C
import math
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import cache8_ref as ref
from attentionengine_b200 import AttentionEngine, CustomIO, PagedCache8, SymbolScalar, Var, examples, meta_tensor, plan_pages
from attentionengine_b200 import runtime as rt
from attentionengine_b200.attn_engine.cache8 import _plan_kernel, _write_kernel, is_softmax

E4M3 = torch.float8_e4m3fn
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parameter_blocks_have_the_header_s_sizes():
    pairs = {"AeAttnPackedParams": rt.AttnPackedParams, "AePlanPagesParams": rt.PlanPagesParams, "AeCache8WriteParams": rt.Cache8WriteParams,
             "AeCache8DecodeParams": rt.Cache8DecodeParams}
    src = '#include <stdio.h>\n#include "ae_b200.h"\nint main(){' + "".join(f'printf("%zu\\n", sizeof({n}));' for n in pairs) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "s.c"), "w") as f:
            f.write(src)
        subprocess.run(["gcc", f"-I{ROOT}/include", os.path.join(d, "s.c"), "-o", os.path.join(d, "s")], check=True)
        out = subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [C.sizeof(m) for m in pairs.values()]


def test_entry_points_refuse_bad_arguments():
    L = rt.lib()
    for name in ("ae_launch_attn_packed", "ae_launch_plan_pages", "ae_launch_cache8_write", "ae_launch_cache8_decode"):
        assert getattr(L, name)(None, None, None) == 1
    plan, write = _plan_kernel(), _write_kernel(16, 64, 64)
    p = rt.PlanPagesParams()
    for n, _ in rt.PlanPagesParams._fields_[:12]:
        setattr(p, n, 16)
    p.head_out = 32
    p.B, p.max_pages, p.page_size, p.n_tokens, p.n_segments = 1, 1, 16, 4, 2
    assert L.ae_launch_plan_pages(write.handle, C.byref(p), None) == 6
    for field, value in (("B", 0), ("B", 5000), ("page_size", 24), ("page_size", 0), ("n_segments", 1), ("head_out", 16), ("max_pages", 0)):
        q = rt.PlanPagesParams.from_buffer_copy(bytes(p))
        setattr(q, field, value)
        assert L.ae_launch_plan_pages(plan.handle, C.byref(q), None) == 1, field
    w = rt.Cache8WriteParams()
    for n, _ in rt.Cache8WriteParams._fields_[:7]:
        setattr(w, n, 64)
    w.n_tokens = w.n_segments = w.num_pages = w.H = 1
    w.k_stride[0] = 4  # not a multiple of 16 bytes
    assert L.ae_launch_cache8_write(write.handle, C.byref(w), None) == 1
    assert L.ae_launch_cache8_write(plan.handle, C.byref(w), None) == 6


def test_cpu_tensors_are_refused():
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(rt.AeError, match="CPU"):
        plan_pages(i, i, i[None], i, i, 16, 1)
    with pytest.raises(rt.AeError, match="CPU"):
        PagedCache8(2, 16, 1, 64, device="cpu")
    eng = examples.softmax_engine("B", 4, 2, "S", 64, 64, torch.float16, True, packed=True)
    x = torch.zeros(3, 4, 64, dtype=torch.float16)
    with pytest.raises(rt.AeError, match="CPU"):
        eng.prefill_packed(x, x[:, :2], x[:, :2], torch.tensor([0, 3], dtype=torch.int32))


class Plain(examples.OnlineSoftmax):
    """A softmax without the running maximum: the same result, another recurrence."""

    @staticmethod
    def online_fwd(scores, online_rowscales, b, h, q_idx):
        p = scores.exp()
        return p, {"m": online_rowscales["m"], "r": online_rowscales["r"] + p.get_reduce("sum")}, SymbolScalar("o_scale", Var("1"))


def test_softmax_is_told_from_other_online_functions():
    assert is_softmax(examples.OnlineSoftmax()) and is_softmax(examples.OnlineSoftmaxSplit()) and is_softmax(Plain())
    assert not is_softmax(examples.OnlineIdentity()) and not is_softmax(examples.OnlineRetention())


def test_engines_that_cannot_be_made():
    E, soft = examples.decode_engine, dict(cache_dtype=E4M3)
    for make in (lambda: E(1, 4, 2, 1, 64, 64, torch.float16, online=examples.OnlineIdentity(), **soft),
                 lambda: E(1, 4, 2, 1, 64, 64, torch.float16, cache_dtype=torch.int8),
                 lambda: E(1, 4, 2, 2, 64, 64, torch.float16, **soft),       # grouped heads, two positions
                 lambda: E(1, 4, 4, 64, 64, 64, torch.float16, **soft),      # q_len == kv_len
                 lambda: E(1, 4, 2, 1, 64, 192, torch.float16, **soft),
                 lambda: E("B", "H", 2, 1, 64, 64, torch.float16, **soft),
                 lambda: examples.softmax_engine("B", 4, 2, "S", 64, 64, torch.float16, True, packed=True, cache_dtype=E4M3),
                 lambda: examples.softmax_engine("B", 4, 2, "S", 64, 64, torch.float16, True, packed=True, extern_block_mask=True)):
        with pytest.raises(NotImplementedError):
            make()
    m = [meta_tensor("B", 2, n, 64, dtype=torch.float16) for n in (1, "S", "S")]
    with pytest.raises(NotImplementedError, match="positions"):
        AttentionEngine(m, CustomIO({"x": ("batch", "heads", 1, "seq_len_kv")}), online_func=examples.OnlineSoftmax(), mask_mod=None,
                        score_mod=lambda s, c, b, h, q, kv: s + c.input_tensors["x"], cache_dtype=E4M3)
    m = [meta_tensor("B", 2, "S", 64, dtype=torch.float16) for _ in range(3)]
    with pytest.raises(NotImplementedError, match="positions"):
        AttentionEngine(m, CustomIO({"x": ("batch", "heads", "seq_len")}), online_func=examples.OnlineSoftmax(), mask_mod=None,
                        score_mod=lambda s, c, b, h, q, kv: s + c.input_tensors["x"], packed=True)
    with pytest.raises(NotImplementedError, match="-inf"):
        AttentionEngine([meta_tensor("B", 2, n, 64, dtype=torch.float16) for n in (1, "S", "S")], CustomIO({}), mask_value="0",
                        score_mod=lambda s, c, b, h, q, kv: s, mask_mod=lambda b, h, q, kv: kv > 3, online_func=examples.OnlineSoftmax(),
                        cache_dtype=E4M3)


def test_masks_of_packed_engines():
    make = lambda mask: AttentionEngine([meta_tensor("B", 2, "S", 64, dtype=torch.float16) for _ in range(3)], CustomIO({}),  # noqa: E731
                                        score_mod=lambda s, c, b, h, q, kv: s, mask_mod=mask, online_func=examples.OnlineSoftmax(), packed=True)
    assert make(None).mask_mode == 0 and make(examples.causal_mask).mask_mode == 1
    assert make(lambda b, h, q, kv: q - kv < 9).mask_mode == 3


def test_the_plain_e4m3_is_torch_s():
    """The reference of the GPU tests, on every half of the range: torch's rounding, which saturates to NaN above 448."""
    x = torch.cat([torch.linspace(-448, 448, 40001), torch.logspace(-4, 2.6, 9001), torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, math.nan])])
    np.testing.assert_array_equal(ref.e4m3(x.double().numpy()), x.to(E4M3).double().numpy())
