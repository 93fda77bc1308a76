"""QKNormRope and the plans over a pool's pages without a GPU: parameter blocks, entry points, what is refused when it is made, CPU tensors, angles."""
import ctypes as C
import math
import os
import subprocess
import tempfile
from fractions import Fraction

import pytest
import torch

import pages_ref
import rope_ref
from attentionengine_b200 import QKNormRope, copy_pages, plan_compaction, plan_forks
from attentionengine_b200 import runtime as rt
from attentionengine_b200.attn_engine import pages, rotary

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parameter_blocks_have_the_header_s_sizes():
    pairs = {"AePlanForksParams": rt.PlanForksParams, "AePlanCompactionParams": rt.PlanCompactionParams, "AePagePool": rt.PagePool,
             "AeCopyPagesParams": rt.CopyPagesParams, "AeQkRopeParams": rt.QkRopeParams}
    src = '#include <stdio.h>\n#include "ae_b200.h"\nint main(){' + "".join(f'printf("%zu\\n", sizeof({n}));' for n in pairs) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "s.c"), "w") as f:
            f.write(src)
        subprocess.run(["gcc", f"-I{ROOT}/include", os.path.join(d, "s.c"), "-o", os.path.join(d, "s")], check=True)
        out = subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [C.sizeof(m) for m in pairs.values()]


def _changed(p, **fields):
    q = type(p).from_buffer_copy(bytes(p))
    for k, v in fields.items():
        setattr(q, k, v)
    return C.byref(q)


def test_entry_points_refuse_bad_arguments():
    L = rt.lib()
    for name in ("ae_launch_plan_forks", "ae_launch_plan_compaction", "ae_launch_copy_pages", "ae_launch_qk_rope"):
        assert getattr(L, name)(None, None, None) == 1
    forks, pack, copy = pages._forks_kernels()[0][0], pages._compaction_kernels()[0][0], pages._copy_kernels()[0][0]
    p = rt.PlanForksParams(*(64 * (i + 1) for i in range(13)))
    p.B, p.max_pages, p.n_free, p.page_size, p.num_pages = 2, 3, 4, 16, 5
    assert L.ae_launch_plan_forks(copy.handle, C.byref(p), None) == 6
    for f in (dict(B=0), dict(B=5000), dict(max_pages=0), dict(page_size=24), dict(num_pages=0), dict(n_free=-1), dict(table_out=p.block_table),
              dict(copies=8), dict(workspace=8), dict(parents=None), dict(max_pages=0x7fffffff)):
        assert L.ae_launch_plan_forks(forks.handle, _changed(p, **f), None) == 1, f
    c = rt.PlanCompactionParams(*(64 * (i + 1) for i in range(8)))
    c.B, c.max_pages, c.page_size, c.num_pages, c.n_copies = 2, 3, 16, 5, 2
    assert L.ae_launch_plan_compaction(forks.handle, C.byref(c), None) == 6
    for f in (dict(B=0), dict(page_size=0), dict(n_copies=1), dict(table_out=c.block_table), dict(free_out=None), dict(copies=None)):
        assert L.ae_launch_plan_compaction(pack.handle, _changed(c, **f), None) == 1, f
    m = rt.CopyPagesParams(copies=64, n_copies=1, n_pools=1, num_pages=4, page_size=16)
    m.pools[0] = rt.PagePool(base=64, page_stride=1024, slot_stride=64, row_stride=64, rows=1, run_bytes=64)
    assert L.ae_launch_copy_pages(forks.handle, C.byref(m), None) == 6
    assert L.ae_launch_copy_pages(copy.handle, _changed(m, n_copies=0), None) == 0
    assert L.ae_launch_copy_pages(copy.handle, _changed(m, n_pools=0), None) == 0
    for f in (dict(n_pools=49), dict(n_copies=-1), dict(copies=8), dict(copies=None), dict(page_size=0), dict(page_size=1 << 30)):
        assert L.ae_launch_copy_pages(copy.handle, _changed(m, **f), None) == 1, f
    for pool in (dict(base=None), dict(rows=0), dict(run_bytes=0), dict(extra=66, extra_bytes=4), dict(extra=64, extra_bytes=6)):
        q = rt.CopyPagesParams.from_buffer_copy(bytes(m))
        for k, v in pool.items():
            setattr(q.pools[0], k, v)
        assert L.ae_launch_copy_pages(copy.handle, C.byref(q), None) == 1, pool
    rows = rt.CopyPagesParams.from_buffer_copy(bytes(m))
    rows.pools[0].rows, rows.pools[0].run_bytes = 2, 32
    assert L.ae_launch_copy_pages(pages._copy_kernels()[0][1].handle, C.byref(rows), None) == 1
    assert L.ae_plan_lists_workspace(3, 5) == 16 * 3 + 12 * 4 + 4 * 5
    assert L.ae_plan_lists_phases(1, 1, 1) == 0 and L.ae_plan_lists_phases(4096, 500, 100000) == 1
    fwd, bwd, dw = rotary._kernels(64, 64, True, False)
    r = rt.QkRopeParams(positions=64, B=1, S=3, pos_stride=(0, 1), H=(2, 0))
    r.x[0] = r.y[0] = r.g[0] = 256
    for i in range(3):
        r.x_stride[0][i] = r.g_stride[0][i] = (0, 128, 64)[i]
    assert L.ae_launch_qk_rope(copy.handle, C.byref(r), None) == 6
    assert L.ae_launch_qk_rope(fwd.handle, _changed(r, S=0), None) == 0
    for mod in (fwd, bwd):
        for f in (dict(B=-1), dict(H=(C.c_int32 * 2)(0, 0)), dict(positions=None), dict(B=65536, S=65536)):
            assert L.ae_launch_qk_rope(mod.handle, _changed(r, **f), None) == 1, f
        for name in ("x", "y", "g") if mod is bwd else ("x", "y"):
            for bad in (None, 8):
                q = rt.QkRopeParams.from_buffer_copy(bytes(r))
                getattr(q, name)[0] = bad
                assert L.ae_launch_qk_rope(mod.handle, C.byref(q), None) == 1, (name, bad)
    q = rt.QkRopeParams.from_buffer_copy(bytes(r))
    q.x_stride[0][1] = 132
    assert L.ae_launch_qk_rope(fwd.handle, C.byref(q), None) == 1
    assert L.ae_qk_rope_workspace(bwd.handle) >= 297 * 64 * 4 and L.ae_qk_rope_workspace(copy.handle) == 0


def test_objects_that_cannot_be_made():
    for kw, err in ((dict(head_dim=96), NotImplementedError), (dict(head_dim=512), NotImplementedError), (dict(rotary_dim=0), ValueError),
                    (dict(rotary_dim=24), ValueError), (dict(rotary_dim=80), ValueError), (dict(rotary_dim=32.0), ValueError), (dict(base=0.0), ValueError),
                    (dict(base=math.inf), ValueError), (dict(eps=-1e-6), ValueError), (dict(eps=math.nan), ValueError), (dict(rotary_scale=math.inf), ValueError),
                    (dict(inv_freq=[1.0] * 31), ValueError), (dict(inv_freq=[math.nan] * 32), ValueError)):
        with pytest.raises(err):
            QKNormRope(**{"head_dim": 64, **kw})


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(3, 4, 64, dtype=torch.float16)
    with pytest.raises(rt.AeError, match="CPU"):
        QKNormRope(64)(x, x, torch.arange(3))
    with pytest.raises(rt.AeError, match="CPU"):
        plan_forks(i, i, i[:, None], i, i[:1], 16, 4)
    with pytest.raises(rt.AeError, match="CPU"):
        plan_compaction(i, i[:, None], 16, 4)
    with pytest.raises(rt.AeError, match="CPU"):
        copy_pages([torch.zeros(4, 16, 8)], torch.zeros(1, 4, dtype=torch.int32))


def test_turns_are_exact():
    """One position's fraction of a turn is off by 2^-65 at most, so wrap-around products give any position's angle."""
    for f in (1.0, 0.25, 1e-4 ** 0.5, 1e6 ** (-126 / 128), 0.0, -0.75, 7.5, 1e-30):
        t = Fraction(f) / (2 * rotary._PI)
        t -= math.floor(t)
        off = abs(Fraction(rotary.turns_of(f), 2 ** 64) - t)
        assert min(off, 1 - off) <= Fraction(1, 2 ** 65)
    for p in (1, 1000, 2 ** 20, 2 ** 31 - 1):
        got = (p * rotary.turns_of(1.0)) % 2 ** 64 / 2 ** 64 * 2 * math.pi
        assert abs(math.cos(got) - math.cos(p)) < 1e-9 and abs(math.sin(got) - math.sin(p)) < 1e-9
    assert abs(float(rotary._PI) - math.pi) == 0.0


def test_the_plain_gradient_is_that_of_the_plain_forward():
    g = torch.Generator().manual_seed(1)
    freq = [10.0 ** -i for i in range(8)]
    for inter, norm in ((False, True), (True, True), (True, False)):
        x, w = torch.randn(5, 3, 32, generator=g, dtype=torch.float64), 1 + torch.rand(32, generator=g, dtype=torch.float64)
        d_y, pos, h = torch.randn(5, 3, 32, generator=g, dtype=torch.float64), torch.tensor([3, 0, 99, -1, 7]), 1e-6
        dx, _, dw, _ = rope_ref.backward(x, w, pos, freq, 16, inter, norm, 1e-6, d_y)
        loss = lambda x, w: float((rope_ref.forward(x, w, pos, freq, 16, inter, norm, 1e-6)[0] * d_y).sum())  # noqa: E731
        for _ in range(5):
            d, e = torch.randn(5, 3, 32, generator=g, dtype=torch.float64), torch.randn(32, generator=g, dtype=torch.float64)
            assert abs((loss(x + h * d, w) - loss(x - h * d, w)) / (2 * h) - float((dx * d).sum())) < 1e-6
            if norm:
                assert abs((loss(x, w + h * e) - loss(x, w - h * e)) / (2 * h) - float((dw * e).sum())) < 1e-6


def test_the_plain_plans():
    """The references of the GPU tests on cases worked out by hand (pages of 4)."""
    f = pages_ref.forks([0, 0, -1, 3], [6, 0, 5, 3], [[0, 1, 0], [0] * 3, [2, 3, 0], [4, 0, 0]], [0, 1, 2, 3, 4, 8, 9], 5, 4)
    assert f["block_table"] == [[0, 1, 0], [0, 8, 0], [0, 0, 0], [4, 0, 0]] and f["seq_lens"] == [6, 6, 0, 3]
    assert f["copies"] == [[1, 8, 2, 0]] + [[0] * 4] * 3 and f["free_head"] == [4] and f["free_pages"] == [0, 1, 2, 3, 2, 3, 9]
    c = pages_ref.compaction([6, 2], [[5, 1], [4, 0]], 4, 8)
    assert c["block_table"] == [[2, 1], [0, 0]] and c["copies"] == [[4, 0, 2, 0], [5, 2, 4, 0]] + [[0] * 4] * 2 and c["free_head"] == [3]
