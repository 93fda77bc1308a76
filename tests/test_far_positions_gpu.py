"""What QKNormRope's angles are: a position times the frequency's fraction of a turn, modulo 2^64 in whole numbers.

Bounds: the upper 32 bits of the product are half turns of 2^-31, rounded to fp32 (2^-25 of a half turn, 1e-7 radians), and sincospif's two units: 2^-20 of
each of the two terms holds them, as in the tests of other positions; half a step of fp16 for the output, 2^-11 of the value."""
import math

import pytest
import torch

from attentionengine_b200 import QKNormRope
from attentionengine_b200.attn_engine.rotary import turns_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_wrap_around(interleaved):
    rope = QKNormRope(64, base=1e4, norm=False, interleaved=interleaved)
    positions = [0, 1, 77, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 32, 2 ** 40 + 12345, 2 ** 53 + 1, 2 ** 62, 2 ** 62 + 2 ** 61 + 987654321, 2 ** 63 - 1]
    x = torch.ones(len(positions), 1, 64, dtype=torch.float16, device="cuda")
    got = rope(x, None, torch.tensor(positions, device="cuda"))[0][:, 0].double().cpu()
    for p, row in zip(positions, got):
        for i, f in enumerate(rope.inv_freq):
            a = (p * turns_of(f)) % 2 ** 64 / 2 ** 64 * 2 * math.pi  # Python divides whole numbers to the nearest double
            at = (2 * i, 2 * i + 1) if interleaved else (i, 32 + i)
            for v, want in ((row[at[0]], math.cos(a) - math.sin(a)), (row[at[1]], math.cos(a) + math.sin(a))):
                assert abs(float(v) - want) <= 2 * 2.0 ** -20 + 2.0 ** -11 * abs(want), (p, i, float(v), want)
