"""GPU: the angle of far positions against exact arithmetic."""
import math
from decimal import Decimal, localcontext

import pytest
import torch

pytestmark = pytest.mark.gpu
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899863")


def _angle(position, freq):
    """position * freq modulo a turn, in [-pi, pi)."""
    with localcontext() as c:
        c.prec = 70
        a = Decimal(position) * Decimal(freq) / (2 * PI)
        a -= a.to_integral_value(rounding="ROUND_HALF_EVEN")
        return float(a * 2 * PI)


@pytest.mark.parametrize("far", [0, 1 << 22, 1 << 32, 1 << 40, -(1 << 40), 1 << 46])
def test_angles(cuda_device, far):
    """x = (1, 0) becomes (cos, sin); positions at which the sine is small show the angle itself, in fp16 to 2^-25.  Allowed: the
    stated error of the angle, the same for the sine and cosine in float32 (2 steps of 2^-24, of 1 at most), half a step of fp16."""
    from unified_cache_management_b200 import ops
    freq = [1.0, 0.03162277660168379, 1.1e-3, 1.154782e-4, 3.3e-6, 2.1e-7, 0.7390851332151607, 1e-4 / 40]
    f = torch.tensor(freq, dtype=torch.float64, device="cuda")
    turns = [2 * math.pi / w for w in freq]
    pos = [far + i for i in (0, 1, 2, 77, 5000)]
    for p in turns:                                            # near whole turns of each pair, around `far`
        pos += [round((round(far / p) + i) * p) for i in (0, 1, 2, 3, 50, 1001)]
    t, n = len(pos), len(freq)
    x = torch.zeros((t, 1, 2 * n), dtype=torch.float16, device="cuda")
    x[..., :n] = 1.0
    y = ops.rotary(x, torch.tensor(pos, device="cuda"), f)[:, 0].double().cpu()
    small = 0
    for i, p in enumerate(pos):
        for j, w in enumerate(freq):
            a = _angle(p, w)
            room = abs(p) * w * 2.0 ** -52 + abs(p) * 2 * math.pi * 2.0 ** -64 + 2.0 ** -23 + 2.0 ** -23
            for got, want in ((float(y[i, j]), math.cos(a)), (float(y[i, n + j]), math.sin(a))):
                assert abs(got - want) <= room + max(abs(want) * 2.0 ** -11, 2.0 ** -25), (p, w, got, want, room)
            small += abs(math.sin(a)) < 2.0 ** -10
    assert small > 20
