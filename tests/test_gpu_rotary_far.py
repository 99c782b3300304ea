"""Rotary positions far out: angles are those of the exact product of position and frequency."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798214808651")


def reduced(position, frequency):
    """The angle within half a turn, from 100 digits."""
    getcontext().prec = 100
    turns = Decimal(position) * Decimal(frequency) / (2 * PI)
    return float((turns - turns.to_integral_value()) * 2 * PI)


@pytest.mark.parametrize("interleaved", [False, True])
def test_any_position(interleaved):
    positions = [0, 1, 12_345_678, 2 ** 33 + 7, -(2 ** 40) - 3, 2 ** 47 + 1, 2 ** 53 - 1, 2 ** 53 + 1, 3 ** 39, -(3 ** 39) + 1, 2 ** 63 - 1, -(2 ** 63)]
    frequencies = [1.0, 0.1, 10_000.0 ** (-5 / 16), 1 / 3, 1e-4, 3.7]
    half = len(frequencies)
    q = torch.zeros(len(positions), 1, 2 * half, device=DEV)
    first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, half), slice(half, None))
    q[:, :, first] = 1.0
    out = F.rotary(q, None, torch.tensor(positions, device=DEV), torch.tensor(frequencies, dtype=torch.float64, device=DEV), 1, interleaved=interleaved)[:, 0].double().cpu()
    for i, p in enumerate(positions):
        for j, f in enumerate(frequencies):
            angle = reduced(p, f)
            # a cosine and a sine within 2^-22, of an angle that float32 has within 2^-24 of half a turn
            assert abs(out[i, first][j] - math.cos(angle)) <= 2.0 ** -21 and abs(out[i, second][j] - math.sin(angle)) <= 2.0 ** -21, (p, f)
