"""lh_q8_silu where gate and up lie at opposite ends of FP32's range: products in its middle of
factors whose own intermediate values would leave it."""
import numpy as np
import pytest

import q8_oracle as q8
from test_gpu_q8 import run_silu

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -149   # the smallest subnormal

# A width of each number of waves, and one that registers do not hold.
WIDTHS = [2, 300, 1000, 3000, 4100, 9216, 20000, 30000, 40000]


def rows_of(width):
    rng = np.random.default_rng(width)

    def some(low, high):
        """Of every size in between, either sign."""
        return rng.choice((-1.0, 1.0), width) * np.exp2(rng.uniform(low, high, width))

    def whole(most):
        """Subnormals of few bits, either sign."""
        return LEAST * rng.integers(-most, most + 1, width)

    gate, up = [], []

    def row(g, u):
        gate.append(np.broadcast_to(np.asarray(g, np.float32), width))
        up.append(np.broadcast_to(np.asarray(u, np.float32), width))

    three = np.where(np.arange(width) % 2 == 0, 3.0, 1.0)
    row(LEAST * three, 2.0 ** 127)
    row(LEAST * (2 + three), 1e35)
    row(-LEAST * three, -2.0 ** 127)
    row(1e-43 * rng.uniform(0.5, 1, width), 1e30 * rng.uniform(0.5, 1, width))
    row(whole(9), some(120, 127.9))
    row(whole(999), some(90, 127.9))
    row(some(-149, -126), some(100, 127.9))
    row(some(-135, -115), some(60, 127.9))
    row(some(-149, -90), some(25, 45))
    row(some(-149, -120), some(60, 72))
    row(some(-149, -125), some(60, 66))
    row(whole(5), some(38, 70))
    row(whole(5), some(64, 70))
    # Subnormal ups under large gates.
    row(np.abs(some(90, 127.9)), whole(9))
    row(np.abs(some(60, 127.9)), some(-149, -115))
    row(-rng.uniform(0, 80, width), some(-149, 127.9))
    # One such product among ordinary ones, the row's largest and not.
    for size in (2.0 ** 127, 2.0 ** 100):
        g, u = rng.normal(size=width), rng.normal(size=width)
        if size < 2.0 ** 127:
            g, u = g * 2.0 ** -30, u * 2.0 ** -30
        g[width // 2], u[width // 2] = 3 * LEAST, size
        row(g, u)
    # Zeros under the largest.
    row(np.where(rng.random(width) < 0.5, 0.0, rng.normal(size=width)), some(-1, 127.9))
    row(0.0, 3e38)
    return np.array(gate), np.array(up)


@pytest.mark.parametrize("width", WIDTHS)
def test_silu_of_far_factors(gpu, width):
    gate, up = rows_of(width)
    codes, scales = run_silu(gpu, gate, up, pad=1, offset=1)
    q8.check_rows(codes, scales, q8.silu(gate, up))
