"""YaRN's ramp where its slow end lies past the last rotated pair: the tables of r97b_rope_tables (csrc/rope.cu) against
angles formed here from the definition. The ramp runs from the floor of the pair that turns beta_fast times over the
original length (0 at least) to the ceiling of the one that turns beta_slow times (rot - 1 at most, the rotated width's
last dim): a ramp that ends past the last pair stays short of 1 there."""
import math

import pytest
import torch

from r97training_b200 import ops
from tests.packed_ref import E32, assert_within

pytestmark = pytest.mark.gpu


def _ramp_ends(rot, theta, original, beta_fast=32.0, beta_slow=1.0):
    """The real pair index i whose angle original * theta^(-2 i / rot) is 2 pi `turns`, solved by bisection."""
    def pair(turns):
        lo, hi = -8.0 * rot, 8.0 * rot
        for _ in range(200):
            mid = 0.5 * (lo + hi)
            if original * theta ** (-2.0 * mid / rot) > 2.0 * math.pi * turns:
                lo = mid
            else:
                hi = mid
        return lo
    fast, slow = pair(beta_fast), pair(beta_slow)
    assert min(abs(v - round(v)) for v in (fast, slow)) > 1e-6  # floor and ceiling do not hang on a rounding
    return max(math.floor(fast), 0), min(math.ceil(slow), rot - 1)


# the ramp's end inside the pairs, past the last one, and past the rotated width's last dim
@pytest.mark.parametrize("rot,theta,original,ends", [(128, 1e4, 4096, (20, 46)), (128, 1e4, 65536, (40, 65)),
                                                     (64, 1e4, 65536, (20, 33)), (16, 1e4, 32768, (4, 8)),
                                                     (64, 1e4, 10 ** 9, (53, 63)), (16, 100.0, 4096, (5, 12))])
def test_yarn_ramp(cuda, rot, theta, original, ends):
    low, high = _ramp_ends(rot, theta, original)
    assert (low, high) == ends
    factor, n = 8.0, 5003
    cos, sin = ops.rope_tables(n, rot, theta, scaling={"type": "yarn", "factor": factor, "original": original},
                               device=cuda)
    inv = []
    for i in range(rot // 2):
        base = theta ** (-2.0 * i / rot)
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        inv.append(base * (1.0 - ramp) + base / factor * ramp)
    ang = torch.arange(n, dtype=torch.float64, device=cuda)[:, None] * torch.tensor(inv, dtype=torch.float64, device=cuda)
    amp = 0.1 * math.log(factor) + 1.0
    slack = n * 2.0 ** -50  # a few f64 roundings of the frequency times the position
    for got, want in ((cos, amp * torch.cos(ang)), (sin, amp * torch.sin(ang))):
        assert_within(got, (want, E32 * want.abs() + slack), "table")
