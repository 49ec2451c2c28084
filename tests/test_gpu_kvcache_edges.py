"""The paged key/value cache operators where their kernels' parts meet: short units next to each other, several CTAs on one
head, few rows of a block (GPU). Cases, definitions in 64 bits and tolerances as in test_gpu_kvcache.py, and half of f16's
least spacing (2^-24) more where an f16 output is below its normal numbers: u |o| is the rounding of normal ones only."""
import math

import pytest
import torch

from technograd_b200 import _lib, kvcache  # noqa: F401
from test_gpu_kvcache import BF16, F16, F32, INF, UNIT, Case, attend, bits, check_attend, near, plain, random_mask  # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, want, dtype):
    """out and lse against plain()'s."""
    near(got[0], want[0], want[2] + (2.0 ** -25 if dtype is F16 else 0), "out")
    near(got[1], want[1], want[3], "lse")


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("lens", [[0] * 200 + [700], [0, 1, 128, 129] * 60, [128] * 300])
def test_short_units_after_each_other(cuda, lens, dtype, dim):
    """Many units of one or two tiles to a CTA of the 128-row kernel: each row's reference and sum are its own unit's. The
    rows' scores differ by hundreds from unit to unit, so that another unit's would show."""
    c = Case(lens, 2, 2, dim, 16, "head", dtype, 20)
    c.q *= torch.tensor([1.0, 20.0, 0.05])[torch.arange(len(lens)) % 3][:, None, None, None]
    mask = random_mask(len(lens), 20, 3)
    out, lse = attend(c, mask)
    check((out, lse), plain(c, mask), dtype)
    for _ in range(20):
        again = attend(c, mask)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
