"""SiLU and the tanh form of GELU in fp32, relative to the value, far out where it is small."""

import pytest
import torch

from moe_bench_b200 import capi
from oracle import ffn_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_tails_keep_the_digits_that_the_exponential_has(act):
    """Both are z s with s = 1 / (1 + exp(-v)).  CUDA gives __expf(v) to 2 + 1.173 |v| units of 2^-23 and __fdividef to 2 of
    them while the divisor is below 2^126, so in steps of 2^-24: 4 + 2.35 |v| for the exponential, 1 for the sum, 4 for the
    quotient, 1 for the product with z, and 1 for what is of second order.  v is z itself, or for GELU a polynomial of which
    4 roundings make the cubic term, 1 the sum, 2 the factor: 7 steps of |v|, which the exponential passes on whole.
    Past a divisor of 2^126 (v below -87.3) s is 0 instead of less than 2^-126."""
    z = torch.cat([torch.linspace(-110, 110, 200001), torch.linspace(-12, 12, 100001), -torch.logspace(-30, 0, 500)]).cuda()
    w = torch.zeros(z.numel(), 8, device=DEV, dtype=torch.bfloat16)
    zd = z.double()
    v, passed_on = (zd, 0) if act == "silu" else (2 * (2 / torch.pi) ** 0.5 * (zd + 0.044715 * zd ** 3), 7)
    ref, _ = F.activation(act, zd)
    bound = (11 + (2.35 + passed_on) * v.abs()) * F.U32 * ref.abs() + 2.0 ** -140
    bound = torch.where(v < -87, bound + zd.abs() * 2.0 ** -125, bound)
    for rows in (1, 40):
        y = capi.linear(torch.zeros(rows, 8, device=DEV, dtype=torch.bfloat16), w, bias=z, activation=act, out_dtype=torch.float32)
        for row in y:
            wrong = F.inside(row, ref, bound)
            assert wrong is None, wrong
