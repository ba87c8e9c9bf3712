"""The expert operators where their values, plans and inputs are at an edge, against their definitions in 64 bits
(tests/experts_ref.py; the roundings that tolerances count are those of tests/test_experts_gpu.py)."""
import math

import pytest
import torch

import experts_ref as ref
from experts_ref import F32_MAX
from test_experts_gpu import C, DEV, FUNCS, gen

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------- routing
@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("K,k", [(32, 3), (129, 1), (256, 9), (512, 1), (512, 5), (1000, 32), (4096, 4)])
def test_route_many_infinities_and_largest_scores(func, K, k):
    """+inf counts as the largest finite value: among many of both, the lowest indices are chosen."""
    inf = math.inf
    z = torch.randn(6, K, generator=gen(K))
    z[0, :K // 3] = F32_MAX; z[0, K * 2 // 3] = inf
    z[1, 1::2] = F32_MAX; z[1, 2::4] = inf
    z[2, ::2] = inf
    z[3, :] = F32_MAX; z[3, K - 1] = inf
    z[4, K // 2:] = inf; z[4, K // 2 - 1] = F32_MAX
    z[5, :] = torch.finfo(torch.float32).min; z[5, K - 2] = inf
    for renorm in (True, False):
        got = C().route_experts(z.to(DEV), k, score_func=func, renormalize=renorm)
        assert torch.equal(got[1].cpu(), ref.route(z, k, func, renormalize=renorm)[1])
