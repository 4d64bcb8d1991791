"""What the entry points for MLPs of experts launch, at sizes that no test runs at: fewer than 2^32 threads (a launch of more runs modulo 2^32 of them, without an error) and
grids that the hardware takes; and that the sizes of GPU tests reach the kernels that they are there for."""
import random

import pytest

from launches import launches
from openvino_contrib_amd import ops_capi
from openvino_contrib_amd.capi import BF16, F16, F32

P = 1 << 20  # (an address that nobody follows)


def product(m, n, k, c_dtype=BF16, offset=0, workspace=0):
    return ("hipops_matmul_fp8", "MatmulFp8Desc", dict(c_dtype=c_dtype, m=m, n=n, k=k), [P + offset, P, P, P, None, None, P, P if workspace else None, workspace, None])


def routing(tokens, experts, top_k, lists):
    return ("hipops_route_experts", "RouteDesc", dict(logits_dtype=F16, renormalise=1, experts=experts, top_k=top_k, scale=1.0, tokens=tokens),
            [P, None, P, P] + [P if lists else None] * 3 + [P, 1 << 50, None])


def fits(launch):
    return 0 < launch.threads < 1 << 32 and launch.grid[1] <= 65535 and launch.grid[2] <= 65535


def sizes(rng, most):
    """A number up to `most`, spread over its logarithm, some of them whole blocks or powers of two."""
    v = max(1, min(most, int(2 ** rng.uniform(0, most.bit_length()))))
    return rng.choice([v, max(1, v // 128 * 128), 1 << (v.bit_length() - 1)])


@pytest.mark.parametrize("m,n,k", [(1 << 30, 1, 1), (1 << 30, 32, 1), (1 << 30, 32, 16), ((1 << 31) - 1, 1, 1), ((1 << 31) - 1, 1, 256), ((1 << 31) - 1, 129, 128), (5000, (1 << 31) - 1, 640)])
def test_products_of_few_columns_or_rows(m, n, k):
    for c_dtype in (BF16, F32):
        for status, error, found in launches(product(m, n, k, c_dtype), product(m, n, k, c_dtype, offset=1)):
            assert status == 0, error
            assert found and all(fits(l) for l in found), [l for l in found if not fits(l)]


def test_products_of_any_size():
    rng, calls = random.Random(1), []
    while len(calls) < 800:
        m, n, k = sizes(rng, (1 << 31) - 1), sizes(rng, (1 << 31) - 1), sizes(rng, 65536)
        if m * n <= 1 << 37:
            calls.append(product(m, n, k, rng.choice((F32, F16, BF16)), rng.choice((0, 1)), rng.choice((0, 1 << 34))))
    for call, (status, error, found) in zip(calls, launches(*calls)):
        assert status == 0, error
        assert found and all(fits(l) for l in found), (call, [l for l in found if not fits(l)])


@pytest.mark.parametrize("tokens", [939524096, (1 << 30) + 1, (1 << 31) - 1])
def test_routing_of_very_many_tokens(tokens):
    for status, error, found in launches(*[routing(tokens, experts, 1, False) for experts in (1, 128, 256, 512, 1024)]):
        assert status == 0, error
        assert len(found) > 1 and all(fits(l) for l in found), found
        assert sum(l.grid[0] for l in found) == -(-tokens // 224)


def test_routing_of_any_size():
    rng = random.Random(2)
    calls = [routing(sizes(rng, 1 << 26), rng.choice((1, 8, 60, 128, 1024)), 1, lists) for lists in (True, False) for _ in range(100)]
    for call, (status, error, found) in zip(calls, launches(*calls)):
        assert status == 0, error
        assert found and all(fits(l) for l in found), (call, found)
