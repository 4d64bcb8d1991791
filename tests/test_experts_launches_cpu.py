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


def experts_product(experts, rows, n, k, c_dtype, gated=0, workspace=1 << 30):
    return ("hipops_matmul_fp8_experts", "MatmulFp8ExpertsDesc", dict(c_dtype=c_dtype, gated=gated, order_divisor=1, experts=experts, rows=rows, n=n, k=k, a_rows=50),
            [P, P, P, P, P, P, P, P, P, workspace, None])


def quantising(rows, width, source=0):
    return ("hipops_quantize_fp8", "QuantizeFp8Desc", dict(source=source, x_dtype=F16, gamma_dtype=F16, rows=rows, width=width), [P, None, P, P, None])


def combining(tokens, n, y_dtype):
    return ("hipops_combine_experts", "CombineDesc", dict(y_dtype=y_dtype, out_dtype=F16, top_k=2, tokens=tokens, rows=5, n=n), [P] * 5 + [None])


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


def test_the_other_calls_of_any_size():
    rng, calls = random.Random(3), []
    while len(calls) < 800:
        rows, n = sizes(rng, (1 << 31) - 1), sizes(rng, 1 << 26)
        if rows * n > 1 << 37:
            continue
        gated, experts, k = rng.choice((0, 1)), sizes(rng, 1024), sizes(rng, 65536)
        c_dtype = rng.choice((F32, F16, BF16, ops_capi.F8_E4M3) if gated else (F32, F16, BF16))
        calls += [experts_product(experts, rows, max(2, n // 2 * 2), k, c_dtype, gated, rng.choice((1 << 30, 1 << 36))), quantising(rows, n, rng.choice((0, 1, 2))),
                  combining(rows, n, rng.choice((F32, F16)))]
    for call, (status, error, found) in zip(calls, launches(*calls)):
        assert status == 0, error
        assert found and all(fits(l) for l in found), (call, [l for l in found if not fits(l)][:3])


def test_sizes_of_gpu_tests_reach_their_kernels():
    deep, tiles, by_row, quantise = "matmul_fp8_deep_kernel<", "matmul_fp8_tiles_kernel<", "quantize_fp8_norm_kernel<", "quantize_fp8_kernel<"
    E4M3 = ops_capi.F8_E4M3
    rows = (1 << 19) + 3001
    cases = [(product(2001, 6245, 2048, c_dtype), [deep, tiles]) for c_dtype in (BF16, F16)]
    cases += [(quantising((1 << 26) + 5000, 3, source), [by_row if source == 1 else quantise] * 2) for source in (0, 1, 2)]
    cases += [(experts_product(4, 2056, n, k, E4M3, 1, 700 * n // 2 * 4), [deep, quantise] * 3) for n, k in ((512, 1024), (256, 640))]
    cases += [(experts_product(6, 3086, n, k, E4M3, 1, 700 * n // 2 * 4), [deep, quantise] * 5) for n, k in ((512, 1024), (256, 640))]
    cases += [(experts_product(4, rows, *how), [kernel] * 2) for how, kernel in (((256, 512, BF16, 0), deep), ((512, 640, F16, 1), deep), ((256, 512, F32, 0), tiles), ((130, 100, BF16, 0), tiles))]
    for (call, kernels), (status, error, found) in zip(cases, launches(*[call for call, _ in cases])):
        assert status == 0, error
        assert len(found) == len(kernels) and all(k in l.kernel for k, l in zip(kernels, found)), (call, found)


def test_results_in_fp32_are_exact_products():
    """Of any size, dense and by expert, but for what becomes codes: kernels whose last choice is the exact one."""
    calls = [product(m, n, k, F32, offset) for m in (1, 40, 300, 8001) for n, k in ((512, 512), (6144, 4096), (6150, 4096), (6144, 640)) for offset in (0, 1)]
    calls += [experts_product(8, rows, 4096, k, F32, gated) for rows in (1, 64, 400, 1000, 9000) for k in (512, 656, 4099) for gated in (0, 1)]
    for call, (status, error, found) in zip(calls, launches(*calls)):
        assert status == 0, error
        products = [l for l in found if "finish" not in l.kernel]
        assert products and all("true>(" in l.kernel for l in products), (call, found)


@pytest.mark.parametrize("a_rows,lda", [(50, 1 << 27), (1 << 20, 4096), ((1 << 31) - 1, 1 << 33), (1 << 24, 1 << 40), (1 << 30, 1 << 34)])
def test_rows_of_experts_that_32_bits_do_not_reach(a_rows, lda):
    """Rows named by an order go to the kernels with whole addresses as soon as one may lie 2^32 bytes behind the first, products that pass 64 bits included."""
    calls = []
    for rows in (4, 400, 4000):
        call = experts_product(8, rows, 512, 512, BF16)
        call[2].update(a_rows=a_rows, lda=lda)
        calls.append(call)
    for status, error, found in launches(*calls):
        assert status == 0, error
        assert len(found) == 1 and "matmul_fp8_tiles_kernel<" in found[0].kernel and found[0].kernel.split("<")[1].split(",")[5].strip() == "false", found
