"""Cases that reach every form of the 4-bit kernels (test_fp4_rules.py says which), against the definition in float64."""
import pytest
import torch

from tests.test_gpu_fp4_experts_terms import _check as check_experts
from tests.test_gpu_fp4_gemm import _check as check_product
from tests.test_gpu_fp4_moe import _layer, _run, _want

pytestmark = pytest.mark.gpu

# tokens, experts, experts a token, hidden, intermediate: 16 and 32 columns with K in whole steps, split over warps or not
EXPERTS = [(48, 4, 2, 1024, 512), (64, 8, 4, 2048, 1024), (24, 2, 1, 512, 1024), (16, 2, 1, 2048, 1024), (64, 2, 2, 256, 2048),
           (40, 4, 2, 2048, 2048), (100, 4, 4, 256, 256), (14, 2, 1, 256, 7168), (8, 1, 1, 288, 352), (16, 3, 2, 288, 3104)]

# rows, columns, K and the width of a pair's tile there: several tiles a pair and ragged ends
PAIRS = [(6400, 640, 544, 128), (6400, 632, 1056, 128), (6391, 608, 288, 128), (3000, 2120, 96, 192), (1024, 10248, 544, 192), (515, 9000, 1056, 192),
         (3000, 9224, 800, 256), (300, 37000, 288, 256), (515, 18944, 96, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,topk,H,I", EXPERTS)
def test_experts(T, E, topk, H, I, dtype):
    args = _layer(T, E, topk, H, I, dtype, T + I)
    check_experts(_run(*args), _want(*args), H, I, dtype)


@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,N,K,columns", PAIRS)
def test_pairs(M, N, K, columns, bias, group):
    check_product(M, N, K, group, torch.float16 if bias else torch.bfloat16, alpha=2.0**-10, bias=bias, seed=M + N)
