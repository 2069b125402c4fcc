"""The bounded waits of the adapters' and the router's kernels, made to run out on a healthy GPU: they return promptly with the status word
set, and the next ordinary call is right."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
GIVE_UP_AT_ONCE = 0xFFFFFFFF


def _check(call):
    from sglang_b200 import ops
    from sglang_b200._lib import check, lib
    good = call()
    torch.cuda.synchronize()
    assert ops.gemm_status() == 0
    lib.sglb200_gemm_set_wait_probes(GIVE_UP_AT_ONCE)
    try:
        t0 = time.perf_counter()
        call()
        torch.cuda.synchronize()  # returns: no role is left waiting
        assert time.perf_counter() - t0 < 5.0
        assert ops.gemm_status() == 1
    finally:
        lib.sglb200_gemm_set_wait_probes(0)
        check(lib.sglb200_gemm_status_clear())
    again = call()
    torch.cuda.synchronize()
    assert ops.gemm_status() == 0 and torch.equal(again, good)


@pytest.mark.parametrize("T,E,K", [(600, 64, 1024), (2000, 256, 2048), (700, 512, 512)])
def test_router(T, E, K):
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T)
    x, w = (torch.randn(n, K, device="cuda", generator=g).bfloat16() for n in (T, E))
    _check(lambda: ops.router_logits(x, w))


# runs of one adapter and of many, ranks of one span and of two, more runs than a CTA has tiles
@pytest.mark.parametrize("T,K,N,R,L,mixed", [(1500, 512, 1024, 16, 2, False), (600, 512, 2560, 64, 40, True), (1500, 256, 136, 128, 3, False)])
def test_adapters(T, K, N, R, L, mixed):
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T + N)
    x, base = (torch.randn(T, n, device="cuda", generator=g).bfloat16() for n in (K, N))
    a, b = torch.randn(L, R, K, device="cuda", generator=g).bfloat16(), torch.randn(L, N, R, device="cuda", generator=g).bfloat16()
    ids = torch.randint(-1, L, (T,), device="cuda", generator=g) if mixed else torch.arange(T, device="cuda") * L // T
    ids = ids.to(torch.int32)
    _check(lambda: ops.lora_add(base, x, a, b, ids))
