"""Where the kernels' bounded waits report that they ran out, from the sources: the expert-parallel layer asks after every exchange, and each word
of its own is a synchronous copy of 12 us."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang_b200", "csrc")


def _code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_the_adapters_and_the_routers_kernels_report_in_the_products_word():
    asked = re.search(r"int sglb200_gemm_status\(void\) \{(.*?)\n\}", _code("gemm.cu"), re.S).group(1)
    assert len(re.findall(r"cudaMemcpyFromSymbol|\w+_status\(\)", asked)) == 5
    for name in ("narrow_tile.cu", "lora_tile.cu"):
        code = _code(name)
        assert not re.search(r"__device__ int \w+", code) and re.search(r"atomicExch\([tp]\.status, 1\)", code)
        assert re.search(r"gemm_status_word\(&[tp]\.status\)", code)
