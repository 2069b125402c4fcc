"""What the adapters, the router's product and the routing refuse (no GPU needed)."""
import ctypes

import pytest
import torch

A = 4096  # an aligned address that is never touched


def _err():
    from sglang_b200._lib import lib
    return lib.sglb200_last_error().decode()


def test_router_logits_refuses():
    from sglang_b200._lib import lib
    fn = lib.sglb200_router_logits
    ok = dict(x=A, w=A, dtype=0, y=A, T=4, E=8, K=64, ld=64)

    def call(**kw):
        a = {**ok, **kw}
        return fn(a["x"], a["w"], a["dtype"], a["y"], a["T"], a["E"], a["K"], a["ld"], None)

    assert call(dtype=2) == -2 and "dtype" in _err()
    assert call(K=60, ld=64) == -1 and "divisible by 8" in _err()
    assert call(ld=68) == -1 and call(ld=56) == -1
    assert call(E=0) == -1 and call(T=-1) == -1 and call(K=0) == -1
    assert call(T=1 << 31) == -1 and "too large" in _err()
    assert call(K=(1 << 20) + 8, ld=(1 << 20) + 8) == -1
    assert call(x=None) == -1 and "null" in _err()
    assert call(w=A + 8) == -1 and "16-byte" in _err()
    assert call(T=0, x=None, w=None, y=None) == 0


def test_route_topk_refuses():
    from sglang_b200._lib import lib
    fn = lib.sglb200_route_topk
    ok = dict(x=A, dtype=0, T=4, E=64, k=8, softmax=1, bias=None, G=8, kept=4, top=2, renorm=1, factor=1.0, w=A, i=A)

    def call(**kw):
        a = {**ok, **kw}
        return fn(a["x"], a["dtype"], a["T"], a["E"], a["k"], a["softmax"], a["bias"], a["G"], a["kept"], a["top"], a["renorm"], a["factor"],
                  a["w"], a["i"], None)

    assert call(dtype=3) == -1 and "dtype" in _err()
    assert call(T=-1) == -1 and call(E=0) == -1 and call(k=0) == -1 and call(k=65) == -1
    assert call(G=7) == -1 and "equal size" in _err()
    assert call(G=0) == -1 and call(kept=9) == -1 and call(kept=0) == -1
    assert call(kept=1, k=9) == -1 and "exceeds" in _err()
    assert call(top=3) == -1 and "group_top" in _err()
    assert call(k=33, G=1, kept=1) == -2 and "at most" in _err()
    assert call(E=128, G=64, kept=32) == -2
    assert call(E=2048, G=1, kept=1) == -2 and "at most" in _err()
    assert call(x=None) == -1 and "null" in _err()
    assert call(T=0, x=None, w=None, i=None) == 0


def test_lora_add_refuses():
    from sglang_b200._lib import lib
    fn = lib.sglb200_lora_add
    ok = dict(x=A, a=A, b=A, base=A, out=A, dtype=0, ids=A, scal=None, ranks=None, T=4, L=2, R=16, N=64, K=128, ldx=128, ldb=64, ldo=64,
              sizes=(64,), ws=A, bytes=1 << 30)

    def call(**kw):
        a = {**ok, **kw}
        sizes = None if a["sizes"] is None else (ctypes.c_int64 * len(a["sizes"]))(*a["sizes"])
        return fn(a["x"], a["a"], a["b"], a["base"], a["out"], a["dtype"], a["ids"], a["scal"], a["ranks"], a["T"], a["L"], a["R"], a["N"], a["K"],
                  a["ldx"], a["ldb"], a["ldo"], 1 if sizes is None else len(sizes), sizes, a["ws"], a["bytes"], None)

    assert call(dtype=2) == -2 and "dtype" in _err()
    assert call(T=-1) == -1 and call(L=0) == -1 and call(N=0, sizes=(0,)) == -1
    assert call(R=12) == -2 and call(R=264) == -2 and call(L=1025) == -2 and call(sizes=(8,) * 9, N=72, ldb=72, ldo=72) == -2
    assert call(K=100, ldx=104) == -1 and "divisible by 8" in _err()
    assert call(ldx=132) == -1 and call(ldx=120) == -1 and call(ldb=56) == -1 and call(ldo=63) == -1
    assert call(sizes=(32, 16)) == -1 and "48 columns of 64" in _err()
    assert call(sizes=(64, 8)) == -1 and call(sizes=(64, 0)) == -1 and call(sizes=None) == -1
    assert call(x=None) == -1 and call(ids=None) == -1 and "null" in _err()
    assert call(a=A + 8) == -1 and "16-byte" in _err()
    assert call(out=A + 1) == -1 and "2 bytes" in _err()
    for kw in (dict(out=A + 2), dict(out=A + 64), dict(out=A - 128), dict(ldo=72), dict(out=A + 100, ldb=200, ldo=200), dict(out=A + 320, ldb=200, ldo=200),
               dict(out=A + 64, T=1), dict(out=A + 504)):
        assert call(**kw) == -1 and "overlaps" in _err(), kw
    # columns of one buffer, arrays behind one another, one row of any stride: no overlap, so the next check speaks
    for kw in (dict(), dict(out=A + 128, ldb=128, ldo=128), dict(out=A + 272, ldb=200, ldo=200), dict(out=A + 512), dict(out=A - 512),
               dict(ldo=72, T=1), dict(out=A + 128, T=1)):
        assert call(ws=None, **kw) == -4, kw
    need = lib.sglb200_lora_add_workspace_bytes(4, 2, 16, 1)
    assert need > 0 and call(bytes=need - 1) == -4 and "workspace" in _err() and call(ws=None) == -4 and call(ws=A + 8) == -4
    assert call(T=0, x=None, base=None) == 0
    assert lib.sglb200_lora_add_workspace_bytes(0, 2, 16, 1) == 0


def test_python_forms_refuse():
    from sglang_b200 import ops
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.router_logits(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.route_topk(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError, match="scoring_func"):
        ops.route_topk(torch.zeros(4, 8), 2, "relu")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.lora_add(x, x, torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 64, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32))
