"""Adapters, router, routing and experts as a decoder layer runs them: together, captured and replayed, on streams of their own."""
import numpy as np
import pytest
import torch

from oracle import more_oracle as O
from tests.util import codes_to_fp8, make_act, make_weight

pytestmark = pytest.mark.gpu

H, I, E, TOPK, SLOTS, R = 512, 256, 16, 4, 5, 16


class Block:
    """Two projections (merged, with adapters; and back) and routed experts."""

    def __init__(self, seed=0):
        from sglang_b200.srt.layers.linear import MergedColumnParallelLinear, RowParallelLinear
        from sglang_b200.srt.layers.moe.fused_moe_triton.layer import FusedMoE
        from sglang_b200.srt.layers.moe.router import Router
        from sglang_b200.srt.layers.quantization.fp8 import Fp8Config
        from sglang_b200.srt.lora import LoRABatch, attach_lora, load_adapter
        cfg = Fp8Config()
        self.batch = LoRABatch(2048, "cuda")
        self.up = MergedColumnParallelLinear(H, [384, 256], quant_config=cfg, device="cuda")
        self.down = RowParallelLinear(640, H, quant_config=cfg, device="cuda")
        g = torch.Generator().manual_seed(seed)
        for n, layer in enumerate((self.up, self.down)):
            q, s = make_weight(layer.weight.shape[0], layer.weight.shape[1], 10 + n)
            layer.load_full_weight(codes_to_fp8(q), torch.from_numpy(s).cuda())
            attach_lora(layer, self.batch, SLOTS, R)
            for slot in range(SLOTS - 1):  # the last stays empty
                rank = (R, 7, 12, 16)[slot]
                a = [torch.randn(rank, layer.weight.shape[1], generator=g) * 0.05 for _ in layer.lora.slices]
                b = [torch.randn(w, rank, generator=g) * 0.1 for w in layer.lora.slices]
                load_adapter(layer, slot, a, b, 0.5 + slot)
        self.router = Router(E, H, TOPK, "sigmoid", num_expert_group=4, topk_group=2, use_correction_bias=True, routed_scaling_factor=2.5, device="cuda")
        self.router.weight.data.copy_(torch.randn(E, H, generator=g) * 0.1)
        self.router.correction_bias.data.copy_(torch.randn(E, generator=g) * 0.1)
        self.moe = FusedMoE(E, H, I, TOPK, quant_config=cfg, device="cuda")
        w13, s13 = make_weight(2 * I, H, 20, std=0.05, experts=E)
        w2, s2 = make_weight(H, I, 21, std=0.05, experts=E)
        self.moe.load_full_weights(codes_to_fp8(w13), torch.from_numpy(s13).cuda(), codes_to_fp8(w2), torch.from_numpy(s2).cuda())

    def __call__(self, x):
        mid, _ = self.up(x)
        y, _ = self.down(mid)
        top = self.router(y)
        return mid, y, top, self.moe(y, top)


def _ids(T, seed):
    return torch.randint(-1, SLOTS, (T,), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("T", [1, 7, 40, 150, 1300])
def test_a_block_against_its_parts(T):
    from sglang_b200 import ops
    blk, x, ids = Block(), make_act(T, H, T).cuda(), _ids(T, T)
    blk.batch.set(ids.cuda())
    mid, y, top, out = blk(x)
    for layer, inp, got in ((blk.up, x, mid), (blk.down, mid, y)):
        s = layer.lora
        base = layer.quant_method.apply(layer, inp, None)
        f = lambda t: t.double().cpu().numpy()
        want, mass = O.lora_add(f(base), f(inp), f(s.lora_a), f(s.lora_b), ids.numpy(), f(s.scalings), s.ranks.cpu().numpy(), s.slices)
        # as in the operator's own test: sums of float32, h in two terms (2^-16 of the row's largest, 16 of which a sum can be short of),
        # one rounding to bf16
        tol = 2.0**-12 * mass + 2.0**-8 * 1.01 * np.abs(want) + 1e-30
        assert (np.abs(f(got) - want) <= tol).all()
        none = (ids.numpy() < 0) | (ids.numpy() == SLOTS - 1)
        assert torch.equal(got.cpu()[none], base.cpu()[none])
    logits = top.router_logits
    want_w, want_i = O.route(logits.double().cpu().numpy(), TOPK, "sigmoid", blk.router.correction_bias.double().cpu().numpy(), 4, 2, 2, True, 2.5)
    np.testing.assert_array_equal(top.topk_ids.cpu().numpy(), want_i)
    exact = y.double() @ blk.router.weight.double().t()
    mass = y.double().abs() @ blk.router.weight.double().abs().t()
    assert ((logits.double() - exact).abs() <= (H // 16 * 2 + 64) * 2.0**-24 * mass).all()
    assert torch.equal(out, blk.moe(y, top)) and ops.gemm_status() == 0


def test_a_block_captured_and_replayed():
    """One graph for all batches: other tokens, other adapters, a slot that is loaded anew between replays."""
    from sglang_b200.srt.lora import load_adapter, unload_adapter
    T, blk = 48, Block()
    static = make_act(T, H, 1).cuda()
    blk.batch.set(_ids(T, 1).cuda())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        blk(static)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mid, y, top, out = blk(static)
    for seed in (5, 6, 7):
        static.copy_(make_act(T, H, seed))
        blk.batch.set(_ids(T - seed, seed).cuda())  # (a padded batch: the last tokens name none)
        if seed == 6:
            gen = torch.Generator().manual_seed(9)
            load_adapter(blk.down, 0, [torch.randn(3, 640, generator=gen) * 0.1], [torch.randn(H, 3, generator=gen) * 0.1], 2.0)
            unload_adapter(blk.up, 2)
        g.replay()
        torch.cuda.synchronize()
        e_mid, e_y, e_top, e_out = blk(static)
        assert torch.equal(mid, e_mid) and torch.equal(y, e_y) and torch.equal(top.topk_ids, e_top.topk_ids)
        assert torch.equal(top.topk_weights, e_top.topk_weights) and torch.equal(out, e_out)


def test_experts_out_of_service():
    """Fewer experts in service than a token takes: the slots that are left over add nothing."""
    blk, x = Block(), make_act(90, H, 3).cuda()
    blk.router.correction_bias.data[3:] = -float("inf")
    top = blk.router(x)
    assert (top.topk_ids[:, 3:] == -1).all() and (top.topk_ids[:, :3] >= 0).all() and not top.topk_weights[:, 3:].any()
    out = blk.moe(x, top)
    zeroed = top._replace(topk_ids=top.topk_ids.clamp_min(0))  # the same weights: 0 for what is not there
    assert torch.equal(out, blk.moe(x, zeroed))


def test_two_streams_and_two_graphs_at_once():
    """Two batches of the same layers in flight at the same time, eagerly and as two graphs."""
    blk = Block()
    T = 200
    xs = [make_act(T, H, s).cuda() for s in (1, 2)]
    ids = [_ids(T, s).to(torch.int32).cuda() for s in (1, 2)]
    from sglang_b200 import ops
    s = blk.up.lora
    w = blk.router.weight

    def step(i):
        base = blk.up.quant_method.apply(blk.up, xs[i], None)
        y = ops.lora_add(base, xs[i], s.lora_a, s.lora_b, ids[i], s.scalings, s.ranks, s.slices)
        return y, ops.router_logits(xs[i], w), ops.route_topk(ops.router_logits(xs[i], w), 3)[1]

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, graphs, held = [torch.cuda.Stream() for _ in range(2)], [], []
    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            held.append(step(i))
        graphs.append(g)
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i, r in got + list(enumerate(held)):
        for a, b in zip(r, want[i]):
            assert torch.equal(a, b)


def test_operands_written_by_the_kernel_in_front():
    """Every operand comes from a kernel of this library that lets the next launch in early."""
    from sglang_b200 import ops
    T, K, N = 40, 512, 320
    g = torch.Generator(device="cuda").manual_seed(0)

    def written(rows, cols):  # values that a quantised product has just made
        x = torch.randn(rows, 256, generator=g, device="cuda").to(torch.bfloat16)
        q, s = ops.per_token_group_quant_fp8(x, 128)
        wq, ws = make_weight(cols, 256, rows + cols)
        wq, ws = codes_to_fp8(wq), torch.from_numpy(ws).cuda()
        return lambda: ops.w8a8_block_fp8_matmul(q, wq, s, ws)

    make = {"x": written(T, K), "a": written(32, K), "b": written(2 * N, 16), "base": written(T, N), "w": written(24, K)}
    ids = torch.randint(-1, 2, (T,), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()

    def lora(v):
        return ops.lora_add(v["base"], v["x"], v["a"].view(2, 16, K), v["b"].view(2, N, 16), ids)

    v = {k: f() for k, f in make.items()}
    torch.cuda.synchronize()
    want_l, want_r = lora(v), ops.router_logits(v["x"], v["w"])
    torch.cuda.synchronize()
    for last in make:  # written right before the call
        for t in v.values():
            t.fill_(float("nan"))  # (what the allocator hands out next)
        v = {k: f() for k, f in make.items() if k != last}
        torch.cuda.synchronize()
        v[last] = make[last]()
        got = lora(v) if last != "w" else ops.router_logits(v["x"], v["w"])
        torch.cuda.synchronize()
        assert torch.equal(got, want_l if last != "w" else want_r), last
        if last == "x":
            v[last] = make[last]()
            assert torch.equal(ops.router_logits(v["x"], v["w"]), want_r)
