"""Slots of low-rank adapters beside the linear layers, without a GPU: what a rank keeps of an adapter, what is refused; and the
dispatcher's negative ids."""
import pytest
import torch


def _as_rank(monkeypatch, rank, world):
    from sglang_b200.srt.layers import linear
    from sglang_b200.srt.layers.quantization import fp8
    for m in (linear, fp8):
        for name, v in (("get_tensor_model_parallel_world_size", world), ("get_tensor_model_parallel_rank", rank)):
            if hasattr(m, name):
                monkeypatch.setattr(m, name, lambda v=v: v)
    from sglang_b200.srt import distributed
    monkeypatch.setattr(distributed, "get_tensor_model_parallel_world_size", lambda: world)


def _mats(rank, inputs, outputs, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rank, inputs, generator=g), torch.randn(outputs, rank, generator=g)


def _product(layer, slot):
    """Per merged projection, the scaled product of what a slot holds."""
    s, row, out = layer.lora, 0, []
    r = int(s.ranks[slot])
    for part, width in enumerate(s.slices):
        a = s.lora_a[slot, part * s.max_rank : part * s.max_rank + r]
        out.append(s.scalings[slot] * s.lora_b[slot, row : row + width, :r] @ a)
        row += width
    return out


@pytest.mark.parametrize("world", [1, 2])
def test_ranks_hold_parts_of_the_whole(monkeypatch, world):
    from sglang_b200.srt.layers.linear import MergedColumnParallelLinear, QKVParallelLinear, ReplicatedLinear, RowParallelLinear
    from sglang_b200.srt.layers.quantization.fp8 import Fp8Config
    from sglang_b200.srt.lora import LoRABatch, attach_lora, load_adapter, unload_adapter
    cfg, batch = Fp8Config(), LoRABatch(8)
    gate, up, down = _mats(12, 512, 256, 1), _mats(12, 512, 256, 2), _mats(12, 512, 384, 3)
    q, k, v = _mats(5, 512, 1024, 4), _mats(5, 512, 128, 5), _mats(5, 512, 128, 6)
    row_sum = torch.zeros(384, 512)
    for rank in range(world):
        _as_rank(monkeypatch, rank, world)
        col = MergedColumnParallelLinear(512, [256, 256], quant_config=cfg)
        attach_lora(col, batch, 3, 16, torch.float32)
        load_adapter(col, 1, [gate[0], up[0]], [gate[1], up[1]], 0.5)
        n = 256 // world
        for got, (a, b) in zip(_product(col, 1), (gate, up)):
            torch.testing.assert_close(got, 0.5 * b[rank * n : (rank + 1) * n] @ a)
        assert int(col.lora.ranks[0]) == 0 and int(col.lora.ranks[1]) == 12
        load_adapter(col, 1, [None, up[0]], [None, up[1]], 2.0)  # a projection that is left alone, in a slot that held another
        first, second = _product(col, 1)
        assert not first.any()
        torch.testing.assert_close(second, 2.0 * up[1][rank * n : (rank + 1) * n] @ up[0])
        unload_adapter(col, 1)
        assert int(col.lora.ranks[1]) == 0

        row = RowParallelLinear(512, 384, quant_config=cfg)
        attach_lora(row, batch, 2, 16, torch.float32)
        load_adapter(row, 0, [down[0]], [down[1]], 1.5)
        kk = 512 // world
        row_sum[:, rank * kk : (rank + 1) * kk] += _product(row, 0)[0]

        qkv = QKVParallelLinear(512, 128, 8, 1, quant_config=cfg)  # one key/value head: every rank has it
        attach_lora(qkv, batch, 2, 8, torch.float32)
        load_adapter(qkv, 1, [q[0], k[0], v[0]], [q[1], k[1], v[1]], 1.0)
        parts = _product(qkv, 1)
        torch.testing.assert_close(parts[0], q[1][rank * 1024 // world : (rank + 1) * 1024 // world] @ q[0])
        torch.testing.assert_close(parts[1], k[1] @ k[0])
        torch.testing.assert_close(parts[2], v[1] @ v[0])

        rep = ReplicatedLinear(512, 256, quant_config=cfg)
        attach_lora(rep, batch, 1, 16, torch.float32)
        load_adapter(rep, 0, [gate[0]], [gate[1]], 1.0)
        torch.testing.assert_close(_product(rep, 0)[0], gate[1] @ gate[0])
    torch.testing.assert_close(row_sum, 1.5 * down[1] @ down[0])


def test_refusals():
    from sglang_b200.srt.layers.linear import MergedColumnParallelLinear
    from sglang_b200.srt.layers.quantization.fp8 import Fp8Config
    from sglang_b200.srt.lora import LoRABatch, attach_lora, load_adapter
    layer, batch = MergedColumnParallelLinear(256, [128, 128], quant_config=Fp8Config()), LoRABatch(4)
    for bad in (0, 12, 264):
        with pytest.raises(RuntimeError, match="max_rank"):
            attach_lora(layer, batch, 2, bad)
    attach_lora(layer, batch, 2, 16)
    a, b = _mats(8, 256, 128, 0)
    for slot, am, bm, what in ((2, [a, a], [b, b], "slot"), (0, [a], [b], "merged"), (0, [a, a[:4]], [b, b], "rank"), (0, [a, None], [b, b], "one matrix"),
                               (0, [None, None], [None, None], "ranks"), (0, [a[:, :128], a], [b, b], "expected"), (0, [a, a], [b[:64], b], "")):
        with pytest.raises(RuntimeError, match=what):
            load_adapter(layer, slot, am, bm, 1.0)
    big = _mats(24, 256, 128, 0)
    with pytest.raises(RuntimeError, match="at most 16"):
        load_adapter(layer, 0, [big[0]] * 2, [big[1]] * 2, 1.0)
    assert not layer.lora.ranks.any() and not layer.lora.lora_a.any()  # nothing of a refused adapter stays
    with pytest.raises(RuntimeError, match="16-bit"):
        layer.lora.add(torch.zeros(1, 256), (torch.zeros(1, 256), torch.zeros(1, 2)))


def test_batch():
    from sglang_b200.srt.lora import LoRABatch
    b = LoRABatch(6)
    assert b.ids(6).tolist() == [-1] * 6
    where = b.buffer.data_ptr()
    b.set(torch.tensor([3, -1, 2]))
    b.set(torch.tensor([[1], [0]], dtype=torch.int64))
    assert b.ids(4).tolist() == [1, 0, -1, -1] and b.buffer.data_ptr() == where
    with pytest.raises(RuntimeError, match="7 tokens"):
        b.set(torch.zeros(7))
    with pytest.raises(RuntimeError, match="7 tokens"):
        b.ids(7)


def test_dispatcher_keeps_negative_ids():
    from sglang_b200.srt.layers.moe.token_dispatcher import StandardDispatcher, StandardTopKOutput
    d = StandardDispatcher(8, ep_size=2, ep_rank=1)
    out = d.dispatch(torch.zeros(2, 4), StandardTopKOutput(torch.ones(2, 3), torch.tensor([[0, 4, -1], [7, -1, 3]], dtype=torch.int32), None))
    assert out.topk_output.topk_ids.tolist() == [[-1, 0, -1], [3, -1, -1]] and out.topk_output.topk_ids.dtype == torch.int32
