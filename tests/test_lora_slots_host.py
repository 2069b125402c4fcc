"""Matrices, slots and ids that a layer with adapters refuses, and what attaching leaves alone (no GPU needed)."""
import pytest
import torch


def _as_rank(monkeypatch, rank, world):
    from sglang_b200.srt import distributed
    from sglang_b200.srt.layers import linear
    from sglang_b200.srt.layers.quantization import fp8
    for m in (linear, fp8, distributed):
        for name, v in (("get_tensor_model_parallel_world_size", world), ("get_tensor_model_parallel_rank", rank)):
            if hasattr(m, name):
                monkeypatch.setattr(m, name, lambda v=v: v)


def _layers():
    from sglang_b200.srt.layers.linear import MergedColumnParallelLinear, QKVParallelLinear, ReplicatedLinear, RowParallelLinear
    from sglang_b200.srt.layers.quantization.fp8 import Fp8Config
    cfg = Fp8Config()
    # with the full sizes of every projection: inputs, outputs
    return [(MergedColumnParallelLinear(512, [256, 512], quant_config=cfg), [(512, 256), (512, 512)]),
            (QKVParallelLinear(512, 128, 8, 1, quant_config=cfg), [(512, 1024), (512, 128), (512, 128)]),
            (QKVParallelLinear(512, 128, 8, 2, quant_config=cfg), [(512, 1024), (512, 256), (512, 256)]),
            (RowParallelLinear(512, 384, quant_config=cfg), [(512, 384)]), (ReplicatedLinear(512, 256, quant_config=cfg), [(512, 256)])]


@pytest.mark.parametrize("rank,world", [(0, 1), (0, 2), (1, 2)])
def test_matrices_that_are_not_the_whole(monkeypatch, rank, world):
    """A and B are the adapter's full ones: a larger, a smaller or an already cut one is refused, and not cut to what fits."""
    from sglang_b200.srt.lora import LoRABatch, attach_lora, load_adapter
    _as_rank(monkeypatch, rank, world)
    for layer, sizes in _layers():
        s = attach_lora(layer, LoRABatch(4), 2, 16, torch.float32)
        good = [(torch.ones(8, i), torch.ones(o, 8)) for i, o in sizes]
        for part, (i, o) in enumerate(sizes):
            for di, do in ((512, 0), (-256, 0), (0, 128), (0, o), (0, -o // 2), (8, 0), (0, 1)):
                bad = list(good)
                bad[part] = (torch.ones(8, i + di), torch.ones(o + do, 8))
                with pytest.raises(RuntimeError, match="expected"):
                    load_adapter(layer, 0, [m[0] for m in bad], [m[1] for m in bad], 1.0)
        assert not s.ranks.any() and not s.lora_a.any() and not s.lora_b.any()
        load_adapter(layer, 1, [m[0] for m in good], [m[1] for m in good], 1.0)
        assert int(s.ranks[1]) == 8 and s.lora_b[1, :, :8].eq(1).all() and s.lora_b[1].sum() == s.lora_b.shape[1] * 8


def test_slots_that_are_not_there():
    """A slot out of range (-1 would be the last one), a layer without slots, numbers of slots that the operator does not take."""
    from sglang_b200.srt.lora import LoRABatch, attach_lora, load_adapter, unload_adapter
    layer, sizes = _layers()[4]
    (i, o), = sizes
    for call in (lambda: unload_adapter(layer, 0), lambda: load_adapter(layer, 0, [torch.ones(8, i)], [torch.ones(o, 8)], 1.0)):
        with pytest.raises(RuntimeError, match="no slots"):
            call()
    for bad in (0, -1, 1025):
        with pytest.raises(RuntimeError, match="num_slots"):
            attach_lora(layer, LoRABatch(4), bad, 16)
        assert layer.lora is None
    s = attach_lora(layer, LoRABatch(4), 3, 16, torch.float32)
    for slot in range(3):
        load_adapter(layer, slot, [torch.ones(8, i)], [torch.ones(o, 8)], 1.0)
    for bad in (-1, 3, -3):
        with pytest.raises(RuntimeError, match="slot"):
            unload_adapter(layer, bad)
        with pytest.raises(RuntimeError, match="slot"):
            load_adapter(layer, bad, [torch.ones(8, i)], [torch.ones(o, 8)], 1.0)
    assert s.ranks.tolist() == [8, 8, 8]
    unload_adapter(layer, 2)
    assert s.ranks.tolist() == [8, 8, 0]
    for a, b in ((torch.ones(8), torch.ones(o, 8)), (torch.ones(8, i), torch.ones(o)), (torch.ones(1, 8, i), torch.ones(1, o, 8))):
        with pytest.raises(RuntimeError, match="matrix"):
            load_adapter(layer, 0, [a], [b], 1.0)


def test_ids_of_any_integer_type():
    """Ids beyond int32 name no adapter (they wrapped around to one), and numbers that are no integers are refused."""
    from sglang_b200.srt.lora import LoRABatch
    b = LoRABatch(6)
    b.set(torch.tensor([1 << 32, (1 << 32) + 3, -(1 << 32) + 2, 5, -(1 << 31) - 1, (1 << 31) + 1]))
    assert [i if 0 <= i < 1024 else None for i in b.ids(6).tolist()] == [None, None, None, 5, None, None]
    b.set(torch.tensor([(1 << 32) + 3, (1 << 63) - 1], dtype=torch.int64).to(torch.uint64))
    assert all(not 0 <= i < 1024 for i in b.ids(6).tolist())
    for dtype in (torch.uint8, torch.int8, torch.uint32, torch.int16, torch.int32, torch.int64):
        b.set(torch.tensor([3, 0, 7], dtype=dtype))
        assert b.ids(6).tolist() == [3, 0, 7, -1, -1, -1]
    for bad in (torch.tensor([1.0]), torch.tensor([True]), torch.tensor([1.0], dtype=torch.bfloat16)):
        with pytest.raises(RuntimeError, match="integer"):
            b.set(bad)
    assert b.ids(6).tolist() == [3, 0, 7, -1, -1, -1]


def test_attaching_leaves_the_state_dict_alone():
    """A checkpoint of the layer loads with and without slots, and holds no adapters: they come and go while a program runs."""
    from sglang_b200.srt.lora import LoRABatch, attach_lora
    for layer, _ in _layers():
        before = layer.state_dict()
        attach_lora(layer, LoRABatch(4), 2, 16, torch.float32)
        assert list(layer.state_dict()) == list(before)
        layer.load_state_dict(before)
        moved = layer.to("meta")  # the slots still go where the layer goes
        assert moved.lora.lora_a.device.type == moved.lora.ranks.device.type == "meta"


def test_trained_matrices_leave_no_history():
    """Matrices that require gradients, as a trained adapter's do: the slots are no part of their graph."""
    from sglang_b200.srt.lora import LoRABatch, attach_lora, load_adapter, unload_adapter
    layer, sizes = _layers()[4]
    (i, o), = sizes
    s = attach_lora(layer, LoRABatch(4), 2, 16, torch.float32)
    a, b = torch.nn.Parameter(torch.ones(8, i)), torch.nn.Parameter(torch.ones(o, 8))
    load_adapter(layer, 1, [a], [b * 2], torch.nn.Parameter(torch.tensor(0.5)))
    unload_adapter(layer, 0)
    for t in s.buffers():
        assert not t.requires_grad and t.grad_fn is None
    assert s.lora_b[1, :, :8].eq(2).all() and float(s.scalings[1]) == 0.5
