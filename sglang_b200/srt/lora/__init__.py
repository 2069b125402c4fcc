"""Low-rank adapters of many requests beside the quantised linear layers (`srt/layers/linear.py`).

A program keeps one `LoRABatch` for all its layers and writes into it, once per batch, which adapter every token names.  A layer
gets its adapters' slots from `attach_lora(layer, ...)`; from then on its `forward` adds

    scaling[l] * B[l] (A[l] x)          l = the adapter that the token names, none: nothing

to what it returns (`ops.lora_add`, in place, before a row-parallel layer's all-reduce).  Slots are loaded and emptied while the
program runs; their buffers stay where they are, so that captured graphs go on working, and are no part of the layer's state_dict.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch
from torch import nn


class LoRABatch:
    """The adapters that the tokens of the batch in flight name: int32, in a buffer that stays where it is."""

    def __init__(self, max_tokens: int, device=None):
        self.buffer = torch.full((max_tokens,), -1, dtype=torch.int32, device=device)

    def set(self, adapter_ids: torch.Tensor) -> None:
        """`adapter_ids` [tokens] (any integer type; negative, or more than int32 holds: no adapter); tokens behind them name none."""
        n = adapter_ids.numel()
        if n > self.buffer.numel():
            raise RuntimeError(f"LoRABatch: {n} tokens, made for {self.buffer.numel()}")
        if adapter_ids.dtype == torch.bool or adapter_ids.is_floating_point() or adapter_ids.is_complex():
            raise RuntimeError(f"LoRABatch: ids of {adapter_ids.dtype}, not of an integer type")
        ids = adapter_ids.reshape(-1)
        self.buffer[:n].copy_(ids.to(torch.int64).clamp(-1, 2**31 - 1) if ids.element_size() == 8 else ids)
        self.buffer[n:].fill_(-1)

    def ids(self, tokens: int) -> torch.Tensor:
        if tokens > self.buffer.numel():
            raise RuntimeError(f"LoRABatch: {tokens} tokens, made for {self.buffer.numel()}")
        return self.buffer[:tokens]


class LoRASlots(nn.Module):
    """This rank's part of the adapters of one layer: `num_slots` of rank up to `max_rank`."""

    def __init__(self, layer, batch: LoRABatch, num_slots: int, max_rank: int, dtype: torch.dtype, device=None):
        super().__init__()
        if not 1 <= num_slots <= 1024:
            raise RuntimeError(f"num_slots is {num_slots}, not 1 to 1024")
        if max_rank % 8 or not 8 <= max_rank <= 256:
            raise RuntimeError(f"max_rank is {max_rank}, not a multiple of 8 up to 256")
        self.batch, self.max_rank, self.num_slots = batch, max_rank, num_slots
        self.slices = tuple(layer.lora_output_sizes())
        n, parts = sum(self.slices), len(self.slices)
        self.register_buffer("lora_a", torch.zeros(num_slots, parts * max_rank, layer.lora_input_size(), dtype=dtype, device=device), persistent=False)
        self.register_buffer("lora_b", torch.zeros(num_slots, n, max_rank, dtype=dtype, device=device), persistent=False)
        self.register_buffer("scalings", torch.zeros(num_slots, dtype=torch.float32, device=device), persistent=False)
        self.register_buffer("ranks", torch.zeros(num_slots, dtype=torch.int32, device=device), persistent=False)

    def add(self, out: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """out += the adapters' part of x, in place."""
        from ... import ops

        if not isinstance(x, torch.Tensor):
            raise RuntimeError("a layer with adapters takes 16-bit activations, not codes and scales")
        ids = self.batch.ids(x.numel() // x.shape[-1]).view(x.shape[:-1])
        return ops.lora_add(out, x, self.lora_a, self.lora_b, ids, self.scalings, self.ranks, self.slices, out=out)


def attach_lora(layer, batch: LoRABatch, num_slots: int, max_rank: int, dtype: torch.dtype = torch.bfloat16) -> LoRASlots:
    """Gives a linear layer `num_slots` empty slots for adapters of rank up to `max_rank`."""
    layer.lora = LoRASlots(layer, batch, num_slots, max_rank, dtype, layer.weight.device)
    return layer.lora


def _slots(layer, slot: int) -> LoRASlots:
    if layer.lora is None:
        raise RuntimeError("the layer has no slots for adapters (attach_lora)")
    if not 0 <= slot < layer.lora.num_slots:
        raise RuntimeError(f"slot {slot} of {layer.lora.num_slots}")
    return layer.lora


@torch.no_grad()
def load_adapter(layer, slot: int, a_parts: Sequence[Optional[torch.Tensor]], b_parts: Sequence[Optional[torch.Tensor]],
                 scaling: float) -> None:
    """An adapter's FULL matrices into `slot` of a layer, of which this rank keeps its part: per merged projection A [rank, inputs] and
    B [its outputs, rank], or None for a projection that the adapter leaves alone."""
    s = _slots(layer, slot)
    if len(a_parts) != len(s.slices) or len(b_parts) != len(s.slices):
        raise RuntimeError(f"{len(a_parts)} and {len(b_parts)} matrices for {len(s.slices)} merged projections")
    for m in (*a_parts, *b_parts):
        if m is not None and m.dim() != 2:
            raise RuntimeError(f"{tuple(m.shape)} is not a matrix")
    ranks = {a.shape[0] for a in a_parts if a is not None} | {b.shape[1] for b in b_parts if b is not None}
    if len(ranks) != 1 or not 0 < max(ranks) <= s.max_rank:
        raise RuntimeError(f"ranks {sorted(ranks)}: one rank of at most {s.max_rank} for all of a layer's projections")
    rank, R, row = ranks.pop(), s.max_rank, 0
    a_new, b_new = torch.zeros_like(s.lora_a[slot]), torch.zeros_like(s.lora_b[slot])
    for part, (a, b, width) in enumerate(zip(a_parts, b_parts, s.slices)):
        if (a is None) != (b is None):
            raise RuntimeError(f"projection {part} has one matrix of two")
        if a is not None:
            want = (rank, layer.input_size), (layer.lora_full_outputs(part), rank)
            if tuple(a.shape) != want[0] or tuple(b.shape) != want[1]:
                raise RuntimeError(f"projection {part}: A {tuple(a.shape)} and B {tuple(b.shape)}, expected {want[0]} and {want[1]}")
            a, b = layer.lora_shard(part, a, b)
            a_new[part * R : part * R + rank].copy_(a)
            b_new[row : row + width, :rank].copy_(b)
        row += width
    s.lora_a[slot].copy_(a_new)
    s.lora_b[slot].copy_(b_new)
    s.scalings[slot] = scaling
    s.ranks[slot] = rank


@torch.no_grad()
def unload_adapter(layer, slot: int) -> None:
    """Empties a slot: tokens that name it get nothing added."""
    _slots(layer, slot).ranks[slot] = 0


__all__: List[str] = ["LoRABatch", "LoRASlots", "attach_lora", "load_adapter", "unload_adapter"]
