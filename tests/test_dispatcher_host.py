"""Ids through the expert-parallel dispatcher (no GPU needed)."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode


class Count(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.ops.append(func.overloadpacket.__name__)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("ep_size", [1, 2, 4])
def test_ids_by_one_gather(ep_size, dtype):
    """A rank's experts become 0, 1, .., all others and negative ids -1, by a conversion and a gather alone."""
    from sglang_b200.srt.layers.moe.token_dispatcher import StandardDispatcher, StandardTopKOutput
    E = 16
    ids = torch.cat([torch.arange(E), torch.tensor([-1, -1, -2, -E])]).to(dtype).view(4, 5)
    n = E // ep_size
    for rank in range(ep_size):
        d = StandardDispatcher(E, ep_size, rank)
        top = StandardTopKOutput(torch.ones(4, 5), ids, None)
        d.dispatch(torch.zeros(4, 8), top)
        with Count() as count:
            got = d.dispatch(torch.zeros(4, 8), top).topk_output.topk_ids
        if ep_size == 1:
            assert got is ids
            continue
        want = torch.where((ids >= rank * n) & (ids < (rank + 1) * n), ids - rank * n, -1)
        assert got.dtype == torch.int32 and got.tolist() == want.tolist()
        assert [o for o in count.ops if o not in ("zeros", "_to_copy")] == ["index"] and count.ops.count("_to_copy") <= 1, count.ops
